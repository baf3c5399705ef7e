// A paged key-value cache: what the kernels that write, read and attend to it share.
//
// Pages [P, H, page, 2, D]: a page holds, for every head, `page` consecutive positions of one sequence, key and value of a position side by side
// (as in the interleaved rings).  table [S, columns] gives the page of positions [c page, (c + 1) page) of a sequence.  In 8 bits a
// row has a scale byte, scale [P, H, page, 2] (dsqg_rows8.cuh).
#pragma once

#include "dsqg_rows8.cuh"

namespace dsqg {

struct PageArgs {
    char* kv; uint8_t* scale; const int32_t* table;
    int dtype, pages, page, columns, H, D, S;

    // Index of the first row of a page for head h, -1 where the table names no page of the cache: nothing is read or written there.
    __device__ __forceinline__ long long rows_of(int s, int h, int column) const {
        const int id = __ldg(table + (long long)s * columns + column);
        return id < 0 || id >= pages ? -1 : ((long long)id * H + h) * page;
    }
};

struct StepArgs {
    PageArgs c;
    const void* q; const void* k_new; const void* v_new; const int32_t* lengths;
    void* out;
    float2* ml;                // per (sequence, query head, part): maximum (in units of log2) and sum; null where nothing is split
    float* acc;                // ... and the sums of values, D each
    int G, q_f32, limit, chunk, parts;
    float scale;               // of the scores, times log2 e
};

// The positions of sequence s that part `part` attends to.  A length outside [0, limit] makes the results of the sequence NaN.
struct Range { int first, end, length; bool bad; };
__device__ __forceinline__ Range range_of(const StepArgs& a, int s, int part) {
    Range r;
    r.length = __ldg(a.lengths + s);
    r.bad = r.length < 0 || r.length > a.limit;
    if (r.bad) r.length = 0;
    r.first = part * a.chunk;
    r.end = r.first + min(r.length - r.first, a.chunk);        // up to 2^31 - 256 positions: first + chunk may be beyond an int
    return r;
}

// The new token's key and value as the cache holds them, by the 32 lanes of a warp: to `row` ([2][D] in shared memory, its scale bytes at
// `bytes`) and, where `store` says so, to the cache.  D <= 128.
__device__ __forceinline__ void new_row(const StepArgs& a, int s, int h, int position, bool store, char* row, uint8_t* bytes) {
    const PageArgs& c = a.c;
    const int lane = threadIdx.x & 31, half = lane >> 4, d = (lane & 15) * 8;
    const bool on = d < c.D;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (on) load8_as(half ? a.v_new : a.k_new, ((long long)s * c.H + h) * c.D + d, a.q_f32 ? DSQG_DTYPE_F32 : DSQG_DTYPE_BF16, x);
    uint32_t byte = 127u;
    if (c.dtype == DSQG_DTYPE_E4M3) {
        uint32_t top = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, abs_bits(x[e]));
        byte = row_scale_byte(group_max<16>(top));
        const float inv = scale_inverse(byte);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= inv;
    }
    const long long first = store ? c.rows_of(s, h, position / c.page) : -1;
    const long long at = (first + position % c.page) * 2 + half;
    if (on) {
        store8_as(row, half * c.D + d, c.dtype, x);
        if (first >= 0) store8_as(c.kv, at * c.D + d, c.dtype, x);
    }
    if (c.dtype == DSQG_DTYPE_E4M3 && (lane & 15) == 0) {
        bytes[half] = (uint8_t)byte;
        if (first >= 0) c.scale[at] = (uint8_t)byte;
    }
}

// The tensor-core form (dsqg_paged_mma.cu): bf16 queries, pages in bf16 or e4m3, D 48, 80 or a multiple of 32, pages of a multiple of 16 positions.
bool paged_mma_supported(const StepArgs& a);
cudaError_t launch_paged_mma(const StepArgs& a, cudaStream_t s);

}  // namespace dsqg
