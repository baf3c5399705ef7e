// Single-token DSQG decode over rings in 8 bits: e4m3 rows with a power-of-two scale each (dsqg_rows8.cuh), key and value of a slot side by side.
//
// As csrc/dsqg_decode.cu: one warp per (sequence, head), a group of TPR lanes takes a tap, every row of up to R rounds of taps is requested before
// one is used.  A row is half as long as in bf16, so a lane holds twice the elements in the same load and a round covers twice the taps: 43 taps of
// 64 columns are six rounds of 16-byte loads, which registers hold (bf16 needs eleven, most of them in shared memory).  The step attends to what the ring
// holds: the new token's rows are quantised first, and tap 0 reads them.
#include "dsqg_rows8.cuh"

namespace dsqg {
namespace {

constexpr int kWarps = 4;

template <int VEC> struct Bytes;                               // VEC e4m3 values of a row
template <> struct Bytes<16> {
    uint4 u;
    __device__ __forceinline__ void load(const uint8_t* p) { u = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void store(uint8_t* p) const { *reinterpret_cast<uint4*>(p) = u; }
    __device__ __forceinline__ void zero() { u = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void get(float (&x)[16]) const { e4m3x4_float(u.x, x); e4m3x4_float(u.y, x + 4); e4m3x4_float(u.z, x + 8); e4m3x4_float(u.w, x + 12); }
    __device__ __forceinline__ void set(const float (&x)[16]) {
        u = make_uint4(pack_e4m3x4(x[0], x[1], x[2], x[3]), pack_e4m3x4(x[4], x[5], x[6], x[7]), pack_e4m3x4(x[8], x[9], x[10], x[11]), pack_e4m3x4(x[12], x[13], x[14], x[15]));
    }
};
template <> struct Bytes<8> {
    uint2 u;
    __device__ __forceinline__ void load(const uint8_t* p) { u = *reinterpret_cast<const uint2*>(p); }
    __device__ __forceinline__ void store(uint8_t* p) const { *reinterpret_cast<uint2*>(p) = u; }
    __device__ __forceinline__ void zero() { u = make_uint2(0u, 0u); }
    __device__ __forceinline__ void get(float (&x)[8]) const { e4m3x4_float(u.x, x); e4m3x4_float(u.y, x + 4); }
    __device__ __forceinline__ void set(const float (&x)[8]) { u = make_uint2(pack_e4m3x4(x[0], x[1], x[2], x[3]), pack_e4m3x4(x[4], x[5], x[6], x[7])); }
};
template <typename T, int VEC> __device__ __forceinline__ void load_row(const void* p, long long i, float (&x)[VEC]) {
#pragma unroll
    for (int b = 0; b < VEC; b += 8) {
        float y[8];
        load8(static_cast<const T*>(p) + i + b, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[b + e] = y[e];
    }
}
// A row's slice in e4m3 and the row's scale byte; all lanes of a group of TPR take part.
template <int TPR, int VEC> __device__ __forceinline__ uint32_t quantize(float (&x)[VEC], Bytes<VEC>& to) {
    uint32_t top = 0u;
#pragma unroll
    for (int e = 0; e < VEC; ++e) top = max(top, abs_bits(x[e]));
    const uint32_t byte = row_scale_byte(group_max<TPR>(top));
    const float inv = scale_inverse(byte);
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[e] *= inv;
    to.set(x);
    return byte;
}

// T: type of q, k_new, v_new, out.  PDL: the overlapped form (dsqg_decode.cu), which reads head, fill and the rows of taps with delta > 0 before it waits.
template <typename T, int TPR, int VEC, int R, bool PDL>
__global__ void __launch_bounds__(kWarps * 32)
decode8_kernel(const DecodeArgs a, uint8_t* __restrict__ scale, const Taps t) {
    if constexpr (!PDL) stream_wait();
    constexpr int GROUPS = 32 / TPR;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sh = blockIdx.x * kWarps + warp;                 // (sequence, head) pair
    if (sh >= a.S * a.H) return;                               // whole warp leaves together
    const int s = sh / a.H, h = sh - s * a.H;
    const int g = lane / TPR, d0 = (lane % TPR) * VEC, D = a.D;
    const bool active = d0 < D;
    const int head = a.head[s], fill = a.fill ? a.fill[s] : a.R;
    uint8_t* const ring = static_cast<uint8_t*>(a.k_ring) + (size_t)sh * a.R * 2 * D;
    uint8_t* const bytes = scale + (size_t)sh * a.R * 2;

    float q[VEC], acc[VEC], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = q[e] = 0.f;
    Bytes<VEC> kn, vn;
    uint32_t new_scale = 0u;
    const int rounds = (t.J + GROUPS - 1) / GROUPS;
#pragma unroll 1
    for (int r0 = 0; r0 < rounds; r0 += R) {                   // one pass for the usual tap counts
        Bytes<VEC> k[R], v[R];
        uint32_t sb[R];
        unsigned exists = 0u;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int j = (r0 + r) * GROUPS + g;
            const int delta = j < t.J ? t.delta(j) : 0;
            int slot = head - delta;
            if (slot < 0) slot += a.R;
            k[r].zero(); v[r].zero(); sb[r] = 127u | 127u << 8;
            if (j < t.J && delta < fill) {
                exists |= 1u << r;
                if (delta) {
                    if (active) { k[r].load(ring + (size_t)slot * 2 * D + d0); v[r].load(ring + (size_t)slot * 2 * D + D + d0); }
                    sb[r] = *reinterpret_cast<const uint16_t*>(bytes + 2 * slot);
                }
            }
        }
        if (r0 == 0) {
            if constexpr (PDL) stream_wait();
            float x[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = 0.f;
            if (active) load_row<T, VEC>(a.k_new, (long long)sh * D + d0, x);
            float y[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[e] = 0.f;
            if (active) { load_row<T, VEC>(a.v_new, (long long)sh * D + d0, y); load_row<T, VEC>(a.q, (long long)sh * D + d0, q); }
            new_scale = quantize<TPR, VEC>(x, kn);
            new_scale |= quantize<TPR, VEC>(y, vn) << 8;
            if (g == 0 && active) {                            // the new token's slot
                kn.store(ring + (size_t)head * 2 * D + d0); vn.store(ring + (size_t)head * 2 * D + D + d0);
                if (d0 == 0) *reinterpret_cast<uint16_t*>(bytes + 2 * head) = (uint16_t)new_scale;
            }
            if (g == 0 && t.delta(0) == 0 && (exists & 1u)) { k[0] = kn; v[0] = vn; sb[0] = new_scale; }      // offsets ascend: only tap 0 can be delta 0
        }
        // ---- scores of the pass, then one softmax step over all of them
        float sc[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float x[VEC];
            k[r].get(x);
            const int j = (r0 + r) * GROUPS + g;
            const float ks = scale_value(sb[r] & 255u);
            float dot = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) dot = fmaf(q[e], x[e], dot);
            dot *= ks;
            if (a.scale_embed != nullptr && (exists >> r & 1u) && active) {
                float se[VEC];
                load_row<float, VEC>(a.scale_embed, (long long)j * D + d0, se);
#pragma unroll
                for (int e = 0; e < VEC; ++e) dot = fmaf(q[e], se[e], dot);
            }
            sc[r] = dot;
        }
#pragma unroll
        for (int o = TPR / 2; o > 0; o >>= 1)
#pragma unroll
            for (int r = 0; r < R; ++r) sc[r] += __shfl_xor_sync(0xffffffffu, sc[r], o);
        float mx = m;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            sc[r] = exists >> r & 1u ? fmaf(sc[r], a.scale, __ldg(a.pos_bias + ((r0 + r) * GROUPS + g) * a.H + h)) : -INFINITY;
            mx = fmaxf(mx, sc[r]);
        }
#pragma unroll
        for (int o = TPR; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float base = mx == -INFINITY ? 0.f : mx, cor = __expf(m - base);
        l *= cor;
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] *= cor;
        m = mx;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float p = __expf(sc[r] - base);
            l += p;
            const float w = p * scale_value(sb[r] >> 8);
            float x[VEC];
            v[r].get(x);
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] = fmaf(w, x[e], acc[e]);
        }
    }
#pragma unroll
    for (int o = TPR; o < 32; o <<= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], o);
    }
    if (g == 0 && active) {
        const float inv = l == 0.f ? 0.f : (a.head_gain ? a.head_gain[h] : 1.f) / l;
#pragma unroll
        for (int b = 0; b < VEC; b += 8) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = acc[b + e] * inv;
            store8(static_cast<T*>(a.out) + (size_t)sh * D + d0 + b, y);
        }
    }
}

template <typename T, int TPR, int VEC> cudaError_t launch_group(const DecodeArgs& a, uint8_t* scale, const Taps& t, cudaStream_t s, bool overlap) {
    const unsigned blocks = (unsigned)((a.S * a.H + kWarps - 1) / kWarps);
    const int rounds = (t.J + 32 / TPR - 1) / (32 / TPR);
    // A pass of three rounds where that is all there is (43 taps of 32 columns), of six otherwise.
    if (rounds <= 3) return launch_after(overlap ? decode8_kernel<T, TPR, VEC, 3, true> : decode8_kernel<T, TPR, VEC, 3, false>, blocks, kWarps * 32, 0, s, a, scale, t);
    return launch_after(overlap ? decode8_kernel<T, TPR, VEC, 6, true> : decode8_kernel<T, TPR, VEC, 6, false>, blocks, kWarps * 32, 0, s, a, scale, t);
}
// 16-byte slices where rows are a multiple of that, 8-byte slices otherwise.
template <typename T> cudaError_t launch_type(const DecodeArgs& a, uint8_t* scale, const Taps& t, cudaStream_t s, bool overlap) {
    if (a.D % 16 == 0) {
        const int n = a.D / 16;
        if (n <= 1) return launch_group<T, 1, 16>(a, scale, t, s, overlap);
        if (n <= 2) return launch_group<T, 2, 16>(a, scale, t, s, overlap);
        if (n <= 4) return launch_group<T, 4, 16>(a, scale, t, s, overlap);
        return launch_group<T, 8, 16>(a, scale, t, s, overlap);
    }
    const int n = a.D / 8;
    if (n <= 1) return launch_group<T, 1, 8>(a, scale, t, s, overlap);
    if (n <= 4) return launch_group<T, 4, 8>(a, scale, t, s, overlap);
    if (n <= 8) return launch_group<T, 8, 8>(a, scale, t, s, overlap);
    return launch_group<T, 16, 8>(a, scale, t, s, overlap);
}

// Ring prefill: position p of the last min(N, R) of every sequence to slot p mod R, quantised.  A group of lanes takes one row.
template <int LPR> __global__ void __launch_bounds__(256)
ring_prefill8_kernel(const void* __restrict__ k, const void* __restrict__ v, uint8_t* ring, uint8_t* scale, int32_t* head, int32_t* fill, int S, int H, int N, int R, int D,
                     int dtype) {
    stream_wait();
    const int keep = N < R ? N : R, d = (threadIdx.x % LPR) * 8;
    const long long at = ((long long)blockIdx.x * 256 + threadIdx.x) / LPR, pair = at / 2, total = (long long)S * H * keep;
    const int which = (int)(at & 1), sh = (int)(pair / keep), p = N - keep + (int)(pair - (long long)sh * keep);
    const bool there = pair < total, on = there && d < D;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (on) load8_as(which ? v : k, ((long long)sh * N + p) * D + d, dtype, x);
    uint32_t top = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, abs_bits(x[e]));
    const uint32_t byte = row_scale_byte(group_max<LPR>(top));
    const float inv = scale_inverse(byte);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= inv;
    const long long row = ((long long)sh * R + p % R) * 2 + which;
    if (on) store8_as(ring, row * D + d, DSQG_DTYPE_E4M3, x);
    if (there && d == 0) scale[row] = (uint8_t)byte;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i < S) { head[i] = (N - 1) % R; fill[i] = keep; }
}

// Rows in 8 bits back to bf16 or fp32: 8 elements a thread.
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ x, const uint8_t* __restrict__ scale, void* out, long long rows, int D, int dtype) {
    stream_wait();
    const int per = D / 8;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, row = i / per;
    if (row >= rows) return;
    const float s = scale_value(__ldg(scale + row));
    float y[8];
    load8_as(x, i * 8, DSQG_DTYPE_E4M3, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= s;
    store8_as(out, i * 8, dtype, y);
}

inline bool bad(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

}  // namespace

cudaError_t launch_decode8(const DecodeArgs& a, uint8_t* scale, const Taps& t, int dtype, cudaStream_t s, bool overlap) {
    return dtype == DSQG_DTYPE_BF16 ? launch_type<__nv_bfloat16>(a, scale, t, s, overlap) : launch_type<float>(a, scale, t, s, overlap);
}

}  // namespace dsqg

using namespace dsqg;

extern "C" {

int dsqg_ring_prefill_e4m3(const void* k, const void* v, void* kv_ring, void* kv_scale, int32_t* head, int32_t* fill, int S, int H, int N, int D, int R, int dtype, void* stream) {
    if (!k || !v || !kv_ring || !kv_scale || !head || !fill) return DSQG_ERR_NULL_POINTER;
    if (dtype != DSQG_DTYPE_BF16 && dtype != DSQG_DTYPE_F32) return DSQG_ERR_BAD_DTYPE;
    if (S < 1 || H < 1 || N < 1 || R < 1 || D < 8 || D > 128 || D % 8 || (long long)S * H * R * 2 > 0x7fffffffLL || (long long)S * H * N > 0x7fffffffLL) return DSQG_ERR_BAD_SHAPE;
    if (bad(k) || bad(v) || bad(kv_ring)) return DSQG_ERR_MISALIGNED;
    const int lanes = D / 8, lpr = lanes <= 1 ? 1 : lanes <= 2 ? 2 : lanes <= 4 ? 4 : lanes <= 8 ? 8 : 16;
    const long long threads = (long long)S * H * (N < R ? N : R) * 2 * lpr;        // at least S
    const unsigned blocks = (unsigned)((threads + 255) / 256);
    auto kern = lpr == 1 ? ring_prefill8_kernel<1> : lpr == 2 ? ring_prefill8_kernel<2> : lpr == 4 ? ring_prefill8_kernel<4> : lpr == 8 ? ring_prefill8_kernel<8> : ring_prefill8_kernel<16>;
    return launch_after(kern, blocks, 256, 0, static_cast<cudaStream_t>(stream), k, v, static_cast<uint8_t*>(kv_ring), static_cast<uint8_t*>(kv_scale), head, fill, S, H, N, R, D, dtype)
        == cudaSuccess ? DSQG_OK : DSQG_ERR_CUDA;
}

int dsqg_dequantize_rows(const void* x, const void* scale, void* out, long long rows, int D, int dtype, void* stream) {
    if (!x || !scale || !out) return DSQG_ERR_NULL_POINTER;
    if (dtype != DSQG_DTYPE_BF16 && dtype != DSQG_DTYPE_F32) return DSQG_ERR_BAD_DTYPE;
    if (rows < 1 || D < 8 || D % 8 || rows * (D / 8) > 0x7fffffffLL * 256) return DSQG_ERR_BAD_SHAPE;
    if (bad(x) || bad(out)) return DSQG_ERR_MISALIGNED;
    return launch_after(dequantize_kernel, (unsigned)((rows * (D / 8) + 255) / 256), 256, 0, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(x),
                        static_cast<const uint8_t*>(scale), out, rows, D, dtype) == cudaSuccess ? DSQG_OK : DSQG_ERR_CUDA;
}

}  // extern "C"
