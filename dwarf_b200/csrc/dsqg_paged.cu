// The paged cache written from and read back to token-major tensors, and one new token's attention to it on CUDA cores, for every type and width.
#include <algorithm>
#include <cmath>

#include "dsqg_paged.cuh"

namespace dsqg {
namespace {

constexpr int kT = 256;

// ---- prompts into pages and back.  Token t of a ragged batch belongs to the sequence s with cu[s] <= t < cu[s+1] and has position
// start[s] + t - cu[s].  A group of lanes (8 elements a lane) takes the key and value rows of one (token, head) pair, so that the 2 D
// elements of a cache slot are written together.  Bound by memory.
struct MoveArgs {
    PageArgs c;
    const int32_t* cu; const int32_t* start;
    void* k; void* v;
    long long k_token, k_head, v_token, v_head;                // element strides
    int tokens, dtype;
};

// (sequence, position) of token t, or s = -1: a row in front of the first sequence or behind the last.  All lanes of a warp take part, LPR of them with the same
// token.  Up to 32 sequences a lane looks at one boundary and the warp counts those at or below its tokens: one load to wait for instead of five.
template <int LPR> __device__ __forceinline__ int sequence_of(const MoveArgs& a, int t, bool there, long long& position) {
    const int S = a.c.S, lane = threadIdx.x & 31;
    int s = -1, from = 0;
    if (S <= 32) {
        const int first = __ldg(a.cu), edge = __ldg(a.cu + 1 + min(lane, S - 1));
        int count = 0;
#pragma unroll
        for (int q = 0; q < 32 / LPR; ++q) {
            const int other = __shfl_sync(0xffffffffu, t, q * LPR);
            const unsigned below = __ballot_sync(0xffffffffu, lane < S && edge <= other);
            if (lane / LPR == q) count = __popc(below);
        }
        from = __shfl_sync(0xffffffffu, edge, max(count - 1, 0));
        if (count == 0) from = first;
        if (there && t >= first && count < S) s = count;
    } else if (there) {
        int lo = 0, hi = S;
        if (t >= __ldg(a.cu) && t < __ldg(a.cu + hi)) {
            while (hi - lo > 1) {                               // cu[lo] <= t < cu[hi]
                const int mid = (lo + hi) >> 1;
                if (__ldg(a.cu + mid) <= t) lo = mid; else hi = mid;
            }
            s = lo; from = __ldg(a.cu + lo);
        }
    }
    if (s >= 0) position = (long long)t - from + (a.start ? __ldg(a.start + s) : 0);
    return s;
}

// Eight elements as they lie in memory, so that the rows of all heads are asked for before one is used.
struct Raw8 {
    uint4 a, b;
    __device__ __forceinline__ void load(const void* p, long long i, int dtype) {
        if (dtype == DSQG_DTYPE_F32) { const uint4* s = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i); a = __ldg(s); b = __ldg(s + 1); }
        else if (dtype == DSQG_DTYPE_BF16) a = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + i));
        else { const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p) + i); a.x = u.x; a.y = u.y; }
    }
    __device__ __forceinline__ void get(float (&x)[8], int dtype) const {
        if (dtype == DSQG_DTYPE_F32) {
            const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(u[e]);
        } else if (dtype == DSQG_DTYPE_BF16) {
            const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) { x[2 * e] = __uint_as_float(u[e] << 16); x[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u); }
        } else { e4m3x4_float(a.x, x); e4m3x4_float(a.y, x + 4); }
    }
};

// HC heads of a token a group of lanes: where the token goes is found once for them, and their rows are on their way together (8 tokens of up to 2048
// positions, 12 heads of 64 into 8 bits, one head a group: 12.5 us, most of it 64-bit divisions; 32-bit ones 11.4).
template <int LPR, int HC, bool WRITE>
__global__ void __launch_bounds__(kT) move_kernel(const MoveArgs a) {
    stream_wait();
    const unsigned group = blockIdx.x * (kT / LPR) + threadIdx.x / LPR, per = (a.c.H + HC - 1) / HC;
    const int d = (threadIdx.x % LPR) * 8, D = a.c.D;
    const int t = (int)(group / per), h0 = (int)(group - (unsigned)t * per) * HC;
    const bool there = t < a.tokens, on = there && d < D, f8 = a.c.dtype == DSQG_DTYPE_E4M3;
    const long long ki = (long long)t * a.k_token + h0 * a.k_head + d, vi = (long long)t * a.v_token + h0 * a.v_head + d, step = 2LL * a.c.page;
    Raw8 k[HC], v[HC];
#pragma unroll
    for (int i = 0; i < HC; ++i) {                             // what is written does not wait for where it goes
        k[i].a = k[i].b = v[i].a = v[i].b = make_uint4(0u, 0u, 0u, 0u);
        if (WRITE && h0 + i < a.c.H && on) { k[i].load(a.k, ki + i * a.k_head, a.dtype); v[i].load(a.v, vi + i * a.v_head, a.dtype); }
    }
    long long position = 0, slot = -1;
    const int s = sequence_of<LPR>(a, t, there, position);
    if (s >= 0 && position >= 0 && position < (long long)a.c.columns * a.c.page) {
        const unsigned at = (unsigned)position, column = at / (unsigned)a.c.page;
        const long long first = a.c.rows_of(s, h0, (int)column);
        if (first >= 0) slot = (first + (at - column * a.c.page)) * 2;
    }
    uint32_t sb[HC];
#pragma unroll
    for (int i = 0; i < HC; ++i) {
        sb[i] = 127u | 127u << 8;
        if (!WRITE && h0 + i < a.c.H && on && slot >= 0) {
            const long long at = slot + i * step;
            k[i].load(a.c.kv, at * D + d, a.c.dtype); v[i].load(a.c.kv, (at + 1) * D + d, a.c.dtype);
            if (f8) sb[i] = *reinterpret_cast<const uint16_t*>(a.c.scale + at);
        }
    }
#pragma unroll
    for (int i = 0; i < HC; ++i) {
        float x[8], y[8];
        const long long at = slot + i * step;
        const bool mine = h0 + i < a.c.H && on;
        if constexpr (WRITE) {
            k[i].get(x, a.dtype); v[i].get(y, a.dtype);
            if (f8) {
                uint32_t kt = 0u, vt = 0u;
#pragma unroll
                for (int e = 0; e < 8; ++e) { kt = max(kt, abs_bits(x[e])); vt = max(vt, abs_bits(y[e])); }
                const uint32_t kb = row_scale_byte(group_max<LPR>(kt)), vb = row_scale_byte(group_max<LPR>(vt));
                const float ik = scale_inverse(kb), iv = scale_inverse(vb);
#pragma unroll
                for (int e = 0; e < 8; ++e) { x[e] *= ik; y[e] *= iv; }
                if (d == 0 && mine && slot >= 0) *reinterpret_cast<uint16_t*>(a.c.scale + at) = (uint16_t)(kb | vb << 8);
            }
            if (mine && slot >= 0) {
                store8_as(a.c.kv, at * D + d, a.c.dtype, x);
                store8_as(a.c.kv, (at + 1) * D + d, a.c.dtype, y);
            }
        } else if (mine) {
            k[i].get(x, a.c.dtype); v[i].get(y, a.c.dtype);
            // a position that the table has no page for is NaN, a row of no sequence (whose bytes are zeros) zeros
            const float nan = __uint_as_float(0x7fc00000u), sk = s >= 0 && slot < 0 ? nan : f8 ? scale_value(sb[i] & 255u) : 1.f, sv = s >= 0 && slot < 0 ? nan : f8 ? scale_value(sb[i] >> 8) : 1.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) { x[e] *= sk; y[e] *= sv; }
            store8_as(a.k, ki + i * a.k_head, a.dtype, x);
            store8_as(a.v, vi + i * a.v_head, a.dtype, y);
        }
    }
}

template <bool WRITE, int HC> cudaError_t launch_move(const MoveArgs& a, cudaStream_t s) {
    const int lanes = a.c.D / 8, lpr = lanes <= 1 ? 1 : lanes <= 2 ? 2 : lanes <= 4 ? 4 : lanes <= 8 ? 8 : 16;
    const unsigned blocks = (unsigned)(((long long)a.tokens * ((a.c.H + HC - 1) / HC) * lpr + kT - 1) / kT);
    switch (lpr) {
        case 1: return launch_after(move_kernel<1, HC, WRITE>, blocks, kT, 0, s, a);
        case 2: return launch_after(move_kernel<2, HC, WRITE>, blocks, kT, 0, s, a);
        case 4: return launch_after(move_kernel<4, HC, WRITE>, blocks, kT, 0, s, a);
        case 8: return launch_after(move_kernel<8, HC, WRITE>, blocks, kT, 0, s, a);
        default: return launch_after(move_kernel<16, HC, WRITE>, blocks, kT, 0, s, a);
    }
}
// Heads a group: three where they divide up evenly, two otherwise (us, write and read back of 6820 tokens, 12 heads of 64, 8 bits: one 9.8 and 8.6, two 9.5 and
// 7.7, three 9.0 and 7.2, four 9.5 and 9.2; read of 14,501 tokens, 8 heads of 128: one 21.3, two 21.9, three 23.8, four 24.3; floor 13.6).
template <bool WRITE> cudaError_t launch_move_heads(const MoveArgs& a, cudaStream_t s) {
    return a.c.H == 1 ? launch_move<WRITE, 1>(a, s) : a.c.H % 3 == 0 ? launch_move<WRITE, 3>(a, s) : launch_move<WRITE, 2>(a, s);
}

// ---- attention of one new token, CUDA cores: fp32 arithmetic for any types, D a multiple of 8 up to 128, pages of any length.
// A block takes a part of one sequence for up to four query heads of one key-value head; a group of LPR lanes takes a position at a time and
// keeps the running maximum and sum of its softmax for each of those heads, the next position on its way; the groups are joined in shared memory in a
// fixed order.  Bound by its instructions: a dot product over LPR lanes by shuffles for every position and head.  16 sequences up to 2048, 8 heads of 64
// in fp32: 20.5 us (four heads a block, three of them idle, and nothing asked for ahead: 32.1; memory's floor 8.6); 64 up to 4096, 8 x 4 heads of 128: 409 (170).
constexpr int kStepThreads = 128;

template <int LPR, int kHeads>
__global__ void __launch_bounds__(kStepThreads) step_kernel(const StepArgs a) {
    __shared__ __align__(16) char fresh[2 * 128 * 4];
    __shared__ uint8_t fresh_scale[2];
    __shared__ float sm[kHeads][kStepThreads / LPR], sl[kHeads][kStepThreads / LPR];
    __shared__ float sacc[kHeads][kStepThreads / LPR][LPR * 8];
    stream_wait();
    const PageArgs& c = a.c;
    const int D = c.D, blocks_h = (a.G + kHeads - 1) / kHeads, hb = blockIdx.y % blocks_h, h = blockIdx.y / blocks_h, s = blockIdx.z, part = blockIdx.x;
    const Range r = range_of(a, s, part);
    if (part && r.first >= r.length) return;                   // part 0 always answers
    const int heads = min(kHeads, a.G - hb * kHeads), q0 = (s * c.H + h) * a.G + hb * kHeads;
    const int group = threadIdx.x / LPR, d = (threadIdx.x % LPR) * 8;
    const bool on = d < D, has_new = a.k_new != nullptr && r.end == r.length && r.length > 0;
    if (has_new) {
        if (threadIdx.x < 32) new_row(a, s, h, r.length - 1, hb == 0, fresh, fresh_scale);
        __syncthreads();
    }
    float q[kHeads][8], acc[kHeads][8], m[kHeads], l[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        m[i] = -INFINITY; l[i] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) q[i][e] = acc[i][e] = 0.f;
        if (on && i < heads) load8_as(a.q, (long long)(q0 + i) * D + d, a.q_f32 ? DSQG_DTYPE_F32 : DSQG_DTYPE_BF16, q[i]);
    }
    bool bad = r.bad;
    const int last = has_new ? r.length - 1 : -1;
    struct Row { float k[8], v[8]; bool valid; };
    const auto fetch = [&](int p) {
        Row x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x.k[e] = x.v[e] = 0.f;
        x.valid = p < r.end;
        if (!x.valid) return x;
        const long long first = c.rows_of(s, h, p / c.page);
        if (first < 0) { bad = true; x.valid = false; return x; }
        if (!on) return x;
        const long long slot = (first + p % c.page) * 2;
        const bool is_new = p == last;
        const void* rows = is_new ? static_cast<const void*>(fresh) : c.kv;
        load8_as(rows, is_new ? d : slot * D + d, c.dtype, x.k);
        load8_as(rows, is_new ? D + d : (slot + 1) * D + d, c.dtype, x.v);
        if (c.dtype == DSQG_DTYPE_E4M3) {
            const uint8_t* b = is_new ? fresh_scale : c.scale + slot;
            const float sk = scale_value(b[0]), sv = scale_value(b[1]);
#pragma unroll
            for (int e = 0; e < 8; ++e) { x.k[e] *= sk; x.v[e] *= sv; }
        }
        return x;
    };
    constexpr int STEP = kStepThreads / LPR;
    Row next = fetch(r.first + group);
    for (int p0 = r.first; p0 < r.end; p0 += STEP) {
        const Row now = next;
        next = fetch(p0 + STEP + group);                       // on its way while this one is used; at most 2^31 - 257 + 255
        const float (&k)[8] = now.k, (&v)[8] = now.v;
        const bool valid = now.valid;
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            float dot = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) dot = fmaf(q[i][e], k[e], dot);
            dot = group_sum<LPR>(dot) * a.scale;
            if (valid) {
                const float mn = fmaxf(m[i], dot), base = mn == -INFINITY ? 0.f : mn;
                const float cor = exp2f(m[i] - base), w = exp2f(dot - base);
                l[i] = fmaf(l[i], cor, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[i][e] = fmaf(acc[i][e], cor, w * v[e]);
                m[i] = mn;
            }
        }
    }
    const bool any_bad = __syncthreads_or(bad);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        if (d == 0) { sm[i][group] = m[i]; sl[i][group] = l[i]; }
#pragma unroll
        for (int e = 0; e < 8; ++e) sacc[i][group][d + e] = acc[i][e];
    }
    __syncthreads();
    for (int o = threadIdx.x; o < heads * D; o += kStepThreads) {
        const int i = o / D, e = o - i * D;
        float M = -INFINITY;
        for (int g = 0; g < kStepThreads / LPR; ++g) M = fmaxf(M, sm[i][g]);
        const float base = M == -INFINITY ? 0.f : M;
        float L = 0.f, A = 0.f;
        for (int g = 0; g < kStepThreads / LPR; ++g) {
            const float w = exp2f(sm[i][g] - base);
            L = fmaf(w, sl[i][g], L); A = fmaf(w, sacc[i][g][e], A);
        }
        if (any_bad) L = A = __uint_as_float(0x7fc00000u);
        if (a.ml) {
            const long long at = (long long)(q0 + i) * a.parts + part;
            if (e == 0) a.ml[at] = make_float2(M, L);
            a.acc[at * D + e] = A;
        } else {
            const float y = L == 0.f ? 0.f : A / L;
            const long long at = (long long)(q0 + i) * D + e;
            if (a.q_f32) static_cast<float*>(a.out)[at] = y;
            else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16(y);
        }
    }
}

// Joins the parts of a sequence: W warps per (sequence, query head), four parts a warp at a time (maximum, sum and values asked for together), the warps
// added in order.  What it waits for is memory: W so that no warp goes round twice up to 32 parts, and not more, for there may be many rows of few parts
// (2048 rows of two parts: 6 us with one warp each, 13 with eight).
// (One warp per row, parts one after the other: 40 us for 128 rows of 98 parts, which is a chain of loads.)
constexpr int kJoinWarps = 8;
template <int W> __global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const StepArgs a) {
    constexpr int kParts = 4;
    __shared__ float4 sums[kJoinWarps][32];
    __shared__ float2 tops[kJoinWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = a.c.D, d = 4 * lane, sub = warp % W, rows = a.c.S * a.c.H * a.G;
    const int row = blockIdx.x * (kJoinWarps / W) + warp / W;
    // The length is read before the wait: this kernel starts when every block of the one in front of it has waited for all that came before.
    int n = 0;
    if (row < rows) {
        const Range r = range_of(a, row / (a.c.H * a.G), 0);
        n = r.length ? (r.length - 1) / a.chunk + 1 : 1;
    }
    stream_wait();
    const float2* ml = a.ml + (long long)row * a.parts;
    const float* acc = a.acc + (long long)row * a.parts * D;
    float M = -INFINITY, L = 0.f;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto add = [&](const float2 v, const float4 x, float base) {
        const float w = exp2f(v.x - base);
        L = fmaf(w, v.y, L);
        A.x = fmaf(w, x.x, A.x); A.y = fmaf(w, x.y, A.y); A.z = fmaf(w, x.z, A.z); A.w = fmaf(w, x.w, A.w);
    };
    const auto rebase = [&](float top) {                       // what the sums are relative to, 0 for -inf
        const float base = top == -INFINITY ? 0.f : top, f = exp2f(M - base);
        L *= f; A.x *= f; A.y *= f; A.z *= f; A.w *= f;
        M = top;
        return base;
    };
    for (int p0 = sub * kParts; p0 < n; p0 += W * kParts) {
        float2 v[kParts];
        float4 x[kParts];
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            const bool on = p0 + i < n;
            v[i] = on ? ml[p0 + i] : make_float2(-INFINITY, 0.f);
            x[i] = on && d < D ? *reinterpret_cast<const float4*>(acc + (long long)(p0 + i) * D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < kParts; ++i) top = fmaxf(top, v[i].x);
        const float base = rebase(top);
#pragma unroll
        for (int i = 0; i < kParts; ++i) add(v[i], x[i], base);
    }
    if constexpr (W > 1) {
        sums[warp][lane] = A;
        if (lane == 0) tops[warp] = make_float2(M, L);
        __syncthreads();
        if (sub) return;
        float top = M;
#pragma unroll
        for (int w = 1; w < W; ++w) top = fmaxf(top, tops[warp + w].x);
        const float base = rebase(top);
#pragma unroll
        for (int w = 1; w < W; ++w) add(tops[warp + w], sums[warp + w][lane], base);
    }
    if (row >= rows || d >= D) return;
    const float z[4] = {L == 0.f ? 0.f : A.x / L, L == 0.f ? 0.f : A.y / L, L == 0.f ? 0.f : A.z / L, L == 0.f ? 0.f : A.w / L};
    if (a.q_f32) *reinterpret_cast<float4*>(static_cast<float*>(a.out) + (long long)row * D + d) = make_float4(z[0], z[1], z[2], z[3]);
    else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + (long long)row * D + d) = make_uint2(pack_bf16x2(z[0], z[1]), pack_bf16x2(z[2], z[3]));
}
cudaError_t launch_join(const StepArgs& a, cudaStream_t s) {
    const long long rows = (long long)a.c.S * a.c.H * a.G;
    const auto grid = [&](int W) { return dim3((unsigned)((rows * W + kJoinWarps - 1) / kJoinWarps)); };
    if (a.parts <= 4) return launch_after(join_kernel<1>, grid(1), kJoinWarps * 32, 0, s, a);
    if (a.parts <= 8) return launch_after(join_kernel<2>, grid(2), kJoinWarps * 32, 0, s, a);
    return launch_after(join_kernel<8>, grid(8), kJoinWarps * 32, 0, s, a);
}

// One query head a block where a key-value head has one, else up to four.
template <int LPR> cudaError_t launch_lanes(const StepArgs& a, cudaStream_t s) {
    if (a.G == 1) return launch_after(step_kernel<LPR, 1>, dim3(a.parts, a.c.H, a.c.S), kStepThreads, 0, s, a);
    return launch_after(step_kernel<LPR, 4>, dim3(a.parts, a.c.H * ((a.G + 3) / 4), a.c.S), kStepThreads, 0, s, a);
}
cudaError_t launch_step(const StepArgs& a, cudaStream_t s) {
    const int lanes = a.c.D / 8;
    if (lanes <= 1) return launch_lanes<1>(a, s);
    if (lanes <= 2) return launch_lanes<2>(a, s);
    if (lanes <= 4) return launch_lanes<4>(a, s);
    if (lanes <= 8) return launch_lanes<8>(a, s);
    return launch_lanes<16>(a, s);
}

inline bool bad(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

// The positions of a part: a multiple of 64, from the sizes alone.  Blocks run in waves of as many as the GPU holds at once (`an_sm` per SM), and one block too
// many takes a wave of its own: about 85 % of one wave, or of two, three, .., shall have work if lengths are spread evenly up to the longest, in as few waves as keep
// a part at 3200 positions or fewer: the longer the parts, the more is lost where lengths differ from that.  One wave against two, us, 4 x 8 heads of 128 in 8 bits,
// lengths spread evenly / all equal: 8 sequences up to 30000 (parts of 1472 positions in one wave) 32.5 : 36.4 / 55.4 : 55.3, 4 up to 77000 (2048) 52.7 : 52.0 / 72.3 :
// 67.6, 100001 (2688) 58.6 : 60.4 / 86.9 : 80.3, 125000 (3328) 74.2 : 70.5 / 108.6 : 95.7, 150000 (4032) 92.9 : 88.0 / 123.5 : 109.2; one of 131072, 8 x 8 heads in bf16
// (2624), 85.0 : 88.8.  Three waves take more than two in all of these.
// From 16 sequences on, which differ more, two waves, and parts of up to 2048 positions then (256 up to 2048, 8 x 4 heads of 64 in bf16, 83; a whole number of
// waves of fewer positions, 88).
// (us, with one part of the longest for every block that runs at once, whatever the lengths / with this: 16 sequences up to 8192, 8 x 4 heads of 128 in 8 bits, 44 /
// 35; 4 up to 20000, 4 x 8 heads in 8 bits, 21.7 / 18.7; one of 4096, 8 x 4 heads in bf16, 10.5 / 7.7.)
struct Split { int chunk, parts; };
inline Split split_for(int S, int H, int G, int limit, int an_sm) {
    const long long most = ((long long)limit + 63) / 64;                       // in units of 64 positions
    const double pairs = (double)S * H * ((G + 15) / 16), share = (S + 1) / (2.0 * S), one_wave = pairs * most * share / (148 * an_sm * 0.85);
    long long units = (long long)std::ceil(S < 16 ? one_wave / std::max(1.0, std::ceil(one_wave / 50.0)) : std::min(one_wave / 2, 32.0));
    const long long least = (most + 1023) / 1024;                              // no more than 1024 parts
    if (units < least) units = least;
    if (units < 1) units = 1;
    Split r;
    r.chunk = (int)(units * 64);
    r.parts = (int)((most + units - 1) / units);
    if (r.parts < 1) r.parts = 1;
    return r;
}
// Blocks of the kernel that a step takes that an SM holds.
inline int blocks_an_sm(bool mma, int G, int D, bool f8) { return !mma ? 4 : G > 8 || !f8 ? 2 : D > 96 ? 3 : 4; }

// A description of a cache that kernels may use.
int page_args(const dsqg_pages* c, PageArgs* a) {
    if (!c || !c->kv || !c->table || (c->dtype == DSQG_DTYPE_E4M3 && !c->scale)) return DSQG_ERR_NULL_POINTER;
    if (c->dtype != DSQG_DTYPE_BF16 && c->dtype != DSQG_DTYPE_F32 && c->dtype != DSQG_DTYPE_E4M3) return DSQG_ERR_BAD_DTYPE;
    if (c->sequences < 1 || c->sequences > 65535 || c->heads < 1 || c->heads > 65535 || c->pages < 1 || c->columns < 1 || c->page_size < 1 || c->D < 8 || c->D > 128 || c->D % 8 ||
        (long long)c->columns * c->page_size > 0x7fffff00LL || (long long)c->pages * c->heads > 0x7fffffffffLL / ((long long)c->page_size * 2))
        return DSQG_ERR_BAD_SHAPE;
    if (bad(c->kv) || (reinterpret_cast<uintptr_t>(c->scale) & 1u)) return DSQG_ERR_MISALIGNED;
    a->kv = static_cast<char*>(c->kv); a->scale = static_cast<uint8_t*>(c->scale); a->table = c->table;
    a->dtype = c->dtype; a->pages = c->pages; a->page = c->page_size; a->columns = c->columns; a->H = c->heads; a->D = c->D; a->S = c->sequences;
    return DSQG_OK;
}

int move_args(const dsqg_pages* c, const int32_t* cu, const int32_t* start, void* k, void* v, long long k_token, long long k_head, long long v_token, long long v_head,
              long long tokens, int dtype, MoveArgs* a) {
    if (!cu || !k || !v) return DSQG_ERR_NULL_POINTER;
    if (int rc = page_args(c, &a->c)) return rc;
    if (dtype != DSQG_DTYPE_BF16 && dtype != DSQG_DTYPE_F32) return DSQG_ERR_BAD_DTYPE;
    if (tokens < 1 || tokens > 0x7fffffffLL / c->heads - kT) return DSQG_ERR_BAD_SHAPE;
    if (bad(k) || bad(v) || k_token % 8 || k_head % 8 || v_token % 8 || v_head % 8) return DSQG_ERR_MISALIGNED;
    a->cu = cu; a->start = start; a->k = k; a->v = v; a->tokens = (int)tokens; a->dtype = dtype;
    a->k_token = k_token; a->k_head = k_head; a->v_token = v_token; a->v_head = v_head;
    return DSQG_OK;
}

}  // namespace
}  // namespace dsqg

using namespace dsqg;

extern "C" {

int dsqg_paged_write(const dsqg_pages* cache, const void* k, const void* v, long long k_token, long long k_head, long long v_token, long long v_head,
                     const int32_t* cu_seqlens, const int32_t* start, long long tokens, int dtype, void* stream) {
    MoveArgs a;
    if (int rc = move_args(cache, cu_seqlens, start, const_cast<void*>(k), const_cast<void*>(v), k_token, k_head, v_token, v_head, tokens, dtype, &a)) return rc;
    return cuda_status(launch_move_heads<true>(a, static_cast<cudaStream_t>(stream)));
}

int dsqg_paged_read(const dsqg_pages* cache, void* k, void* v, const int32_t* cu_seqlens, const int32_t* start, long long tokens, int dtype, void* stream) {
    MoveArgs a;
    const long long D = cache ? cache->D : 0, HD = cache ? D * cache->heads : 0;
    if (int rc = move_args(cache, cu_seqlens, start, k, v, HD, D, HD, D, tokens, dtype, &a)) return rc;
    return cuda_status(launch_move_heads<false>(a, static_cast<cudaStream_t>(stream)));
}

size_t dsqg_paged_step_scratch_bytes(int sequences, int heads, int q_heads, int D, int max_length) {
    if (sequences < 1 || heads < 1 || q_heads < heads || q_heads % heads || D < 1 || max_length < 0) return 0;
    int parts = 1;                                             // whatever the types
    for (int n = 2; n <= 4; ++n) parts = std::max(parts, split_for(sequences, heads, q_heads / heads, max_length, n).parts);
    return parts == 1 ? 0 : (size_t)sequences * q_heads * parts * (D + 2) * 4;
}

int dsqg_paged_step(const dsqg_pages* cache, const void* q, const void* k_new, const void* v_new, const int32_t* lengths, int q_heads, int max_length, float scale,
                    void* out, void* scratch, size_t scratch_bytes, int dtype, void* stream) {
    StepArgs a;
    if (!q || !lengths || !out || !k_new != !v_new) return DSQG_ERR_NULL_POINTER;
    if (int rc = page_args(cache, &a.c)) return rc;
    if (dtype != DSQG_DTYPE_BF16 && dtype != DSQG_DTYPE_F32) return DSQG_ERR_BAD_DTYPE;
    if (q_heads < a.c.H || q_heads % a.c.H || (long long)a.c.S * q_heads > 0x7fffffffLL / 128 || max_length < 0 || a.c.H * ((q_heads / a.c.H + 3) / 4) > 65535) return DSQG_ERR_BAD_SHAPE;
    if (!(scale < 3.0e38f)) return DSQG_ERR_UNSUPPORTED;
    if (bad(q) || bad(k_new) || bad(v_new) || bad(out) || bad(scratch)) return DSQG_ERR_MISALIGNED;
    if (max_length > (long long)a.c.columns * a.c.page) return DSQG_ERR_BAD_SHAPE;
    a.limit = max_length;
    a.q = q; a.k_new = k_new; a.v_new = v_new; a.lengths = lengths; a.out = out; a.G = q_heads / a.c.H; a.q_f32 = dtype == DSQG_DTYPE_F32;
    a.scale = (scale > 0.f ? scale : 1.0f / sqrtf((float)a.c.D)) * 1.4426950408889634f;
    const bool mma = paged_mma_supported(a);
    const Split p = split_for(a.c.S, a.c.H, a.G, a.limit, blocks_an_sm(mma, a.G, a.c.D, a.c.dtype == DSQG_DTYPE_E4M3));
    a.chunk = p.chunk; a.parts = p.parts; a.ml = nullptr; a.acc = nullptr;
    if (p.parts > 1) {
        const size_t rows = (size_t)a.c.S * q_heads * p.parts;
        if (!scratch) return DSQG_ERR_NULL_POINTER;
        if (scratch_bytes < rows * (a.c.D + 2) * 4) return DSQG_ERR_SCRATCH_TOO_SMALL;
        a.acc = static_cast<float*>(scratch); a.ml = reinterpret_cast<float2*>(a.acc + rows * a.c.D);
    }
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = mma ? launch_paged_mma(a, s) : launch_step(a, s);
    if (e == cudaSuccess && a.ml) e = launch_join(a, s);
    return cuda_status(e);
}

}  // extern "C"
