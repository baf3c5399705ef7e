// Single-token DSQG decode over rings in 8 bits: e4m3 rows with a power-of-two scale each (dsqg_rows8.cuh), key and value of a slot side by side.
//
// As csrc/dsqg_decode.cu: one warp per (sequence, head), a group of TPR lanes takes a tap, every row of up to R rounds of taps is requested before one is
// used: with cp.async into shared memory, no register held while in flight, and each lane reads back only the bytes it requested itself, so no barrier is
// needed after the wait.  A row is half as long as in bf16, so a lane holds twice the elements in the same load and a round covers twice the taps: 43 taps
// of 64 columns are six rounds.  The step attends to what the ring holds: the new token's rows are quantised first, and tap 0 reads them.
//
// 256 sequences, 12 heads of 64, 43 taps: HBM's floor is 2.9 us, the dependent chain of one wave of warps (write head, rows, softmax, result) the rest.
// With the rows of a step in registers (157 of them, 12 warps an SM, two waves) this form took 10.6.  bf16 queries without scale_embed take the form on tensor
// cores further down: 7.9.
#include "dsqg_rows8.cuh"

namespace dsqg {
namespace {

constexpr int kWarps = 4;

template <int VEC> struct Bytes {                               // VEC e4m3 values of a row (to load and store: 8 or 16)
    uint32_t u[VEC / 4];
    __device__ __forceinline__ void load(const void* p) {
        if constexpr (VEC == 16) { const uint4 v = *static_cast<const uint4*>(p); u[0] = v.x; u[1] = v.y; u[2] = v.z; u[3] = v.w; }
        else { const uint2 v = *static_cast<const uint2*>(p); u[0] = v.x; u[1] = v.y; }
    }
    __device__ __forceinline__ void store(void* p) const {
        if constexpr (VEC == 16) *static_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
        else *static_cast<uint2*>(p) = make_uint2(u[0], u[1]);
    }
    __device__ __forceinline__ f32x2 get(int i) const {        // values 2 i, 2 i + 1
        const float2 v = __half22float2(e4m3x2_half2(i & 1 ? u[i / 2] >> 16 : u[i / 2] & 0xffffu));
        return pair(v.x, v.y);
    }
    __device__ __forceinline__ void set(const float (&x)[VEC]) {
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i) u[i] = pack_e4m3x4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    }
};
// BYTES from global to shared memory, zeros where `on` is false
template <int BYTES> __device__ __forceinline__ void copy_async(void* to, const void* from, bool on) {
    const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(to));
    const int n = on ? BYTES : 0;
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(d), "l"(from), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" :: "r"(d), "l"(from), "n"(BYTES), "r"(n) : "memory");
}
// scale_value of a byte from 1 on (0, which no row of this library has: 0)
__device__ __forceinline__ float row_scale(uint32_t byte) { return byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23); }
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
__global__ void __launch_bounds__(kWarps * 32, 6)
decode8_kernel(const DecodeArgs a, uint8_t* __restrict__ scale, const Taps t) {
    if constexpr (!PDL) stream_wait();
    constexpr int GROUPS = 32 / TPR;
    __shared__ __align__(16) char rows[kWarps][R][2][32 * VEC];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sh = blockIdx.x * kWarps + warp;                 // (sequence, head) pair
    if (sh >= a.S * a.H) return;                               // whole warp leaves together
    const int s = sh / a.H, h = sh - s * a.H;
    const int g = lane / TPR, d0 = (lane % TPR) * VEC, D = a.D;
    const bool active = d0 < D;
    const int head = a.head[s], fill = a.fill ? a.fill[s] : a.R;
    uint8_t* const ring = static_cast<uint8_t*>(a.k_ring) + (size_t)sh * a.R * 2 * D;
    uint8_t* const bytes = scale + (size_t)sh * a.R * 2;

    f32x2 q[VEC / 2], acc[VEC / 2];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) acc[e] = q[e] = pair(0.f, 0.f);
    const int rounds = (t.J + GROUPS - 1) / GROUPS;
#pragma unroll 1
    for (int r0 = 0; r0 < rounds; r0 += R) {                   // one pass for the usual tap counts
        uint32_t sb[R];
        unsigned exists = 0u;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int j = (r0 + r) * GROUPS + g;
            const int delta = j < t.J ? t.delta(j) : 0;
            int slot = head - delta;
            if (slot < 0) slot += a.R;
            const bool tap = j < t.J && delta < fill;
            if (tap) exists |= 1u << r;
            const bool old = tap && delta > 0;
            const uint8_t* const from = ring + (size_t)(old && active ? slot : 0) * 2 * D + (active ? d0 : 0);
            copy_async<VEC>(&rows[warp][r][0][lane * VEC], from, old && active);
            copy_async<VEC>(&rows[warp][r][1][lane * VEC], from + D, old && active);
            sb[r] = 127u | 127u << 8;
            if (old) sb[r] = *reinterpret_cast<const uint16_t*>(bytes + 2 * slot);
        }
        if (r0 == 0) {
            if constexpr (PDL) stream_wait();
            float x[VEC], y[VEC], z[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = y[e] = z[e] = 0.f;
            if (active) {
                load_row<T, VEC>(a.k_new, (long long)sh * D + d0, x); load_row<T, VEC>(a.v_new, (long long)sh * D + d0, y);
                load_row<T, VEC>(a.q, (long long)sh * D + d0, z);
            }
#pragma unroll
            for (int e = 0; e < VEC / 2; ++e) q[e] = pair(z[2 * e], z[2 * e + 1]);
            Bytes<VEC> kn, vn;
            uint32_t new_scale = quantize<TPR, VEC>(x, kn);
            new_scale |= quantize<TPR, VEC>(y, vn) << 8;
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (g == 0) {
                if (active) {                                  // the new token's slot
                    kn.store(ring + (size_t)head * 2 * D + d0); vn.store(ring + (size_t)head * 2 * D + D + d0);
                    if (d0 == 0) *reinterpret_cast<uint16_t*>(bytes + 2 * head) = (uint16_t)new_scale;
                }
                if (t.delta(0) == 0 && (exists & 1u)) {        // offsets ascend: only tap 0 can be delta 0
                    kn.store(&rows[warp][0][0][lane * VEC]); vn.store(&rows[warp][0][1][lane * VEC]);
                    sb[0] = new_scale;
                }
            }
        } else asm volatile("cp.async.wait_all;" ::: "memory");
        // ---- scores of the pass, then one softmax step over all of them
        float sc[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            Bytes<VEC> k;
            k.load(&rows[warp][r][0][lane * VEC]);
            f32x2 dot = pair(0.f, 0.f);
#pragma unroll
            for (int e = 0; e < VEC / 2; ++e) dot = fma2(q[e], k.get(e), dot);
            float lo, hi;
            unpair(dot, lo, hi);
            sc[r] = (lo + hi) * row_scale(sb[r] & 255u);
            if (a.scale_embed != nullptr && (exists >> r & 1u) && active) {
                float se[VEC];
                load_row<float, VEC>(a.scale_embed, (long long)((r0 + r) * GROUPS + g) * D + d0, se);
                dot = pair(0.f, 0.f);
#pragma unroll
                for (int e = 0; e < VEC / 2; ++e) dot = fma2(q[e], pair(se[2 * e], se[2 * e + 1]), dot);
                unpair(dot, lo, hi);
                sc[r] += lo + hi;
            }
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
        const float base = mx == -INFINITY ? 0.f : mx;
        if (r0) {
            const float cor = __expf(m - base);
            const f32x2 cc = pair(cor, cor);
            l *= cor;
#pragma unroll
            for (int e = 0; e < VEC / 2; ++e) acc[e] = mul2(acc[e], cc);
        }
        m = mx;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float p = __expf(sc[r] - base), w = p * row_scale(sb[r] >> 8);
            l += p;
            const f32x2 ww = pair(w, w);
            Bytes<VEC> v;
            v.load(&rows[warp][r][1][lane * VEC]);
#pragma unroll
            for (int e = 0; e < VEC / 2; ++e) acc[e] = fma2(ww, v.get(e), acc[e]);
        }
    }
    float out[VEC];
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) unpair(acc[e], out[2 * e], out[2 * e + 1]);
#pragma unroll
    for (int o = TPR; o < 32; o <<= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
        for (int e = 0; e < VEC; ++e) out[e] += __shfl_xor_sync(0xffffffffu, out[e], o);
    }
    if (g == 0 && active) {
        const float inv = l == 0.f ? 0.f : (a.head_gain ? a.head_gain[h] : 1.f) / l;
#pragma unroll
        for (int b = 0; b < VEC; b += 8) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = out[b + e] * inv;
            store8(static_cast<T*>(a.out) + (size_t)sh * D + d0 + b, y);
        }
    }
}

// ---- the same step on tensor cores: bf16 queries, no scale_embed, D = 32, 64 or 128.
//
// Taps are the 16 rows of mma.sync (m16n8k16, f16 in, fp32 sums), the query stands in all eight columns: scores = K q without a shuffle, and after the softmax
// O^T += V^T p without one, p turned from a result into an operand by movmatrix.  e4m3 becomes f16 exactly; the query becomes f16 after a power of two
// that brings its largest element to [1, 2); the keys' scales multiply the scores.  An operand of the second product is 2^(score + exponent of the value row's
// scale - w), w such that the largest is at 2^12: what is largest in the result is largest in f16, whatever scales other rows have.  It stands as two f16 numbers,
// itself in the even columns and what its rounding left in the odd ones, off by 2^-22 together.  What bounds the step is instructions, not memory: some 1180 a warp instead of the 1730 of the form above, whose rows go to fp32 one by one.
// A lane asks for the pieces of key rows g and g + 8 that it needs itself (lane (g, t): piece t); value rows go to shared memory as rows, even ones in
// front of odd ones and pieces exchanged so that rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9 are read without bank conflicts.
template <int D> struct Mma {
    static constexpr int KB = D >= 64 ? 16 : 8, KP = D / (4 * KB);           // bytes of a piece of a row, pieces a lane
    static constexpr int VB = D / 8;                                         // bytes of a value row for a lane
    static constexpr int TILES = 3, W = D == 128 ? 2 : 4;                    // 16-tap tiles a pass; warps a block
    // Blocks an SM: us at 256 x 12 x 64 with five, six, seven 8.3, 7.9, 9.2 (spills); at 256 x 8 x 32 5.7, 6.0, 5.0, a launch's blocks then fit beside the last one's
    static constexpr int CTAS = D == 32 ? 7 : 6;
    static constexpr int KTILE = 16 * D, STAGE = TILES * 2 * KTILE;          // key rows, then value rows
    __device__ static __forceinline__ int value_at(int row, int byte) {
        const int r = (row & 8) | (row & 1) << 2 | (row >> 1 & 3);
        return r * D + (D == 128 ? byte ^ (r & 3) << 5 : D == 64 ? byte ^ (r >> 1 & 1) << 5 : byte);
    }
};
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) { const __half2 h = __floats2half2_rn(lo, hi); return *reinterpret_cast<const uint32_t*>(&h); }
template <int WORDS> __device__ __forceinline__ void words_of(const void* p, uint32_t (&w)[WORDS]) {
    if constexpr (WORDS == 4) { const uint4 v = *static_cast<const uint4*>(p); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
    else if constexpr (WORDS == 2) { const uint2 v = *static_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
    else w[0] = *static_cast<const uint32_t*>(p);
}

template <int D, bool PDL>
__global__ void __launch_bounds__(Mma<D>::W * 32, Mma<D>::CTAS) decode8_mma_kernel(const DecodeArgs a, uint8_t* __restrict__ scale, const Taps t) {
    using C = Mma<D>;
    constexpr int TILES = C::TILES, KP = C::KP, KB = C::KB, VEC = D / 4, STEPS = D / 16, E = KB / 4;
    if constexpr (!PDL) stream_wait();
    __shared__ __align__(16) char smem[C::W][C::STAGE];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tig = lane & 3;
    const int sh = blockIdx.x * C::W + warp;                   // (sequence, head) pair
    if (sh >= a.S * a.H) return;                               // whole warp leaves together
    const int s = sh / a.H, h = sh - s * a.H;
    const int head = a.head[s], fill = a.fill ? a.fill[s] : a.R;
    uint8_t* const ring = static_cast<uint8_t*>(a.k_ring) + (size_t)sh * a.R * 2 * D;
    uint8_t* const bytes = scale + (size_t)sh * a.R * 2;
    char* const keys = smem[warp];
    char* const values = smem[warp] + TILES * C::KTILE;

    uint32_t qb[STEPS][2];
    float fs = 0.f, m = -INFINITY, l = 0.f, wbase = -1e30f, o[STEPS][4];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
        qb[k][0] = qb[k][1] = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[k][e] = 0.f;
    }
#pragma unroll 1
    for (int j0 = 0; j0 < t.J; j0 += 16 * TILES) {             // one pass for the usual tap counts
        uint32_t sb[TILES][2];
        bool tap[TILES][2];
#pragma unroll
        for (int i = 0; i < TILES; ++i)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int row = g + 8 * x, j = j0 + 16 * i + row, delta = j < t.J ? t.delta(j) : 0;
                int slot = head - delta;
                if (slot < 0) slot += a.R;
                tap[i][x] = j < t.J && delta < fill;
                const bool old = tap[i][x] && delta > 0;
                if (!old) slot = 0;
                const uint8_t* const from = ring + (size_t)slot * (2 * D) + tig * KB;
#pragma unroll
                for (int k = 0; k < KP; ++k) {
                    copy_async<KB>(keys + (((i * 2 + x) * KP + k) * 32 + lane) * KB, from + 4 * k * KB, old);
                    copy_async<KB>(values + i * C::KTILE + C::value_at(row, (4 * k + tig) * KB), from + D + 4 * k * KB, old);
                }
                sb[i][x] = 127u | 127u << 8;
                if (old) sb[i][x] = *reinterpret_cast<const uint16_t*>(bytes + 2 * slot);
            }
        if (j0 == 0) {
            if constexpr (PDL) stream_wait();
            // the query, and the new token's rows in e4m3: piece 4 k + tig of each, by every group of four lanes
            float x[VEC], y[VEC];
            uint32_t top = 0u;
#pragma unroll
            for (int k = 0; k < KP; ++k) {
                const long long at = (long long)sh * D + (4 * k + tig) * KB;
#pragma unroll
                for (int b = 0; b < KB; b += 8) {
                    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + at + b);
                    qb[k * E + b / 4][0] = u.x; qb[k * E + b / 4][1] = u.y; qb[k * E + b / 4 + 1][0] = u.z; qb[k * E + b / 4 + 1][1] = u.w;
                    float z[8];
                    load8(static_cast<const __nv_bfloat16*>(a.k_new) + at + b, z);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[k * KB + b + e] = z[e];
                    load8(static_cast<const __nv_bfloat16*>(a.v_new) + at + b, z);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[k * KB + b + e] = z[e];
                }
            }
#pragma unroll
            for (int k = 0; k < STEPS; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e) top = max(top, max(qb[k][e] << 16 & 0x7fff0000u, qb[k][e] & 0x7fff0000u));
            top = group_max<4>(top);
            int ex = (int)(top >> 23);                         // NaN and infinity stay what they are
            ex = ex == 0 ? 127 : ex >= 254 ? 253 : ex;
            const float down = __uint_as_float((254u - ex) << 23);
            fs = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)ex << 23);
#pragma unroll
            for (int k = 0; k < STEPS; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e) qb[k][e] = f16x2(__uint_as_float(qb[k][e] << 16) * down, __uint_as_float(qb[k][e] & 0xffff0000u) * down);
            Bytes<VEC> kn, vn;
            const uint32_t fresh = quantize<4, VEC>(x, kn) | quantize<4, VEC>(y, vn) << 8;
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (g == 0) {
                const bool here = t.delta(0) == 0 && tap[0][0];               // offsets ascend: only tap 0 can be delta 0
                if (here) sb[0][0] = fresh;
#pragma unroll
                for (int k = 0; k < KP; ++k) {
                    const int at = (4 * k + tig) * KB;
                    uint8_t* const to = ring + (size_t)head * (2 * D) + at;
#pragma unroll
                    for (int b = 0; b < KB; b += 8) {
                        const uint2 ku = make_uint2(kn.u[(k * KB + b) / 4], kn.u[(k * KB + b) / 4 + 1]), vu = make_uint2(vn.u[(k * KB + b) / 4], vn.u[(k * KB + b) / 4 + 1]);
                        *reinterpret_cast<uint2*>(to + b) = ku; *reinterpret_cast<uint2*>(to + D + b) = vu;
                        if (here) {
                            *reinterpret_cast<uint2*>(keys + (k * 32 + lane) * KB + b) = ku;
                            *reinterpret_cast<uint2*>(values + C::value_at(0, at) + b) = vu;
                        }
                    }
                }
                if (tig == 0) *reinterpret_cast<uint16_t*>(bytes + 2 * head) = (uint16_t)fresh;
            }
        } else asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        // ---- scores: taps g and g + 8 of a tile, the same in every column
        float sc[TILES][2], vlog[TILES][2], mx = m, top = -INFINITY;
        bool one = false;
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KP; ++k) {
                uint32_t w[2][E];
                words_of(keys + (((i * 2) * KP + k) * 32 + lane) * KB, w[0]);
                words_of(keys + (((i * 2 + 1) * KP + k) * 32 + lane) * KB, w[1]);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    uint32_t ka[4];
                    e4m3x4_half2(w[0][e], ka[0], ka[2]); e4m3x4_half2(w[1][e], ka[1], ka[3]);
                    mma(c, ka, qb[k * E + e][0], qb[k * E + e][1]);
                }
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float bias = tap[i][x] ? __ldg(a.pos_bias + (j0 + 16 * i + g + 8 * x) * a.H + h) * 1.4426950408889634f : -INFINITY;
                sc[i][x] = tap[i][x] ? fmaf(c[2 * x] * row_scale(sb[i][x] & 255u), fs, bias) : -INFINITY;
                mx = fmaxf(mx, sc[i][x]);
                const uint32_t vb = sb[i][x] >> 8;
                vlog[i][x] = vb == 255u ? __uint_as_float(0x7fc00000u) : log2_scale(vb);
                one |= tap[i][x] && vb == 127u;
            }
        }
        if (__any_sync(0xffffffffu, one)) {                    // a value row of zeros has a scale of 1 but no weight in the sum: left out
#pragma unroll
            for (int i = 0; i < TILES; ++i)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    uint32_t any = 0u;
#pragma unroll
                    for (int k = 0; k < KP; ++k) {
                        uint32_t u[E];
                        words_of(values + i * C::KTILE + C::value_at(g + 8 * x, (4 * k + tig) * KB), u);
#pragma unroll
                        for (int e = 0; e < E; ++e) any |= u[e] & 0x7f7f7f7fu;
                    }
                    any |= __shfl_xor_sync(0xffffffffu, any, 1); any |= __shfl_xor_sync(0xffffffffu, any, 2);
                    if (any == 0u) vlog[i][x] -= INFINITY;
                }
        }
#pragma unroll
        for (int i = 0; i < TILES; ++i)
#pragma unroll
            for (int x = 0; x < 2; ++x) top = fmaxf(top, sc[i][x] + vlog[i][x]);
#pragma unroll
        for (int b = 4; b < 32; b <<= 1) {
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, b));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, b));
        }
        const float moved = fmaxf(wbase, rintf(top) - 12.f);
        const float base = mx == -INFINITY ? 0.f : mx;
        if (j0) {                                              // a later pass: what was summed so far is against the old maximum and the old w
            const float fv = exp2f(wbase - moved);
            l *= exp2f(m - base);
#pragma unroll
            for (int k = 0; k < STEPS; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[k][e] *= fv;
        }
        m = mx; wbase = moved;
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            uint32_t pb[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                l += exp2_fast(sc[i][x] - base);
                const float w = tap[i][x] ? exp2_fast(sc[i][x] + (vlog[i][x] - wbase)) : 0.f;
                const __half hi = __float2half_rn(w);
                asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pb[x]) : "r"(f16x2(w, w - __half2float(hi))));
            }
            uint32_t w[4][C::VB / 4];
#pragma unroll
            for (int x = 0; x < 4; ++x) words_of(values + i * C::KTILE + C::value_at(2 * tig + (x & 1) + 8 * (x >> 1), g * C::VB), w[x]);
#pragma unroll
            for (int e = 0; e < C::VB / 4; ++e)
#pragma unroll
                for (int y = 0; y < 2; ++y) {                  // values 2 y, 2 y + 1 of the word: rows g and g + 8 of m-tile 2 e + y
                    uint32_t va[4];
                    e4m3x4_half2(__byte_perm(w[0][e], w[1][e], y ? 0x7362 : 0x5140), va[0], va[1]);
                    e4m3x4_half2(__byte_perm(w[2][e], w[3][e], y ? 0x7362 : 0x5140), va[2], va[3]);
                    mma(o[2 * e + y], va, pb[0], pb[1]);
                }
        }
        __syncwarp();                                          // every lane has read the rows that the next pass replaces
    }
#pragma unroll
    for (int b = 4; b < 32; b <<= 1) l += __shfl_xor_sync(0xffffffffu, l, b);
    if (tig == 0) {                                            // d = VB g + 2 (m-tile), + 1
        const float inv = l == 0.f ? 0.f : (a.head_gain ? a.head_gain[h] : 1.f) / l;
        const float unit = exp2f(0.5f * (wbase - (m == -INFINITY ? 0.f : m)));         // twice, for 2^(w - m) alone may be out of range
        uint32_t y[STEPS];
#pragma unroll
        for (int k = 0; k < STEPS; ++k) y[k] = pack_bf16x2((o[k][0] + o[k][1]) * unit * unit * inv, (o[k][2] + o[k][3]) * unit * unit * inv);
        uint32_t* const to = reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.out) + (size_t)sh * D + g * C::VB);
#pragma unroll
        for (int k = 0; k < STEPS; k += 2) *reinterpret_cast<uint2*>(to + k) = make_uint2(y[k], y[k + 1]);
    }
}

template <int D> cudaError_t launch_mma(const DecodeArgs& a, uint8_t* scale, const Taps& t, cudaStream_t s, bool overlap) {
    const unsigned blocks = (unsigned)((a.S * a.H + Mma<D>::W - 1) / Mma<D>::W);
    return launch_after(overlap ? decode8_mma_kernel<D, true> : decode8_mma_kernel<D, false>, blocks, Mma<D>::W * 32, 0, s, a, scale, t);
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
    if (dtype == DSQG_DTYPE_BF16 && !a.scale_embed) {
        if (a.D == 64) return launch_mma<64>(a, scale, t, s, overlap);
        if (a.D == 32) return launch_mma<32>(a, scale, t, s, overlap);
        if (a.D == 128) return launch_mma<128>(a, scale, t, s, overlap);
    }
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
    return cuda_status(launch_after(kern, blocks, 256, 0, static_cast<cudaStream_t>(stream), k, v, static_cast<uint8_t*>(kv_ring), static_cast<uint8_t*>(kv_scale), head, fill, S, H, N, R, D, dtype));
}

int dsqg_dequantize_rows(const void* x, const void* scale, void* out, long long rows, int D, int dtype, void* stream) {
    if (!x || !scale || !out) return DSQG_ERR_NULL_POINTER;
    if (dtype != DSQG_DTYPE_BF16 && dtype != DSQG_DTYPE_F32) return DSQG_ERR_BAD_DTYPE;
    if (rows < 1 || D < 8 || D % 8 || rows * (D / 8) > 0x7fffffffLL * 256) return DSQG_ERR_BAD_SHAPE;
    if (bad(x) || bad(out)) return DSQG_ERR_MISALIGNED;
    return cuda_status(launch_after(dequantize_kernel, (unsigned)((rows * (D / 8) + 255) / 256), 256, 0, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(x),
                        static_cast<const uint8_t*>(scale), out, rows, D, dtype));
}

}  // extern "C"
