// One new token's attention to a paged cache on tensor cores: bf16 queries, pages in bf16 or e4m3, D = 32, 64, 96 or 128.
//
// A block takes a part of one sequence for up to 16 query heads of one key-value head, a warp every fourth tile of 16 positions of it.  The query
// heads are the 16 rows of mma.sync (m16n8k16, fp32 accumulators): S = Q K^T, softmax with a running maximum and sum per row, O += P V.  The
// contraction of a product may be permuted freely as long as both operands agree, so every lane reads exactly the 16-byte pieces of a tile that it
// needs itself: it copies them into shared memory with cp.async some tiles ahead and reads back its own bytes, with no barrier and no bank
// conflict, and no register is held by a load in flight.  Key rows are the B operand as they lie (lane (g, t): row g, every fourth piece from t);
// of the value rows a lane takes four positions and an eighth of the columns, and pairs of positions are put together by byte permutation.
//
// 8 bits: e4m3 becomes f16 exactly.  Queries become f16 after a power of two that brings their largest element near 1; the keys' scales multiply the
// scores; the values' scales multiply the probabilities, relative to the largest scale seen so far (another running maximum), so that f16 holds them.
//
// mma.sync and not tcgen05: an operand of 128 rows would be at most an eighth full (query heads of one key-value head), and what is in question is memory.
#include "dsqg_paged.cuh"

namespace dsqg {
namespace {

constexpr int kWarps = 4, kTile = 16;

template <bool F16> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// BYTES from global to shared memory, zeros where `on` is false.
template <int BYTES> __device__ __forceinline__ void copy_async(char* to, const char* from, bool on) {
    const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(to));
    const int n = on ? BYTES : 0;
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(d), "l"(from), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" :: "r"(d), "l"(from), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) { return half2_bits(__floats2half2_rn(lo, hi)); }

template <int D, bool F8, bool WIDE, int STAGES>
struct Cfg {
    static constexpr int SZ = F8 ? 1 : 2;
    static constexpr int KB = F8 ? (D % 64 == 0 ? 16 : 8) : 16;          // bytes of a piece of a key row: four lanes take 4 KB bytes
    static constexpr int KP = D * SZ / (4 * KB);                         // pieces a lane and key row
    static constexpr int VB = F8 ? (D % 128 == 0 ? 16 : D % 64 == 0 ? 8 : 4) : (D % 64 == 0 ? 16 : 8);     // of a value row: eight lanes take 8 VB
    static constexpr int VE = VB / SZ, VP = D / (8 * VE);                // elements of it, pieces a lane and value row
    static constexpr int VOFF = 2 * KP * KB * 32;
    static constexpr int SOFF = VOFF + 4 * VP * VB * 32;
    static constexpr int STAGE = SOFF + (F8 ? 2 * 4 * 32 : 0);
    static constexpr int ROWS = WIDE ? 16 : 8;
    static constexpr int FIFO = kWarps * STAGES * STAGE, MERGE = kWarps * ROWS * (D + 2) * 4;
    static constexpr int BUF = FIFO > MERGE ? FIFO : MERGE;
    static constexpr int SMEM = BUF + 2 * D * SZ + 16;
    static constexpr int NT = D / 8;                                     // n-tiles of the output
    static constexpr int KS = D / 16;                                    // steps of the contraction over D
};

template <int D, bool F8, bool WIDE, int STAGES, int CTAS>
__global__ void __launch_bounds__(kWarps * 32, CTAS) step_mma_kernel(const StepArgs a) {
    using C = Cfg<D, F8, WIDE, STAGES>;
    extern __shared__ __align__(16) char smem[];
    char* const fresh = smem + C::BUF;
    uint8_t* const fresh_scale = reinterpret_cast<uint8_t*>(fresh + 2 * D * C::SZ);
    stream_wait();
    const PageArgs& c = a.c;
    const int blocks_h = (a.G + 15) / 16, hb = blockIdx.y % blocks_h, h = blockIdx.y / blocks_h, s = blockIdx.z, part = blockIdx.x;
    const Range r = range_of(a, s, part);
    if (part && r.first >= r.length) return;                   // part 0 always answers
    const int heads = min(16, a.G - hb * 16);
    const long long q0 = ((long long)s * c.H + h) * a.G + hb * 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const bool has_new = a.k_new != nullptr && r.end == r.length && r.length > 0;
    const int last = has_new ? r.length - 1 : -1, old_end = has_new ? r.length - 1 : r.end;     // rows in front of old_end come from the pages

    char* const fifo = smem + warp * STAGES * C::STAGE;
    const int first_tile = r.first + warp * kTile, tiles = r.end > first_tile ? (r.end - first_tile + kWarps * kTile - 1) / (kWarps * kTile) : 0;
    bool bad = r.bad;

    const auto page_rows = [&](int i) -> long long {           // first row of tile i, -1: no page
        const int p = first_tile + i * (kWarps * kTile);
        if (i >= tiles) return 0;
        const long long rows = c.rows_of(s, h, p / c.page);
        return rows < 0 ? -1 : rows + p % c.page;
    };
    const auto issue = [&](int i, long long row0) {
        if (i < tiles) {
            char* const st = fifo + (i % STAGES) * C::STAGE;
            const int p = first_tile + i * (kWarps * kTile), n = row0 < 0 ? 0 : old_end - p;      // rows of the tile that exist
            if (row0 < 0) { bad = true; row0 = 0; }
            const char* const base = c.kv + row0 * (2 * D * C::SZ);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int k = 0; k < C::KP; ++k)
                    copy_async<C::KB>(st + ((j * C::KP + k) * 32 + lane) * C::KB, base + (g + 8 * j) * (2 * D * C::SZ) + (4 * k + t) * C::KB, g + 8 * j < n);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = 2 * t + (j & 1) + 8 * (j >> 1);
#pragma unroll
                for (int k = 0; k < C::VP; ++k)
                    copy_async<C::VB>(st + C::VOFF + ((j * C::VP + k) * 32 + lane) * C::VB, base + key * (2 * D * C::SZ) + D * C::SZ + (8 * k + g) * C::VB, key < n);
            }
            if constexpr (F8) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    copy_async<4>(st + C::SOFF + (j * 32 + lane) * 4, reinterpret_cast<const char*>(c.scale) + (row0 + 8 * j + 2 * t) * 2, true);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    long long next = page_rows(0);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
        const long long row0 = next;
        next = page_rows(i + 1);
        issue(i, row0);
    }

    // ---- queries as the A operand: registers 0 and 2 row g, 1 and 3 row g + 8
    uint32_t qa[C::KS][4];
    float fs[2] = {a.scale, a.scale};
    {
        const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + q0 * D;
        constexpr int E = C::KB / C::SZ;                       // elements of a piece: E / 4 steps
#pragma unroll
        for (int row = 0; row < 2; ++row) {
            const int hr = g + 8 * row;
            const bool on = hr < heads && (WIDE || row == 0);
#pragma unroll
            for (int k = 0; k < C::KP; ++k)
#pragma unroll
                for (int e = 0; e < E / 4; ++e) {
                    uint2 u = make_uint2(0u, 0u);
                    if (on) u = *reinterpret_cast<const uint2*>(q + hr * D + (4 * k + t) * E + 4 * e);
                    qa[k * (E / 4) + e][row] = u.x; qa[k * (E / 4) + e][2 + row] = u.y;
                }
            if constexpr (F8) {
                uint32_t top = 0u;
#pragma unroll
                for (int k = 0; k < C::KS; ++k)
#pragma unroll
                    for (int e = 0; e < 2; ++e) top = max(top, max(qa[k][row + 2 * e] << 16 & 0x7fff0000u, qa[k][row + 2 * e] & 0x7fff0000u));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1)); top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // largest element to [1, 2): nothing is lost but what is below 2^-25 of it.  NaN and infinity stay what they are.
                int ex = (int)(top >> 23);
                ex = ex == 0 ? 127 : ex >= 254 ? 253 : ex;
                const float down = __uint_as_float((254u - ex) << 23);
                fs[row] = a.scale * __uint_as_float((uint32_t)ex << 23);
#pragma unroll
                for (int k = 0; k < C::KS; ++k)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t& w = qa[k][row + 2 * e];
                        w = pack_f16x2(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xffff0000u) * down);
                    }
            }
        }
    }
    if (has_new) {
        if (warp == 0) new_row(a, s, h, last, hb == 0, fresh, fresh_scale);
        __syncthreads();
    }

    float o[C::NT][4];
#pragma unroll
    for (int n = 0; n < C::NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
    constexpr int HALVES = WIDE ? 2 : 1;                       // rows g, and g + 8
    float m[HALVES], l[HALVES];
#pragma unroll
    for (int i = 0; i < HALVES; ++i) { m[i] = -INFINITY; l[i] = 0.f; }
    uint32_t vtop = 0u;                                        // largest scale byte of a value row so far

#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
        {
            const long long row0 = next;
            next = page_rows(i + STAGES);
            issue(i + STAGES - 1, row0);
        }
        asm volatile("cp.async.wait_group %0;" :: "n"(STAGES - 1) : "memory");
        char* const st = fifo + (i % STAGES) * C::STAGE;
        const int p = first_tile + i * (kWarps * kTile);
        if (last >= p && last < p + kTile) {                   // the new token's row: from where new_row left it
            const int key = last - p;
            if (g == (key & 7)) {
                const int j = key >> 3;
#pragma unroll
                for (int k = 0; k < C::KP; ++k)
#pragma unroll
                    for (int b = 0; b < C::KB; b += 8)
                        *reinterpret_cast<uint2*>(st + ((j * C::KP + k) * 32 + lane) * C::KB + b) = *reinterpret_cast<const uint2*>(fresh + (4 * k + t) * C::KB + b);
            }
            if (t == (key & 7) >> 1) {
                const int j = (key & 1) + 2 * (key >> 3);
#pragma unroll
                for (int k = 0; k < C::VP; ++k)
#pragma unroll
                    for (int b = 0; b < C::VB; b += 4)
                        *reinterpret_cast<uint32_t*>(st + C::VOFF + ((j * C::VP + k) * 32 + lane) * C::VB + b) =
                            *reinterpret_cast<const uint32_t*>(fresh + D * C::SZ + (8 * k + g) * C::VB + b);
                if constexpr (F8) {
                    uint8_t* b = reinterpret_cast<uint8_t*>(st + C::SOFF + ((key >> 3) * 32 + lane) * 4) + 2 * (key & 1);
                    b[0] = fresh_scale[0]; b[1] = fresh_scale[1];
                }
            }
        }
        // ---- scores of 16 positions: column 2 t and 2 t + 1 of each half
        float sc[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[j][e] = 0.f;
#pragma unroll
            for (int k = 0; k < C::KP; ++k) {
                uint32_t w[C::KB / 4];
                const char* from = st + ((j * C::KP + k) * 32 + lane) * C::KB;
                if constexpr (C::KB == 16) { const uint4 u = *reinterpret_cast<const uint4*>(from); w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w; }
                else { const uint2 u = *reinterpret_cast<const uint2*>(from); w[0] = u.x; w[1] = u.y; }
                if constexpr (F8) {
#pragma unroll
                    for (int e = 0; e < C::KB / 4; ++e)
                        mma<true>(sc[j], qa[k * (C::KB / 4) + e], half2_bits(e4m3x2_half2(w[e] & 0xffffu)), half2_bits(e4m3x2_half2(w[e] >> 16)));
                } else {
                    mma<false>(sc[j], qa[2 * k], w[0], w[1]);
                    mma<false>(sc[j], qa[2 * k + 1], w[2], w[3]);
                }
            }
        }
        // ---- softmax: the scale bytes of positions 2 t, 2 t + 1 (+ 8) are {k, v, k, v}
        uint32_t sb[2];
        bool valid[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if constexpr (F8) sb[j] = *reinterpret_cast<const uint32_t*>(st + C::SOFF + (j * 32 + lane) * 4);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                valid[j][e] = p + 8 * j + 2 * t + e < r.end;
                if constexpr (F8) {
                    const float ks = scale_value(sb[j] >> (16 * e) & 255u);
                    sc[j][e] *= ks; sc[j][2 + e] *= ks;
                }
            }
        }
        float vs[2][2];
        if constexpr (F8) {
            uint32_t top = 0u;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t b = sb[j] >> (16 * e + 8) & 255u;
                    if (valid[j][e] && b != 255u) top = max(top, b);
                }
            top = __reduce_max_sync(0xffffffffu, top);
            if (top > vtop) {                                  // rarely: the scales of a head's values are much alike
                const int e = 127 + (int)vtop - (int)top;
                const float f = e > 0 ? __uint_as_float((uint32_t)e << 23) : 0.f;
#pragma unroll
                for (int n = 0; n < C::NT; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[n][x] *= f;
                vtop = top;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t b = sb[j] >> (16 * e + 8) & 255u;
                    const int x = 127 + (int)b - (int)vtop;
                    vs[j][e] = !valid[j][e] ? 0.f : b == 255u ? __uint_as_float(0x7fc00000u) : x > 0 ? __uint_as_float((uint32_t)x << 23) : 0.f;
                }
        }
        uint32_t pa[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i2 = 0; i2 < HALVES; ++i2) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float& x = sc[j][2 * i2 + e];
                    x = valid[j][e] ? x * fs[i2] : -INFINITY;
                    mx = fmaxf(mx, x);
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1)); mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            if (__any_sync(0xffffffffu, mx > m[i2])) {
                const float mn = fmaxf(m[i2], mx), f = mn == -INFINITY ? 1.f : exp2f(m[i2] - mn);
                l[i2] *= f;
#pragma unroll
                for (int n = 0; n < C::NT; ++n) { o[n][2 * i2] *= f; o[n][2 * i2 + 1] *= f; }
                m[i2] = mn;
            }
            const float base = m[i2] == -INFINITY ? 0.f : m[i2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float x[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    x[e] = exp2f(sc[j][2 * i2 + e] - base);
                    l[i2] += x[e];
                    if constexpr (F8) x[e] *= vs[j][e];
                }
                // to 16 bits, as the operand of the product: relative 2^-9 (bf16) or 2^-12 (f16) on terms that add up, within the result's own rounding
                pa[2 * j + i2] = F8 ? pack_f16x2(x[0], x[1]) : pack_bf16x2(x[0], x[1]);
            }
        }
        // ---- O += P V: n-tile k VE + e has column n at d = 8 VE k + VE n + e
#pragma unroll
        for (int k = 0; k < C::VP; ++k) {
            uint32_t w[4][C::VB / 4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const char* from = st + C::VOFF + ((j * C::VP + k) * 32 + lane) * C::VB;
                if constexpr (C::VB == 16) { const uint4 u = *reinterpret_cast<const uint4*>(from); w[j][0] = u.x; w[j][1] = u.y; w[j][2] = u.z; w[j][3] = u.w; }
                else if constexpr (C::VB == 8) { const uint2 u = *reinterpret_cast<const uint2*>(from); w[j][0] = u.x; w[j][1] = u.y; }
                else w[j][0] = *reinterpret_cast<const uint32_t*>(from);
            }
            // pairs of columns of four positions -> the B operands of two n-tiles
            const auto two = [&](int n, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
                mma<F8>(o[n], pa, __byte_perm(w0, w1, 0x5410), __byte_perm(w2, w3, 0x5410));
                mma<F8>(o[n + 1], pa, __byte_perm(w0, w1, 0x7632), __byte_perm(w2, w3, 0x7632));
            };
#pragma unroll
            for (int x = 0; x < C::VB / 4; ++x) {
                if constexpr (F8) {
                    two(k * C::VE + 4 * x, half2_bits(e4m3x2_half2(w[0][x] & 0xffffu)), half2_bits(e4m3x2_half2(w[1][x] & 0xffffu)),
                        half2_bits(e4m3x2_half2(w[2][x] & 0xffffu)), half2_bits(e4m3x2_half2(w[3][x] & 0xffffu)));
                    two(k * C::VE + 4 * x + 2, half2_bits(e4m3x2_half2(w[0][x] >> 16)), half2_bits(e4m3x2_half2(w[1][x] >> 16)),
                        half2_bits(e4m3x2_half2(w[2][x] >> 16)), half2_bits(e4m3x2_half2(w[3][x] >> 16)));
                } else two(k * C::VE + 2 * x, w[0][x], w[1][x], w[2][x], w[3][x]);
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // ---- the four warps' results, joined in warp order
    const bool any_bad = __syncthreads_or(bad);
    float* const sml = reinterpret_cast<float*>(smem);         // [warps][rows][2]
    float* const so = sml + kWarps * C::ROWS * 2;              // [warps][rows][D]
    const float unit = F8 ? scale_value(vtop) : 1.f;
#pragma unroll
    for (int i = 0; i < HALVES; ++i) {
        const int row = g + 8 * i;
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1); l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if (t == 0) { sml[(warp * C::ROWS + row) * 2] = m[i]; sml[(warp * C::ROWS + row) * 2 + 1] = l[i]; }
#pragma unroll
        for (int k = 0; k < C::VP; ++k)
#pragma unroll
            for (int e = 0; e < C::VE; ++e)
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    so[(warp * C::ROWS + row) * D + 8 * C::VE * k + C::VE * (2 * t + x) + e] = o[k * C::VE + e][2 * i + x] * unit;
    }
    __syncthreads();
    for (int z = threadIdx.x; z < heads * D; z += kWarps * 32) {
        const int row = z / D, d = z - row * D;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sml[(w * C::ROWS + row) * 2]);
        const float base = M == -INFINITY ? 0.f : M;
        float L = 0.f, A = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = exp2f(sml[(w * C::ROWS + row) * 2] - base);
            L = fmaf(f, sml[(w * C::ROWS + row) * 2 + 1], L); A = fmaf(f, so[(w * C::ROWS + row) * D + d], A);
        }
        if (any_bad) L = A = __uint_as_float(0x7fc00000u);
        if (a.ml) {
            const long long at = (q0 + row) * a.parts + part;
            if (d == 0) a.ml[at] = make_float2(M, L);
            a.acc[at * D + d] = A;
        } else static_cast<__nv_bfloat16*>(a.out)[(q0 + row) * D + d] = __float2bfloat16(L == 0.f ? 0.f : A / L);
    }
}

template <int D, bool F8, bool WIDE, int STAGES, int CTAS> cudaError_t launch_one(const StepArgs& a, cudaStream_t s) {
    using C = Cfg<D, F8, WIDE, STAGES>;
    auto kern = step_mma_kernel<D, F8, WIDE, STAGES, CTAS>;
    static bool ready[64] = {};                                // per device: the attribute is set once
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return e;
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)) { cudaGetLastError(); return e; }
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    return launch_after(kern, dim3(a.parts, a.c.H * ((a.G + 15) / 16), a.c.S), kWarps * 32, C::SMEM, s, a);
}
template <int D, bool F8> cudaError_t launch_width(const StepArgs& a, cudaStream_t s) {
    constexpr int STAGES = F8 ? 4 : D > 64 ? 3 : 4;
    return a.G > 8 ? launch_one<D, F8, true, STAGES, 2>(a, s) : launch_one<D, F8, false, STAGES, 2>(a, s);
}
template <bool F8> cudaError_t launch_type(const StepArgs& a, cudaStream_t s) {
    switch (a.c.D) {
        case 32: return launch_width<32, F8>(a, s);
        case 64: return launch_width<64, F8>(a, s);
        case 96: return launch_width<96, F8>(a, s);
        default: return launch_width<128, F8>(a, s);
    }
}

}  // namespace

bool paged_mma_supported(const StepArgs& a) {
    return !a.q_f32 && (a.c.dtype == DSQG_DTYPE_BF16 || a.c.dtype == DSQG_DTYPE_E4M3) && a.c.D % 32 == 0 && a.c.page % kTile == 0 &&
           (reinterpret_cast<uintptr_t>(a.c.scale) & 3u) == 0;
}
cudaError_t launch_paged_mma(const StepArgs& a, cudaStream_t s) { return a.c.dtype == DSQG_DTYPE_E4M3 ? launch_type<true>(a, s) : launch_type<false>(a, s); }

}  // namespace dsqg
