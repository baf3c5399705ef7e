// Products with 4-bit weights: y = x W^T + b, W[n][k] = (nibble - 8) * scales[n][k / group], for few rows of x (the tokens of a decode step).
//
// What counts is reading the weights once.  A block takes 16 RT rows of W, its warps every W-th tile of 128 columns; tiles come by cp.async some
// stages ahead.  The weights are the A operand of mma.sync (m16n8k16), eight tokens the B operand, fp32 accumulators: a nibble becomes
// a 16-bit float by setting it into the mantissa of 128 (bf16) or 1024 (f16) and subtracting 136 or 1032, which rounds nothing; x is bf16, or
// e4m3 which f16 holds exactly.  The contraction may be permuted freely as long as both operands agree: a lane takes words of eight nibbles, and
// a pair of an operand is nibbles i and i + 4 of a word, so that one mask serves both.  A step of the contraction lies inside one group of 32 columns,
// so a group's products are summed unscaled and its scale is applied to the fp32 sum.  Warps are added in order through shared memory.
#include "dsqg_rows8.cuh"

namespace dsqg {
namespace {

constexpr int kWarps = 8, kCols = 128;                         // columns of a tile: four chunks of 32

struct Int4Args {
    const void* x; const uint8_t* x_scale; const uint8_t* w; const __nv_bfloat16* scales; const float* bias; __nv_bfloat16* y;
    int M, N, K, groups;                                       // groups: K / group
};

template <bool F16> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Nibbles i and i + 4 of w, less 8, as two 16-bit floats.
template <bool F16> __device__ __forceinline__ uint32_t weights(uint32_t w, int i) {
    const uint32_t u = (w >> (4 * i) & 0x000f000fu) | (F16 ? 0x64006400u : 0x43004300u);
    if constexpr (F16) {
        const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), __float2half2_rn(1032.f));
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), __float2bfloat162_rn(136.f));
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}
template <int BYTES> __device__ __forceinline__ void copy_async(char* to, const void* from, bool on) {
    const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(to));
    const int n = on ? BYTES : 0;
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(d), "l"(from), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" :: "r"(d), "l"(from), "n"(BYTES), "r"(n) : "memory");
}

// F8: x in e4m3.  NT: tiles of eight tokens.  RT: tiles of 16 rows of W.  GC: chunks of 32 columns in a group.
template <bool F8, int NT, int RT, int GC, int STAGES>
__global__ void __launch_bounds__(kWarps * 32) int4_kernel(const Int4Args a) {
    constexpr int XB = F8 ? 8 : 16;                            // bytes of eight elements of x
    constexpr int WSTAGE = RT * 16 * (kCols / 2), STAGE = WSTAGE + NT * 4 * 32 * XB;
    extern __shared__ __align__(16) char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16 * RT, m0 = blockIdx.y * 8 * NT;
    char* const fifo = smem + warp * STAGES * STAGE;
    const int all = (a.K + kCols - 1) / kCols, tiles = warp < all ? (all - warp + kWarps - 1) / kWarps : 0;
    stream_wait();

    float sr[STAGES][RT][2];                                   // scales of rows g, g + 8, chunk t of a tile
    const auto issue = [&](int i, int stage) {
        const int k0 = (warp + i * kWarps) * kCols;
        if (i < tiles) {
            char* const st = fifo + stage * STAGE;
#pragma unroll
            for (int j = 0; j < 2 * RT; ++j) {                 // 16 bytes a lane: row 8 j + g, chunk t, placed so that the words are read without bank conflicts
                const int row = 8 * j + g, k = k0 + 32 * t;
                const bool on = k < a.K;
                copy_async<16>(st + row * 64 + ((t ^ (row >> 1)) & 3) * 16, a.w + (size_t)min(n0 + row, a.N - 1) * (a.K / 2) + (on ? k / 2 : 0), on);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) {                  // token 8 j + g, eight elements of chunk c
                    const int token = m0 + 8 * j + g, k = k0 + 32 * c + 8 * t;
                    const bool on = token < a.M && k < a.K;
                    copy_async<XB>(st + WSTAGE + ((j * 4 + c) * 32 + lane) * XB, static_cast<const char*>(a.x) + (on ? ((size_t)token * a.K + k) * (F8 ? 1 : 2) : 0), on);
                }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = k0 + 32 * t;
                sr[stage][j][e] = i < tiles && k < a.K ? __bfloat162float(a.scales[(size_t)min(n0 + 16 * j + 8 * e + g, a.N - 1) * a.groups + k / (32 * GC)]) : 0.f;
            }
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(i, i);

    float total[RT][NT][4];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) total[r][n][e] = 0.f;

    for (int base = 0; base < tiles; base += STAGES) {
#pragma unroll
        for (int stage = 0; stage < STAGES; ++stage) {
            const int i = base + stage;
            if (i >= tiles) break;
            issue(i + STAGES - 1, (stage + STAGES - 1) % STAGES);
            asm volatile("cp.async.wait_group %0;" :: "n"(STAGES - 1) : "memory");
            __syncwarp();
            const char* const st = fifo + stage * STAGE;
            float part[RT][NT][4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (c % GC == 0) {
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) part[r][n][e] = 0.f;
                }
                uint32_t xb[NT][4];                            // pairs (0, 4), (1, 5), (2, 6), (3, 7) of the lane's eight elements
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint32_t w[4];
                    const char* from = st + WSTAGE + ((n * 4 + c) * 32 + lane) * XB;
                    if constexpr (F8) {
                        const uint2 u = *reinterpret_cast<const uint2*>(from);
                        const __half2 h[4] = {e4m3x2_half2(u.x & 0xffffu), e4m3x2_half2(u.x >> 16), e4m3x2_half2(u.y & 0xffffu), e4m3x2_half2(u.y >> 16)};
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = *reinterpret_cast<const uint32_t*>(&h[e]);
                    } else { const uint4 u = *reinterpret_cast<const uint4*>(from); w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w; }
                    xb[n][0] = __byte_perm(w[0], w[2], 0x5410); xb[n][1] = __byte_perm(w[0], w[2], 0x7632);
                    xb[n][2] = __byte_perm(w[1], w[3], 0x5410); xb[n][3] = __byte_perm(w[1], w[3], 0x7632);
                }
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const char* row = st + (16 * r + g) * 64 + ((c ^ (g >> 1)) & 3) * 16 + 4 * t;       // row g + 8: the same place, (g + 8) >> 1 = g >> 1 mod 4
                    const uint32_t w0 = *reinterpret_cast<const uint32_t*>(row), w1 = *reinterpret_cast<const uint32_t*>(row + 8 * 64);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t wa[4] = {weights<F8>(w0, 2 * h), weights<F8>(w1, 2 * h), weights<F8>(w0, 2 * h + 1), weights<F8>(w1, 2 * h + 1)};
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma<F8>(part[r][n], wa, xb[n][2 * h], xb[n][2 * h + 1]);
                    }
                    if (c % GC == GC - 1) {
                        const float s0 = __shfl_sync(0xffffffffu, sr[stage][r][0], (lane & ~3) | c), s1 = __shfl_sync(0xffffffffu, sr[stage][r][1], (lane & ~3) | c);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            total[r][n][0] = fmaf(s0, part[r][n][0], total[r][n][0]); total[r][n][1] = fmaf(s0, part[r][n][1], total[r][n][1]);
                            total[r][n][2] = fmaf(s1, part[r][n][2], total[r][n][2]); total[r][n][3] = fmaf(s1, part[r][n][3], total[r][n][3]);
                        }
                    }
                }
            }
            __syncwarp();                                      // the stage is free for the next copies
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    // ---- [warp][token][row], added in warp order
    constexpr int ROWS = 16 * RT, TOKENS = 8 * NT, PITCH = ROWS + 1;
    float* const red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[(warp * TOKENS + 8 * n + 2 * t + (e & 1)) * PITCH + 16 * r + g + 8 * (e >> 1)] = total[r][n][e];
    __syncthreads();
    for (int z = threadIdx.x; z < ROWS * TOKENS; z += kWarps * 32) {
        const int row = z % ROWS, token = z / ROWS, n = n0 + row, m = m0 + token;
        if (n >= a.N || m >= a.M) continue;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) s += red[(w * TOKENS + token) * PITCH + row];
        if constexpr (F8) s *= scale_value(a.x_scale[m]);
        if (a.bias) s += a.bias[n];
        a.y[(size_t)m * a.N + n] = __float2bfloat16(s);
    }
}

template <bool F8, int NT, int RT, int GC, int STAGES> cudaError_t launch_one(const Int4Args& a, cudaStream_t s) {
    constexpr int FIFO = kWarps * STAGES * (RT * 16 * (kCols / 2) + NT * 4 * 32 * (F8 ? 8 : 16)), RED = kWarps * 8 * NT * (16 * RT + 1) * 4;
    constexpr int SMEM = FIFO > RED ? FIFO : RED;
    auto kern = int4_kernel<F8, NT, RT, GC, STAGES>;
    if (SMEM > 48 * 1024) {
        static bool ready[64] = {};                            // per device: the attribute is set once
        int dev = 0;
        if (cudaError_t e = cudaGetDevice(&dev)) return e;
        if (dev < 0 || dev >= 64 || !ready[dev]) {
            if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM)) { cudaGetLastError(); return e; }
            if (dev >= 0 && dev < 64) ready[dev] = true;
        }
    }
    return launch_after(kern, dim3((a.N + 16 * RT - 1) / (16 * RT), (a.M + 8 * NT - 1) / (8 * NT)), kWarps * 32, SMEM, s, a);
}
template <bool F8, int NT, int RT> cudaError_t launch_group(const Int4Args& a, int group, cudaStream_t s) {
    return group == 32 ? launch_one<F8, NT, RT, 1, 4>(a, s) : group == 64 ? launch_one<F8, NT, RT, 2, 4>(a, s) : launch_one<F8, NT, RT, 4, 4>(a, s);
}
template <bool F8> cudaError_t launch_type(const Int4Args& a, int group, cudaStream_t s) {
    return a.M <= 8 ? launch_group<F8, 1, 1>(a, group, s) : launch_group<F8, 2, 1>(a, group, s);
}

inline bool bad(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

}  // namespace
}  // namespace dsqg

using namespace dsqg;

extern "C" {

int dsqg_int4_linear(const void* x, const void* x_scale, const void* weight, const void* scales, const float* bias, void* y, int M, int N, int K, int group, int dtype,
                     void* stream) {
    if (!x || !weight || !scales || !y || (dtype == DSQG_DTYPE_E4M3 && !x_scale)) return DSQG_ERR_NULL_POINTER;
    if (dtype != DSQG_DTYPE_BF16 && dtype != DSQG_DTYPE_E4M3) return DSQG_ERR_BAD_DTYPE;
    if (group != 32 && group != 64 && group != 128) return DSQG_ERR_UNSUPPORTED;
    if (M < 1 || N < 1 || K < group || K % group || M > 65535 * 8) return DSQG_ERR_BAD_SHAPE;
    if (bad(x) || bad(weight)) return DSQG_ERR_MISALIGNED;
    const Int4Args a = {x, static_cast<const uint8_t*>(x_scale), static_cast<const uint8_t*>(weight), static_cast<const __nv_bfloat16*>(scales), bias,
                        static_cast<__nv_bfloat16*>(y), M, N, K, K / group};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return (dtype == DSQG_DTYPE_E4M3 ? launch_type<true>(a, group, s) : launch_type<false>(a, group, s)) == cudaSuccess ? DSQG_OK : DSQG_ERR_CUDA;
}

}  // extern "C"
