// Root-mean-square norm of a residual stream with the addition in front of it, forward and backward.
//
//   h = x + r (rounded to r's type: the stream the next layer reads), rstd = 1 / sqrt(mean(h^2) + eps), y = h rstd w
//   dh = dh_out + rstd (w dy - x^ mean(w dy x^)), x^ = h rstd;  dx = dr = dh;  dw = sum over rows of dy x^
//
// The norm is of h as it is stored, which is what the backward pass and the next layer see.  fp32 arithmetic throughout.  y leaves in bf16,
// fp32 or e4m3 with a power-of-two scale per row (dsqg_rows8.cuh).  Bound by memory: every tensor is read and written once, a row stays
// in registers between its reduction and its result.
#include "dsqg_rows8.cuh"

namespace dsqg {
namespace {

constexpr int kThreads = 256;

// W consecutive elements as they lie in memory (bf16 or fp32), so that every load of a row is under way before one is used.
template <int W> struct Piece;
template <> struct Piece<8> {
    uint4 a, b;
    __device__ __forceinline__ void load(const void* p, long long i, bool f32) {
        const uint4* s = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + i * (f32 ? 4 : 2));
        a = __ldg(s);
        if (f32) b = __ldg(s + 1);
    }
    __device__ __forceinline__ void get(float (&x)[8], bool f32) const {
        const uint32_t u[4] = {a.x, a.y, a.z, a.w}, v[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (f32) { x[i] = __uint_as_float(u[i]); x[4 + i] = __uint_as_float(v[i]); }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!f32) { x[2 * i] = __uint_as_float(u[i] << 16); x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
        }
    }
};
template <> struct Piece<1> {
    uint32_t a;
    __device__ __forceinline__ void load(const void* p, long long i, bool f32) {
        if (f32) a = __ldg(static_cast<const uint32_t*>(p) + i);
        else a = (uint32_t)__ldg(static_cast<const unsigned short*>(p) + i) << 16;
    }
    __device__ __forceinline__ void get(float (&x)[1], bool) const { x[0] = __uint_as_float(a); }
};
template <int W> __device__ __forceinline__ void put(void* p, long long i, int dtype, const float (&x)[W]) {
    if constexpr (W == 8) store8_as(p, i, dtype, x);
    else if (dtype == DSQG_DTYPE_F32) static_cast<float*>(p)[i] = x[0];
    else if (dtype == DSQG_DTYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16(x[0]);
    else static_cast<uint8_t*>(p)[i] = (uint8_t)__nv_cvt_float_to_fp8(x[0], __NV_SATFINITE, __NV_E4M3);
}

// Sum, or maximum, over the TPR threads of a row.  red: two slots a warp, used in turn, so that one barrier an exchange is enough.
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* red, int& turn) {
    v = group_sum<(TPR < 32 ? TPR : 32)>(v);
    if constexpr (TPR > 32) {
        float* slot = red + (turn ^= 1) * 32;
        if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < TPR / 32; ++w) v += slot[w];
    }
    return v;
}
template <int TPR> __device__ __forceinline__ uint32_t row_max(uint32_t v, float* red, int& turn) {
    v = group_max<(TPR < 32 ? TPR : 32)>(v);
    if constexpr (TPR > 32) {
        uint32_t* slot = reinterpret_cast<uint32_t*>(red + (turn ^= 1) * 32);
        if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0u;
#pragma unroll
        for (int w = 0; w < TPR / 32; ++w) v = max(v, slot[w]);
    }
    return v;
}

struct NormArgs {
    const void* x; const void* r; const float* w; void* h; void* y; uint8_t* scale; float* rstd;
    long long rows; int D; float eps; int x_f32, s_dt, y_dt;
};

// TPR threads a row (a block of max(TPR, kThreads) threads), V pieces of W elements a thread.
template <int W, int TPR, int V>
__global__ void __launch_bounds__(TPR < kThreads ? kThreads : TPR) rms_fwd_kernel(const NormArgs a) {
    constexpr int kBlock = TPR < kThreads ? kThreads : TPR;
    __shared__ float red[64];
    int turn = 0;
    const int t = threadIdx.x % TPR;
    const long long row0 = (long long)blockIdx.x * (kBlock / TPR) + threadIdx.x / TPR;
    const bool live = row0 < a.rows;
    const long long at = (live ? row0 : a.rows - 1) * a.D;
    const bool s_f32 = a.s_dt == DSQG_DTYPE_F32;
    stream_wait();
    Piece<W> px[V], pr[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (v * TPR + t) * W;
        if (c < a.D) {
            px[v].load(a.x, at + c, a.x_f32);
            if (a.r) pr[v].load(a.r, at + c, s_f32);
        }
    }
    float h[V][W], ss = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (v * TPR + t) * W;
        if (c < a.D) {
            px[v].get(h[v], a.x_f32);
            if (a.r) {
                float r[W];
                pr[v].get(r, s_f32);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    h[v][e] += r[e];
                    if (!s_f32) h[v][e] = __bfloat162float(__float2bfloat16(h[v][e]));
                }
                if (live) put<W>(a.h, at + c, a.s_dt, h[v]);
            }
#pragma unroll
            for (int e = 0; e < W; ++e) ss = fmaf(h[v][e], h[v][e], ss);
        }
    }
    const float rstd = rsqrtf(row_sum<TPR>(ss, red, turn) / a.D + a.eps);
    if (a.rstd && live && t == 0) a.rstd[row0] = rstd;
    uint32_t top = 0u;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (v * TPR + t) * W;
        if (c < a.D) {
            float w[W];
            if constexpr (W == 8) load8(a.w + c, w); else w[0] = __ldg(a.w + c);
#pragma unroll
            for (int e = 0; e < W; ++e) { h[v][e] = h[v][e] * rstd * w[e]; top = max(top, abs_bits(h[v][e])); }
        }
    }
    float inv = 1.f;
    if (a.y_dt == DSQG_DTYPE_E4M3) {
        const uint32_t byte = row_scale_byte(row_max<TPR>(top, red, turn));
        inv = scale_inverse(byte);
        if (live && t == 0) a.scale[row0] = (uint8_t)byte;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (v * TPR + t) * W;
        if (c < a.D && live) {
#pragma unroll
            for (int e = 0; e < W; ++e) h[v][e] *= inv;
            put<W>(a.y, at + c, a.y_dt, h[v]);
        }
    }
}

// Rows of any width, re-read where a block's registers do not hold them.
__global__ void __launch_bounds__(1024) rms_fwd_wide_kernel(const NormArgs a) {
    __shared__ float red[64];
    int turn = 0;
    stream_wait();
    const long long at = (long long)blockIdx.x * a.D;
    const bool s_f32 = a.s_dt == DSQG_DTYPE_F32;
    const auto value = [&](int c) {
        Piece<1> p;
        float x[1], r[1];
        p.load(a.x, at + c, a.x_f32); p.get(x, a.x_f32);
        if (a.r) {
            p.load(a.r, at + c, s_f32); p.get(r, s_f32);
            x[0] += r[0];
            if (!s_f32) x[0] = __bfloat162float(__float2bfloat16(x[0]));
        }
        return x[0];
    };
    float ss = 0.f;
    for (int c = threadIdx.x; c < a.D; c += 1024) { const float x = value(c); ss = fmaf(x, x, ss); }
    const float rstd = rsqrtf(row_sum<1024>(ss, red, turn) / a.D + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[blockIdx.x] = rstd;
    float inv = 1.f;
    if (a.y_dt == DSQG_DTYPE_E4M3) {
        uint32_t top = 0u;
        for (int c = threadIdx.x; c < a.D; c += 1024) top = max(top, abs_bits(value(c) * rstd * __ldg(a.w + c)));
        const uint32_t byte = row_scale_byte(row_max<1024>(top, red, turn));
        inv = scale_inverse(byte);
        if (threadIdx.x == 0) a.scale[blockIdx.x] = (uint8_t)byte;
    }
    for (int c = threadIdx.x; c < a.D; c += 1024) {
        const float x[1] = {value(c)}, y[1] = {x[0] * rstd * __ldg(a.w + c) * inv};
        if (a.r) put<1>(a.h, at + c, a.s_dt, x);
        put<1>(a.y, at + c, a.y_dt, y);
    }
}

struct NormGradArgs {
    const void* h; const float* rstd; const float* w; const void* dy; const void* dh; void* dx; void* dr; float* part;
    long long rows; int D; int s_dt, y_dt, x_dt;
};

// Blocks of the backward kernel that an SM holds: the grid is that many times 148, so that all of them start at once and walk the same number of rows
// (four an SM where registers allow three took a second wave of blocks that then had a quarter of the rows to itself: 53 us instead of 44 at 65,536 x 256).
constexpr int grad_blocks_an_sm(int W, int TPR, int V) { return TPR > 256 ? 1 : W * V >= 32 ? 1 : W * V >= 16 ? 2 : 3; }

// A block walks rows a grid apart; a thread keeps the sums of its columns of dw.  The partial sums of a block's rows go to part[block],
// added by dw_kernel: the order follows from the sizes alone.
template <int W, int TPR, int V>
__global__ void __launch_bounds__(TPR < kThreads ? kThreads : TPR, grad_blocks_an_sm(W, TPR, V)) rms_bwd_kernel(const NormGradArgs a) {
    constexpr int kBlock = TPR < kThreads ? kThreads : TPR, kRows = kBlock / TPR;
    __shared__ float red[64];
    extern __shared__ float sums[];
    int turn = 0;
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const bool s_f32 = a.s_dt == DSQG_DTYPE_F32, y_f32 = a.y_dt == DSQG_DTYPE_F32;
    float dw[V][W];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < W; ++e) dw[v][e] = 0.f;
    stream_wait();
    for (long long first = (long long)blockIdx.x * kRows; first < a.rows; first += (long long)gridDim.x * kRows) {
        const bool live = first + group < a.rows;
        const long long row = live ? first + group : a.rows - 1, at = row * a.D;
        Piece<W> ph[V], py[V], pd[V];
        const float rstd = __ldg(a.rstd + row);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * TPR + t) * W;
            if (c < a.D) {
                ph[v].load(a.h, at + c, s_f32);
                py[v].load(a.dy, at + c, y_f32);
                if (a.dh) pd[v].load(a.dh, at + c, s_f32);
            }
        }
        float xh[V][W], g[V][W], s = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * TPR + t) * W;
            if (c < a.D) {
                float w[W];
                if constexpr (W == 8) load8(a.w + c, w); else w[0] = __ldg(a.w + c);
                ph[v].get(xh[v], s_f32); py[v].get(g[v], y_f32);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    xh[v][e] *= rstd;
                    if (live) dw[v][e] = fmaf(g[v][e], xh[v][e], dw[v][e]);
                    g[v][e] *= w[e];
                    s = fmaf(g[v][e], xh[v][e], s);
                }
            }
        }
        s = row_sum<TPR>(s, red, turn) / a.D;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * TPR + t) * W;
            if (c < a.D && live) {
                float d[W];
                if (a.dh) pd[v].get(d, s_f32);
#pragma unroll
                for (int e = 0; e < W; ++e) d[e] = fmaf(rstd, g[v][e] - xh[v][e] * s, a.dh ? d[e] : 0.f);
                if (a.dx) put<W>(a.dx, at + c, a.x_dt, d);
                if (a.dr) put<W>(a.dr, at + c, a.s_dt, d);
            }
        }
    }
    if (!a.part) return;
    float* out = a.part + (size_t)blockIdx.x * a.D;
    if constexpr (kRows == 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * TPR + t) * W;
            if (c < a.D)
#pragma unroll
                for (int e = 0; e < W; ++e) out[c + e] = dw[v][e];
        }
    } else {
        for (int k = 0; k < kRows; ++k) {                      // row groups in turn: fixed order of additions
            if (group == k) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const int c = (v * TPR + t) * W;
                    if (c < a.D)
#pragma unroll
                        for (int e = 0; e < W; ++e) sums[c + e] = k ? sums[c + e] + dw[v][e] : dw[v][e];
                }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < a.D; c += kBlock) out[c] = sums[c];
    }
}

// Rows of any width: dx and dr first, then the partial sums of dw by columns.
__global__ void __launch_bounds__(1024) rms_bwd_wide_kernel(const NormGradArgs a) {
    __shared__ float red[64];
    int turn = 0;
    stream_wait();
    const bool s_f32 = a.s_dt == DSQG_DTYPE_F32, y_f32 = a.y_dt == DSQG_DTYPE_F32;
    const long long at = (long long)blockIdx.x * a.D;
    const float rstd = __ldg(a.rstd + blockIdx.x);
    const auto get = [&](const void* p, int c, bool f32) { Piece<1> q; float x[1]; q.load(p, at + c, f32); q.get(x, f32); return x[0]; };
    float s = 0.f;
    for (int c = threadIdx.x; c < a.D; c += 1024) s = fmaf(get(a.dy, c, y_f32) * __ldg(a.w + c), get(a.h, c, s_f32) * rstd, s);
    s = row_sum<1024>(s, red, turn) / a.D;
    for (int c = threadIdx.x; c < a.D; c += 1024) {
        const float g = get(a.dy, c, y_f32) * __ldg(a.w + c), xh = get(a.h, c, s_f32) * rstd;
        const float d[1] = {fmaf(rstd, g - xh * s, a.dh ? get(a.dh, c, s_f32) : 0.f)};
        if (a.dx) put<1>(a.dx, at + c, a.x_dt, d);
        if (a.dr) put<1>(a.dr, at + c, a.s_dt, d);
    }
}
__global__ void __launch_bounds__(kThreads) dw_part_kernel(const NormGradArgs a) {
    stream_wait();
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= a.D) return;
    const bool s_f32 = a.s_dt == DSQG_DTYPE_F32, y_f32 = a.y_dt == DSQG_DTYPE_F32;
    float s = 0.f;
    for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        Piece<1> p;
        float h[1], g[1];
        p.load(a.h, row * a.D + c, s_f32); p.get(h, s_f32);
        p.load(a.dy, row * a.D + c, y_f32); p.get(g, y_f32);
        s = fmaf(g[0], h[0] * __ldg(a.rstd + row), s);
    }
    a.part[(size_t)blockIdx.y * a.D + c] = s;
}

// dw[c] = sum over the n rows of part: 32 columns a block, every 128th row a thread, all of them on their way together; added in row order of the threads.
__global__ void __launch_bounds__(1024) dw_kernel(const float* __restrict__ part, float* __restrict__ dw, int n, int D) {
    stream_wait();
    __shared__ float red[128][33];
    const int col = threadIdx.x & 7, row = threadIdx.x >> 3, c = blockIdx.x * 32 + 4 * col;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (D % 4 == 0 && c < D) {
#pragma unroll 8
        for (int b = row; b < n; b += 128) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(part + (size_t)b * D + c));
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
    } else {
        for (int b = row; b < n; b += 128) {
            const float* p = part + (size_t)b * D + c;
            if (c < D) s.x += p[0];
            if (c + 1 < D) s.y += p[1];
            if (c + 2 < D) s.z += p[2];
            if (c + 3 < D) s.w += p[3];
        }
    }
    red[row][4 * col] = s.x; red[row][4 * col + 1] = s.y; red[row][4 * col + 2] = s.z; red[row][4 * col + 3] = s.w;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) t += red[warp * 4 + i][lane];
    __syncthreads();
    red[warp][lane] = t;
    __syncthreads();
    if (warp) return;
    t = 0.f;
#pragma unroll
    for (int w = 0; w < 32; ++w) t += red[w][lane];
    if (blockIdx.x * 32 + lane < D) dw[blockIdx.x * 32 + lane] = t;
}

inline bool bad(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }
inline int status(cudaError_t e) { return e == cudaSuccess ? DSQG_OK : DSQG_ERR_CUDA; }
inline bool bad_rows(long long rows, int D) { return rows < 1 || D < 1 || rows > 0x7fffffffLL || rows * D > 0x7fffffffffLL; }
inline bool bad_type(int t) { return t != DSQG_DTYPE_BF16 && t != DSQG_DTYPE_F32; }

// Threads and pieces of a row: pieces of eight elements where rows start on 16 bytes, single elements otherwise; a warp (or a part of one) a row up to
// 1024 columns, a block beyond; rows that registers do not hold are read again.
enum Shape { kWide, k8x8, k8x16, k8x32, k8x32x2, k8x32x4, k8x256, k8x256x2, k8x256x4, k8x1024x4, k1x32x8, k1x256x4, k1x256x16 };
inline Shape shape_for(int D, bool vector) {
    if (vector) {
        if (D <= 64) return k8x8;
        if (D <= 128) return k8x16;
        if (D <= 256) return k8x32;
        if (D <= 512) return k8x32x2;
        if (D <= 1024) return k8x32x4;
        if (D <= 2048) return k8x256;
        if (D <= 4096) return k8x256x2;
        if (D <= 8192) return k8x256x4;
        return D <= 32768 ? k8x1024x4 : kWide;
    }
    return D <= 256 ? k1x32x8 : D <= 1024 ? k1x256x4 : D <= 4096 ? k1x256x16 : kWide;
}
inline int rows_per_block(Shape s) {
    switch (s) { case k8x8: return kThreads / 8; case k8x16: return kThreads / 16; case k8x32: case k8x32x2: case k8x32x4: case k1x32x8: return kThreads / 32; default: return 1; }
}
// Blocks of the backward kernel, which follow from the sizes alone.
inline int grad_blocks(long long rows, Shape s) {
    int an_sm = 3;
    switch (s) {
        case k8x32x2: case k8x256x2: case k1x256x16: an_sm = 2; break;
        case k8x32x4: case k8x256x4: case k8x1024x4: an_sm = 1; break;
        case kWide: an_sm = 4; break;
        default: break;
    }
    const long long b = (rows + rows_per_block(s) - 1) / rows_per_block(s);
    return (int)(b < 148 * an_sm ? b : 148 * an_sm);
}

}  // namespace
}  // namespace dsqg

using namespace dsqg;

#define DSQG_NORM_SHAPES(SHAPE, RUN)                                       \
    switch (SHAPE) {                                                       \
        case k8x8: RUN(8, 8, 1); break;                                    \
        case k8x16: RUN(8, 16, 1); break;                                  \
        case k8x32: RUN(8, 32, 1); break;                                  \
        case k8x32x2: RUN(8, 32, 2); break;                                \
        case k8x32x4: RUN(8, 32, 4); break;                                \
        case k8x256: RUN(8, 256, 1); break;                                \
        case k8x256x2: RUN(8, 256, 2); break;                              \
        case k8x256x4: RUN(8, 256, 4); break;                              \
        case k8x1024x4: RUN(8, 1024, 4); break;                            \
        case k1x32x8: RUN(1, 32, 8); break;                                \
        case k1x256x4: RUN(1, 256, 4); break;                              \
        case k1x256x16: RUN(1, 256, 16); break;                            \
        default: break;                                                    \
    }

extern "C" {

int dsqg_rms_norm_fwd(const dsqg_rms_norm* p, void* stream) {
    if (!p || !p->x || !p->weight || !p->y || (p->residual && !p->h) || (p->y_dtype == DSQG_DTYPE_E4M3 && !p->y_scale)) return DSQG_ERR_NULL_POINTER;
    if (bad_rows(p->rows, p->D)) return DSQG_ERR_BAD_SHAPE;
    if (bad_type(p->x_dtype) || (p->residual && bad_type(p->stream_dtype)) || (bad_type(p->y_dtype) && p->y_dtype != DSQG_DTYPE_E4M3)) return DSQG_ERR_BAD_DTYPE;
    if (bad(p->x) || bad(p->residual) || bad(p->weight) || bad(p->h) || bad(p->y)) return DSQG_ERR_MISALIGNED;
    const NormArgs a = {p->x, p->residual, p->weight, p->h, p->y, static_cast<uint8_t*>(p->y_scale), p->rstd, p->rows, p->D, p->eps, p->x_dtype == DSQG_DTYPE_F32, p->stream_dtype, p->y_dtype};
    const Shape shape = shape_for(p->D, p->D % 8 == 0);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const long long per = rows_per_block(shape);
    const unsigned blocks = (unsigned)((p->rows + per - 1) / per);
    if (shape == kWide) return status(launch_after(rms_fwd_wide_kernel, blocks, 1024, 0, s, a));
    cudaError_t e = cudaSuccess;
#define DSQG_RUN(W, TPR, V) e = launch_after(rms_fwd_kernel<W, TPR, V>, blocks, TPR < kThreads ? kThreads : TPR, 0, s, a)
    DSQG_NORM_SHAPES(shape, DSQG_RUN)
#undef DSQG_RUN
    return status(e);
}

size_t dsqg_rms_norm_bwd_scratch_bytes(long long rows, int D) {
    if (bad_rows(rows, D)) return 0;
    const int v = grad_blocks(rows, shape_for(D, true)), s = grad_blocks(rows, shape_for(D, false));
    return (size_t)(v > s ? v : s) * D * 4;
}

int dsqg_rms_norm_bwd(const dsqg_rms_norm* p, const void* dy, const void* dh, void* dx, void* dresidual, float* dweight, void* scratch, size_t scratch_bytes,
                      void* stream) {
    if (!p || !p->weight || !p->rstd || !dy || (!dx && !dresidual && !dweight) || (dweight && !scratch)) return DSQG_ERR_NULL_POINTER;
    const void* h = p->residual ? p->h : p->x;
    const int s_dt = p->residual ? p->stream_dtype : p->x_dtype;
    if (!h) return DSQG_ERR_NULL_POINTER;
    if (bad_rows(p->rows, p->D)) return DSQG_ERR_BAD_SHAPE;
    if (bad_type(p->x_dtype) || bad_type(s_dt) || bad_type(p->y_dtype)) return DSQG_ERR_BAD_DTYPE;
    if (bad(h) || bad(p->weight) || bad(dy) || bad(dh) || bad(dx) || bad(dresidual) || bad(scratch)) return DSQG_ERR_MISALIGNED;
    if (dweight && scratch_bytes < dsqg_rms_norm_bwd_scratch_bytes(p->rows, p->D)) return DSQG_ERR_SCRATCH_TOO_SMALL;
    const NormGradArgs a = {h, p->rstd, p->weight, dy, dh, dx, dresidual, dweight ? static_cast<float*>(scratch) : nullptr, p->rows, p->D, s_dt, p->y_dtype, p->x_dtype};
    const Shape shape = shape_for(p->D, p->D % 8 == 0);
    const int blocks = grad_blocks(p->rows, shape);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    if (shape == kWide) {
        if (dx || dresidual) e = launch_after(rms_bwd_wide_kernel, (unsigned)p->rows, 1024, 0, s, a);
        if (e == cudaSuccess && dweight) e = launch_after(dw_part_kernel, dim3((p->D + kThreads - 1) / kThreads, blocks), kThreads, 0, s, a);
    } else {
#define DSQG_RUN(W, TPR, V) e = launch_after(rms_bwd_kernel<W, TPR, V>, (unsigned)blocks, TPR < kThreads ? kThreads : TPR, TPR < kThreads ? (size_t)p->D * 4 : 0, s, a)
        DSQG_NORM_SHAPES(shape, DSQG_RUN)
#undef DSQG_RUN
    }
    if (e == cudaSuccess && dweight) e = launch_after(dw_kernel, (p->D + 31) / 32, 1024, 0, s, static_cast<const float*>(scratch), dweight, blocks, p->D);
    return status(e);
}

}  // extern "C"
