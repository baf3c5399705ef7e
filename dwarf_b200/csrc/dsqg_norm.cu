// Root-mean-square norm of a residual stream with the addition in front of it, forward and backward.
//
//   h = x + r (rounded to r's type: the stream the next layer reads), rstd = 1 / sqrt(mean(h^2) + eps), y = h rstd w
//   dh = dh_out + rstd (w dy - x^ mean(w dy x^)), x^ = h rstd;  dx = dr = dh;  dw = sum over rows of dy x^
//
// The norm is of h as it is stored, which is what the backward pass and the next layer see.  fp32 arithmetic throughout.  y leaves in bf16,
// fp32 or e4m3 with a power-of-two scale per row (dsqg_rows8.cuh).  Bound by memory: every tensor is read and written once, a row stays
// in registers between its reduction and its result, as it lies in memory (unpacked to fp32 and with room for either type, the backward pass of
// 1024 x 16,384 in bf16 spilled: 162 us instead of 74 forward and backward).
#include "dsqg_rows8.cuh"

namespace dsqg {
namespace {

constexpr int kThreads = 256;

// Eight consecutive elements as they lie in memory (bf16 or fp32), so that every load of a row is under way before one is used.
template <bool F32> struct Piece {
    uint4 a[F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* p, long long i) {
        const uint4* s = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + i * (F32 ? 4 : 2));
#pragma unroll
        for (int k = 0; k < (F32 ? 2 : 1); ++k) a[k] = __ldg(s + k);
    }
    // the first `n` of them, one by one
    __device__ __forceinline__ void load_first(const void* p, long long i, int n) {
        uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) {
                if (F32) w[e] = __ldg(static_cast<const uint32_t*>(p) + i + e);
                else w[e / 2] |= (uint32_t)__ldg(static_cast<const unsigned short*>(p) + i + e) << 16 * (e & 1);
            }
#pragma unroll
        for (int k = 0; k < (F32 ? 2 : 1); ++k) a[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int k = 0; k < (F32 ? 2 : 1); ++k) {
            const uint32_t u[4] = {a[k].x, a[k].y, a[k].z, a[k].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (F32) x[4 * k + i] = __uint_as_float(u[i]);
                else { x[2 * i] = __uint_as_float(u[i] << 16); x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
            }
        }
    }
};
__device__ __forceinline__ float load_one(const void* p, long long i, bool f32) {
    return f32 ? __ldg(static_cast<const float*>(p) + i) : __uint_as_float((uint32_t)__ldg(static_cast<const unsigned short*>(p) + i) << 16);
}
__device__ __forceinline__ void store_one(void* p, long long i, int dtype, float x) {
    if (dtype == DSQG_DTYPE_F32) static_cast<float*>(p)[i] = x;
    else if (dtype == DSQG_DTYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16(x);
    else static_cast<uint8_t*>(p)[i] = (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

// Rows of a width that is no multiple of eight: the whole tensor is cut into pieces of eight elements all the same, and a row is the pieces that it touches,
// the first from element -shift on, shift = row D mod 8.  A piece's elements in front of the row or behind it count as zeros and are not stored.
// (4096 x 1111 in bf16 forward and backward: 36 us, 134 element by element.)
template <bool ODD> struct Cut {
    long long first;           // element of the row's first piece
    int shift, D;
    long long total;
    __device__ __forceinline__ Cut(long long row, int D, long long rows) : D(D), total(rows * D) {
        const long long at = row * D;
        shift = ODD ? (int)(at & 7) : 0;
        first = at - shift;
    }
    __device__ __forceinline__ int column(int piece) const { return piece * 8 - shift; }       // of the piece's first element; the row has it if below D
    __device__ __forceinline__ bool has(int column, int e) const { return !ODD || (unsigned)(column + e) < (unsigned)D; }
    template <bool F32> __device__ __forceinline__ void load(Piece<F32>& p, const void* from, int piece) const {
        const long long i = first + piece * 8;
        if (!ODD || i + 8 <= total) p.load(from, i);
        else p.load_first(from, i, (int)(total - i));
    }
    __device__ __forceinline__ void store(void* to, int piece, int dtype, const float (&x)[8]) const {
        const long long i = first + piece * 8;
        const int c = column(piece);
        if (!ODD || (c >= 0 && c + 8 <= D)) store8_as(to, i, dtype, x);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (has(c, e)) store_one(to, i + e, dtype, x[e]);
    }
    __device__ __forceinline__ void weights(const float* w, int piece, float (&x)[8]) const {
        const int c = column(piece);
        if constexpr (!ODD) load8(w + c, x);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = has(c, e) ? __ldg(w + c + e) : 0.f;
    }
    __device__ __forceinline__ void mask(int piece, float (&x)[8]) const {
        if constexpr (ODD) {
            const int c = column(piece);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = has(c, e) ? x[e] : 0.f;
        }
    }
};

// Sum, or maximum, over the TPR threads of a row.  red: two slots a warp, used in turn, so that one barrier an exchange is enough.
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* red, int& turn) {
    v = group_sum<(TPR < 32 ? TPR : 32)>(v);
    if constexpr (TPR > 32) {
        float* slot = red + (turn ^= 1) * 32;
        if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < TPR / 32; ++w) v += slot[threadIdx.x / TPR * (TPR / 32) + w];
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
        for (int w = 0; w < TPR / 32; ++w) v = max(v, slot[threadIdx.x / TPR * (TPR / 32) + w]);
    }
    return v;
}

struct NormArgs {
    const void* x; const void* r; const float* w; void* h; void* y; uint8_t* scale; float* rstd;
    long long rows; int D; float eps; int x_f32, s_dt, y_dt;
};

// TPR threads a row (a block of max(TPR, kThreads) threads), V pieces a thread.
template <bool ODD, bool X32, bool S32, int TPR, int V>
__global__ void __launch_bounds__(TPR < kThreads ? kThreads : TPR) rms_fwd_kernel(const NormArgs a) {
    constexpr int kBlock = TPR < kThreads ? kThreads : TPR;
    __shared__ float red[64];
    int turn = 0;
    const int t = threadIdx.x % TPR;
    const long long row0 = (long long)blockIdx.x * (kBlock / TPR) + threadIdx.x / TPR;
    const bool live = row0 < a.rows;
    const Cut<ODD> cut(live ? row0 : a.rows - 1, a.D, a.rows);
    stream_wait();
    Piece<X32> px[V];
    Piece<S32> pr[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int p = v * TPR + t;
        if (cut.column(p) < a.D) {
            cut.load(px[v], a.x, p);
            if (a.r) cut.load(pr[v], a.r, p);
        }
    }
    float h[V][8], ss = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int p = v * TPR + t;
        if (cut.column(p) < a.D) {
            px[v].get(h[v]);
            if (a.r) {
                float r[8];
                pr[v].get(r);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h[v][e] += r[e];
                    if (!S32) h[v][e] = __bfloat162float(__float2bfloat16(h[v][e]));
                }
                if (live) cut.store(a.h, p, S32 ? DSQG_DTYPE_F32 : DSQG_DTYPE_BF16, h[v]);
            }
            cut.mask(p, h[v]);
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(h[v][e], h[v][e], ss);
        }
    }
    const float rstd = rsqrtf(row_sum<TPR>(ss, red, turn) / a.D + a.eps);
    if (a.rstd && live && t == 0) a.rstd[row0] = rstd;
    uint32_t top = 0u;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int p = v * TPR + t;
        if (cut.column(p) < a.D) {
            float w[8];
            cut.weights(a.w, p, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[v][e] = h[v][e] * rstd * w[e];
            cut.mask(p, h[v]);                                 // a row that is not finite has NaN in the products with zeros
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, abs_bits(h[v][e]));
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
        const int p = v * TPR + t;
        if (cut.column(p) < a.D && live) {
#pragma unroll
            for (int e = 0; e < 8; ++e) h[v][e] *= inv;
            cut.store(a.y, p, a.y_dt, h[v]);
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
        float x = load_one(a.x, at + c, a.x_f32);
        if (a.r) {
            x += load_one(a.r, at + c, s_f32);
            if (!s_f32) x = __bfloat162float(__float2bfloat16(x));
        }
        return x;
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
        const float x = value(c);
        if (a.r) store_one(a.h, at + c, a.s_dt, x);
        store_one(a.y, at + c, a.y_dt, x * rstd * __ldg(a.w + c) * inv);
    }
}

struct NormGradArgs {
    const void* h; const float* rstd; const float* w; const void* dy; const void* dh; void* dx; void* dr; float* part;
    long long rows; int D; int s_dt, y_dt, x_dt;
};

// Blocks of the backward kernel that an SM holds: the grid is that many times 148, so that all of them start at once and walk the same number of rows
// (four an SM where registers allowed three took a second wave of blocks that then had a quarter of the rows to itself: 53 us instead of 43 at 65,536 x 256).
// A row is read while others of the SM are reduced, so the more the better until values leave the registers.  Forward and backward at 16,384 x 1024 in bf16:
// 62.8 us with three, 57.4 with four, 55.8 with five, 62.4 with six.  With an fp32 tensor three hold their values: 78.2 us at 65,536 x 256, 80.3 with four.
__host__ __device__ constexpr int grad_blocks_an_sm(int TPR, int V, bool wide) {
    return TPR == 1024 ? 1 : TPR == 512 ? (wide ? 1 : 2) : V == 2 ? (wide ? 2 : 4) : wide ? 3 : 5;
}

// A block walks rows a grid apart; a thread keeps the sums of its columns of dw (rows of one shift only: rows a grid apart are a multiple of eight apart).
// The partial sums of a block's rows go to part[block], added by dw_kernel: the order follows from the sizes alone.
template <bool ODD, bool S32, bool Y32, int TPR, int V>
__global__ void __launch_bounds__(TPR < kThreads ? kThreads : TPR, grad_blocks_an_sm(TPR, V, S32 || Y32)) rms_bwd_kernel(const NormGradArgs a) {
    constexpr int kBlock = TPR < kThreads ? kThreads : TPR, kRows = kBlock / TPR;
    __shared__ float red[64];
    extern __shared__ float sums[];
    int turn = 0;
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    float dw[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[v][e] = 0.f;
    stream_wait();
    for (long long first = (long long)blockIdx.x * kRows; first < a.rows; first += (long long)gridDim.x * kRows) {
        const bool live = first + group < a.rows;
        const long long row = live ? first + group : a.rows - 1;
        const Cut<ODD> cut(row, a.D, a.rows);
        const float rstd = __ldg(a.rstd + row);
        Piece<S32> ph[V], pd[V];
        Piece<Y32> py[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int p = v * TPR + t;
            if (cut.column(p) < a.D) {
                cut.load(ph[v], a.h, p);
                cut.load(py[v], a.dy, p);
                if (a.dh) cut.load(pd[v], a.dh, p);
            }
        }
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int p = v * TPR + t;
            if (cut.column(p) < a.D) {
                float xh[8], g[8], w[8];
                cut.weights(a.w, p, w);
                ph[v].get(xh); py[v].get(g);
                cut.mask(p, xh); cut.mask(p, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    xh[e] *= rstd;
                    if (live) dw[v][e] = fmaf(g[e], xh[e], dw[v][e]);
                    s = fmaf(g[e] * w[e], xh[e], s);
                }
            }
        }
        s = row_sum<TPR>(s, red, turn) / a.D;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int p = v * TPR + t;
            if (cut.column(p) < a.D && live) {
                float xh[8], g[8], w[8], d[8];
                cut.weights(a.w, p, w);
                ph[v].get(xh); py[v].get(g);
                if (a.dh) pd[v].get(d);
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] = fmaf(rstd, g[e] * w[e] - xh[e] * rstd * s, a.dh ? d[e] : 0.f);
                if (a.dx) cut.store(a.dx, p, a.x_dt, d);
                if (a.dr) cut.store(a.dr, p, S32 ? DSQG_DTYPE_F32 : DSQG_DTYPE_BF16, d);
            }
        }
    }
    if (!a.part) return;
    float* out = a.part + (size_t)blockIdx.x * a.D;
    const Cut<ODD> cut((long long)blockIdx.x * kRows + group, a.D, a.rows);
    if constexpr (kRows == 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = cut.column(v * TPR + t);
            if (c < a.D)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (cut.has(c, e)) out[c + e] = dw[v][e];
        }
    } else {
        for (int k = 0; k < kRows; ++k) {                      // row groups in turn: fixed order of additions
            if (group == k) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const int c = cut.column(v * TPR + t);
                    if (c < a.D)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (cut.has(c, e)) sums[c + e] = k ? sums[c + e] + dw[v][e] : dw[v][e];
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
    const auto get = [&](const void* p, int c, bool f32) { return load_one(p, at + c, f32); };
    float s = 0.f;
    for (int c = threadIdx.x; c < a.D; c += 1024) s = fmaf(get(a.dy, c, y_f32) * __ldg(a.w + c), get(a.h, c, s_f32) * rstd, s);
    s = row_sum<1024>(s, red, turn) / a.D;
    for (int c = threadIdx.x; c < a.D; c += 1024) {
        const float g = get(a.dy, c, y_f32) * __ldg(a.w + c), xh = get(a.h, c, s_f32) * rstd;
        const float d = fmaf(rstd, g - xh * s, a.dh ? get(a.dh, c, s_f32) : 0.f);
        if (a.dx) store_one(a.dx, at + c, a.x_dt, d);
        if (a.dr) store_one(a.dr, at + c, a.s_dt, d);
    }
}
__global__ void __launch_bounds__(kThreads) dw_part_kernel(const NormGradArgs a) {
    stream_wait();
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= a.D) return;
    const bool s_f32 = a.s_dt == DSQG_DTYPE_F32, y_f32 = a.y_dt == DSQG_DTYPE_F32;
    float s = 0.f;
    for (long long row = blockIdx.y; row < a.rows; row += gridDim.y)
        s = fmaf(load_one(a.dy, row * a.D + c, y_f32), load_one(a.h, row * a.D + c, s_f32) * __ldg(a.rstd + row), s);
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
// A column index may go 1024 beyond a row.
inline bool bad_rows(long long rows, int D) { return rows < 1 || D < 1 || D > 0x7ffff000 || rows > 0x7fffffffLL || rows * D > 0x7fffffffffLL; }
inline bool bad_type(int t) { return t != DSQG_DTYPE_BF16 && t != DSQG_DTYPE_F32; }

// Threads and pieces of a row, forward and backward: one piece a thread up to 2048 columns, two beyond, from 16,384 columns on four; wider than 32,768 a row
// is read again instead of held.  4096 x 4096 in bf16 forward and backward took 62 us with 256 threads of two pieces, 64 with 512 of one, 150 with 128 of four.
struct Shape { int tpr, v; };
inline Shape shape_of(int D) {
    const int n = D % 8 ? (D + 14) / 8 : D / 8;                // a row that starts anywhere touches up to (D + 14) / 8 pieces
    Shape s = {8, n > 4096 ? 0 : n > 2048 ? 4 : n > 256 ? 2 : 1};
    while (s.tpr < 1024 && s.tpr * s.v < n) s.tpr *= 2;
    return s;
}
inline int rows_per_block(Shape s) { return s.tpr < kThreads ? kThreads / s.tpr : 1; }
// Blocks of the backward kernel, which follow from the sizes and types alone; of an odd width, rows a grid apart are a multiple of eight rows apart.
inline int grad_blocks(long long rows, int D, bool wide = false) {
    const Shape s = shape_of(D);
    const int per = rows_per_block(s), most = 148 * (s.v ? grad_blocks_an_sm(s.tpr, s.v, wide) : 4), step = D % 8 && per < 8 ? 8 / per : 1;
    const long long b = (rows + per - 1) / per, up = (b + step - 1) / step * step;
    return (int)(up < most ? up : most / step * step);
}

}  // namespace
}  // namespace dsqg

using namespace dsqg;

#define DSQG_NORM_SHAPES(SHAPE, ODD, A, B, RUN)                             \
    switch (SHAPE.tpr * 8 + SHAPE.v) {                                      \
        case 8 * 8 + 1: RUN(ODD, A, B, 8, 1); break;                        \
        case 16 * 8 + 1: RUN(ODD, A, B, 16, 1); break;                      \
        case 32 * 8 + 1: RUN(ODD, A, B, 32, 1); break;                      \
        case 64 * 8 + 1: RUN(ODD, A, B, 64, 1); break;                      \
        case 128 * 8 + 1: RUN(ODD, A, B, 128, 1); break;                    \
        case 256 * 8 + 1: RUN(ODD, A, B, 256, 1); break;                    \
        case 256 * 8 + 2: RUN(ODD, A, B, 256, 2); break;                    \
        case 512 * 8 + 2: RUN(ODD, A, B, 512, 2); break;                    \
        case 1024 * 8 + 2: RUN(ODD, A, B, 1024, 2); break;                  \
        case 1024 * 8 + 4: RUN(ODD, A, B, 1024, 4); break;                  \
        default: break;                                                     \
    }
#define DSQG_NORM_TYPES(SHAPE, ODD, A32, B32, RUN)                         \
    if (A32) { if (B32) { DSQG_NORM_SHAPES(SHAPE, ODD, true, true, RUN) } else { DSQG_NORM_SHAPES(SHAPE, ODD, true, false, RUN) } }    \
    else { if (B32) { DSQG_NORM_SHAPES(SHAPE, ODD, false, true, RUN) } else { DSQG_NORM_SHAPES(SHAPE, ODD, false, false, RUN) } }

extern "C" {

int dsqg_rms_norm_fwd(const dsqg_rms_norm* p, void* stream) {
    if (!p || !p->x || !p->weight || !p->y || (p->residual && !p->h) || (p->y_dtype == DSQG_DTYPE_E4M3 && !p->y_scale)) return DSQG_ERR_NULL_POINTER;
    if (bad_rows(p->rows, p->D)) return DSQG_ERR_BAD_SHAPE;
    if (bad_type(p->x_dtype) || (p->residual && bad_type(p->stream_dtype)) || (bad_type(p->y_dtype) && p->y_dtype != DSQG_DTYPE_E4M3)) return DSQG_ERR_BAD_DTYPE;
    if (bad(p->x) || bad(p->residual) || bad(p->weight) || bad(p->h) || bad(p->y)) return DSQG_ERR_MISALIGNED;
    const NormArgs a = {p->x, p->residual, p->weight, p->h, p->y, static_cast<uint8_t*>(p->y_scale), p->rstd, p->rows, p->D, p->eps, p->x_dtype == DSQG_DTYPE_F32, p->stream_dtype, p->y_dtype};
    const Shape shape = shape_of(p->D);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const long long per = rows_per_block(shape);
    const unsigned blocks = (unsigned)((p->rows + per - 1) / per);
    if (!shape.v) return cuda_status(launch_after(rms_fwd_wide_kernel, blocks, 1024, 0, s, a));
    cudaError_t e = cudaSuccess;
    const bool s32 = p->residual && p->stream_dtype == DSQG_DTYPE_F32;
#define DSQG_RUN(ODD, X32, S32, TPR, V) e = launch_after(rms_fwd_kernel<ODD, X32, S32, TPR, V>, blocks, TPR < kThreads ? kThreads : TPR, 0, s, a)
    if (p->D % 8) { DSQG_NORM_TYPES(shape, true, a.x_f32, s32, DSQG_RUN) } else { DSQG_NORM_TYPES(shape, false, a.x_f32, s32, DSQG_RUN) }
#undef DSQG_RUN
    return cuda_status(e);
}

size_t dsqg_rms_norm_bwd_scratch_bytes(long long rows, int D) {
    if (bad_rows(rows, D)) return 0;
    return (size_t)grad_blocks(rows, D) * D * 4;
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
    const Shape shape = shape_of(p->D);
    const bool s32 = s_dt == DSQG_DTYPE_F32, y32 = p->y_dtype == DSQG_DTYPE_F32;
    const int blocks = grad_blocks(p->rows, p->D, s32 || y32);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    if (!shape.v) {
        if (dx || dresidual) e = launch_after(rms_bwd_wide_kernel, (unsigned)p->rows, 1024, 0, s, a);
        if (e == cudaSuccess && dweight) e = launch_after(dw_part_kernel, dim3((p->D + kThreads - 1) / kThreads, blocks), kThreads, 0, s, a);
    } else {
#define DSQG_RUN(ODD, S32, Y32, TPR, V) e = launch_after(rms_bwd_kernel<ODD, S32, Y32, TPR, V>, (unsigned)blocks, TPR < kThreads ? kThreads : TPR, TPR < kThreads ? (size_t)p->D * 4 : 0, s, a)
        if (p->D % 8) { DSQG_NORM_TYPES(shape, true, s32, y32, DSQG_RUN) } else { DSQG_NORM_TYPES(shape, false, s32, y32, DSQG_RUN) }
#undef DSQG_RUN
    }
    if (e == cudaSuccess && dweight) e = launch_after(dw_kernel, (p->D + 31) / 32, 1024, 0, s, static_cast<const float*>(scratch), dweight, blocks, p->D);
    return cuda_status(e);
}

}  // extern "C"
