// Products with 4-bit weights: y = x W^T + b, W[n][k] = (nibble - 8) * scales[n][k / group], for few rows of x (the tokens of a decode step).
//
// What counts is reading the weights once.  A warp takes 16 RT rows of W and a part of the columns, the warps of a block that share rows every ks-th tile
// of 128 SUBS columns; they are added in order through shared memory.  A tile comes by cp.async, 64 SUBS bytes of a row after the other, pieces of 16
// bytes exchanged by row so that words are read without bank conflicts.  The weights are the A operand of mma.sync (m16n8k16), eight tokens the B
// operand, fp32 accumulators: a nibble becomes a 16-bit float by setting it into the mantissa of 128 (bf16) or of 1024 or 64 (f16) and subtracting 136, 1032 or
// 72, which rounds nothing; x is bf16, or e4m3 which f16 holds exactly.  The contraction may be permuted freely as long as both operands agree: a lane
// takes words of eight nibbles, and a pair of an operand is nibbles i and i + 4 of a word, so that one mask serves both.  A step of the contraction lies
// inside one group of 32 columns, so a group's products are summed unscaled and its scale is applied to the fp32 sum.  x goes straight to registers,
// 128 columns ahead of its use (it is small and stays in L1), the scales a tile ahead.
//
// What bounds it is waiting: 1 x 4096 x 16384 takes 12.2 us where the copies alone take 6 (HBM's floor 5.3), with the issue slots at 52 %, the pipe of shifts and
// logic at 51 % (some 180 instructions for 16 rows of 128 columns, half of them there), DRAM at 28 % and a fifth of the warps there could be: a warp has 3.5
// tiles, one ahead, behind a first copy that nothing hides.  Where N is small it is also few blocks (64 of them for 1 x 8192 x 1024, 4.7 us, floor 0.7).  Built and taken back: x brought to f16 and into the
// order of the pairs in shared memory, with the columns of a row block shared out over a cluster (11.5, but 3.3 instead of 2.3 us for 1 x 256 x 768 and
// 9.5 instead of 7.7 for 8 x 8192 x 4096); four warps a block (13.5); 64-byte pieces of eight rows a copy (18.4); scales fetched 128 columns ahead (16.4).
#include "dsqg_rows8.cuh"

namespace dsqg {
namespace {

constexpr int kWarps = 8, kStages = 2;

struct Int4Args {
    const void* x; const uint8_t* x_scale; const uint8_t* w; const __nv_bfloat16* scales; const float* bias; __nv_bfloat16* y;
    int M, N, K, groups;                                       // groups: K / group
    int ks;                                                    // warps that share the columns of a row tile
};

template <bool F16> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (x & mask) | base in one instruction: the constants are kept in registers, for an instruction holds one constant only.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t base) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(x), "r"(mask), "r"(base));
    return r;
}
template <bool F16> struct Magic {
    uint32_t low, high, low_base, high_base;
    __device__ __forceinline__ Magic() {
        asm volatile("mov.b32 %0, 0x000f000f;\n\tmov.b32 %1, 0x00f000f0;\n\tmov.b32 %2, %4;\n\tmov.b32 %3, 0x54005400;"
                     : "=r"(low), "=r"(high), "=r"(low_base), "=r"(high_base) : "n"(F16 ? 0x64006400 : 0x43004300));
    }
};
// Nibbles i and i + 4 of w, less 8, as two 16-bit floats.
template <bool F16> __device__ __forceinline__ uint32_t weights(uint32_t w, int i, const Magic<F16>& k) {
    if constexpr (F16) {                                       // an odd nibble stays where it is, in the mantissa of 64
        const uint32_t u = i & 1 ? and_or(w >> (4 * i - 4), k.high, k.high_base) : and_or(w >> (4 * i), k.low, k.low_base);
        const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), __float2half2_rn(i & 1 ? 72.f : 1032.f));
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const uint32_t u = and_or(w >> (4 * i), k.low, k.low_base);
        const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), __float2bfloat162_rn(136.f));
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}
__device__ __forceinline__ void copy_async16(uint32_t to, const void* from, bool on) {
    const int n = on ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(to), "l"(from), "r"(n) : "memory");
}
// Where piece p of a row lies among the row's 4 SUBS: the same piece of eight rows (a word of it each lane), and four pieces of two neighbouring rows, then
// meet no bank twice.
template <int SUBS> __device__ __forceinline__ int place(int row, int p) {
    return SUBS == 1 ? p ^ (row >> 1 & 3) : p ^ ((row & 1) << 2 ^ (row >> 1 & 3));
}

// F8: x in e4m3.  NT: tiles of eight tokens.  RT: tiles of 16 rows of W.  GC: chunks of 32 columns in a group.  SUBS: 128-column parts of a tile.
template <bool F8, int NT, int RT, int GC, int SUBS>
__global__ void __launch_bounds__(kWarps * 32, 2) int4_kernel(const Int4Args a) {
    constexpr int KT = 128 * SUBS, ROW = KT / 2, STAGE = RT * 16 * ROW;
    constexpr bool WIDE = GC == 4;                             // a group is 128 columns: lane t takes whole chunk t; otherwise word t of every chunk
    extern __shared__ __align__(16) char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int ks = a.ks, part_of_k = warp % ks, n0 = (blockIdx.x * (kWarps / ks) + warp / ks) * 16 * RT, m0 = blockIdx.y * 8 * NT;
    const uint32_t fifo = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * kStages * STAGE;
    const int all = (a.K + KT - 1) / KT, tiles = part_of_k < all && n0 < a.N ? (all - part_of_k + ks - 1) / ks : 0;
    stream_wait();

    // A lane copies one piece of 16 bytes of every (512 / ROW)-th row.  Rows behind the last repeat it.
    constexpr int COPIES = STAGE / 512, ROWS_A_COPY = 512 / ROW;
    const int row_l = lane * 16 / ROW, piece_l = lane * 16 % ROW / 16;
    const size_t row_bytes = a.K / 2;
    const uint8_t* const wp = a.w + (size_t)min(n0 + row_l, a.N - 1) * row_bytes + piece_l * 16;
    const bool whole = n0 + 16 * RT <= a.N;
    uint32_t to[SUBS];                                         // where a piece goes: copies SUBS apart are whole groups of eight rows apart
#pragma unroll
    for (int j = 0; j < SUBS; ++j) to[j] = fifo + (j * ROWS_A_COPY + row_l) * ROW + place<SUBS>(j * ROWS_A_COPY + row_l, piece_l) * 16;
    const auto issue = [&](int i) {
        if (i < tiles) {
            const int k0 = (part_of_k + i * ks) * KT;
            const bool on = k0 + 32 * piece_l < a.K;
            const uint8_t* const from = on ? wp + k0 / 2 : a.w;
            const uint32_t stage = (i % kStages) * STAGE;
#pragma unroll
            for (int j = 0; j < COPIES; ++j) {
                const size_t ahead = whole ? j * ROWS_A_COPY * row_bytes : (size_t)max(min(j * ROWS_A_COPY, a.N - 1 - n0 - row_l), 0) * row_bytes;
                copy_async16(to[j % SUBS] + j / SUBS * SUBS * 512 + stage, on ? from + ahead : from, on);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);

    // x of 128 columns from k on, eight elements a chunk: token 8 n + g, and of lane t those of the words that it takes of W (below)
    const char* xp[NT];                                        // a column behind the last token repeats it: columns do not meet, and it is not stored
#pragma unroll
    for (int n = 0; n < NT; ++n) xp[n] = static_cast<const char*>(a.x) + ((size_t)min(m0 + 8 * n + g, a.M - 1) * a.K + (WIDE ? 32 : 8) * t) * (F8 ? 1 : 2);
    const auto fetch = [&](uint32_t (&x)[NT][4][F8 ? 2 : 4], int k) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                constexpr int STEP = WIDE ? 8 : 32;
                const bool on = WIDE ? k < a.K : k + 32 * c < a.K;        // the same for the whole warp
                const char* const from = xp[n] + (k + STEP * c) * (F8 ? 1 : 2);
                if constexpr (F8) {
                    uint2 u = make_uint2(0u, 0u);
                    if (on) u = __ldg(reinterpret_cast<const uint2*>(from));
                    x[n][c][0] = u.x; x[n][c][1] = u.y;
                } else {
                    uint4 u = make_uint4(0u, 0u, 0u, 0u);
                    if (on) u = __ldg(reinterpret_cast<const uint4*>(from));
                    x[n][c][0] = u.x; x[n][c][1] = u.y; x[n][c][2] = u.z; x[n][c][3] = u.w;
                }
            }
    };
    // Scales of a tile: SC groups a row.  A lane holds PL pairs (rows r and r + 8 of a row tile): pair r SC + group belongs to lane (r SC + group) / PL.
    constexpr int SC = 4 * SUBS / GC, PL = SC < 4 ? 1 : SC / 4;
    const auto fetch_scales = [&](uint32_t (&s)[RT][PL], int i) {
        const int k0 = (part_of_k + i * ks) * KT;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int j = 0; j < PL; ++j) {
                const int q = lane * PL + j, row = q / SC, k = k0 + q % SC * (32 * GC);
                s[r][j] = 0u;
                if (i < tiles && row < 8 && k < a.K) {
                    const unsigned short* const p = reinterpret_cast<const unsigned short*>(a.scales) + k / (32 * GC);
                    const int n = n0 + 16 * r + row;
                    s[r][j] = __ldg(p + (size_t)min(n, a.N - 1) * a.groups) | (uint32_t)__ldg(p + (size_t)min(n + 8, a.N - 1) * a.groups) << 16;
                }
            }
    };

    // place() exchanges pieces by lane, so an address is a lane's offset, of which there are few, and a constant.
    constexpr int PAR = SUBS == 1 ? 1 : 2;
    uint32_t w_at[PAR][WIDE ? 1 : 4];
#pragma unroll
    for (int b = 0; b < PAR; ++b)
#pragma unroll
        for (int c = 0; c < (WIDE ? 1 : 4); ++c) w_at[b][c] = fifo + g * ROW + (WIDE ? place<SUBS>(g, 4 * b + t) * 16 : place<SUBS>(g, 4 * b + c) * 16 + 4 * t);
    const Magic<F8> magic;
    float total[RT][NT][4];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) total[r][n][e] = 0.f;

    uint32_t x_next[NT][4][F8 ? 2 : 4], s_now[RT][PL], s_next[RT][PL];
    fetch_scales(s_next, 0);
    if (tiles > 0) fetch(x_next, part_of_k * KT);
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
        __syncwarp();                                          // every lane has read the tile that the next copies replace
        issue(i + kStages - 1);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int j = 0; j < PL; ++j) s_now[r][j] = s_next[r][j];
        fetch_scales(s_next, i + 1);
        asm volatile("cp.async.wait_group %0;" :: "n"(kStages - 1) : "memory");
        __syncwarp();
        const int k0 = (part_of_k + i * ks) * KT;
        const uint32_t stage = (i % kStages) * STAGE;
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub) {
            uint32_t x[NT][4][F8 ? 2 : 4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int e = 0; e < (F8 ? 2 : 4); ++e) x[n][c][e] = x_next[n][c][e];
            if (sub + 1 < SUBS) fetch(x_next, k0 + 128 * (sub + 1));
            else if (i + 1 < tiles) fetch(x_next, k0 + ks * KT);
            float part[RT][NT][4];
            uint32_t wide[RT][2][4];                           // WIDE: chunk t of rows g, g + 8, its four words
            if constexpr (WIDE) {
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(wide[r][e][0]), "=r"(wide[r][e][1]), "=r"(wide[r][e][2]), "=r"(wide[r][e][3])
                                     : "r"(w_at[sub % PAR][0] + stage + (16 * r + 8 * e) * ROW + sub / PAR * 128) : "memory");
            }
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
                    if constexpr (F8) { e4m3x4_half2(x[n][c][0], w[0], w[1]); e4m3x4_half2(x[n][c][1], w[2], w[3]); }
                    else { w[0] = x[n][c][0]; w[1] = x[n][c][1]; w[2] = x[n][c][2]; w[3] = x[n][c][3]; }
                    xb[n][0] = __byte_perm(w[0], w[2], 0x5410); xb[n][1] = __byte_perm(w[0], w[2], 0x7632);
                    xb[n][2] = __byte_perm(w[1], w[3], 0x5410); xb[n][3] = __byte_perm(w[1], w[3], 0x7632);
                }
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    uint32_t w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if constexpr (WIDE) w[e] = wide[r][e][c];
                        else
                            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[e]) : "r"(w_at[sub % PAR][WIDE ? 0 : c] + stage + (16 * r + 8 * e) * ROW + sub / PAR * 128) : "memory");
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t wa[4] = {weights<F8>(w[0], 2 * h, magic), weights<F8>(w[1], 2 * h, magic), weights<F8>(w[0], 2 * h + 1, magic), weights<F8>(w[1], 2 * h + 1, magic)};
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma<F8>(part[r][n], wa, xb[n][2 * h], xb[n][2 * h + 1]);
                    }
                    if (c % GC == GC - 1) {
                        const int group = (4 * sub + c) / GC;
                        const uint32_t pair = __shfl_sync(0xffffffffu, s_now[r][group % PL], SC < 4 ? g * SC + group : 4 * g + group / PL);
                        const float s0 = __uint_as_float(pair << 16), s1 = __uint_as_float(pair & 0xffff0000u);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            total[r][n][0] = fmaf(s0, part[r][n][0], total[r][n][0]); total[r][n][1] = fmaf(s0, part[r][n][1], total[r][n][1]);
                            total[r][n][2] = fmaf(s1, part[r][n][2], total[r][n][2]); total[r][n][3] = fmaf(s1, part[r][n][3], total[r][n][3]);
                        }
                    }
                }
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    // ---- [warp][token][row]; the warps of a row tile are added in order
    constexpr int ROWS = 16 * RT, TOKENS = 8 * NT, PITCH = ROWS + 1;
    float* const red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[(warp * TOKENS + 8 * n + 2 * t + (e & 1)) * PITCH + 16 * r + g + 8 * (e >> 1)] = total[r][n][e];
    __syncthreads();
    const int tokens = min(TOKENS, a.M - m0), rows = kWarps / ks * ROWS;       // rows of the block, next to one another
    for (int z = threadIdx.x; z < rows * tokens; z += kWarps * 32) {
        const int row = z % rows, token = z / rows, n = blockIdx.x * rows + row, m = m0 + token;
        if (n >= a.N) continue;
        float s = 0.f;
        const float* from = red + (row / ROWS * ks * TOKENS + token) * PITCH + row % ROWS;
        for (int w = 0; w < ks; ++w) s += from[w * TOKENS * PITCH];
        if constexpr (F8) s *= scale_value(a.x_scale[m]);
        if (a.bias) s += a.bias[n];
        a.y[(size_t)m * a.N + n] = __float2bfloat16(s);
    }
}

template <bool F8, int NT, int RT, int GC, int SUBS> cudaError_t launch_one(Int4Args a, cudaStream_t s) {
    constexpr int FIFO = kWarps * kStages * RT * 16 * 64 * SUBS, RED = kWarps * 8 * NT * (16 * RT + 1) * 4;
    constexpr int SMEM = FIFO > RED ? FIFO : RED;
    auto kern = int4_kernel<F8, NT, RT, GC, SUBS>;
    static std::atomic<unsigned long long> done{0};
    if (SMEM > 48 * 1024)
        if (cudaError_t e = allow_shared(reinterpret_cast<const void*>(kern), SMEM, done)) return e;
    const int units = (a.N + 16 * RT - 1) / (16 * RT), cols = (a.K + 128 * SUBS - 1) / (128 * SUBS);
    a.ks = 1;
    while (a.ks < kWarps && a.ks < cols && units * a.ks < 148 * 12) a.ks *= 2;
    return launch_after(kern, dim3((units + kWarps / a.ks - 1) / (kWarps / a.ks), (a.M + 8 * NT - 1) / (8 * NT)), kWarps * 32, SMEM, s, a);
}
// Two row tiles a warp, which then share what unpacking x costs, where that leaves a warp for every SM's schedulers and tiles of 256 columns keep two
// blocks on an SM; one row tile and 512 columns below (us, two : one: 1 x 4096 x 16384 12.2 : 12.7, 8 x 4096 x 8192 e4m3 6.7 : 7.1, 1 x 1024 x 16384 4.8 : 6.7,
// but 1 x 4096 x 4096 4.6 : 4.5, 1 x 8192 x 1024 7.1 : 4.7, 1 x 256 x 768 2.6 : 2.3).  128 columns where there are few.
template <bool F8, int NT, int GC> cudaError_t launch_shape(const Int4Args& a, cudaStream_t s) {
    if (NT == 2 || a.N >= 148 * 32) return a.K >= 4096 ? launch_one<F8, NT, 2, GC, 2>(a, s) : launch_one<F8, NT, 2, GC, 1>(a, s);
    if constexpr (NT == 1) return a.K >= 4096 ? launch_one<F8, 1, 1, GC, 4>(a, s) : launch_one<F8, 1, 1, GC, 1>(a, s);
    else return cudaErrorInvalidValue;
}
template <bool F8, int NT> cudaError_t launch_group(const Int4Args& a, int group, cudaStream_t s) {
    return group == 32 ? launch_shape<F8, NT, 1>(a, s) : group == 64 ? launch_shape<F8, NT, 2>(a, s) : launch_shape<F8, NT, 4>(a, s);
}
template <bool F8> cudaError_t launch_type(const Int4Args& a, int group, cudaStream_t s) {
    return a.M <= 8 ? launch_group<F8, 1>(a, group, s) : launch_group<F8, 2>(a, group, s);
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
    // a block's last row may be 255 beyond N, a warp's next tile eight of 512 columns beyond K
    if (M < 1 || N < 1 || N > 0x7fffff00 || K < group || K > 0x7fffc000 || K % group) return DSQG_ERR_BAD_SHAPE;
    if (bad(x) || bad(weight)) return DSQG_ERR_MISALIGNED;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    constexpr int kRows = 65535 * 16;                          // of x, that a grid's second dimension has room for
    for (long long m = 0; m < M; m += kRows) {
        const int rows = (int)(M - m < kRows ? M - m : kRows);
        const bool f8 = dtype == DSQG_DTYPE_E4M3;
        const Int4Args a = {static_cast<const char*>(x) + m * K * (f8 ? 1 : 2), f8 ? static_cast<const uint8_t*>(x_scale) + m : nullptr, static_cast<const uint8_t*>(weight),
                            static_cast<const __nv_bfloat16*>(scales), bias, static_cast<__nv_bfloat16*>(y) + m * N, rows, N, K, K / group};
        if (cudaError_t e = f8 ? launch_type<true>(a, group, s) : launch_type<false>(a, group, s)) return cuda_status(e);
    }
    return DSQG_OK;
}

}  // extern "C"
