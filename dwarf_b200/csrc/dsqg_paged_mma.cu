// One new token's attention to a paged cache on tensor cores: bf16 queries, pages in bf16 or e4m3, D = 32, 48, 64, 80, 96 or 128.
//
// A block takes a part of one sequence for up to 8 HT query heads of one key-value head, a warp every fourth tile of 16 positions of it.  Positions are
// the 16 rows of mma.sync (m16n8k16, fp32 accumulators) and the query heads its 8 columns: S^T = K Q^T, softmax with a running maximum and sum per
// column, O^T += V^T P^T.  A tile is one run of memory (a page keeps key and value of a position side by side): a warp copies its tiles to shared memory
// with cp.async, two tiles ahead, 512 consecutive bytes an instruction, and waits for nobody but itself.  (Every lane copying the pieces that
// it needs itself, 64 to 128 bytes a row: 68 us of copies alone for 4 sequences of 100001 positions, 4 x 8 heads of 128 in 8 bits, against 51.)  The
// 16-byte pieces of a row are exchanged by s(row), so that the reads below are free of bank conflicts.  The contraction of a product, and the rows of
// its result, may be permuted freely: key rows are the A operand as they lie (lane (g, t): rows g and g + 8, every fourth piece from t); of the value
// rows a lane takes four positions and an eighth of the columns, and pairs of positions are put together by byte permutation.
// P^T turns from a result into an operand by movmatrix.
//
// 8 bits: e4m3 becomes f16 exactly.  Queries become f16 after a power of two that brings their largest element near 1; the keys' scales multiply the
// scores; the values' scales multiply the probabilities, as exponents: an operand is 2^(score + exponent of its value row's scale - w), w a running base of
// each column that follows the largest of these sums, so that what is largest in the result is largest in f16, whatever scales other rows have.  (Relative to the
// largest scale alone, a value row 2^20 above the others took the bits of all that came with or after it, even one that no query looks at.)
//
// (Keys in 8 bits as they lie, through m16n8k32 with e4m3 operands and the query as two e4m3 numbers, when a probability was one number: 61 us instead of 58 for
// 4 sequences of 100001 positions.  Query heads as the 16 rows of the product instead: half of every accumulator idle up to 8 heads, 179 registers, 8 warps an SM and 636 instructions a
// tile of 8-bit rows of 128 columns; 160 us for 4 sequences of 100001 positions, 4 x 8 heads.)
//
// mma.sync and not tcgen05: an operand of 128 rows would be at most an eighth full (query heads of one key-value head), and what is in question is memory.
#include "dsqg_paged.cuh"

namespace dsqg {
namespace {

constexpr int kWarps = 4, kTile = 16;
// A new maximum rescales what was summed so far only if it is above the old one by more than this (in powers of two): probabilities stay below 2^8, which
// f16, bf16 and the fp32 sums hold as well as those below 1.  A warp then rescales once or twice; at every new maximum of any of eight heads it did so at
// 13 of its first 16 tiles.
constexpr float kSlack = 8.f;
// The operands of 8-bit pages: rescaled when one would be above 2^15 (f16 ends at 65504), the largest then to about 2^10.  Two f16 numbers hold 2^-22 of an
// operand from 2^-3 on, and 2^-25 below: 2^-34.5 of the largest since the last rescaling, times the 2 that maxima of e4m3 rows are apart.
constexpr float kTop = 15.f, kLevel = 10.f;

template <bool F16> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// BYTES from global to shared memory, zeros where `on` is false.
template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t to, const char* from, bool on) {
    const int n = on ? BYTES : 0;
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(to), "l"(from), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" :: "r"(to), "l"(from), "n"(BYTES), "r"(n) : "memory");
}
template <int WORDS> __device__ __forceinline__ void load_shared(uint32_t from, uint32_t (&w)[WORDS]) {
    if constexpr (WORDS == 4) asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(from) : "memory");
    else if constexpr (WORDS == 2) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(from) : "memory");
    else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(from) : "memory");
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// 8 x 8 elements of 16 bits, a pair of a row a lane: transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// DR: columns of the cache; D: of the products, DR rounded up to 32.  What is behind the DR columns of a key or value row is zero in shared memory, from the start on.
template <int DR, bool F8, int HT, int STAGES>
struct Cfg {
    static constexpr int D = (DR + 31) / 32 * 32;
    static constexpr int SZ = F8 ? 1 : 2, ROW = 2 * D * SZ, HELD = 2 * DR * SZ;           // bytes of an element, of a position in shared memory and in the cache
    static constexpr int PAD = (D - DR) * SZ / 16;                       // 16-byte pieces of zeros behind a row
    static constexpr int KB = F8 ? (D % 64 == 0 ? 16 : 8) : 16;          // bytes of a piece of a key row: four lanes take 4 KB bytes
    static constexpr int KP = D * SZ / (4 * KB);                         // pieces a lane and key row
    static constexpr int VB = F8 ? (D % 128 == 0 ? 16 : D % 64 == 0 ? 8 : 4) : (D % 64 == 0 ? 16 : 8);     // of a value row: eight lanes take 8 VB
    static constexpr int VE = VB / SZ, VP = D / (8 * VE);                // elements of it, pieces a lane and value row
    static constexpr int SOFF = kTile * ROW;                             // a tile's scale bytes behind its rows
    static constexpr int STAGE = SOFF + (F8 ? 2 * kTile : 0);
    static constexpr bool EXCHANGE = ROW % 128 == 0;                     // rows of whole 128-byte lines
    static constexpr int HEADS = 8 * HT;
    static constexpr int FIFO = kWarps * STAGES * STAGE, MERGE = kWarps * HEADS * (D + 2) * 4;
    static constexpr int BUF = FIFO > MERGE ? FIFO : MERGE;
    static constexpr int SMEM = BUF + HELD + 16;
    static constexpr int MT = D / 16;                                    // m-tiles of the output, and steps of the contraction over D

    // A position's byte in the cache, in shared memory
    __device__ static __forceinline__ int spread(int byte) { return PAD && byte >= DR * SZ ? byte + PAD * 16 : byte; }
    // Where a tile's byte `byte` of row `row` lies: pieces exchanged by s(row) in 0 .. 7.  The eight lanes of a read's phase ask for pieces x, .., x + 3 of two
    // neighbouring rows (keys: bit 2 of s tells them apart) or two pieces of four rows two apart (values: bits 1 and 2).
    __device__ static __forceinline__ int at(int row, int byte) {
        return row * ROW + (EXCHANGE ? byte ^ ((row & 1) << 6 ^ (row >> 1 & 3) << 5) : byte);
    }
};

// STAGES - 1 tiles of copies ahead.
template <int DR, bool F8, int HT, int STAGES, int CTAS>
__global__ void __launch_bounds__(kWarps * 32, CTAS) step_mma_kernel(const StepArgs a) {
    using C = Cfg<DR, F8, HT, STAGES>;
    constexpr int D = C::D;
    extern __shared__ __align__(16) char smem[];
    char* const fresh = smem + C::BUF;
    uint8_t* const fresh_scale = reinterpret_cast<uint8_t*>(fresh + C::HELD);
    stream_wait();
    const PageArgs& c = a.c;
    const int blocks_h = (a.G + C::HEADS - 1) / C::HEADS, hb = blockIdx.y % blocks_h, h = blockIdx.y / blocks_h, s = blockIdx.z, part = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

    // (column, row) of the table walk ahead of the tile that is asked for, so that the page's index is there when it is needed: the first while the length is
    // on its way.
    constexpr int STEP = kWarps * kTile;                       // positions from a warp's tile to its next
    const int first_tile = part * a.chunk + warp * kTile;
    const int32_t* const table = c.table + (long long)s * c.columns;
    const int step_columns = STEP / c.page, step_rows = STEP % c.page;
    int column = first_tile / c.page, row = first_tile % c.page, next_id = 0, next_row = 0;
    const auto look = [&] {                                    // the page of the next tile
        if (column < c.columns) next_id = __ldg(table + column);
        next_row = row;
        column += step_columns; row += step_rows;
        if (row >= c.page) { row -= c.page; ++column; }
    };
    look();
    const Range r = range_of(a, s, part);
    if (part && r.first >= r.length) return;                   // part 0 always answers
    const int heads = min(C::HEADS, a.G - hb * C::HEADS);
    const long long q0 = ((long long)s * c.H + h) * a.G + hb * C::HEADS;
    const bool has_new = a.k_new != nullptr && r.end == r.length && r.length > 0;
    const int last = has_new ? r.length - 1 : -1, old_end = has_new ? r.length - 1 : r.end;     // rows in front of old_end come from the pages

    const uint32_t fifo = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * STAGES * C::STAGE;
    const int tiles = r.end > first_tile ? (r.end - first_tile + STEP - 1) / STEP : 0;
    bool bad = r.bad;

    if constexpr (C::PAD > 0) {
        for (int z = lane; z < STAGES * kTile * 2 * C::PAD; z += 32) {
            const int piece = z % C::PAD, half = z / C::PAD % 2, r = z / (2 * C::PAD) % kTile, stage = z / (2 * C::PAD * kTile);
            const uint32_t to = fifo + stage * C::STAGE + C::at(r, half * D * C::SZ + DR * C::SZ + piece * 16);
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" :: "r"(to), "r"(0) : "memory");
        }
        __syncwarp();
    }

    // ---- copies
    const auto issue = [&](int i, uint32_t st) {
        const int id = next_id, row_in = next_row;
        look();
        if (i < tiles) {
            const bool there = id >= 0 && id < c.pages;
            bad |= !there;
            const int n = there ? old_end - (first_tile + i * STEP) : 0;         // rows of the tile that exist
            const long long row0 = ((long long)(there ? id : 0) * c.H + h) * c.page + (there ? row_in : 0);
            const char* const from = c.kv + row0 * C::HELD + lane * 16;
#pragma unroll
            for (int j = 0; j < kTile * C::HELD / 512; ++j) {
                const int byte = j * 512 + lane * 16, r = byte / C::HELD;
                copy_async<16>(st + C::at(r, C::spread(byte % C::HELD)), from + j * 512, r < n);
            }
            if constexpr (F8)
                if (lane < kTile / 2) copy_async<4>(st + C::SOFF + lane * 4, reinterpret_cast<const char*>(c.scale) + row0 * 2 + lane * 4, true);
        }
    };
    const auto issue_tile = [&](int first, int slot) {
        issue(first, fifo + slot * C::STAGE);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue_tile(i, i);

    // ---- queries as the B operand: column g of tile n
    uint32_t qb[HT][C::MT][2];
    float fs[HT][2];                                           // what the scores of columns 2 t, 2 t + 1 are multiplied by
    {
        const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + q0 * DR;
        constexpr int E = C::KB / C::SZ;                       // elements of a piece: E / 4 steps
#pragma unroll
        for (int n = 0; n < HT; ++n) {
            const bool on = g + 8 * n < heads;
#pragma unroll
            for (int k = 0; k < C::KP; ++k)
#pragma unroll
                for (int e = 0; e < E / 4; ++e) {
                    uint2 u = make_uint2(0u, 0u);
                    if (on && (4 * k + t) * E + 4 * e < DR) u = *reinterpret_cast<const uint2*>(q + (g + 8 * n) * DR + (4 * k + t) * E + 4 * e);
                    qb[n][k * (E / 4) + e][0] = u.x; qb[n][k * (E / 4) + e][1] = u.y;
                }
            fs[n][0] = fs[n][1] = a.scale;
            if constexpr (F8) {
                uint32_t top = 0u;
#pragma unroll
                for (int k = 0; k < C::MT; ++k)
#pragma unroll
                    for (int e = 0; e < 2; ++e) top = max(top, max(qb[n][k][e] << 16 & 0x7fff0000u, qb[n][k][e] & 0x7fff0000u));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1)); top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // largest element to [1, 2): nothing is lost but what is below 2^-25 of it.  NaN and infinity stay what they are.
                int ex = (int)(top >> 23);
                ex = ex == 0 ? 127 : ex >= 254 ? 253 : ex;
                // not 0, for what is masked is -inf times it
                const float down = __uint_as_float((254u - ex) << 23), up = fmaxf(a.scale * __uint_as_float((uint32_t)ex << 23), 1.17549435e-38f);
#pragma unroll
                for (int k = 0; k < C::MT; ++k)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t& w = qb[n][k][e];
                        w = pack_f16x2(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xffff0000u) * down);
                    }
                fs[n][0] = __shfl_sync(0xffffffffu, up, 8 * t); fs[n][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
            }
        }
    }
    if (has_new) {
        if (warp == 0) new_row(a, s, h, last, hb == 0, fresh, fresh_scale);
        __syncthreads();
    }

    float o[HT][C::MT][4];
    // m: what the exponentials are taken against, at least the running maximum less kSlack / fs; base: m fs, 0 where m is still -inf
    float m[HT][2], l[HT][2], base[HT][2], lim[HT][2], wbase[HT][2];          // wbase: w above, a whole number
#pragma unroll
    for (int n = 0; n < HT; ++n) {
#pragma unroll
        for (int k = 0; k < C::MT; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][k][e] = 0.f;
        m[n][0] = m[n][1] = lim[n][0] = lim[n][1] = -INFINITY; l[n][0] = l[n][1] = base[n][0] = base[n][1] = 0.f; wbase[n][0] = wbase[n][1] = -1e30f;
    }
    int slot = 0;

#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
        __syncwarp();                                          // every lane has read the tile that the next copies replace
        issue_tile(i + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
        asm volatile("cp.async.wait_group %0;" :: "n"(STAGES - 1) : "memory");
        __syncwarp();
        const uint32_t st0 = fifo + slot * C::STAGE;
        slot = slot == STAGES - 1 ? 0 : slot + 1;
        const int p0 = first_tile + i * STEP;                  // the tile has positions p0 on
        if (last >= p0 && last < p0 + kTile) {                 // the new token's row: from where new_row left it
            const int key = last - p0;
            char* const to = smem + (st0 - static_cast<uint32_t>(__cvta_generic_to_shared(smem)));
            if (lane * 16 < C::HELD) *reinterpret_cast<uint4*>(to + C::at(key, C::spread(lane * 16))) = *reinterpret_cast<const uint4*>(fresh + lane * 16);
            if (F8 && lane < 2) to[C::SOFF + 2 * key + lane] = fresh_scale[lane];
            __syncwarp();
        }
        // ---- scores: positions g and g + 8 of a tile, heads 2 t and 2 t + 1; two chains of products each, for they wait for one another
        float sc[HT][4], odd[HT][4];
#pragma unroll
        for (int n = 0; n < HT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][e] = odd[n][e] = 0.f;
#pragma unroll
        for (int k = 0; k < C::KP; ++k) {
            uint32_t w[2][C::KB / 4];
            load_shared(st0 + C::at(g, (4 * k + t) * C::KB), w[0]);
            load_shared(st0 + C::at(g, (4 * k + t) * C::KB) + 8 * C::ROW, w[1]);      // s(g + 8) = s(g)
            constexpr int N = F8 ? C::KB / 4 : 2;              // steps of a piece
#pragma unroll
            for (int e = 0; e < N; ++e) {
                uint32_t ka[4];
                if constexpr (F8) { e4m3x4_half2(w[0][e], ka[0], ka[2]); e4m3x4_half2(w[1][e], ka[1], ka[3]); }
                else { ka[0] = w[0][2 * e]; ka[1] = w[1][2 * e]; ka[2] = w[0][2 * e + 1]; ka[3] = w[1][2 * e + 1]; }
#pragma unroll
                for (int n = 0; n < HT; ++n) mma<F8>(e & 1 ? odd[n] : sc[n], ka, qb[n][k * N + e][0], qb[n][k * N + e][1]);
            }
        }
#pragma unroll
        for (int n = 0; n < HT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][e] += odd[n][e];
        // ---- softmax.  A score is the product times its row's scale (ks), in units of 1 / fs; m is in the same units.
        bool valid[2];
        float ks[2], vlog[2];                                  // vlog: log2 of the value rows' scales
#pragma unroll
        for (int j = 0; j < 2; ++j) { valid[j] = p0 + 8 * j + g < r.end; ks[j] = 1.f; vlog[j] = 0.f; }
        if constexpr (F8) {
            uint32_t kb[2], vb[2];
            bool nan = false;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint16_t b;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(b) : "r"(st0 + C::SOFF + 2 * (8 * j + g)) : "memory");
                if (!valid[j]) b = 0;
                kb[j] = b & 255u; vb[j] = b >> 8;
                nan |= kb[j] == 255u || vb[j] == 255u;
                ks[j] = __uint_as_float(kb[j] << 23);              // a byte of 0 (2^-127, which no row of this library has): 0
                vlog[j] = log2_scale(vb[j]);
            }
            if (__any_sync(0xffffffffu, nan)) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (kb[j] == 255u) ks[j] = __uint_as_float(0x7fc00000u);
                    if (vb[j] == 255u) vlog[j] = __uint_as_float(0x7fc00000u);
                }
            }
        }
        uint32_t pb[HT][2], pl[HT][2];                         // P^T in two numbers of 16 bits
#pragma unroll
        for (int n = 0; n < HT; ++n) {
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float& v = sc[n][2 * j + x];
                    if constexpr (F8) v *= ks[j];
                    v = valid[j] ? v : -INFINITY;
                    mx[x] = fmaxf(mx[x], v);
                }
            if (__any_sync(0xffffffffu, mx[0] > lim[n][0] || mx[1] > lim[n][1])) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
#pragma unroll
                    for (int b = 4; b < 32; b <<= 1) mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], b));
                    const float mn = fmaxf(m[n][x], mx[x]), f = mn == -INFINITY ? 1.f : exp2_fast((m[n][x] - mn) * fs[n][x]);
                    m[n][x] = mn;
                    lim[n][x] = mn + kSlack / fs[n][x];
                    base[n][x] = mn == -INFINITY ? 0.f : mn * fs[n][x];
                    l[n][x] *= f;
                    if constexpr (!F8) {                           // in 8 bits the sums of values have a base of their own
#pragma unroll
                        for (int k = 0; k < C::MT; ++k) { o[n][k][x] *= f; o[n][k][2 + x] *= f; }
                    }
                }
            }
            float w[2][2];                                     // 8 bits: log2 of the operands
            if constexpr (F8) {
                const auto operands = [&] {
                    bool over = false;
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            w[j][e] = fmaf(sc[n][2 * j + e], fs[n][e], vlog[j] - wbase[n][e]);
                            over |= w[j][e] > kTop;
                        }
                    return __any_sync(0xffffffffu, over);
                };
                if (operands()) {
                    // a value row of zeros has a scale of 1 but no weight in the sum: left out
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t any = 0u;
#pragma unroll
                        for (int b = 0; b < D; b += 64) {
                            uint32_t u[4] = {0u, 0u, 0u, 0u};
                            if (b + 16 * t < D) load_shared(st0 + C::at(g, D + b + 16 * t) + 8 * j * C::ROW, u);
                            any |= (u[0] | u[1] | u[2] | u[3]) & 0x7f7f7f7fu;
                        }
                        any |= __shfl_xor_sync(0xffffffffu, any, 1); any |= __shfl_xor_sync(0xffffffffu, any, 2);
                        if (any == 0u) vlog[j] -= INFINITY;
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(fmaf(sc[n][e], fs[n][e], vlog[0]), fmaf(sc[n][2 + e], fs[n][e], vlog[1]));
#pragma unroll
                        for (int b = 4; b < 32; b <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, b));
                        const float moved = fmaxf(wbase[n][e], rintf(top) - kLevel), f = exp2_fast(wbase[n][e] - moved);
                        wbase[n][e] = moved;
#pragma unroll
                        for (int k = 0; k < C::MT; ++k) { o[n][k][e] *= f; o[n][k][2 + e] *= f; }
                    }
                    operands();
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float x[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    x[e] = exp2_fast(fmaf(sc[n][2 * j + e], fs[n][e], -base[n][e]));
                    l[n][e] += x[e];
                    if constexpr (F8) x[e] = exp2_fast(w[j][e]);
                }
                // Two operands of 16 bits, the number and what its rounding left: together off by 2^-15 of it (bf16) or 2^-22 (f16, see kTop).  One alone (2^-8 or
                // 2^-11) is seen in the result: in bf16 0.0023 from 64 bits (2-norms, 64 sequences up to 4096, 8 x 4 heads of 128), where the result's own
                // rounding to bf16 is 0.0017.
                uint32_t hi, lo;
                if constexpr (F8) {
                    hi = pack_f16x2(x[0], x[1]);
                    const float2 held = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                    lo = pack_f16x2(x[0] - held.x, x[1] - held.y);
                } else {
                    // cut off and not rounded, so that nothing of it is negative, and never 0: an infinity in a value row is one in the result, and no NaN
                    hi = __byte_perm(__float_as_uint(x[0]), __float_as_uint(x[1]), 0x7632);
                    lo = pack_bf16x2(fmaxf(x[0] - __uint_as_float(hi << 16), 1.17549435e-38f), fmaxf(x[1] - __uint_as_float(hi & 0xffff0000u), 1.17549435e-38f));
                }
                pb[n][j] = transposed(hi); pl[n][j] = transposed(lo);
            }
        }
        // ---- O^T += V^T P^T: rows g and g + 8 of m-tile (k VE + e) / 2 are d = 8 VE k + VE g + e and the next
#pragma unroll
        for (int k = 0; k < C::VP; ++k) {
            uint32_t w[4][C::VB / 4];
#pragma unroll
            for (int j = 0; j < 4; ++j)                    // positions 2 t, 2 t + 1 (+ 8)
                load_shared(st0 + C::at(2 * t + (j & 1), D * C::SZ + (8 * k + g) * C::VB) + 8 * (j >> 1) * C::ROW, w[j]);
#pragma unroll
            for (int x = 0; x < C::VB / 4; ++x) {
                if constexpr (F8) {
#pragma unroll
                    for (int y = 0; y < 2; ++y) {          // columns 2 y, 2 y + 1 of the word: {position, next position} of each
                        uint32_t va[4];
                        e4m3x4_half2(__byte_perm(w[0][x], w[1][x], y ? 0x7362 : 0x5140), va[0], va[1]);
                        e4m3x4_half2(__byte_perm(w[2][x], w[3][x], y ? 0x7362 : 0x5140), va[2], va[3]);
#pragma unroll
                        for (int n = 0; n < HT; ++n) {
                            mma<true>(o[n][(k * C::VE + 4 * x) / 2 + y], va, pb[n][0], pb[n][1]);
                            mma<true>(o[n][(k * C::VE + 4 * x) / 2 + y], va, pl[n][0], pl[n][1]);
                        }
                    }
                } else {
                    const uint32_t va[4] = {__byte_perm(w[0][x], w[1][x], 0x5410), __byte_perm(w[0][x], w[1][x], 0x7632),
                                            __byte_perm(w[2][x], w[3][x], 0x5410), __byte_perm(w[2][x], w[3][x], 0x7632)};
#pragma unroll
                    for (int n = 0; n < HT; ++n) {
                        mma<false>(o[n][(k * C::VE + 2 * x) / 2], va, pb[n][0], pb[n][1]);
                        mma<false>(o[n][(k * C::VE + 2 * x) / 2], va, pl[n][0], pl[n][1]);
                    }
                }
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // ---- the four warps' results, joined in warp order
    const bool any_bad = __syncthreads_or(bad);
    float* const sml = reinterpret_cast<float*>(smem);         // [warps][heads][2]
    float* const so = sml + kWarps * C::HEADS * 2;             // [warps][heads][D]
#pragma unroll
    for (int n = 0; n < HT; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int at = warp * C::HEADS + 8 * n + 2 * t + x;
#pragma unroll
            for (int b = 4; b < 32; b <<= 1) l[n][x] += __shfl_xor_sync(0xffffffffu, l[n][x], b);
            const float top = m[n][x] == -INFINITY ? 0.f : base[n][x];
            const float unit = F8 ? exp2f(0.5f * (wbase[n][x] - top)) : 1.f;         // twice, for 2^(w - base) alone may be out of range
            if (g == 0) { sml[at * 2] = m[n][x] == -INFINITY ? -INFINITY : base[n][x]; sml[at * 2 + 1] = l[n][x]; }
#pragma unroll
            for (int k = 0; k < C::VP; ++k)
#pragma unroll
                for (int e = 0; e < C::VE; ++e) so[at * D + 8 * C::VE * k + C::VE * g + e] = o[n][(k * C::VE + e) / 2][2 * (e & 1) + x] * unit * unit;
        }
    __syncthreads();
    for (int z = threadIdx.x; z < heads * DR; z += kWarps * 32) {
        const int row = z / DR, d = z - row * DR;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sml[(w * C::HEADS + row) * 2]);
        const float base = M == -INFINITY ? 0.f : M;
        float L = 0.f, A = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = exp2f(sml[(w * C::HEADS + row) * 2] - base);
            L = fmaf(f, sml[(w * C::HEADS + row) * 2 + 1], L); A = fmaf(f, so[(w * C::HEADS + row) * D + d], A);
        }
        if (any_bad) L = A = __uint_as_float(0x7fc00000u);
        if (a.ml) {
            const long long at = (q0 + row) * a.parts + part;
            if (d == 0) a.ml[at] = make_float2(M, L);
            a.acc[at * DR + d] = A;
        } else static_cast<__nv_bfloat16*>(a.out)[(q0 + row) * DR + d] = __float2bfloat16(L == 0.f ? 0.f : A / L);
    }
}

template <int D, bool F8, int HT, int STAGES, int CTAS> cudaError_t launch_one(const StepArgs& a, cudaStream_t s) {
    using C = Cfg<D, F8, HT, STAGES>;
    auto kern = step_mma_kernel<D, F8, HT, STAGES, CTAS>;
    static std::atomic<unsigned long long> done{0};
    if (cudaError_t e = allow_shared(reinterpret_cast<const void*>(kern), C::SMEM, done)) return e;
    return launch_after(kern, dim3(a.parts, a.c.H * ((a.G + C::HEADS - 1) / C::HEADS), a.c.S), kWarps * 32, C::SMEM, s, a);
}
template <int D, bool F8> cudaError_t launch_width(const StepArgs& a, cudaStream_t s) {
    // Two CTAs of four warps and 8-KB tiles in bf16, three in 8 bits, four up to 96 columns, two tiles ahead each: 88 us for 64 sequences up to 4096, 8 x 4 heads
    // of 128 in bf16 (84 at the rate of a copy), 55 us for 4 up to 100001, 4 x 8 heads of 128 in 8 bits (44).  With one number a probability, four CTAs in 8 bits: 17.7 -> 19.0
    // for 4 up to 20000, 33.1 -> 33.9 for 16 up to 8192; three at 80 columns 31.7 -> 32.7.  Three tiles ahead: the same.  bf16 with three CTAs and one tile ahead 1 % more, two tiles
    // a round 14 % more in 8 bits; tiles by the copy engine through a swizzled tensor map 2 % more in bf16 and 2 % less in 8 bits.
    if (a.G > 8) return launch_one<D, F8, 2, 3, 2>(a, s);
    return launch_one<D, F8, 1, 3, (!F8 ? 2 : D > 96 ? 3 : 4)>(a, s);
}
template <bool F8> cudaError_t launch_type(const StepArgs& a, cudaStream_t s) {
    switch (a.c.D) {
        case 32: return launch_width<32, F8>(a, s);
        case 48: return launch_width<48, F8>(a, s);
        case 64: return launch_width<64, F8>(a, s);
        case 80: return launch_width<80, F8>(a, s);
        case 96: return launch_width<96, F8>(a, s);
        default: return launch_width<128, F8>(a, s);
    }
}

}  // namespace

bool paged_mma_supported(const StepArgs& a) {
    return !a.q_f32 && (a.c.dtype == DSQG_DTYPE_BF16 || a.c.dtype == DSQG_DTYPE_E4M3) && (a.c.D % 32 == 0 || a.c.D == 48 || a.c.D == 80) && a.c.page % kTile == 0 &&
           (reinterpret_cast<uintptr_t>(a.c.scale) & 3u) == 0;
}
cudaError_t launch_paged_mma(const StepArgs& a, cudaStream_t s) { return a.c.dtype == DSQG_DTYPE_E4M3 ? launch_type<true>(a, s) : launch_type<false>(a, s); }

}  // namespace dsqg
