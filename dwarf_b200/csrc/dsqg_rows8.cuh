// Rows held in 8 bits: e4m3 values and one power-of-two scale per row.
//
// scale = the smallest 2^e (e >= -126) with max|row| <= 448 * 2^e, 1 for a row of zeros, held as its exponent field
// (float8_e8m0fnu: byte b stands for 2^(b-127), 255 for NaN).  Dividing by a power of two rounds nothing, so a stored value is the
// row's value rounded once, to e4m3's four significant bits, and what a row holds does not depend on the order of any sum.  A scale
// with a mantissa would use the topmost binade better but changes no rounding error of a floating-point format by more than a binade's
// position; it would cost a second rounding and three more bytes.  A row with a NaN or an infinity in it is NaN as a whole.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "dsqg_common.cuh"

namespace dsqg {

// max|x| as the bits of a non-negative float: an integer maximum keeps NaN (above infinity) where fmaxf would drop it.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The scale's byte for a row whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t row_scale_byte(uint32_t top) {
    if (top >= 0x7f800000u) return 255u;
    if (top == 0u) return 127u;
    const int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u);     // 448 = 1.75 * 2^8
    return (uint32_t)(e < 1 ? 1 : e);
}
__device__ __forceinline__ float scale_value(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte ? byte << 23 : 0x00400000u);
}
// log2 of the scale that a byte below 255 stands for (of 0: -127)
__device__ __forceinline__ float log2_scale(uint32_t byte) { return __uint_as_float(0x4b000000u | byte) - 8388735.f; }
// 1 / scale of a byte that row_scale_byte gave (1 .. 247, or 255: NaN)
__device__ __forceinline__ float scale_inverse(uint32_t byte) { return byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float((254u - byte) << 23); }

__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}
// two e4m3 values (the low 16 bits) as half2: exact
__device__ __forceinline__ __half2 e4m3x2_half2(uint32_t two) {
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
    return __half2(r);
}
// four of them as two half2, in the bits of 32-bit words
__device__ __forceinline__ void e4m3x4_half2(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;}" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ void e4m3x4_float(uint32_t w, float* x) {
    const float2 a = __half22float2(e4m3x2_half2(w & 0xffffu)), b = __half22float2(e4m3x2_half2(w >> 16));
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}

// 2^x (2 ulp; results below 2^-126 become 0)
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

template <int WIDTH> __device__ __forceinline__ uint32_t group_max(uint32_t x) {
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1) x = max(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}

// Eight elements of a row at element i of a tensor in bf16, fp32 or e4m3 (its scale apart).
__device__ __forceinline__ void load8_as(const void* p, long long i, int dtype, float (&x)[8]) {
    if (dtype == DSQG_DTYPE_F32) load8(static_cast<const float*>(p) + i, x);
    else if (dtype == DSQG_DTYPE_BF16) load8(static_cast<const __nv_bfloat16*>(p) + i, x);
    else {
        const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p) + i);
        e4m3x4_float(u.x, x); e4m3x4_float(u.y, x + 4);
    }
}
__device__ __forceinline__ void store8_as(void* p, long long i, int dtype, const float (&x)[8]) {
    if (dtype == DSQG_DTYPE_F32) store8(static_cast<float*>(p) + i, x);
    else if (dtype == DSQG_DTYPE_BF16) store8(static_cast<__nv_bfloat16*>(p) + i, x);
    else *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p) + i) = make_uint2(pack_e4m3x4(x[0], x[1], x[2], x[3]), pack_e4m3x4(x[4], x[5], x[6], x[7]));
}

}  // namespace dsqg
