// Rows of a cache entry held in eight bits.
//
// A row is one token's keys (or values) of one head: D numbers x_d, kept as D codes c_d and one exponent e with
// x_d ~ c_d * 2^e.  e4m3: c_d the e4m3 number nearest to x_d 2^-e (ties to even), e the smallest with max|x| <= 448 2^e.
// int8: c_d the whole number nearest to it, e the smallest with max|x| <= 127 2^e.  The scale is a power of two, so that a
// code times its scale is exact in bfloat16 (four or seven significant bits of eight) and the quantisation rounds once;
// e4m3 loses nothing by it, int8 up to one bit against a scale of max|x| / 127.
// e lies within -50..50 - beyond, codes saturate above and vanish below - and is 0 for a row of zeros; the byte e + 127 is what a
// float32's exponent field holds for 2^e.  Two rows' scales then lie within 2^100, inside float32's range however they meet.
// A row with an infinity or NaN has the byte 255 and codes of zero, and reads back as NaN.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>
#include <cuda_fp8.h>

enum { KVB_E4M3 = 0, KVB_INT8 = 1 };

namespace cq {

constexpr int EXP_MIN = -50, EXP_MAX = 50, BIAS = 127, NOT_FINITE = 255;

// The scale byte of a row whose largest magnitude has these float32 bits (sign cleared).
template <int STORE>
__device__ __forceinline__ int scale_byte(uint32_t top) {
    if (top >= 0x7f800000u) return NOT_FINITE;
    if (top == 0u) return BIAS;
    // top = (1 + frac) 2^p: 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6.
    const int p = (int)(top >> 23) - 127;
    const uint32_t frac = top & 0x7fffffu;
    const int e = STORE == KVB_E4M3 ? p - 8 + (frac > 0x600000u) : p - 6 + (frac > 0x7e0000u);
    return min(EXP_MAX, max(EXP_MIN, e)) + BIAS;
}
// 2^-e (0 for a row that is not finite: its codes are zeros) and 2^e (NaN for such a row) of a scale byte.
__device__ __forceinline__ float scale_down(int byte) { return byte == NOT_FINITE ? 0.f : __int_as_float((2 * BIAS - byte) << 23); }
__device__ __forceinline__ float scale_up(int byte) { return __int_as_float(byte == NOT_FINITE ? 0x7fffffff : byte << 23); }

// The code of a finite x times 2^-e, in the low byte, rounded once: on the way to e4m3 a float32 whose last bit says that something was left out.
template <int STORE>
__device__ __forceinline__ uint32_t code_of(double x, float down) {
    const double y = x * (double)down;
    if (STORE == KVB_INT8) {
        // Whole numbers by the sum with 1.5 * 2^52; |y| is far below 2^31 but for rows beyond 2^EXP_MAX, which saturate.
        const int c = __double2loint(fmin(fmax(y, -127.0), 127.0) + 6755399441055744.0);
        return (uint32_t)c & 0xffu;
    }
    const uint32_t left = (__double2loint(y) & 0x1fffffff) != 0 ? 1u : 0u;         // the 29 bits that a float32 has not
    return (uint32_t)__nv_cvt_float_to_fp8(__uint_as_float(__float_as_uint(__double2float_rz(y)) | left), __NV_SATFINITE, __NV_E4M3);
}
template <int STORE>
__device__ __forceinline__ float code_value(uint32_t code) {
    if (STORE == KVB_E4M3) return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3)));
    return (float)(int8_t)code;
}

}  // namespace cq
