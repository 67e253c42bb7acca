// Rows of keys and values held in 8 bits: e4m3 codes and one power of two for the row (a head's entries of one token, of keys
// or of values).
//
//   amax = max |x_i|;  e = the smallest whole number with amax <= 448 * 2^e, at least -60;
//   code_i = x_i * 2^-e rounded to e4m3 (ties to even);  scale byte = e + 127;  the entry stands for code_i * 2^e.
//
// A power of two costs nothing against amax / 448: e4m3 has floating steps, so an entry's relative rounding is 2^-4 at most
// wherever the entry is at least 2^-6 * 2^e, whatever the scale; and a product with it is exact: writing needs no division whose
// rounding could break a tie, reading gives numbers that bfloat16 holds exactly, and in the attention kernels the scale is an
// addition to an exponent.  What 8 bits cannot hold (a row with an infinity or a NaN, or beyond 448 * 2^60) keeps scale byte
// 255 and codes 0, and reads back as NaN in all its entries: the row's one byte says it, no code does, so a masked row can
// never reach a sum.  Rows below 448 * 2^-60 keep e = -60 (they are off by up to 2^-70).
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

#define FP8_MIN_EXP (-60)
#define FP8_LIMIT 0x1.cp68f  // 448 * 2^60, to the last bit
#define FP8_BAD 255

// 2^e for -126 <= e <= 127
__device__ __forceinline__ float fp8_pow2(int e) { return __int_as_float((e + 127) << 23); }

// The scale's exponent for a row of this amax (finite, not above FP8_LIMIT): 448 = 1.75 * 2^8.
__device__ __forceinline__ int fp8_row_exp(float amax) {
  const uint32_t b = __float_as_uint(amax);
  return max((int)(b >> 23) - 127 - 8 + ((b & 0x7fffff) > 0x600000), FP8_MIN_EXP);
}

// What a scale byte stands for (255: NaN).  Byte 0, a row that was never written (no row is kept with it; its codes are 0), gives 0.
__device__ __forceinline__ float fp8_scale(int byte) { return byte == FP8_BAD ? __int_as_float(0x7fc00000) : __int_as_float(byte << 23); }
// The byte whose exponent goes into the weights of the values: a row that was never written is one of zeros, which is kept with
// the smallest scale.  (With 2^-127 its weight would leave the 32-bit range and its share of the softmax's sum be lost, with 2^0
// it could set the reference of rows that hold far smaller values.)
__device__ __forceinline__ int fp8_weight_byte(int byte) { return byte == 0 ? FP8_MIN_EXP + 127 : byte; }

// Four codes -> two pairs of float16 (exact: float16 holds every e4m3 number).
__device__ __forceinline__ void fp8x4_to_half(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(codes));
}

// Four numbers -> four codes, ties to even.
__device__ __forceinline__ uint32_t fp8x4_from_float(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
