// Activations as sums of 6-bit floats under shared powers of two, the form in
// which the scaled matrix instructions take them beside 4-bit weights.
//
// A group of 32 values gets a power of two 2^e that brings its largest
// magnitude into [4, 8), and each value a is written as
//
//   a = 2^e (p0 + p1 / 16 + p2 / 1024) + rest    (tokens)
//   a = 2^e (p0 + p1 / 32) + rest                (intermediates)
//
// with p0 and p1 of 1 sign, 2 exponent and 3 mantissa bits (E2M3: steps of 1/8 up
// to 2, 1/4 up to 4, 1/2 up to 7.5) and p2 of 1 mantissa bit (E2M1, the weights'
// format), each the nearest to what the ones before leave over.
//
// Tokens are bf16.  Two pieces hold a value of at least an eighth of the
// group's largest exactly and any other to 2^-8 2^e, i.e. to 2^-10 of the
// largest, the rest of a value being at most 4 / 1024 2^e.  p2 is kept only where one value stands out of its group
// (its square is more than the sum of the other 31's, in trained models the few
// channels with huge activations), so that the others are not rounded to a
// step that it sets: they are then off by at most 2^-10 2^e, 2^-12 of the largest.
//
// Intermediates are fp32.  The second piece's smaller unit makes its steps half
// as wide where most values are (2^-9 2^e below 2, 2^-8 2^e below 4, 2^-7 2^e above,
// and 2^-6 2^e where a value all but halves two steps of p0 and p1 ends at
// 7.5): off by 2^-8 of the group's largest at most and by as much as a
// rounding to bf16 would be on average.  A largest value of 7.75 2^e and more
// takes the next power of two, since p0 ends at 7.5 and p1 could not reach
// the rest.
//
// A group that holds an infinity or a NaN gets the scale 255 (not a number).
#pragma once

#include "pmoe_internal.h"

namespace pmoe {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x32 __attribute__((ext_vector_type(32)));
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));

constexpr int kMxGroup = 32;
// A row of pieces goes by steps of 128 values (4 groups, the last step padded):
// p0 and p1 of a group are 48 bytes, chunk i of the step's groups side by side
// in 64 bytes, so that lanes side by side fetch whole 64-byte stretches.
constexpr int kMxStepGroups = 4;
constexpr int kMxStepPair = 192;      // 3 chunks of 4 x 16 bytes
constexpr int kMxStepThird = 64;      // p2: 4 x 16 bytes
constexpr int kMxChunk = 64;
// Their scales go by 512 values, 16 bytes: byte 4 q + i is group 4 i + q's, so
// that a lane finds its group's scales of four steps in one word.
constexpr int kMxScaleSteps = 4;
constexpr int kMxScaleBlock = 16;

__host__ __device__ constexpr int mx_steps(int cols) {
  return (cols / kMxGroup + kMxStepGroups - 1) / kMxStepGroups;
}

constexpr int kMxTokenShift = 4;      // p1's power of two below p0's
constexpr int kMxThirdShift = 10;     // p2's
constexpr int kMxInterShift = 5;
// The least scale byte of p0: the last piece's is at least 1.
constexpr int kMxMinToken = kMxThirdShift + 1, kMxMinInter = kMxInterShift + 1;

// 32 floats over 2^x to E2M3, nearest even.  The instruction takes the even
// and the odd values apart, and writes its result while it still reads its
// operands, which the compiler does not know: the empty statement keeps the
// operands alive so that the result gets registers of its own.
__device__ __forceinline__ u32x6 mx_to_fp6(const float (&v)[32], float scale) {
  f32x16 even, odd;
#pragma unroll
  for (int i = 0; i < 16; ++i) even[i] = v[2 * i], odd[i] = v[2 * i + 1];
  u32x6 r = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, scale);
  asm volatile("" : "+v"(r) : "v"(even), "v"(odd), "v"(scale));
  return r;
}

__device__ __forceinline__ f32x32 mx_from_fp6(u32x6 q, float scale) {
  f32x32 r = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(q, scale);
  asm volatile("" : "+v"(r) : "v"(q), "v"(scale));  // as above
  return r;
}

__device__ __forceinline__ float mx_pow2(int biased) {
  return __uint_as_float(uint32_t(biased) << 23);
}

// The scale byte of a group and its pieces; v is left with the rest.  THIRD: a
// token's, with p2 (zeros where no value stands out, and then false).
template <bool THIRD>
__device__ __forceinline__ bool mx_split(float (&v)[32], int& scale, u32x6& p0, u32x6& p1,
                                         uint4& p2) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  const int e = int(top >> 23);
  // intermediates: 7.75 = 4 * 1.9375, the mantissa 0xf8 over 8 bits
  const int up = !THIRD && (top & 0x7fffffu) >= 0x780000u ? 1 : 0;
  const int s = max(e - 2 + up, THIRD ? kMxMinToken : kMxMinInter);
  bool peak = false;
  if constexpr (THIRD) {
    // in units of 2^s the squares neither overflow nor vanish
    const float inv = mx_pow2(254 - s);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float t = v[i] * inv;
      sum = __builtin_fmaf(t, t, sum);
    }
    const float t = __uint_as_float(top) * inv;
    peak = 2.0f * t * t > sum;
  }
  const float f = mx_pow2(s);
  p0 = mx_to_fp6(v, f);
  f32x32 b = mx_from_fp6(p0, f);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] -= b[i];
  const float f1 = mx_pow2(s - (THIRD ? kMxTokenShift : kMxInterShift));
  p1 = mx_to_fp6(v, f1);
  p2 = make_uint4(0, 0, 0, 0);
  if constexpr (THIRD) {
    if (peak) {
      b = mx_from_fp6(p1, f1);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] -= b[i];
      const float f2 = mx_pow2(s - kMxThirdShift);
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], v[8 * i], v[8 * i + 1], f2, 0);
        w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], v[8 * i + 2], v[8 * i + 3], f2, 1);
        w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], v[8 * i + 4], v[8 * i + 5], f2, 2);
        w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], v[8 * i + 6], v[8 * i + 7], f2, 3);
      }
      p2 = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  scale = e == 255 ? 255 : s;
  return peak;
}

__host__ __device__ constexpr int mx_scale_row(int cols) {
  return (mx_steps(cols) + kMxScaleSteps - 1) / kMxScaleSteps * kMxScaleBlock;
}

// Where group g's scale lies in a row of scales.
__device__ __forceinline__ int mx_scale_at(int g) {
  return (g & ~15) + 4 * (g & 3) + (g >> 2 & 3);
}

// Group g's pieces into a row of pieces.
__device__ __forceinline__ void mx_store_pair(uint8_t* row, int g, u32x6 p0, u32x6 p1) {
  uint8_t* d = row + (g >> 2) * kMxStepPair + (g & 3) * 16;
  *reinterpret_cast<uint4*>(d) = make_uint4(p0[0], p0[1], p0[2], p0[3]);
  *reinterpret_cast<uint4*>(d + kMxChunk) = make_uint4(p0[4], p0[5], p1[0], p1[1]);
  *reinterpret_cast<uint4*>(d + 2 * kMxChunk) = make_uint4(p1[2], p1[3], p1[4], p1[5]);
}

__device__ __forceinline__ void mx_store_third(uint8_t* row, int g, uint4 p2) {
  *reinterpret_cast<uint4*>(row + (g >> 2) * kMxStepThird + (g & 3) * 16) = p2;
}

}  // namespace pmoe
