// Microscaled 4-bit format: quantize and dequantize kernels.
//
// Groups of 32 values along a row share one power of two, stored as a uint8
// exponent biased by 127 (255: not a number), and each value is a 4-bit float
// of 1 sign, 2 exponent and 1 mantissa bit: +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}
// (the Open Compute MX format with E2M1 elements and E8M0 scales).  Words u32
// [rows, cols / 8] hold value i of a group in bits 4i, low first; scales are
// [rows, cols / 32].
//
//   scale   2^(floor(log2 max|w|) - 2), no less than 2^-127: the largest value
//           lands in [4, 8)
//   code    w / scale to the nearest of the eight magnitudes, ties to the one
//           with an even mantissa bit, above 6 to 6
//   a group with an infinity or a NaN gets the scale 255, so all of its
//   values read back as NaN
//
// Every step is exact but the code's rounding: the quotient is a product with
// a power of two.  Rows are whole groups, so both kernels work on the flat
// list of groups, a few lanes a group, a wave's groups contiguous in every array.
// Both are bound by HBM: 24576 x 4096 quantize 78 us from fp32 (5.8 TB/s) and 49
// from bf16 (5.2 TB/s), dequant 64 us to fp32 and 36 to bf16 (7.1 TB/s).
#include <hip/hip_fp16.h>

#include "pmoe_internal.h"

namespace pmoe {

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int DT>
struct Elem;
template <>
struct Elem<PMOE_F32> {
  typedef float type;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Elem<PMOE_BF16> {
  typedef uint16_t type;
  static __device__ __forceinline__ float get(uint16_t v) { return bf16f(v); }
  static __device__ __forceinline__ uint16_t put(float v) { return f2bf(v); }
};
template <>
struct Elem<PMOE_F16> {
  typedef uint16_t type;
  static __device__ __forceinline__ float get(uint16_t v) {
    return __half2float(__ushort_as_half(v));
  }
  static __device__ __forceinline__ uint16_t put(float v) {
    return __half_as_ushort(__float2half_rn(v));
  }
};

// 8 elements, as 16-byte words where the array allows it.
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const typename Elem<DT>::type* src, float (&v)[8]) {
  typename Elem<DT>::type e[8];
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < int(sizeof(e) / 16); ++i)
      reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(src)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = src[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = Elem<DT>::get(e[i]);
}

// VEC: w is 16-byte aligned.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(
    const typename Elem<DT>::type* __restrict__ w, size_t groups, uint32_t* __restrict__ q,
    uint8_t* __restrict__ scales) {
  const size_t gid = size_t(blockIdx.x) * 64 + (threadIdx.x >> 2);
  const int sub = threadIdx.x & 3;
  float v[8];
  load8<DT, VEC>(w + (gid < groups ? gid : groups - 1) * 32 + sub * 8, v);
  // the largest magnitude by its bits: a NaN's are above every other's
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  top = max(top, uint32_t(__float_as_int(xor_lane<1>(__int_as_float(int(top))))));
  top = max(top, uint32_t(__float_as_int(xor_lane<2>(__int_as_float(int(top))))));
  const int e = int(top >> 23);  // 0: zero or denormal, below any scale's reach
  const bool bad = e == 255;
  const int s = e > 2 ? e - 2 : 0;
  // 2^(127 - s): s <= 252, and 2^127 at s = 0
  const float inv = __uint_as_float(uint32_t(254 - s) << 23);
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = fabsf(v[i]) * inv;  // in [0, 8)
    // rounded to steps of 1/2 below 2, of 1 below 4 and of 2 above, ties to
    // even: each step's own ties are the codes' ties
    const float r = t < 2.0f   ? __builtin_rintf(t * 2.0f)
                    : t < 4.0f ? __builtin_rintf(t) + 2.0f
                               : fminf(__builtin_rintf(t * 0.5f), 3.0f) + 4.0f;
    const uint32_t c = uint32_t(r) | (__float_as_uint(v[i]) >> 28 & 8u);
    word |= c << (4 * i);
  }
  if (gid >= groups) return;
  q[gid * 4 + sub] = bad ? 0u : word;
  if (sub == 0) scales[gid] = bad ? uint8_t(255) : uint8_t(s);
}

// A lane writes 16 bytes, so that a wave's stores are contiguous: 8 values of 16
// bits (4 lanes a group) or 4 of 32 (8 lanes).  VEC: out is 16-byte aligned.  NT:
// stores past the caches, for results that they would not hold anyway (24576 x 4096
// to fp32 97 -> 64 us, to bf16 41 -> 36).
template <int DT, bool VEC, bool NT>
__global__ __launch_bounds__(256) void mx4_dequant_kernel(
    const uint32_t* __restrict__ q, const uint8_t* __restrict__ scales, size_t groups,
    typename Elem<DT>::type* __restrict__ out) {
  constexpr int kVals = 16 / sizeof(typename Elem<DT>::type), kLanes = 32 / kVals;
  const size_t gid = size_t(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  const int sub = threadIdx.x % kLanes;
  if (gid >= groups) return;
  const uint32_t word = q[gid * 4 + sub * kVals / 8] >> (sub * kVals % 8 * 4);
  const uint32_t s = scales[gid];
  const float scale =
      __uint_as_float(s == 255 ? 0x7fc00000u : s == 0 ? 0x00400000u : s << 23);
  // the codes as they are (scale 1), then one product: exact in fp32 unless it
  // leaves fp32's range
  f32x2 p[4];
  p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 0);
  p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 1);
  p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 2);
  p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 3);
  typename Elem<DT>::type e[kVals];
#pragma unroll
  for (int i = 0; i < kVals; ++i) e[i] = Elem<DT>::put((i & 1 ? p[i / 2].y : p[i / 2].x) * scale);
  auto* dst = out + gid * 32 + sub * kVals;
  if constexpr (VEC) {
    const u32x4 v = *reinterpret_cast<const u32x4*>(e);
    if constexpr (NT)
      __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(dst));
    else
      *reinterpret_cast<u32x4*>(dst) = v;
  } else {
#pragma unroll
    for (int i = 0; i < kVals; ++i) dst[i] = e[i];
  }
}

// A launch holds at most 2^32 - 1 threads, 8 to a group at most: longer arrays go
// out in several.  go(first group, groups, blocks of `per` groups).
template <class Go>
void each_launch(size_t groups, int per, Go go) {
  constexpr size_t kMost = size_t(1) << 28;
  for (size_t g0 = 0; g0 < groups; g0 += kMost) {
    const size_t n = groups - g0 < kMost ? groups - g0 : kMost;
    go(g0, n, unsigned((n + per - 1) / per));
  }
}

constexpr size_t kPastCaches = size_t(64) << 20;  // bytes of a result

int check_format(const char* what, const void* a, const void* q, const void* s, int dtype,
                 int rows, int cols) {
  PMOE_REQUIRE(a && q && s, std::string(what) + ": null pointer");
  PMOE_REQUIRE(dtype == PMOE_F32 || dtype == PMOE_BF16 || dtype == PMOE_F16,
               std::string(what) + ": unknown dtype");
  PMOE_REQUIRE(rows >= 0 && cols > 0 && cols % 32 == 0,
               std::string(what) + ": cols must be a positive multiple of 32");
  PMOE_REQUIRE(reinterpret_cast<uintptr_t>(q) % 4 == 0 &&
                   reinterpret_cast<uintptr_t>(a) % (dtype == PMOE_F32 ? 4 : 2) == 0,
               std::string(what) + ": misaligned array");
  return PMOE_OK;
}

template <int DT>
void quantize_any(const void* w, size_t n, uint32_t* q, uint8_t* scales, hipStream_t st) {
  const auto* src = static_cast<const typename Elem<DT>::type*>(w);
  const bool vec = reinterpret_cast<uintptr_t>(w) % 16 == 0;
  each_launch(n, 64, [&](size_t g0, size_t groups, unsigned blocks) {
    if (vec)
      mx4_quantize_kernel<DT, true>
          <<<blocks, 256, 0, st>>>(src + g0 * 32, groups, q + g0 * 4, scales + g0);
    else
      mx4_quantize_kernel<DT, false>
          <<<blocks, 256, 0, st>>>(src + g0 * 32, groups, q + g0 * 4, scales + g0);
  });
}

template <int DT>
void dequant_any(const uint32_t* q, const uint8_t* scales, size_t n, void* out, hipStream_t st) {
  auto* dst = static_cast<typename Elem<DT>::type*>(out);
  const bool vec = reinterpret_cast<uintptr_t>(out) % 16 == 0;
  each_launch(n, DT == PMOE_F32 ? 32 : 64, [&](size_t g0, size_t groups, unsigned blocks) {
    const auto go = [&](auto kernel) {
      kernel<<<blocks, 256, 0, st>>>(q + g0 * 4, scales + g0, groups, dst + g0 * 32);
    };
    if (!vec)
      go(mx4_dequant_kernel<DT, false, false>);
    else if (n * 32 * sizeof(*dst) >= kPastCaches)
      go(mx4_dequant_kernel<DT, true, true>);
    else
      go(mx4_dequant_kernel<DT, true, false>);
  });
}

}  // namespace

}  // namespace pmoe

extern "C" int pmoe_mx4_quantize(const void* w, int dtype, int rows, int cols, uint32_t* q,
                                 uint8_t* scales, void* stream) {
  pmoe::clear_error();
  if (int rc = pmoe::check_format("mx4_quantize", w, q, scales, dtype, rows, cols)) return rc;
  const size_t n = size_t(rows) * (cols / 32);
  if (n == 0) return PMOE_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == PMOE_F32)
    pmoe::quantize_any<PMOE_F32>(w, n, q, scales, st);
  else if (dtype == PMOE_BF16)
    pmoe::quantize_any<PMOE_BF16>(w, n, q, scales, st);
  else
    pmoe::quantize_any<PMOE_F16>(w, n, q, scales, st);
  PMOE_LAUNCH_CHECK("mx4_quantize_kernel");
  return PMOE_OK;
}

extern "C" int pmoe_mx4_dequant(const uint32_t* q, const uint8_t* scales, int rows, int cols,
                                int dtype, void* out, void* stream) {
  pmoe::clear_error();
  if (int rc = pmoe::check_format("mx4_dequant", out, q, scales, dtype, rows, cols)) return rc;
  const size_t n = size_t(rows) * (cols / 32);
  if (n == 0) return PMOE_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == PMOE_F32)
    pmoe::dequant_any<PMOE_F32>(q, scales, n, out, st);
  else if (dtype == PMOE_BF16)
    pmoe::dequant_any<PMOE_BF16>(q, scales, n, out, st);
  else
    pmoe::dequant_any<PMOE_F16>(q, scales, n, out, st);
  PMOE_LAUNCH_CHECK("mx4_dequant_kernel");
  return PMOE_OK;
}
