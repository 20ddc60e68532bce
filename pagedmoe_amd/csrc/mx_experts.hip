// Routed SwiGLU experts over microscaled 4-bit weights (group 32 geometries).
//
// y = W_down (silu(W_gate x) * (W_up x)) for the rows of each expert.  The
// weights go into the scaled matrix instructions as they lie in the slab: a
// lane of mfma_scale_f32_16x16x128 takes 32 consecutive 4-bit values of one
// row, which is one group of the format, and that group's scale byte, so
// nothing is unpacked.  The activations come beside them as 6-bit pieces
// (mx_pieces.h), two products for each step, three for the few steps in which
// a value stands out; the sums are fp32.
//
// Three forms, by the rows of the call:
//   few tokens,   one by one, two launches without a dispatch: gate/up from x itself,
//   small experts and the down projection with the columns' weighted sum inside
//   few rows an   dispatch and activation pieces in one launch (mx_prepare_kernel),
//   expert        tiles of 16 rows bound by the weights' stream, a combine
//   many          tiles of 128 rows bound by the matrix instructions and the loads
//                 beside them
// The lines between them stand at mx_one_tokens and mx_tile_rows.
//
// An activation that is infinite or NaN, or an intermediate that leaves fp32,
// makes the outputs of its row NaN.
#include <hip/hip_fp16.h>
#include <math.h>
#include <stdlib.h>

#include <algorithm>
#include <type_traits>

#include "dispatch_small.h"
#include "mx_experts.h"
#include "mx_pieces.h"
#include "pmoe_internal.h"
#include "pmoe_kernels.h"

namespace pmoe {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kFp4 = 4, kFp6 = 2;  // operand formats of the scaled MFMA
constexpr int kStretch = 512;      // values of a row whose scales are 16 bytes

__device__ __forceinline__ const uint8_t* uniform_ptr(const uint8_t* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(uint32_t(v >> 32));
  return reinterpret_cast<const uint8_t*>(uint64_t(lo) | uint64_t(hi) << 32);
}

// Four groups' scale bytes, of which `left` are there; 127 (one) for the others.
__device__ __forceinline__ uint32_t scale_word(const uint8_t* at, int left) {
  uint32_t v = 0x7f7f7f7f;
  if (left >= 4) {
    __builtin_memcpy(&v, at, 4);
  } else {
#pragma unroll
    for (int b = 0; b < 3; ++b)
      if (b < left) v = (v & ~(0xffu << 8 * b)) | uint32_t(at[b]) << 8 * b;
  }
  return v;
}

// acc += W (16 rows x 128) times a piece of 16 activation rows; sw, sp: the
// lane's scale bytes.
__device__ __forceinline__ void mx_mma(f32x4& acc, const uint4& w, int sw, const uint32_t (&p)[6],
                                       int sp) {
  const i32x8 a = {int(w.x), int(w.y), int(w.z), int(w.w), 0, 0, 0, 0};
  const i32x8 b = {int(p[0]), int(p[1]), int(p[2]), int(p[3]), int(p[4]), int(p[5]), 0, 0};
  acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, kFp4, kFp6, 0, sw, 0, sp);
}

// The same with a third piece, in the weights' format.
__device__ __forceinline__ void mx_mma_third(f32x4& acc, const uint4& w, int sw, const uint4& p,
                                             int sp) {
  const i32x8 a = {int(w.x), int(w.y), int(w.z), int(w.w), 0, 0, 0, 0};
  const i32x8 b = {int(p.x), int(p.y), int(p.z), int(p.w), 0, 0, 0, 0};
  acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, kFp4, kFp4, 0, sw, 0,
                                                         sp - kMxThirdShift);
}

// ---------------------------------------------------------------- slot outputs
//
// Outputs that go on to the combine are held in 16 bits: fp16 under a power of
// two for each 32 features of a row (scale byte s: value 2^(s - 127)), which
// leaves 2^-12 of a value where bf16 would leave 2^-9.  The largest of the 32 is
// brought into [2^14, 2^15).  255: an infinity or a NaN among them.

__device__ __forceinline__ int half_scale(uint32_t top) {
  const int e = int(top >> 23);
  return e == 255 ? 255 : max(e - 14, 1);
}

__device__ __forceinline__ uint16_t half_of(float v, int s) {
  return __half_as_ushort(__float2half_rn(v * mx_pow2(254 - min(s, 253))));
}

__device__ __forceinline__ float half_unit(int s) {
  return s == 255 ? __uint_as_float(0x7fc00000u) : mx_pow2(s);
}

// The largest over the lane's half of the wave (32 lanes).
__device__ __forceinline__ uint32_t half_wave_max(uint32_t v) {
  auto other = [&](auto d) {
    return uint32_t(__float_as_int(xor_lane<decltype(d)::value>(__int_as_float(int(v)))));
  };
  v = max(v, other(std::integral_constant<int, 16>{}));
  v = max(v, other(std::integral_constant<int, 8>{}));
  v = max(v, other(std::integral_constant<int, 4>{}));
  v = max(v, other(std::integral_constant<int, 2>{}));
  v = max(v, other(std::integral_constant<int, 1>{}));
  return v;
}

// Slot outputs of this size are written and read past the caches, which would not
// hold them.
inline bool past_caches(int64_t values) { return values >= int64_t(128) << 20; }

// out[n] = bf16(fma over k of weight * y, then the shared expert's times 1 or
// sigmoid(shared_logit[n])), in column order; 8 features a thread.  Bound by HBM:
// 16384 tokens x 8 columns x 4096 features 195 us (6.2 TB/s; 242 with ordinary loads,
// one column at a time); of few tokens by its launch and two rounds of loads (5 us).
template <bool PAST>
__global__ __launch_bounds__(256) void mx_combine_kernel(
    const uint16_t* __restrict__ y, const uint8_t* __restrict__ yscale,
    const float* __restrict__ w, const int32_t* __restrict__ inv,
    const float* __restrict__ shared_logit, int k, int kk, int d, int blocks_row,
    uint16_t* __restrict__ out) {
  const int n = blockIdx.x / blocks_row;
  const int d0 = ((blockIdx.x - n * blocks_row) * 256 + threadIdx.x) * 8;
  if (d0 >= d) return;
  float a[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int kBatch = 4;  // columns whose loads are in flight together
  for (int c0 = 0; c0 < kk; c0 += kBatch) {
    u32x4 v[kBatch];
    float wt[kBatch], unit[kBatch];
    bool in[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int c = min(c0 + j, kk - 1);
      const size_t r = size_t(n) * kk + c;
      const u32x4* src = reinterpret_cast<const u32x4*>(y + r * d + d0);
      if constexpr (PAST)
        v[j] = __builtin_nontemporal_load(src);
      else
        v[j] = *src;
      unit[j] = half_unit(yscale[r * (d / kMxGroup) + d0 / kMxGroup]);
      wt[j] = c < k ? w[size_t(n) * k + c] : shared_logit ? psigmoid(shared_logit[n]) : 1.0f;
      in[j] = c0 + j < kk && inv[r] >= 0;  // a dropped id's row holds anything
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (!in[j]) continue;
      const uint32_t p[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[2 * i] = __builtin_fmaf(
            wt[j], __half2float(__ushort_as_half(uint16_t(p[i]))) * unit[j], a[2 * i]);
        a[2 * i + 1] = __builtin_fmaf(
            wt[j], __half2float(__ushort_as_half(uint16_t(p[i] >> 16))) * unit[j], a[2 * i + 1]);
      }
    }
  }
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = uint32_t(f2bf(a[2 * i])) | uint32_t(f2bf(a[2 * i + 1])) << 16;
  *reinterpret_cast<uint4*>(out + size_t(n) * d + d0) = make_uint4(o[0], o[1], o[2], o[3]);
}

// ---------------------------------------------------------------- activations

struct MxSplit {
  const uint16_t* x;  // bf16 [n, 32 * groups]
  int n, groups, steps, scale_row;
  uint8_t *pair, *third, *scales;
  uint16_t* masks;              // [n, 4]
  const uint16_t* shared_gate;  // or null: shared_logit[n] = x . shared_gate
  float* shared_logit;
  const int32_t* ids;           // [n, k]
  int k, n_experts;
  uint16_t* y;                  // or null: rows [n, k, d] of ids out of range become zero
};

// A token by 256 threads, a lane a group: its pieces, scales and the mask of the
// 128-wide steps that hold a third piece (16 bits a wave), the shared expert's gate
// logit, the zero rows of ids that are dropped.  s_sum: 4 floats of the token's.
// 16384 x 4096: 134 MB in, 280 MB out, 64 us beside the dispatch's scan.  Splitting
// in the products instead would repeat these ~20 operations a value for every block of features.
__device__ __forceinline__ void split_token(const MxSplit& a, int token, int g, float* s_sum) {
  bool peak = false;
  float dot = 0.0f;
  if (token < a.n && g < a.groups) {
    const size_t row = size_t(token) * a.steps;
    const uint4* src =
        reinterpret_cast<const uint4*>(a.x + (size_t(token) * a.groups + g) * kMxGroup);
    float v[32];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 u = src[i];
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[8 * i + 2 * j] = bf16lo(w[j]), v[8 * i + 2 * j + 1] = bf16hi(w[j]);
    }
    if (a.shared_gate)
#pragma unroll
      for (int i = 0; i < 32; ++i)
        dot = __builtin_fmaf(v[i], bf16f(a.shared_gate[g * kMxGroup + i]), dot);
    int s;
    u32x6 p0, p1;
    uint4 p2;
    peak = mx_split<true>(v, s, p0, p1, p2);
    mx_store_pair(a.pair + row * kMxStepPair, g, p0, p1);
    mx_store_third(a.third + row * kMxStepThird, g, p2);
    a.scales[size_t(token) * a.scale_row + mx_scale_at(g)] = uint8_t(s);
  } else if (token < a.n && g < a.steps * kMxStepGroups) {  // zeros to the end of the step
    const size_t row = size_t(token) * a.steps;
    mx_store_pair(a.pair + row * kMxStepPair, g, u32x6{}, u32x6{});
    mx_store_third(a.third + row * kMxStepThird, g, make_uint4(0, 0, 0, 0));
    a.scales[size_t(token) * a.scale_row + mx_scale_at(g)] = 127;
  }
  const uint64_t m = __ballot(peak);
  if (token < a.n && (g & 63) == 0) {
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) bits |= (m >> (4 * i) & 15) ? 1u << i : 0u;
    a.masks[size_t(token) * 4 + (g >> 6)] = uint16_t(bits);
  }
  if (a.shared_gate) {
    dot = wave_sum_bfly(dot);
    if ((g & 63) == 0) s_sum[g >> 6] = dot;
    __syncthreads();
    if (token < a.n && g == 0) a.shared_logit[token] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
  }
  if (a.y && token < a.n) {
    const int d = a.groups * kMxGroup;
    for (int c = 0; c < a.k; ++c) {
      const size_t row = size_t(token) * a.k + c;
      const int e = a.ids[row];
      if (e >= 0 && e < a.n_experts) continue;
      for (int i = g * 8; i < d; i += 256 * 8)
        *reinterpret_cast<uint4*>(a.y + row * d + i) = make_uint4(0, 0, 0, 0);
    }
  }
}

// The dispatch of a small call beside its split: block 0 dispatches, the others
// take four tokens each.  5 us for 24 rows, 7 for 800: the dispatching block's
// barriers, under which the split hides (two launches took 4 us more).
struct MxDispatch {
  IdSrc src;
  int rows, n_ids;
  int32_t* hist;  // large calls: the counts of each kDispatchChunk rows
  int32_t *order, *counts, *offsets, *inv, *active, *n_active;
  TileSink tiles;
};

__global__ __launch_bounds__(1024) void mx_prepare_kernel(const MxSplit a, const MxDispatch d) {
  __shared__ DispatchLds lds;
  if (blockIdx.x == 0) {
    dispatch_small(lds, d.src, d.rows, d.n_ids, d.order, d.counts, d.offsets, d.inv, d.active,
                   d.n_active, d.tiles);
    return;
  }
  const int quarter = threadIdx.x >> 8;
  split_token(a, (blockIdx.x - 1) * 4 + quarter, threadIdx.x & 255,
              reinterpret_cast<float*>(lds.tmp) + 4 * quarter);
}

// The same of a large call, between the dispatch's count and its scatter: block 0
// scans (4096 tokens x 10 of 2048, the whole call 456 -> 443 us against two launches;
// 16384 x 8 of 4096: 48 + 39 -> 64).
__global__ __launch_bounds__(1024) void mx_scan_split_kernel(const MxSplit a, const MxDispatch d) {
  __shared__ ScanLds lds;
  if (blockIdx.x == 0) {
    dispatch_scan(lds, d.hist, (d.rows + kDispatchChunk - 1) / kDispatchChunk, d.n_ids, d.counts,
                  d.offsets, d.active, d.n_active, d.tiles);
    return;
  }
  const int quarter = threadIdx.x >> 8;
  split_token(a, (blockIdx.x - 1) * 4 + quarter, threadIdx.x & 255,
              reinterpret_cast<float*>(lds.tmp) + 4 * quarter);
}

// ---------------------------------------------------------------- memory to LDS

// 16 bytes (4 bytes) a lane from base + voff to LDS [lds, lds + 1024) ([.., +
// 256)), lane l at 16 l (4 l).  base and lds are the wave's.  ONCE: nobody reads
// them again (non-temporal).
template <bool ONCE = false>
__device__ __forceinline__ void dma16(uint32_t lds, uint32_t voff, const uint8_t* base) {
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(uniform_ptr(base))
                 : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(uniform_ptr(base))
                 : "memory");
}

__device__ __forceinline__ void dma4(uint32_t lds, uint32_t voff, const uint8_t* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(uniform_ptr(base))
               : "memory");
}

// Rows of 4, 8 or 16 chunks of 16 bytes lie in LDS with chunk p of row r at place
// p ^ swizzle(r).  A 16-byte LDS read takes its lanes in sets of 16: 0-3, 12-15,
// 20-23, 24-27 and so on, which here are rows 0-3 and 12-15 of one chunk and 4-11
// of the next (lane 16 q + r reads chunk 4 i + q of row r); with these the 16
// meet the 16 groups of four banks once each.
__device__ __forceinline__ int swizzle4(int r) { return -(r >> 2) & 3; }
__device__ __forceinline__ int swizzle8(int r) { return (r >> 1 & 4) | (r & 2); }
__device__ __forceinline__ int swizzle16(int r) { return (r & 3) << 1 | (r & 8); }

// ---------------------------------------------------------------- streamed tiles

constexpr int kFewRows = 16;                       // activation rows a tile
constexpr int kMaxWaves = 8;
constexpr int kStreamStep = 256;                   // reduction that a wave takes at a time
constexpr int kStreamRows = 64;                    // weight rows a block
constexpr int kStreamWave = kStreamRows * 128 + 2 * kStreamRows * 4;  // LDS of a wave

// One tile of at most 16 rows of an expert times 64 weight rows (DUAL: 32 gate and
// the same 32 up features; 64 features otherwise).  The waves share the reduction:
// wave w takes steps w, w + waves, ... of 256, and the partial sums meet in LDS.
// Bound by the weights' stream: a wave's 64 rows x 128
// bytes go straight into its own LDS, 8 lanes side by side on a row's 128 bytes,
// so that nothing waits for registers and the fetches are whole lines; two
// blocks a CU keep 136 KB in flight.  (Loads into registers in the products' own
// lane order, 16 bytes of 64 different rows an instruction, reached 3 TB/s.)  7168x2048
// experts, 3 tokens: 573 MB in 76 + 39 us, 5.0 TB/s; 4096x1536, 100 tokens seam: 435 MB
// in 64 + 33, 4.5 TB/s; 2048x512, 29 tokens: 375 MB in 55 + 25, 4.7 TB/s.
// ONCE: an expert has one tile on average, and its weights need no place in the
// caches (us, gate/up + down, without / with it: 4096x1536 8 tokens 66 + 36 / 62 + 33,
// 7168x2048 3 tokens 80 + 42 / 76 + 40).
// WHOLE: the reduction is whole steps of 128, and its scales lie on 4 bytes, so that
// they come the weights' way; otherwise through registers, and groups past the
// row's end count as zeros.
template <bool DUAL, bool HALF, bool ONCE, bool WHOLE>
__global__ __launch_bounds__(64 * kMaxWaves, 4) void mx_stream_kernel(const MxArgs a) {
  constexpr int NF = 4;
  constexpr int kCols = DUAL ? kStreamRows / 2 : kStreamRows;  // features a block
  extern __shared__ __attribute__((aligned(1024))) uint8_t dyn[];
  const int fblocks = (a.features + kCols - 1) / kCols;
  const int t = blockIdx.x / fblocks;
  const int fb = blockIdx.x - t * fblocks;
  if (t >= *a.n_tiles) return;
  const int4 tile = a.tiles[t];  // {slot, first row, rows of the expert, offset}
  const int m = min(kFewRows, tile.z - tile.y);
  const int p0 = tile.w + tile.y;
  const int waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int cols_in = min(kCols, a.features - fb * kCols);
  if (tile.x < 0) {  // not resident: exact zero rows
    if constexpr (!DUAL) {
      for (int i = threadIdx.x; i < m * kCols; i += blockDim.x) {
        const int c = i % kCols;
        if (c >= cols_in) continue;
        const size_t at = size_t(a.order[p0 + i / kCols]) * a.features + fb * kCols + c;
        a.y[at] = 0;
        if (HALF && c % kMxGroup == 0) a.yscale[at / kMxGroup] = 1;
      }
    }
    return;
  }
  const int r = lane & 15, q = lane >> 4;
  const int groups = a.cols / kMxGroup;
  const int steps = (groups + kMxStepGroups - 1) / kMxStepGroups;
  const uint8_t* base = a.slab + size_t(tile.x) * size_t(a.expert_bytes);
  const uint32_t row_bytes = a.cols / 2;
  // weight tile f: 16 features from f16 of projection f / 2 (DUAL); tiles past the
  // projection load its last one and are not used
  const auto feature0 = [&](int f) {
    return min(fb * kCols + 16 * (DUAL ? f & 1 : f), a.features - 16);
  };
  const uint8_t* wbase[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f)
    wbase[f] = base + (DUAL && f > 1 ? a.w1 : a.w0) + size_t(feature0(f)) * row_bytes;
  // rows 8 i + lane / 8 of a tile; their chunks' order goes by the row
  const int lrow = lane >> 3;
  const int lp[2] = {(lane & 7) ^ swizzle8(lrow), (lane & 7) ^ swizzle8(lrow + 8)};
  const uint8_t* sbase = base + (DUAL && q > 1 ? a.s1 : a.s0) + size_t(feature0(q) + r) * groups;
  uint8_t* own = dyn + wave * kStreamWave;
  const uint32_t own_lds = __builtin_amdgcn_readfirstlane(
      uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)own)));
  const bool live = r < m;
  const size_t arow = live ? (DUAL ? size_t(a.order[p0 + r] / a.kk) : size_t(p0 + r)) : 0;
  const uint8_t* pair = a.pair + arow * steps * kMxStepPair + q * 16;
  const uint8_t* third = DUAL ? a.third + arow * steps * kMxStepThird + q * 16 : nullptr;
  const uint8_t* ascale = a.ascale + arow * mx_scale_row(a.cols) + q * 4;

  f32x4 acc[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int j = wave; 2 * j < steps; j += waves) {
    const bool two = 2 * j + 1 < steps;  // the step's second half is there
    const auto group_in = [&](int i) {   // the lane's group of half i is there
      return WHOLE ? i == 0 || two : 8 * j + 4 * i + q < groups;
    };
    // this step's activations (rows that are not there: zeros)
    uint4 c[2][3], d[2];
    uint32_t sa4 = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int k = 0; k < 3; ++k) c[i][k] = make_uint4(0, 0, 0, 0);
      d[i] = make_uint4(0, 0, 0, 0);
    }
    if (live) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (group_in(i)) {
          const uint8_t* src = pair + (2 * j + i) * kMxStepPair;
#pragma unroll
          for (int k = 0; k < 3; ++k) c[i][k] = *reinterpret_cast<const uint4*>(src + k * kMxChunk);
          if constexpr (DUAL)
            d[i] = *reinterpret_cast<const uint4*>(third + (2 * j + i) * kMxStepThird);
        }
      }
      sa4 = *reinterpret_cast<const uint32_t*>(ascale + (j >> 1) * kMxScaleBlock);
    }
    uint32_t sword[2];
    if constexpr (!WHOLE)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        sword[i] = scale_word(sbase + 8 * j + 4 * i, groups - 8 * j - 4 * i);
    // the LDS reads of the step before are done
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int f = 0; f < NF; ++f) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (WHOLE ? two || lp[i] < 4 : 8 * j + lp[i] < groups)
          dma16<ONCE>(own_lds + f * 2048 + i * 1024, lrow * row_bytes + lp[i] * 16,
                      wbase[f] + size_t(8 * i) * row_bytes + j * 128);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (WHOLE && (i == 0 || two))
        dma4(own_lds + NF * 2048 + i * 256, uint32_t(sbase - base) + (2 * j + i) * 4, base);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (!WHOLE)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<uint32_t*>(own + NF * 2048 + i * 256 + lane * 4) = sword[i];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i && !two) break;
      const int at = (r * 8 + ((4 * i + q) ^ swizzle8(r))) * 16;
      // (an absent group's scale byte was never written)
      const int sa = group_in(i) ? int(sa4 >> (8 * (2 * (j & 1) + i))) : 127;
      uint4 w[NF];
      int sw[NF];
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        w[f] = *reinterpret_cast<const uint4*>(own + f * 2048 + at);
        sw[f] = own[NF * 2048 + i * 256 + (16 * f + r) * 4 + q];
      }
      const uint32_t b0[6] = {c[i][0].x, c[i][0].y, c[i][0].z, c[i][0].w, c[i][1].x, c[i][1].y};
      const uint32_t b1[6] = {c[i][1].z, c[i][1].w, c[i][2].x, c[i][2].y, c[i][2].z, c[i][2].w};
#pragma unroll
      for (int f = 0; f < NF; ++f) mx_mma(acc[f], w[f], sw[f], b0, sa);
#pragma unroll
      for (int f = 0; f < NF; ++f)
        mx_mma(acc[f], w[f], sw[f], b1, sa - (DUAL ? kMxTokenShift : kMxInterShift));
      if constexpr (DUAL)
#pragma unroll
        for (int f = 0; f < NF; ++f) mx_mma_third(acc[f], w[f], sw[f], d[i], sa);
    }
  }
  // partial sums meet in LDS: [wave][4 f + i][lane]
  float(*red)[16][64] = reinterpret_cast<float(*)[16][64]>(dyn);
  float(*hs)[kCols + 1] = reinterpret_cast<float(*)[kCols + 1]>(dyn + waves * sizeof(red[0]));
  __syncthreads();
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) red[wave][4 * f + i][lane] = acc[f][i];
  __syncthreads();
  for (int i = threadIdx.x; i < kFewRows * kCols; i += blockDim.x) {
    const int row = i / kCols, c = i % kCols;
    if (row >= m) break;  // whole halves of a wave
    const int src = (c & 15) / 4 * 16 + row;
    float v = 0.0f, u = 0.0f;
    for (int k = 0; k < waves; ++k) {
      v += red[k][4 * (c >> 4) + (c & 3)][src];
      if constexpr (DUAL) u += red[k][4 * (2 + (c >> 4)) + (c & 3)][src];
    }
    if constexpr (DUAL) {
      hs[row][c] = silu_fast(v) * u;
    } else if (c < cols_in) {  // (a multiple of 32)
      const size_t at = size_t(a.order[p0 + row]) * a.features + fb * kCols + c;
      if constexpr (HALF) {
        const int sc = half_scale(half_wave_max(__float_as_uint(v) & 0x7fffffffu));
        a.y[at] = half_of(v, sc);
        if (c % kMxGroup == 0) a.yscale[at / kMxGroup] = uint8_t(sc);
      } else {
        a.y[at] = f2bf(v);
      }
    }
  }
  if constexpr (DUAL) {
    __syncthreads();
    if (int(threadIdx.x) < m) {
      float v[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) v[c] = hs[threadIdx.x][c];
      int s;
      u32x6 h0, h1;
      uint4 none;
      mx_split<false>(v, s, h0, h1, none);
      const size_t row = p0 + threadIdx.x;
      mx_store_pair(a.hpair + row * mx_steps(a.features) * kMxStepPair, fb, h0, h1);
      a.hscale[row * mx_scale_row(a.features) + mx_scale_at(fb)] = uint8_t(s);
    }
  }
}

template <bool DUAL, bool HALF>
int launch_stream(const MxArgs& a, int max_tiles, bool once, bool whole, hipStream_t st) {
  constexpr int kCols = DUAL ? kStreamRows / 2 : kStreamRows;
  const int steps = (a.cols + kStreamStep - 1) / kStreamStep;
  const int rounds = (steps + kMaxWaves - 1) / kMaxWaves;
  const int waves = (steps + rounds - 1) / rounds;
  const int64_t blocks = int64_t(max_tiles) * ((a.features + kCols - 1) / kCols);
  const size_t lds = std::max<size_t>(size_t(waves) * kStreamWave,
                                      size_t(waves) * 4096 + kFewRows * (kCols + 1) * 4);
  ProfScope prof_scope(DUAL ? K_MX_GATEUP : K_MX_DOWN, st);
  const auto go = [&](auto kernel) { kernel<<<unsigned(blocks), 64 * waves, lds, st>>>(a); };
  if (!whole)
    go(once ? mx_stream_kernel<DUAL, HALF, true, false>
            : mx_stream_kernel<DUAL, HALF, false, false>);
  else
    go(once ? mx_stream_kernel<DUAL, HALF, true, true>
            : mx_stream_kernel<DUAL, HALF, false, true>);
  PMOE_LAUNCH_CHECK("mx_stream_kernel");
  return PMOE_OK;
}

// ---------------------------------------------------------------- single tokens

constexpr int kOneCols = 16;   // features a block
constexpr int kOneBatch = 3;   // (column, stretch) items of the down projection in flight a wave

// Every token by itself (blockIdx.z), its experts' weights read for it alone.
struct MxOne {
  const uint8_t* slab;
  int64_t expert_bytes;
  const int32_t* table;
  int n_experts;
  const int32_t* ids;   // [n, k]
  const float* wts;     // [n, k], or null: uncombined
  int k, kk, shared_slot;
  const uint16_t* shared_gate;  // or null
  float* shared_logit;  // [n]
  int32_t* slots;       // [n, kk], found by the first launch for the second
  int64_t w0, s0, w1, s1, wd, sd;
  const uint16_t* x;    // [n, hidden]
  int hidden, inter;
  float* h;             // fp32 [n, kk, inter]
  uint16_t* out;        // bf16: [n, hidden], or [n, kk, hidden] uncombined

  // the same with the arrays of one token
  __device__ __forceinline__ MxOne of(int token) const {
    MxOne a = *this;
    a.ids += size_t(token) * k;
    if (wts) a.wts += size_t(token) * k;
    if (shared_logit) a.shared_logit += token;
    a.slots += size_t(token) * kk;
    a.x += size_t(token) * hidden;
    a.h += size_t(token) * kk * inter;
    a.out += size_t(token) * (wts ? 1 : kk) * hidden;
    return a;
  }
};

// Slot of column c, -1 where nothing is held.
__device__ __forceinline__ int one_slot(const MxOne& a, int c) {
  if (c >= a.k) return a.shared_slot;
  const int e = a.ids[c];
  return e >= 0 && e < a.n_experts ? a.table[e] : -1;
}

// 16 rows x 512 values of a projection into LDS at `to`: 16 lanes side by side on
// a row's 256 bytes, 4 rows an instruction; then the rows' scales, 4 words each,
// at to + 4096 (word i of row r at 64 i + 4 r).  In stretch j of `groups` groups,
// fetched by one wave.  WHOLE as in mx_stream_kernel: otherwise returns the lane's
// word of scales, which belongs at to + 4096 + 4 lane.
template <bool WHOLE>
__device__ __forceinline__ uint32_t one_fetch(uint32_t to, const uint8_t* w, const uint8_t* s,
                                              uint32_t row_bytes, int groups, int j, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 4 * i + (lane >> 4);
    const int p = (lane & 15) ^ swizzle16(row);
    if (16 * j + p < groups)
      dma16(to + i * 1024, uint32_t(lane >> 4) * row_bytes + p * 16,
            w + size_t(4 * i) * row_bytes + j * 256);
  }
  const int r = lane & 15, i = lane >> 4;
  if constexpr (!WHOLE)
    return scale_word(s + size_t(r) * groups + 16 * j + 4 * i, groups - 16 * j - 4 * i);
  if (16 * j + 4 * i < groups) dma4(to + 4096, uint32_t(r) * groups + 4 * i, s + 16 * j);
  return 0;
}
constexpr int kOneFetch = 4096 + 256;
// A stretch's pieces in LDS: 16 groups of 64 bytes (p0 and p1 48), their scales
// behind them.
constexpr int kOnePieces = 16 * 64 + 16;
// LDS of an item: whole 256 bytes
constexpr int kOneItem = (kOneFetch + kOnePieces + 255) / 256 * 256;

__device__ __forceinline__ void one_put(uint8_t* to, int g, u32x6 p0, u32x6 p1, uint4 p2) {
  uint4* d = reinterpret_cast<uint4*>(to + g * 64);
  d[0] = make_uint4(p0[0], p0[1], p0[2], p0[3]);
  d[1] = make_uint4(p0[4], p0[5], p1[0], p1[1]);
  d[2] = make_uint4(p1[2], p1[3], p1[4], p1[5]);
  d[3] = p2;
}

// acc += 16 rows of weights at `w` (one_fetch) times a stretch's pieces.
__device__ __forceinline__ void one_mma(f32x4& acc, const uint8_t* w, const uint8_t* pieces,
                                        int groups_in, int lane) {
  const int r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (4 * i >= groups_in) break;  // whole steps of 128
    const int p = 4 * i + q;
    const uint4 v = *reinterpret_cast<const uint4*>(w + (r * 16 + (p ^ swizzle16(r))) * 16);
    const int sw = w[4096 + 64 * i + 4 * r + q];
    const uint4* src = reinterpret_cast<const uint4*>(pieces + p * 64);
    const uint4 c0 = src[0], c1 = src[1], c2 = src[2];
    const int sa = pieces[16 * 64 + p];
    const uint32_t b0[6] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y};
    const uint32_t b1[6] = {c1.z, c1.w, c2.x, c2.y, c2.z, c2.w};
    mx_mma(acc, v, sw, b0, sa);
    mx_mma(acc, v, sw, b1, sa - kMxInterShift);
  }
}

// h[c, f] = silu(gate) * up for 32 features of one column, the weights streamed as
// in mx_stream_kernel.  Each wave splits its own stretches of x into pieces, a
// lane a group, while the slot is looked up and its first weights are on their
// way.  All 16 columns of the products hold the same row.  4096x1536, 8 columns:
// 53 MB in 13.0 us, 4.1 TB/s: the two lookups, then two rounds of loads a wave (16
// features a block were slower).
template <bool WHOLE>
__global__ __launch_bounds__(64 * kMaxWaves, 4) void mx_one_gateup_kernel(const MxOne all,
                                                                          int wave_lds) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t dyn[];
  const MxOne a = all.of(blockIdx.z);
  constexpr int NF = 4, kCols = kStreamRows / 2;
  const int c = blockIdx.y, fb = blockIdx.x;
  const int waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int r = lane & 15, q = lane >> 4;
  const int groups = a.hidden / kMxGroup;
  const int steps = (groups + kMxStepGroups - 1) / kMxStepGroups;
  uint8_t* own = dyn + wave * wave_lds;
  uint8_t* pieces = own + kStreamWave;  // [round][8 groups][64 bytes], then their scales
  const int rounds = (steps + 2 * waves - 1) / (2 * waves);
  uint8_t* pscale = pieces + rounds * 8 * 64;

  // lane 8 i + k: group k of this wave's i-th step of 256
  const int mine = 8 * (wave + (lane >> 3) * waves) + (lane & 7);
  const bool has = (lane >> 3) < rounds && mine < groups;
  uint4 xin[4];
  if (has) {
    const uint4* src = reinterpret_cast<const uint4*>(a.x + size_t(mine) * kMxGroup);
#pragma unroll
    for (int i = 0; i < 4; ++i) xin[i] = src[i];
  }
  const int slot = one_slot(a, c);
  if (fb == 0 && threadIdx.x == 0) a.slots[c] = slot;
  if (slot >= 0) {
    const uint8_t* base = a.slab + size_t(slot) * size_t(a.expert_bytes);
    const uint32_t row_bytes = a.hidden / 2;
    const uint8_t* wbase[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f)
      wbase[f] = base + (f > 1 ? a.w1 : a.w0) + size_t(fb * kCols + 16 * (f & 1)) * row_bytes;
    const int lrow = lane >> 3;
    const int lp[2] = {(lane & 7) ^ swizzle8(lrow), (lane & 7) ^ swizzle8(lrow + 8)};
    const uint32_t s_off =
        uint32_t(q > 1 ? a.s1 : a.s0) + uint32_t(fb * kCols + 16 * (q & 1) + r) * groups;
    const uint8_t* srow = base + (q > 1 ? a.s1 : a.s0) +
                          size_t(fb * kCols + 16 * (q & 1) + r) * groups;
    uint32_t sword[2];
    const uint32_t own_lds = __builtin_amdgcn_readfirstlane(
        uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)own)));
    const auto fetch = [&](int j) {
      const bool two = 2 * j + 1 < steps;
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (WHOLE ? two || lp[i] < 4 : 8 * j + lp[i] < groups)
            dma16(own_lds + f * 2048 + i * 1024, lrow * row_bytes + lp[i] * 16,
                  wbase[f] + size_t(8 * i) * row_bytes + j * 128);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if constexpr (!WHOLE)
          sword[i] = scale_word(srow + 8 * j + 4 * i, groups - 8 * j - 4 * i);
        else if (i == 0 || two)
          dma4(own_lds + NF * 2048 + i * 256, s_off + (2 * j + i) * 4, base);
    };
    if (2 * wave < steps) fetch(wave);
    if (has) {
      float v[32];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t t[4] = {xin[i].x, xin[i].y, xin[i].z, xin[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          v[8 * i + 2 * k] = bf16lo(t[k]), v[8 * i + 2 * k + 1] = bf16hi(t[k]);
      }
      int s;
      u32x6 p0, p1;
      uint4 p2;
      mx_split<true>(v, s, p0, p1, p2);
      one_put(pieces, lane, p0, p1, p2);
      pscale[lane] = uint8_t(s);
    } else if (!WHOLE && (lane >> 3) < rounds) {  // past the row's end
      one_put(pieces, lane, u32x6{}, u32x6{}, make_uint4(0, 0, 0, 0));
      pscale[lane] = 127;
    }
    f32x4 acc[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    int round = 0;
    for (int j = wave; 2 * j < steps; j += waves, ++round) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      if constexpr (!WHOLE)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<uint32_t*>(own + NF * 2048 + i * 256 + lane * 4) = sword[i];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (2 * j + i >= steps) break;
        const int at = (r * 8 + ((4 * i + q) ^ swizzle8(r))) * 16;
        const int g = round * 8 + 4 * i + q;
        const uint4* src = reinterpret_cast<const uint4*>(pieces + g * 64);
        const uint4 c0 = src[0], c1 = src[1], c2 = src[2], d = src[3];
        const int sa = pscale[g];
        const uint32_t b0[6] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y};
        const uint32_t b1[6] = {c1.z, c1.w, c2.x, c2.y, c2.z, c2.w};
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          const uint4 w = *reinterpret_cast<const uint4*>(own + f * 2048 + at);
          const int sw = own[NF * 2048 + i * 256 + (16 * f + r) * 4 + q];
          mx_mma(acc[f], w, sw, b0, sa);
          mx_mma(acc[f], w, sw, b1, sa - kMxTokenShift);
          mx_mma_third(acc[f], w, sw, d, sa);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (2 * (j + waves) < steps) fetch(j + waves);
    }
    // lanes 16 q: features 16 f + 4 q + i of the gate (f < 2) and up tiles
    float(*red)[NF * 16] = reinterpret_cast<float(*)[NF * 16]>(dyn);
    __syncthreads();
    if (r == 0)
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[wave][16 * f + 4 * q + i] = acc[f][i];
    __syncthreads();
    if (threadIdx.x < kCols) {
      float g = 0.0f, u = 0.0f;
      for (int w = 0; w < waves; ++w)
        g += red[w][threadIdx.x], u += red[w][kCols + threadIdx.x];
      a.h[size_t(c) * a.inter + fb * kCols + threadIdx.x] = silu_fast(g) * u;
    }
  }
  if (a.shared_gate && fb == 0 && c == a.kk - 1) {  // the shared expert's gate logit
    float sum = 0.0f;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x)
      sum = __builtin_fmaf(bf16f(a.x[i]), bf16f(a.shared_gate[i]), sum);
    sum = wave_sum_bfly(sum);
    float* red = reinterpret_cast<float*>(dyn);
    __syncthreads();
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      float t = 0.0f;
      for (int w = 0; w < waves; ++w) t += red[w];
      *a.shared_logit = t;
    }
  }
}

// 16 features of the down projection.  MIX: of the weighted sum over all columns,
// in fp32 (each wave adds up its own (column, stretch) items, the waves meet in
// LDS, always in the same order); otherwise of column blockIdx.y.  4096x1536, 8
// columns: 27 MB in 8.9 us, every load of a block in flight at once; what is left is
// the launch, the slots' lookup and the sum at the end.
template <bool MIX, bool WHOLE>
__global__ __launch_bounds__(64 * kMaxWaves, 2) void mx_one_down_kernel(const MxOne all,
                                                                        int batch) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t dyn[];
  const MxOne a = all.of(blockIdx.z);
  const int f0 = blockIdx.x * kOneCols;
  const int waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int groups = a.inter / kMxGroup;
  const int stretches = (groups + 15) / 16;
  const int first = MIX ? 0 : blockIdx.y, columns = MIX ? a.kk : 1;
  const int items = columns * stretches;
  const uint32_t row_bytes = a.inter / 2;
  uint8_t* own = dyn + wave * batch * kOneItem;
  const uint32_t own_lds = __builtin_amdgcn_readfirstlane(
      uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)own)));
  // lane c: column c's slot and weight, all looked up at once
  int my_slot = -1;
  float my_weight = 1.0f;
  if (lane < a.kk) {
    my_slot = a.slots[lane];
    if constexpr (MIX)
      my_weight = lane < a.k ? a.wts[lane] : a.shared_gate ? psigmoid(*a.shared_logit) : 1.0f;
  }
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int t0 = wave; t0 < items; t0 += waves * batch) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    uint32_t sword[kOneBatch] = {};
#pragma unroll
    for (int b = 0; b < kOneBatch; ++b) {
      const int t = t0 + b * waves;
      if (b >= batch || t >= items) break;
      const int c = first + t / stretches, j = t % stretches;
      const int slot = __builtin_amdgcn_readlane(my_slot, c);
      if (slot < 0) continue;
      const uint8_t* base = a.slab + size_t(slot) * size_t(a.expert_bytes);
      sword[b] = one_fetch<WHOLE>(own_lds + b * kOneItem, base + a.wd + size_t(f0) * row_bytes,
                                  base + a.sd + size_t(f0) * groups, row_bytes, groups, j, lane);
    }
    {  // 16 lanes an item: a group of its column's h each
      const int b = lane >> 4, t = min(t0 + b * waves, items - 1);
      const int c = first + t / stretches, gi = 16 * (t % stretches) + (lane & 15);
      const int held = __shfl(my_slot, c, 64);  // of every lane: any may be asked
      if (b < batch && t0 + b * waves < items) {
        if (gi < groups && held >= 0) {
          const float4* src = reinterpret_cast<const float4*>(a.h + size_t(c) * a.inter + gi * kMxGroup);
          float v[32];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 x = src[i];
            v[4 * i] = x.x, v[4 * i + 1] = x.y, v[4 * i + 2] = x.z, v[4 * i + 3] = x.w;
          }
          int s;
          u32x6 p0, p1;
          uint4 none;
          mx_split<false>(v, s, p0, p1, none);
          uint8_t* to = own + b * kOneItem + kOneFetch;
          one_put(to, lane & 15, p0, p1, none);
          to[16 * 64 + (lane & 15)] = uint8_t(s);
        } else if (!WHOLE && held >= 0) {  // past the row's end
          uint8_t* to = own + b * kOneItem + kOneFetch;
          one_put(to, lane & 15, u32x6{}, u32x6{}, make_uint4(0, 0, 0, 0));
          to[16 * 64 + (lane & 15)] = 127;
        }
      }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    if constexpr (!WHOLE)
#pragma unroll
      for (int b = 0; b < kOneBatch; ++b)
        if (b < batch) *reinterpret_cast<uint32_t*>(own + b * kOneItem + 4096 + lane * 4) = sword[b];
    for (int b = 0; b < batch; ++b) {
      const int t = t0 + b * waves;
      if (t >= items) break;
      const int c = first + t / stretches, j = t % stretches;
      if (__builtin_amdgcn_readlane(my_slot, c) < 0) continue;
      f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
      one_mma(acc, own + b * kOneItem, own + b * kOneItem + kOneFetch, min(16, groups - 16 * j),
                     lane);
      const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(my_weight), c));
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = MIX ? __builtin_fmaf(w, acc[i], sum[i]) : sum[i] + acc[i];
    }
  }
  float(*red)[16] = reinterpret_cast<float(*)[16]>(dyn);
  __syncthreads();
  if ((lane & 15) == 0)
#pragma unroll
    for (int i = 0; i < 4; ++i) red[wave][(lane >> 4) * 4 + i] = sum[i];
  __syncthreads();
  if (threadIdx.x < kOneCols) {
    float v = 0.0f;
    for (int w = 0; w < waves; ++w) v += red[w][threadIdx.x];
    a.out[size_t(MIX ? 0 : blockIdx.y) * a.hidden + f0 + threadIdx.x] = f2bf(v);
  }
}

// ---------------------------------------------------------------- large tiles

constexpr int kTileRows = 128;    // activation rows a block
constexpr int kTileCols = 512;    // weight rows a block (DUAL: 256 gate, 256 up)
constexpr int kTileWaves = 8;     // 2 halves of the rows x 4 quarters of the weights
constexpr int kActBytes = 8 * 3 * 1024;             // 8 row tiles x 3 chunks a lane
constexpr int kWeightBytes = kTileCols / 16 * 1024;  // 32 row tiles x 1 chunk a lane
constexpr int kThirdBytes = 8 * 1024;                // 8 row tiles x 1 chunk a lane
constexpr int kStageBytes = kActBytes + kWeightBytes + kThirdBytes;
// 16 scale bytes a row, of four steps
constexpr int kActScaleBytes = kTileRows * kMxScaleBlock;
constexpr int kScaleBytes = kActScaleBytes + kTileCols * kMxScaleBlock;
constexpr int kTileLds = 2 * (kStageBytes + kScaleBytes);

// The steps of a tile's reduction: s done of n.
struct Steps {
  int s, n;
  // whether the step's scales are not in the block of the step before
  __device__ __forceinline__ bool fresh() const { return s % kMxScaleSteps == 0; }
  __device__ __forceinline__ bool done() const { return s >= n; }
};

// One tile of at most 128 rows of an expert times 512 weight rows (DUAL: 256
// gate and the same 256 up features).  Each wave holds 64 rows times 128 weight
// rows in its accumulators.  A step of 128 goes from memory straight into LDS,
// 16 rows of 64 bytes an instruction: four lanes side by side fetch one 64-byte
// stretch (lanes in the products' own order, 16 rows side by side, cost the
// cache four times the accesses and bound the kernel), in an order that keeps the
// reads back free of bank conflicts (swizzle4).  The next step's loads are in
// flight while this one's products run.
// 4096x1536, 16384 tokens x 8 columns: gate/up 2.1 to 2.2 ms, down 1.2 (1.5 and 1.35
// PFLOP/s of the layer's products, twice that and the third pieces on the matrix
// units).  Gate/up without its loads takes 1.74 ms, near the 1.63 of its matrix
// instructions alone, and the loads without the products 1.64: what is left is
// where one waits for the other.  The down projection's 12 steps leave a third of
// its time to the first loads and the stores.
// Scales come 16 bytes a row, those of four steps.  The weights' do so where the
// reduction is whole stretches of 512 (kBlocks), so that they lie on 16 bytes;
// where it is whole steps of 128 they are fetched 4 bytes a row for each step
// (kWords; those fetches alone took a sixth of the kernel's time where every step
// did so); otherwise a step's words go through registers, a step ahead, and the
// last step's groups past the row's end count as zeros (kRegs).
enum TileScales { kBlocks, kWords, kRegs };
template <bool DUAL, TileScales SC, bool HALF>
__global__ __launch_bounds__(64 * kTileWaves, 2) void mx_tile_kernel(const MxArgs a) {
  constexpr bool BLOCKS = SC == kBlocks;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kTileLds];
  __shared__ unsigned long long s_third;
  __shared__ int32_t s_order[DUAL ? 1 : kTileRows];  // flat rows, for the stores
  constexpr int kCols = DUAL ? kTileCols / 2 : kTileCols;  // features a block
  const int fblocks = (a.features + kCols - 1) / kCols;
  // XCD x takes a contiguous range of the work, a tile's feature blocks side by
  // side: they share its rows, and an expert's tiles its weights, in one L2
  const int work = *a.n_tiles * fblocks;
  const int per = (work + 7) / 8;
  const int at = int(blockIdx.x & 7) * per + int(blockIdx.x >> 3);
  if (int(blockIdx.x >> 3) >= per || at >= work) return;
  const int t = at / fblocks;
  const int fb = at - t * fblocks;
  const int4 tile = a.tiles[t];  // {slot, first row, rows of the expert, offset}
  const int m = min(kTileRows, tile.z - tile.y);
  const int p0 = tile.w + tile.y;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (tile.x < 0) {  // not resident: exact zero rows
    if constexpr (!DUAL) {
      const int cols = min(kCols, a.features - fb * kCols);
      for (int row = wave; row < m; row += kTileWaves) {
        const size_t flat = a.order[p0 + row];
        for (int c = lane; c < cols; c += 64) a.y[flat * a.features + fb * kCols + c] = 0;
        if (HALF && lane < cols / kMxGroup)
          a.yscale[(flat * a.features + fb * kCols) / kMxGroup + lane] = 1;
      }
    }
    return;
  }
  const int r = lane & 15, q = lane >> 4;
  const int groups = a.cols / kMxGroup;
  const uint8_t* base = a.slab + size_t(tile.x) * size_t(a.expert_bytes);

  // What this wave loads each step: row tile `wave` of the activations and
  // weight tiles 4 wave .. + 3, now and then their scales.  Offsets from the
  // wave's own bases; a tile's intermediate rows follow each other, tokens lie
  // anywhere in less than 4 GiB (mx_tile_rows).
  const int lr = lane >> 2, lq = (lane & 3) ^ swizzle4(lr);
  const int steps = (groups + kMxStepGroups - 1) / kMxStepGroups;
  const auto act_row = [&](int row) {
    const int k = row < m ? row : 0;
    return uint32_t(DUAL ? a.order[p0 + k] / a.kk : k);
  };
  const size_t arow0 = DUAL ? 0 : size_t(p0);
  const uint8_t* apair = a.pair + arow0 * steps * kMxStepPair;
  const uint8_t* ascale = a.ascale + arow0 * mx_scale_row(a.cols);
  const uint32_t arow = act_row(16 * wave + lr) * uint32_t(steps);
  const uint32_t pair_off = arow * kMxStepPair + lq * 16;
  const uint32_t third_off = arow * kMxStepThird + lq * 16;
  const uint32_t ascale_off = act_row(16 * wave + r) * uint32_t(mx_scale_row(a.cols));
  // the block's weight tile i: its gate (0..15) or up features; tiles past the
  // projection load its last one and are not used
  const auto tile_row = [&](int i) {
    return min(fb * kCols + (DUAL ? 16 * i & (kCols - 1) : 16 * i), a.features - 16);
  };
  const bool second = DUAL && wave >= kTileWaves / 2;
  const uint8_t* wbase = base + (second ? a.w1 : a.w0);
  const uint8_t* wscale = base + (second ? a.s1 : a.s0);
  const uint32_t w_off = uint32_t(lr) * uint32_t(a.cols / 2) + lq * 16;
  const uint32_t wscale_off = uint32_t(tile_row(4 * wave + q) + r) * uint32_t(groups);

  if constexpr (!DUAL) {  // (the loop's barriers come before the reads)
    if (int(threadIdx.x) < m) s_order[threadIdx.x] = a.order[p0 + threadIdx.x];
  }

  Steps todo{0, steps};
  uint64_t thirds = 0;  // bit s: a row of the tile has a third piece in step s
  if constexpr (DUAL) {
    if (threadIdx.x == 0) s_third = 0;
    __syncthreads();
    uint64_t mask = 0;
    if (int(threadIdx.x) < m)
      mask = reinterpret_cast<const uint64_t*>(a.asteps)[a.order[p0 + threadIdx.x] / a.kk];
    if (mask) atomicOr(&s_third, static_cast<unsigned long long>(mask));
    __syncthreads();
    const uint64_t v = s_third;
    const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(v));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(uint32_t(v >> 32));
    thirds = uint64_t(lo) | uint64_t(hi) << 32;
  }
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(
      uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds)));
  // scales: LDS buffer of the block that a step is in
  const auto scale_lds = [&](int block) { return 2 * kStageBytes + (block & 1) * kScaleBytes; };
  uint32_t sword = 0;  // kRegs: scales of row 64 wave + lane in the step that is loading
  const uint8_t* wscale_row = wscale + wscale_off;
  // A step's loads in four parts, so that they can be spread over the products of
  // the step before.
  const auto issue = [&](const Steps& st, int buf, int block, int part) {
    const int s = st.s;
    const uint32_t to = lds0 + buf * kStageBytes;
    if (part == 0) {
      const uint32_t act = to + wave * 3 * 1024;
      const uint8_t* p = apair + s * kMxStepPair;
      dma16(act, pair_off, p);
      dma16(act + 1024, pair_off, p + kMxChunk);
      dma16(act + 2048, pair_off, p + 2 * kMxChunk);
    } else if (part < 3) {
#pragma unroll
      for (int i = 2 * part - 2; i < 2 * part; ++i)
        if (SC != kRegs || 4 * s + lq < groups)
          dma16(to + kActBytes + (wave * 4 + i) * 1024, w_off,
                wbase + size_t(tile_row(4 * wave + i)) * (a.cols / 2) + s * 64);
    } else {
      if (DUAL && (thirds >> s & 1))
        dma16(to + kActBytes + kWeightBytes + wave * 1024, third_off, a.third + s * kMxStepThird);
      const uint32_t sc = lds0 + scale_lds(block);
      const int at16 = s / kMxScaleSteps * kMxScaleBlock;
      if (st.fresh()) {
        if (lane < 16) dma16(sc + wave * 16 * kMxScaleBlock, ascale_off, ascale + at16);
        if constexpr (BLOCKS)
          dma16(sc + kActScaleBytes + wave * 64 * kMxScaleBlock, wscale_off, wscale + at16);
      }
      if constexpr (SC == kRegs) sword = scale_word(wscale_row + 4 * s, groups - 4 * s);
      if constexpr (SC == kWords)  // step i of a block: rows' words side by side
        dma4(sc + kActScaleBytes + (s % kMxScaleSteps) * (kTileCols * 4) + wave * 256, wscale_off,
             wscale + s * 4);
    }
  };

  // Which part goes out with row tile i.  The down projection's activations follow
  // each other and come sooner than its weights, which go first (16384 tokens 1218 ->
  // 1180 us; gate/up gathers its activations, and loses 3% of 2048 tokens by it).
  const auto turn = [](int i) { return DUAL ? i : i ^ 2; };

  const int rh = wave & 1, wq = wave >> 1;  // this wave's half of the rows, quarter of the weights
  f32x4 acc[8][4];
#pragma unroll
  for (int f = 0; f < 8; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[f][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // its weight tiles: DUAL 4 gate and the same 4 up ones
  const auto weight_tile = [&](int f) {
    return DUAL ? (f < 4 ? 4 * wq + f : 16 + 4 * wq + f - 4) : 8 * wq + f;
  };
  const int tiles_in = min(4, max(0, (m - 64 * rh + 15) / 16));  // row tiles that hold rows

  const int slot = (r * 4 + (q ^ swizzle4(r))) * 16;  // where chunk q of a tile's row r lies

  // The loop over the steps, for the row tiles of this wave that hold rows: known
  // when compiled, so that no branch keeps the reads of one row tile from running
  // under the products of another (branches cost a fifth).  Every wave passes
  // the same barriers, whichever form its own half of the rows takes.
  const auto run = [&](auto row_tiles) {
  constexpr int NT = decltype(row_tiles)::value;
#pragma unroll
  for (int part = 0; part < 4; ++part) issue(todo, 0, 0, part);
  Steps ahead = todo;
  ++ahead.s;
  int block = 0, block_ahead = 0;
  uint32_t sw4[8], sa4[4];  // the lane's scales of a block's steps, this one's lowest
  for (int buf = 0; !todo.done(); buf ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (SC == kRegs)  // (where kWords' fetches put them)
      *reinterpret_cast<uint32_t*>(lds + scale_lds(block) + kActScaleBytes +
                                   (todo.s % kMxScaleSteps) * (kTileCols * 4) + wave * 256 +
                                   lane * 4) = sword;
    __syncthreads();  // this step is in LDS, and the other buffer has been read
    const bool more = !ahead.done();
    if (more) block_ahead += ahead.fresh() ? 1 : 0;
    if constexpr (NT > 0) {
    const uint8_t* from = lds + buf * kStageBytes;
    const int si = todo.s % kMxScaleSteps;
    const uint8_t* ss = lds + scale_lds(block);
    if (!todo.fresh()) {
#pragma unroll
      for (int i = 0; i < NT; ++i) sa4[i] >>= 8;
      if constexpr (BLOCKS)
#pragma unroll
        for (int f = 0; f < 8; ++f) sw4[f] >>= 8;
    } else {
#pragma unroll
      for (int i = 0; i < NT; ++i)
        sa4[i] = *reinterpret_cast<const uint32_t*>(ss + (64 * rh + 16 * i + r) * kMxScaleBlock +
                                                    4 * q);
      if constexpr (BLOCKS) {
        // bytes q, 4 + q, 8 + q and 12 + q of the row's 16
        const uint32_t pick = uint32_t(q) | uint32_t(4 + q) << 8;
#pragma unroll
        for (int f = 0; f < 8; ++f) {
          const uint4 v = *reinterpret_cast<const uint4*>(
              ss + kActScaleBytes + (16 * weight_tile(f) + r) * kMxScaleBlock);
          sw4[f] = __builtin_amdgcn_perm(v.y, v.x, pick) & 0xffffu |
                   __builtin_amdgcn_perm(v.w, v.z, pick) << 16;
        }
      }
    }
    uint4 w[8];
#pragma unroll
    for (int f = 0; f < 8; ++f) {
      const int wt = weight_tile(f);
      w[f] = *reinterpret_cast<const uint4*>(from + kActBytes + wt * 1024 + slot);
      if constexpr (!BLOCKS)
        sw4[f] = ss[kActScaleBytes + si * (kTileCols * 4) + (16 * wt + r) * 4 + q];
    }
    uint4 c[2][3];
    const auto read = [&](int i) {
      const uint8_t* src = from + (4 * rh + i) * 3 * 1024 + slot;
#pragma unroll
      for (int j = 0; j < 3; ++j) c[i & 1][j] = *reinterpret_cast<const uint4*>(src + j * 1024);
    };
    read(0);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      // the next row tile's reads and a part of the next step's loads go out
      // before this row tile's products
      if (i + 1 < NT) read(i + 1);
      __builtin_amdgcn_sched_barrier(0);
      if (more) issue(ahead, buf ^ 1, block_ahead, turn(i));
      const uint4(&d)[3] = c[i & 1];
      const int sa = int(sa4[i]);
      const uint32_t b0[6] = {d[0].x, d[0].y, d[0].z, d[0].w, d[1].x, d[1].y};
      const uint32_t b1[6] = {d[1].z, d[1].w, d[2].x, d[2].y, d[2].z, d[2].w};
#pragma unroll
      for (int f = 0; f < 8; ++f) mx_mma(acc[f][i], w[f], int(sw4[f]), b0, sa);
#pragma unroll
      for (int f = 0; f < 8; ++f)
        mx_mma(acc[f][i], w[f], int(sw4[f]), b1, sa - (DUAL ? kMxTokenShift : kMxInterShift));
      __builtin_amdgcn_sched_barrier(0);
    }
    if (DUAL && (thirds >> todo.s & 1)) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint4 d = *reinterpret_cast<const uint4*>(from + kActBytes + kWeightBytes +
                                                        (4 * rh + i) * 1024 + slot);
#pragma unroll
        for (int f = 0; f < 8; ++f) mx_mma_third(acc[f][i], w[f], int(sw4[f]), d, int(sa4[i]));
      }
    }
    }
    if (more) {
#pragma unroll
      for (int i = NT; i < 4; ++i) issue(ahead, buf ^ 1, block_ahead, turn(i));
      ++ahead.s;
    }
    ++todo.s;
    block += todo.fresh() ? 1 : 0;
  }
  };
  switch (tiles_in) {
    case 0: run(std::integral_constant<int, 0>{}); break;
    case 1: run(std::integral_constant<int, 1>{}); break;
    case 2: run(std::integral_constant<int, 2>{}); break;
    case 3: run(std::integral_constant<int, 3>{}); break;
    default: run(std::integral_constant<int, 4>{}); break;
  }

  if constexpr (DUAL) {
    // h of 32 rows x 64 features at a time through LDS, then a lane a group
    constexpr int kPitch = 68;
    float* hs = reinterpret_cast<float*>(lds) + wave * 32 * kPitch;
    static_assert(kTileWaves * 32 * kPitch * 4 <= kTileLds, "h staging");
    const int f0 = fb * kCols + 64 * wq;
    __syncthreads();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          const f32x4 g = acc[f][2 * half + i], u = acc[f + 4][2 * half + i];
          *reinterpret_cast<float4*>(hs + (16 * i + r) * kPitch + 16 * f + 4 * q) =
              make_float4(silu_fast(g[0]) * u[0], silu_fast(g[1]) * u[1], silu_fast(g[2]) * u[2],
                          silu_fast(g[3]) * u[3]);
        }
      __syncthreads();
      const int row = 64 * rh + 32 * half + (lane >> 1);
      const int f = f0 + 32 * (lane & 1);
      if (row < m && f < a.features) {
        float v[32];
        const float* src = hs + (lane >> 1) * kPitch + 32 * (lane & 1);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float4 x = *reinterpret_cast<const float4*>(src + 4 * c);
          v[4 * c] = x.x, v[4 * c + 1] = x.y, v[4 * c + 2] = x.z, v[4 * c + 3] = x.w;
        }
        int s;
        u32x6 h0, h1;
        uint4 none;
        mx_split<false>(v, s, h0, h1, none);
        const size_t to = size_t(p0 + row) * mx_steps(a.features);
        mx_store_pair(a.hpair + to * kMxStepPair, f / kMxGroup, h0, h1);
        uint8_t* hs_row = a.hscale + size_t(p0 + row) * mx_scale_row(a.features);
        hs_row[mx_scale_at(f / kMxGroup)] = uint8_t(s);
        if (SC == kRegs && f + kMxGroup == a.features)  // zeros to the end of the step
          for (int g = a.features / kMxGroup; g % kMxStepGroups; ++g) {
            mx_store_pair(a.hpair + to * kMxStepPair, g, u32x6{}, u32x6{});
            hs_row[mx_scale_at(g)] = 127;
          }
      }
      __syncthreads();
    }
  } else {
    // 16 rows x 128 features at a time through the wave's own LDS, so that 16
    // lanes store one row's 256 bytes (8-byte stores from the accumulators took a
    // third of the kernel's time)
    constexpr int kPitch = 272;
    uint8_t* ys = lds + wave * 16 * kPitch;
    const int f0 = fb * kCols + 128 * wq;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row0 = 64 * rh + 16 * i;
      if (row0 >= m || f0 >= a.features) break;
      const size_t own = row0 + r < m ? s_order[row0 + r] : 0;
      uint16_t o[32];
      if constexpr (HALF) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {  // 32 features: two tiles over the row's four lanes
          uint32_t top = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            top = max(top, __float_as_uint(acc[2 * g + j / 4][i][j & 3]) & 0x7fffffffu);
          top = max(top, uint32_t(__float_as_int(xor_lane<16>(__int_as_float(int(top))))));
          top = max(top, uint32_t(__float_as_int(xor_lane<32>(__int_as_float(int(top))))));
          const int sc = half_scale(top);
#pragma unroll
          for (int j = 0; j < 8; ++j) o[8 * g + j] = half_of(acc[2 * g + j / 4][i][j & 3], sc);
          if (q == g && row0 + r < m && f0 + 32 * g < a.features)
            a.yscale[(own * a.features + f0) / kMxGroup + g] = uint8_t(sc);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = f2bf(acc[j / 4][i][j & 3]);
      }
#pragma unroll
      for (int f = 0; f < 8; ++f)
        *reinterpret_cast<uint2*>(ys + r * kPitch + (16 * f + 4 * q) * 2) =
            make_uint2(uint32_t(o[4 * f]) | uint32_t(o[4 * f + 1]) << 16,
                       uint32_t(o[4 * f + 2]) | uint32_t(o[4 * f + 3]) << 16);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = 4 * j + (lane >> 4), c = f0 + 8 * (lane & 15);
        const u32x4 v = *reinterpret_cast<const u32x4*>(ys + row * kPitch + (lane & 15) * 16);
        if (row0 + row < m && c < a.features) {
          u32x4* to = reinterpret_cast<u32x4*>(a.y + size_t(s_order[row0 + row]) * a.features + c);
          if (a.past_caches)
            __builtin_nontemporal_store(v, to);
          else
            *to = v;
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }
}

template <bool DUAL, bool HALF>
int launch_tile(const MxArgs& a, int max_tiles, bool whole, hipStream_t st) {
  constexpr int kCols = DUAL ? kTileCols / 2 : kTileCols;
  const int64_t blocks = (int64_t(max_tiles) * ((a.features + kCols - 1) / kCols) + 7) / 8 * 8;
  ProfScope prof_scope(DUAL ? K_MX_GATEUP : K_MX_DOWN, st);
  const int64_t scales = DUAL ? a.s0 | a.s1 : a.s0;
  const auto go = [&](auto kernel) {
    kernel<<<unsigned(blocks), 64 * kTileWaves, 0, st>>>(a);
  };
  if (!whole)
    go(mx_tile_kernel<DUAL, kRegs, HALF>);
  else if (a.cols % kStretch == 0 && (scales | a.expert_bytes) % 16 == 0)
    go(mx_tile_kernel<DUAL, kBlocks, HALF>);
  else
    go(mx_tile_kernel<DUAL, kWords, HALF>);
  PMOE_LAUNCH_CHECK("mx_tile_kernel");
  return PMOE_OK;
}

}  // namespace

namespace {

// Reductions of whole steps of 128, scales that a lane can fetch four at a time,
// components within 32-bit offsets of their slot: where scales need no way through
// registers.
bool mx_aligned(const pmoe_geom* g) {
  if (g->hidden % 128 || g->inter % 128) return false;
  const int comps[] = {PMOE_GATE_S, PMOE_UP_S, PMOE_DOWN_S};
  for (int c : comps)
    if (g->off[c] % 4 || g->off[c] < 0 ||
        g->off[c] + int64_t(g->hidden) * g->inter / kMxGroup >= int64_t(1) << 31)
      return false;
  return true;
}

// PMOE_MX_TILE=0 / 1 pins tiles of 16 / 128 rows (read per call).
int mx_pinned_rows() {
  const char* v = getenv("PMOE_MX_TILE");
  return !v ? 0 : v[0] == '0' ? kFewRows : v[0] == '1' ? kTileRows : 0;
}

}  // namespace

// Rows of a tile: 16 (streamed tiles, which read an expert's weights again for
// every 16 rows) or 128.  The large tiles pay from 12 rows an expert where their
// blocks, one a CU at a time, fill the GPU one and a half times, and from
// proportionally more where they do not.  us, gate/up + down, 16 / 128 rows a tile:
//   4096x1536, 128 experts  9 rows an expert 301 / 319, 13: 343 / 322, 25: 523 / 344
//   2048x512, 512 experts   9: 225 / 258, 13: 259 / 266, 17: 306 / 272
//   7168x2048, 385 experts  7: 1960 / 1993, 12: 2324 / 2135
//   2048x768, 128 experts   9: 94 / 106, 13: 105 / 107, 19: 134 / 114
//   1024x512, 32 experts    50: 37 / 46, 75: 47 / 48, 100: 55 / 50
//   4096x1536, 8 experts    50: 74 / 97, 100: 121 / 103
// Reductions that are no whole steps of 128 have dearer large tiles (their scales
// go through registers) and pay from 18:
//   4128x1568, 128 experts  14: 535 / 644, 20: 604 / 657, 62: 1372 / 720
//   2880x2880, 32 experts   12: 162 / 194, 19: 197 / 197
//   1056x480, 32 experts    50: 43 / 44, 100: 68 / 47
int mx_tile_rows(const pmoe_geom* g, int n, int kk, int n_experts) {
  // the tokens' pieces within the large tiles' 32-bit offsets
  if (int64_t(n) * mx_steps(g->hidden) * kMxStepPair >= int64_t(1) << 32) return kFewRows;
  if (const int pinned = mx_pinned_rows()) return pinned;
  const int64_t rows = int64_t(n) * kk;
  const int64_t blocks =
      (n_experts + rows / kTileRows) * ((g->inter + kTileCols / 2 - 1) / (kTileCols / 2));
  constexpr int64_t kFull = 384;
  const int64_t least = (mx_aligned(g) ? 12 : 18) * kFull * n_experts;
  return rows * std::min(blocks, kFull) >= least ? kTileRows : kFewRows;
}
int mx_min_tile_rows() { return kFewRows; }

int mx_experts(const MxPlan& p, hipStream_t st) {
  const pmoe_geom* g = p.geom;
  const bool shared = p.kk > p.k;
  const int n_ids = p.n_experts + (shared ? 1 : 0), rows = p.n * p.kk;
  const bool large = p.tile_rows == kTileRows;
  const bool whole = mx_aligned(g);
  PMOE_REQUIRE(n_ids <= kMaxExperts, "dispatch: experts must be 1..1024");
  {  // a launch holds less than 2^32 threads: the split's, the combine's, the products'
    const int up_cols = (large ? kTileCols : kStreamRows) / 2;
    const int down_cols = large ? kTileCols : kStreamRows;
    const int64_t blocks = std::max((g->inter + up_cols - 1) / up_cols,
                                    (g->hidden + down_cols - 1) / down_cols);
    const int64_t row_blocks = (g->hidden + 2047) / 2048;
    PMOE_REQUIRE(p.n * row_blocks < int64_t(1) << 24 &&
                     p.max_tiles * blocks <= (int64_t(1) << 23) - 8,
                 "experts: too many rows for one call");
  }
  MxSplit sp{};
  sp.x = p.x;
  sp.n = p.n, sp.groups = g->hidden / kMxGroup, sp.steps = mx_steps(g->hidden);
  sp.scale_row = mx_scale_row(g->hidden);
  sp.pair = p.xpair, sp.third = p.xthird, sp.scales = p.xscale, sp.masks = p.xsteps;
  sp.shared_gate = p.shared_gate, sp.shared_logit = p.shared_logit;
  sp.ids = p.ids, sp.k = p.k, sp.n_experts = p.n_experts;
  sp.y = p.yscale ? nullptr : p.y;
  MxDispatch d{};
  d.src = IdSrc{p.ids, p.k, p.kk, p.n_experts};
  d.rows = rows, d.n_ids = n_ids;
  d.order = p.order, d.counts = p.counts, d.offsets = p.offsets, d.inv = p.inv;
  d.active = p.active, d.n_active = p.n_active;
  d.tiles = TileSink{p.tiles, p.n_tiles, p.tile_rows, p.table, p.n_experts, p.shared_slot};
  const int split_blocks = (p.n + 3) / 4;
  if (rows <= kSmallRows) {
    ProfScope prof_scope(K_MX_SPLIT, st);
    mx_prepare_kernel<<<1 + split_blocks, 1024, 0, st>>>(sp, d);
    PMOE_LAUNCH_CHECK("mx_prepare_kernel");
  } else {
    PMOE_REQUIRE(p.dws != nullptr && p.dws_bytes >= dispatch_workspace(rows, n_ids),
                 "dispatch: workspace too small");
    d.hist = static_cast<int32_t*>(p.dws);
    int32_t* rank = d.hist + size_t((rows + kDispatchChunk - 1) / kDispatchChunk) * n_ids;
    {
      ProfScope prof_scope(K_DISPATCH, st);
      if (int rc = dispatch_count(d.src, rows, n_ids, d.hist, rank, st)) return rc;
    }
    {
      ProfScope prof_scope(K_MX_SPLIT, st);
      mx_scan_split_kernel<<<1 + split_blocks, 1024, 0, st>>>(sp, d);
      PMOE_LAUNCH_CHECK("mx_scan_split_kernel");
    }
    ProfScope prof_scope(K_DISPATCH, st);
    if (int rc = dispatch_scatter(d.src, rows, n_ids, d.hist, rank, p.order, p.inv, st)) return rc;
  }
  const bool once = rows <= int64_t(kFewRows) * p.n_experts;
  MxArgs a{};
  a.slab = p.slab;
  a.expert_bytes = g->expert_bytes;
  a.tiles = p.tiles;
  a.n_tiles = p.n_tiles;
  a.order = p.order;
  a.kk = p.kk;
  a.w0 = g->off[PMOE_GATE_W], a.s0 = g->off[PMOE_GATE_S];
  a.w1 = g->off[PMOE_UP_W], a.s1 = g->off[PMOE_UP_S];
  a.features = g->inter;
  a.cols = g->hidden;
  a.pair = p.xpair, a.third = p.xthird, a.ascale = p.xscale, a.asteps = p.xsteps;
  a.hpair = p.hpair, a.hscale = p.hscale;
  if (int rc = large ? launch_tile<true, false>(a, p.max_tiles, whole, st)
                     : launch_stream<true, false>(a, p.max_tiles, once, whole, st))
    return rc;
  a.w0 = g->off[PMOE_DOWN_W], a.s0 = g->off[PMOE_DOWN_S];
  a.features = g->hidden;
  a.cols = g->inter;
  a.pair = p.hpair, a.third = nullptr, a.ascale = p.hscale, a.asteps = nullptr;
  a.y = p.y;
  a.yscale = p.yscale;
  a.past_caches = past_caches(int64_t(rows) * g->hidden);
  if (p.yscale)
    return large ? launch_tile<false, true>(a, p.max_tiles, whole, st)
                 : launch_stream<false, true>(a, p.max_tiles, once, whole, st);
  return large ? launch_tile<false, false>(a, p.max_tiles, whole, st)
               : launch_stream<false, false>(a, p.max_tiles, once, whole, st);
}

// How many of n tokens may go one by one (0: none), in two launches instead of a
// dispatch, the tiles' two and a combine.  What that saves, some 7 us and the combine,
// pays for the weights that several of the tokens read (by expectation over
// independent ids, and the shared expert's), and for a stream that is a tenth slower
// than the tiles'.  us, tiles / one by one:
//   1024x512 32 experts, 4 columns    8 tokens 19.0 / 11.8, 16: 20.2 / 14.4, 32: 22.1 / 22.4
//   2048x512 512 experts, 10 + shared 2: 23.9 / 15.7, 4: 31.2 / 21.1, 8: 43.8 / 41.1
//     seam, 10                        2: 19.3 / 14.2, 8: 36.6 / 35.7, 12: 46.6 / 49.0
//   4096x1536 128 experts, 8          2: 43.8 / 39.2, 3: 56.5 / 56.6, 4: 66.6 / 70.6
//     seam                            2: 40.2 / 38.5, 3: 53.3 / 53.8
//   7168x2048 384 experts, 8 + shared 2: 91.7 / 94.0; seam, 8: 79.1 / 80.2
// Up to 64 columns: a lane looks one up.
int mx_one_tokens(const pmoe_geom* g, int n, int k, int shared, int n_experts, bool combined) {
  if (k + shared > 64) return 0;
  if (n <= 1) return n;
  const double bytes = double(g->hidden) * g->inter / kMxGroup * 17 * 3;
  const double most = double((combined ? 36 : 24) << 20) / bytes;  // in experts
  const double absent = pow(1.0 - 1.0 / n_experts, k);  // an expert of one token's
  double none = absent;
  int t = 1;
  for (; t < n && t < 64; ++t) {  // would t + 1 do?
    none *= absent;
    const double repeated =
        double(t + 1) * k - n_experts * (1.0 - none) + double(shared) * t;
    if (repeated + 0.1 * (t + 1) * (k + shared) > most) break;
  }
  return t;
}

bool mx_one_wanted(const pmoe_geom* g, int n, int k, int shared, int n_experts, bool combined) {
  if (n > 1 && mx_pinned_rows()) return false;
  return n <= mx_one_tokens(g, n, k, shared, n_experts, combined);
}

int mx_one(const pmoe_geom* g, const uint8_t* slab, const int32_t* table, int n_experts,
           const uint16_t* x, const int32_t* ids, const float* wts, int n, int k, int shared_slot,
           const uint16_t* shared_gate, float* shared_logit, int32_t* slots, float* h,
           uint16_t* out, hipStream_t st) {
  MxOne a{};
  a.slab = slab;
  a.expert_bytes = g->expert_bytes;
  a.table = table;
  a.n_experts = n_experts;
  a.ids = ids, a.wts = wts;
  a.k = k, a.kk = k + (shared_slot >= 0 ? 1 : 0);
  a.shared_slot = shared_slot;
  a.shared_gate = shared_slot >= 0 ? shared_gate : nullptr;
  a.shared_logit = shared_logit;
  a.slots = slots;
  a.w0 = g->off[PMOE_GATE_W], a.s0 = g->off[PMOE_GATE_S];
  a.w1 = g->off[PMOE_UP_W], a.s1 = g->off[PMOE_UP_S];
  a.wd = g->off[PMOE_DOWN_W], a.sd = g->off[PMOE_DOWN_S];
  a.x = x;
  a.hidden = g->hidden, a.inter = g->inter;
  a.h = h, a.out = out;
  const bool whole = mx_aligned(g);
  const auto waves_for = [](int items) {
    const int rounds = (items + kMaxWaves - 1) / kMaxWaves;
    return (items + rounds - 1) / rounds;
  };
  {
    const int steps = (a.hidden + kStreamStep - 1) / kStreamStep;
    const int waves = waves_for(steps);
    const int rounds = (steps + waves - 1) / waves;  // 8192 / 256 / 8 at most: a lane a group
    const int wave_lds = (kStreamWave + rounds * 8 * (64 + 1) + 255) / 256 * 256;
    ProfScope prof_scope(K_MX_GATEUP, st);
    const auto go = [&](auto kernel) {
      kernel<<<dim3(a.inter / (kStreamRows / 2), a.kk, n), 64 * waves, waves * wave_lds, st>>>(
          a, wave_lds);
    };
    go(whole ? mx_one_gateup_kernel<true> : mx_one_gateup_kernel<false>);
    PMOE_LAUNCH_CHECK("mx_one_gateup_kernel");
  }
  const int stretches = (a.inter + kStretch - 1) / kStretch;
  const int items = wts ? a.kk * stretches : stretches;
  const int waves = waves_for(items);
  const int batch = std::min((items + waves - 1) / waves, kOneBatch);
  const size_t lds = size_t(waves) * batch * kOneItem;
  ProfScope prof_scope(K_MX_DOWN, st);
  const auto go = [&](auto kernel) {
    kernel<<<dim3(a.hidden / kOneCols, wts ? 1 : a.kk, n), 64 * waves, lds, st>>>(a, batch);
  };
  if (wts)
    go(whole ? mx_one_down_kernel<true, true> : mx_one_down_kernel<true, false>);
  else
    go(whole ? mx_one_down_kernel<false, true> : mx_one_down_kernel<false, false>);
  PMOE_LAUNCH_CHECK("mx_one_down_kernel");
  return PMOE_OK;
}

int mx_combine(const uint16_t* y, const uint8_t* yscale, const float* w, const int32_t* inv,
               const float* shared_logit, int n, int k, int kk, int d, uint16_t* out,
               hipStream_t st) {
  const int blocks_row = (d / 8 + 255) / 256;
  ProfScope prof_scope(K_COMBINE, st);
  const auto go = [&](auto kernel) {
    kernel<<<unsigned(n) * blocks_row, 256, 0, st>>>(y, yscale, w, inv, shared_logit, k, kk, d,
                                                     blocks_row, out);
  };
  if (past_caches(int64_t(n) * kk * d))
    go(mx_combine_kernel<true>);
  else
    go(mx_combine_kernel<false>);
  PMOE_LAUNCH_CHECK("mx_combine_kernel");
  return PMOE_OK;
}

}  // namespace pmoe
