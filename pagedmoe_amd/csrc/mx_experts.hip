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
// An activation that is infinite or NaN, or an intermediate that leaves fp32,
// makes the outputs of its row NaN.
#include <stdlib.h>

#include "mx_experts.h"
#include "mx_pieces.h"
#include "pmoe_internal.h"
#include "pmoe_kernels.h"

namespace pmoe {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kFp4 = 4, kFp6 = 2;  // operand formats of the scaled MFMA

// acc += W (16 rows x 128) times a piece of 16 activation rows; sw, sp: the
// lane's scale bytes.
__device__ __forceinline__ void mx_mma(f32x4& acc, const uint4& w, int sw, const uint32_t (&p)[6],
                                       int sp) {
  const i32x8 a = {int(w.x), int(w.y), int(w.z), int(w.w), 0, 0, 0, 0};
  const i32x8 b = {int(p[0]), int(p[1]), int(p[2]), int(p[3]), int(p[4]), int(p[5]), 0, 0};
  acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, kFp4, kFp6, 0, sw, 0, sp);
}

// ---------------------------------------------------------------- activations

// One lane a group: x bf16 [n, d] into pieces, scales and each token's mask of
// the 128-wide steps that hold a third piece (16 bits a wave, 4 waves a token).
__global__ __launch_bounds__(256) void mx_split_kernel(const uint16_t* __restrict__ x, int n,
                                                       int groups, uint8_t* __restrict__ pair,
                                                       uint8_t* __restrict__ third,
                                                       uint8_t* __restrict__ scales,
                                                       uint16_t* __restrict__ steps) {
  const int token = blockIdx.x;
  const int g = threadIdx.x;
  bool peak = false;
  if (g < groups) {
    const size_t at = size_t(token) * groups + g;
    const uint4* src = reinterpret_cast<const uint4*>(x + at * kMxGroup);
    float v[32];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 u = src[i];
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[8 * i + 2 * j] = bf16lo(w[j]), v[8 * i + 2 * j + 1] = bf16hi(w[j]);
    }
    int s;
    u32x6 p0, p1, p2;
    peak = mx_split<true>(v, s, p0, p1, p2);
    mx_store_pair(pair + at * kMxPairBytes, p0, p1);
    mx_store_third(third + at * kMxThirdBytes, p2);
    scales[at] = uint8_t(s);
  }
  const uint64_t m = __ballot(peak);
  if ((threadIdx.x & 63) == 0) {
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) bits |= (m >> (4 * i) & 15) ? 1u << i : 0u;
    steps[size_t(token) * 4 + (threadIdx.x >> 6)] = uint16_t(bits);
  }
}

// ---------------------------------------------------------------- small tiles

constexpr int kSmallRows = 16;   // activation rows a tile
constexpr int kSmallCols = 32;   // features a block (one group of the next product)
constexpr int kStep = 512;       // reduction that a wave takes at a time
constexpr int kMaxWaves = 8;

// One tile of at most 16 rows of an expert times 32 features (DUAL: 32 gate
// and the same 32 up features).  The waves share the reduction: wave w takes
// steps w, w + waves, ... of 512, all loads of a step in flight at once, and
// the partial sums meet in LDS.  FULL: the reduction is whole steps.
template <bool DUAL, bool FULL>
__global__ __launch_bounds__(64 * kMaxWaves) void mx_small_kernel(const MxArgs a) {
  constexpr int NF = DUAL ? 4 : 2;  // 16-feature tiles: gate, gate, up, up
  __shared__ float s_red[kMaxWaves][NF * 4][64];
  __shared__ float s_h[kSmallRows][kSmallCols + 1];
  const int fblocks = a.features / kSmallCols;
  const int t = blockIdx.x / fblocks;
  const int fb = blockIdx.x - t * fblocks;
  if (t >= *a.n_tiles) return;
  const int4 tile = a.tiles[t];  // {slot, first row, rows of the expert, offset}
  const int m = min(kSmallRows, tile.z - tile.y);
  const int p0 = tile.w + tile.y;
  const int waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (tile.x < 0) {  // not resident: exact zero rows
    if constexpr (!DUAL) {
      for (int i = threadIdx.x; i < m * kSmallCols; i += blockDim.x)
        a.y[size_t(a.order[p0 + i / kSmallCols]) * a.features + fb * kSmallCols +
            i % kSmallCols] = 0;
    }
    return;
  }
  const int r = lane & 15, q = lane >> 4;
  const int pos = p0 + (r < m ? r : 0);
  const size_t arow = DUAL ? size_t(a.order[pos] / a.kk) : size_t(pos);
  const int groups = a.cols / kMxGroup;
  const uint8_t* base = a.slab + size_t(tile.x) * size_t(a.expert_bytes);
  const uint8_t* wrow[NF];
  const uint8_t* srow[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const size_t row = size_t(fb) * kSmallCols + (f & 1) * 16 + r;
    wrow[f] = base + (f < 2 ? a.w0 : a.w1) + row * size_t(a.cols / 2);
    srow[f] = base + (f < 2 ? a.s0 : a.s1) + row * size_t(groups);
  }
  const uint8_t* pair = a.pair + arow * groups * kMxPairBytes;
  const uint8_t* third = DUAL ? a.third + arow * groups * kMxThirdBytes : nullptr;
  const uint8_t* ascale = a.ascale + arow * groups;
  f32x4 acc[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int steps = (groups + 15) / 16;
  for (int j = wave; j < steps; j += waves) {
    uint4 w[NF][4];
    int sw[NF][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int g = 16 * j + 4 * i + q;
      const bool in = FULL || g < groups;
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        w[f][i] = in ? *reinterpret_cast<const uint4*>(wrow[f] + size_t(g) * 16)
                     : make_uint4(0, 0, 0, 0);
        sw[f][i] = in ? srow[f][g] : 127;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int g = 16 * j + 4 * i + q;
      const bool in = FULL || g < groups;
      const int gc = in ? g : 0;
      const uint4* src = reinterpret_cast<const uint4*>(pair + size_t(gc) * kMxPairBytes);
      const uint4 c0 = src[0], c1 = src[1], c2 = src[2];
      const int sa = in ? ascale[gc] : 127;
      const uint32_t b0[6] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y};
      const uint32_t b1[6] = {c1.z, c1.w, c2.x, c2.y, c2.z, c2.w};
#pragma unroll
      for (int f = 0; f < NF; ++f) mx_mma(acc[f], w[f][i], sw[f][i], b0, sa);
#pragma unroll
      for (int f = 0; f < NF; ++f)
        mx_mma(acc[f], w[f][i], sw[f][i], b1, sa - (DUAL ? kMxTokenShift : kMxInterShift));
      if constexpr (DUAL) {
        const uint4* s3 = reinterpret_cast<const uint4*>(third + size_t(gc) * kMxThirdBytes);
        const uint4 d0 = s3[0], d1 = s3[1];
        const uint32_t b2[6] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y};
#pragma unroll
        for (int f = 0; f < NF; ++f) mx_mma(acc[f], w[f][i], sw[f][i], b2, sa - 2 * kMxTokenShift);
      }
    }
  }
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) s_red[wave][4 * f + i][lane] = acc[f][i];
  __syncthreads();
  // feature c of row s_r: accumulator c % 4 of lane 16 (c % 16 / 4) + row
  for (int i = threadIdx.x; i < m * kSmallCols; i += blockDim.x) {
    const int row = i / kSmallCols, c = i % kSmallCols;
    const int src = (c & 15) / 4 * 16 + row;
    float v = 0.0f, u = 0.0f;
    for (int k = 0; k < waves; ++k) {
      v += s_red[k][4 * (c >> 4) + (c & 3)][src];
      if constexpr (DUAL) u += s_red[k][4 * (2 + (c >> 4)) + (c & 3)][src];
    }
    if constexpr (DUAL)
      s_h[row][c] = silu_fast(v) * u;
    else
      a.y[size_t(a.order[p0 + row]) * a.features + fb * kSmallCols + c] = f2bf(v);
  }
  if constexpr (DUAL) {
    __syncthreads();
    if (int(threadIdx.x) < m) {
      float v[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) v[c] = s_h[threadIdx.x][c];
      int s;
      u32x6 h0, h1, h2;
      mx_split<false>(v, s, h0, h1, h2);
      const size_t at = size_t(p0 + threadIdx.x) * fblocks + fb;
      mx_store_pair(a.hpair + at * kMxPairBytes, h0, h1);
      a.hscale[at] = uint8_t(s);
    }
  }
}

template <bool DUAL>
int launch_small(const MxArgs& a, int max_tiles, hipStream_t st) {
  const int steps = (a.cols + kStep - 1) / kStep;
  const int rounds = (steps + kMaxWaves - 1) / kMaxWaves;
  const int waves = (steps + rounds - 1) / rounds;
  const int64_t blocks = int64_t(max_tiles) * (a.features / kSmallCols);
  PMOE_REQUIRE(blocks < (int64_t(1) << 31) / 1, "experts: too many tiles for one call");
  ProfScope prof_scope(DUAL ? K_MX_GATEUP : K_MX_DOWN, st);
  if (a.cols % kStep == 0)
    mx_small_kernel<DUAL, true><<<unsigned(blocks), 64 * waves, 0, st>>>(a);
  else
    mx_small_kernel<DUAL, false><<<unsigned(blocks), 64 * waves, 0, st>>>(a);
  PMOE_LAUNCH_CHECK("mx_small_kernel");
  return PMOE_OK;
}

// ---------------------------------------------------------------- large tiles

constexpr int kTileRows = 128;    // activation rows a block
constexpr int kTileCols = 512;    // weight rows a block (DUAL: 256 gate, 256 up)
constexpr int kTileWaves = 8;     // 2 halves of the rows x 4 quarters of the weights
constexpr int kActBytes = 8 * 3 * 1024;             // 8 row tiles x 3 chunks a lane
constexpr int kWeightBytes = kTileCols / 16 * 1024;  // 32 row tiles x 1 chunk a lane
constexpr int kActScaleBytes = kTileWaves * 256;
constexpr int kWeightScaleBytes = kTileWaves * 256;
constexpr int kStageBytes = kActBytes + kWeightBytes + kActScaleBytes + kWeightScaleBytes;
constexpr int kTileLds = 2 * kStageBytes;

// 16 bytes (4 bytes) a lane from p to LDS [lds, lds + 1024) ([.., + 256)), lane l
// at 16 l (4 l).
__device__ __forceinline__ void dma16(uint32_t lds, const uint8_t* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(lds), "v"(p)
               : "memory");
}

__device__ __forceinline__ void dma4(uint32_t lds, const uint8_t* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
               :
               : "s"(lds), "v"(p)
               : "memory");
}

// The steps of a tile's reduction, in order: every 128-wide step with the first
// two pieces, then, for tokens, those steps in which a row of the tile has a
// third piece.
struct Steps {
  int s, n;
  uint64_t left;
  __device__ __forceinline__ bool third() const { return s >= n; }
  __device__ __forceinline__ int step() const {
    return third() ? __builtin_ctzll(left) : s;
  }
  __device__ __forceinline__ void next() {
    if (third())
      left &= left - 1;
    else
      ++s;
  }
  __device__ __forceinline__ bool done() const { return third() && left == 0; }
};

// One tile of at most 128 rows of an expert times 512 weight rows (DUAL: 256
// gate and the same 256 up features).  Each wave holds 64 rows times 128 weight
// rows in its accumulators.  A step of 128 goes from memory straight into LDS
// in the order in which the lanes read it back, 16 bytes a lane, so that no
// read has a bank conflict; the next step's loads are in flight while this
// one's products run.
template <bool DUAL>
__global__ __launch_bounds__(64 * kTileWaves, 2) void mx_tile_kernel(const MxArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kTileLds];
  __shared__ unsigned long long s_third;
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
      for (int row = wave; row < m; row += kTileWaves)
        for (int c = lane; c < cols; c += 64)
          a.y[size_t(a.order[p0 + row]) * a.features + fb * kCols + c] = 0;
    }
    return;
  }
  const int r = lane & 15, q = lane >> 4;
  const int groups = a.cols / kMxGroup;
  const uint8_t* base = a.slab + size_t(tile.x) * size_t(a.expert_bytes);

  // What this wave loads each step: row tile `wave` of the activations (and its
  // scales), weight tiles 4 wave .. + 3 and the scales of those 64 rows.
  const int lrow = 16 * wave + r;
  const int lpos = p0 + (lrow < m ? lrow : 0);
  const size_t arow = DUAL ? size_t(a.order[lpos] / a.kk) : size_t(lpos);
  const uint8_t* pair = a.pair + (arow * groups + q) * kMxPairBytes;
  const uint8_t* third = DUAL ? a.third + (arow * groups + q) * kMxThirdBytes : nullptr;
  const uint8_t* ascale = a.ascale + arow * groups;
  // weight row w of the block: its gate (0..255) or up feature; rows past the
  // projection load its last ones and are not used
  const auto weight_row = [&](int w) {
    const int f = fb * kCols + (DUAL ? w & (kCols - 1) : w);
    return size_t(min(f, a.features - 1));
  };
  const bool second = DUAL && wave >= kTileWaves / 2;
  const uint8_t* wbase = base + (second ? a.w1 : a.w0);
  const uint8_t* wsrc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    wsrc[i] = wbase + weight_row(64 * wave + 16 * i + r) * size_t(a.cols / 2) + q * 16;
  const uint8_t* wscale =
      base + (second ? a.s1 : a.s0) + weight_row(64 * wave + lane) * size_t(groups);

  Steps todo{0, groups / 4, 0};
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
    todo.left = uint64_t(lo) | uint64_t(hi) << 32;
  }
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(
      uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds)));
  const auto issue = [&](const Steps& st, int buf) {
    const size_t s = size_t(st.step());
    const uint32_t to = lds0 + buf * kStageBytes;
    const uint32_t act = to + wave * 3 * 1024;
    if (!DUAL || !st.third()) {
      const uint8_t* p = pair + s * (4 * kMxPairBytes);
      dma16(act, p);
      dma16(act + 1024, p + 16);
      dma16(act + 2048, p + 32);
    } else {
      const uint8_t* p = third + s * (4 * kMxThirdBytes);
      dma16(act, p);
      dma16(act + 1024, p + 16);
    }
    const uint32_t wt = to + kActBytes + wave * 4 * 1024;
#pragma unroll
    for (int i = 0; i < 4; ++i) dma16(wt + i * 1024, wsrc[i] + s * 64);
    dma4(to + kActBytes + kWeightBytes + wave * 256, ascale + s * 4);
    dma4(to + kActBytes + kWeightBytes + kActScaleBytes + wave * 256, wscale + s * 4);
  };

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

  issue(todo, 0);
  Steps ahead = todo;
  ahead.next();
  for (int buf = 0; !todo.done(); buf ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // this step is in LDS, and the other buffer has been read
    if (!ahead.done()) {
      issue(ahead, buf ^ 1);
      ahead.next();
    }
    const uint8_t* from = lds + buf * kStageBytes;
    const uint8_t* as = from + kActBytes + kWeightBytes;
    const uint8_t* ws = as + kActScaleBytes;
    uint4 w[8];
    int sw[8];
#pragma unroll
    for (int f = 0; f < 8; ++f) {
      const int wt = weight_tile(f);
      w[f] = *reinterpret_cast<const uint4*>(from + kActBytes + wt * 1024 + lane * 16);
      sw[f] = ws[(wt >> 2) * 256 + ((wt & 3) * 16 + r) * 4 + q];
    }
    const bool third_step = DUAL && todo.third();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i >= tiles_in) break;
      const int rt = 4 * rh + i;
      const uint8_t* src = from + rt * 3 * 1024 + lane * 16;
      const int sa = as[rt * 256 + r * 4 + q];
      const uint4 c0 = *reinterpret_cast<const uint4*>(src);
      const uint4 c1 = *reinterpret_cast<const uint4*>(src + 1024);
      const uint32_t b0[6] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y};
      if (third_step) {
#pragma unroll
        for (int f = 0; f < 8; ++f) mx_mma(acc[f][i], w[f], sw[f], b0, sa - 2 * kMxTokenShift);
      } else {
        const uint4 c2 = *reinterpret_cast<const uint4*>(src + 2048);
        const uint32_t b1[6] = {c1.z, c1.w, c2.x, c2.y, c2.z, c2.w};
#pragma unroll
        for (int f = 0; f < 8; ++f) mx_mma(acc[f][i], w[f], sw[f], b0, sa);
#pragma unroll
        for (int f = 0; f < 8; ++f)
          mx_mma(acc[f][i], w[f], sw[f], b1, sa - (DUAL ? kMxTokenShift : kMxInterShift));
      }
    }
    todo.next();
  }

  if constexpr (DUAL) {
    // h of 32 rows x 64 features at a time through LDS, then a lane a group
    constexpr int kPitch = 68;
    float* hs = reinterpret_cast<float*>(lds) + wave * 32 * kPitch;
    static_assert(kTileWaves * 32 * kPitch * 4 <= kTileLds, "h staging");
    const int f0 = fb * kCols + 64 * wq;
    const int hgroups = a.features / kMxGroup;
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
        u32x6 h0, h1, h2;
        mx_split<false>(v, s, h0, h1, h2);
        const size_t to = size_t(p0 + row) * hgroups + f / kMxGroup;
        mx_store_pair(a.hpair + to * kMxPairBytes, h0, h1);
        a.hscale[to] = uint8_t(s);
      }
      __syncthreads();
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 64 * rh + 16 * i + r;
      if (row >= m) continue;
      uint16_t* y = a.y + size_t(a.order[p0 + row]) * a.features;
#pragma unroll
      for (int f = 0; f < 8; ++f) {
        const int c = fb * kCols + 128 * wq + 16 * f + 4 * q;
        if (c >= a.features) continue;
        const f32x4 v = acc[f][i];
        *reinterpret_cast<uint2*>(y + c) = make_uint2(uint32_t(f2bf(v[0])) | uint32_t(f2bf(v[1])) << 16,
                                                      uint32_t(f2bf(v[2])) | uint32_t(f2bf(v[3])) << 16);
      }
    }
  }
}

template <bool DUAL>
int launch_tile(const MxArgs& a, int max_tiles, hipStream_t st) {
  constexpr int kCols = DUAL ? kTileCols / 2 : kTileCols;
  const int64_t blocks = (int64_t(max_tiles) * ((a.features + kCols - 1) / kCols) + 7) / 8 * 8;
  PMOE_REQUIRE(blocks < (int64_t(1) << 31), "experts: too many tiles for one call");
  ProfScope prof_scope(DUAL ? K_MX_GATEUP : K_MX_DOWN, st);
  mx_tile_kernel<DUAL><<<unsigned(blocks), 64 * kTileWaves, 0, st>>>(a);
  PMOE_LAUNCH_CHECK("mx_tile_kernel");
  return PMOE_OK;
}

}  // namespace

int mx_tile_rows(const pmoe_geom* g, int n, int kk, int n_experts) {
  const char* v = getenv("PMOE_MX_TILE");
  // whole steps, and scales that a lane can fetch four at a time
  if (g->hidden % 128 || g->inter % 128 ||
      (g->off[PMOE_GATE_S] | g->off[PMOE_UP_S] | g->off[PMOE_DOWN_S]) % 4)
    return kSmallRows;
  if (v && v[0] == '0') return kSmallRows;
  if (v && v[0] == '1') return kTileRows;
  return int64_t(n) * kk >= 16L * n_experts ? kTileRows : kSmallRows;
}
int mx_min_tile_rows() { return kSmallRows; }

int mx_experts(const MxPlan& p, hipStream_t st) {
  const pmoe_geom* g = p.geom;
  {
    ProfScope prof_scope(K_MX_SPLIT, st);
    mx_split_kernel<<<p.n, 256, 0, st>>>(p.x, p.n, g->hidden / kMxGroup, p.xpair, p.xthird,
                                         p.xscale, p.xsteps);
    PMOE_LAUNCH_CHECK("mx_split_kernel");
  }
  const bool large = p.tile_rows == kTileRows;
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
  if (int rc = large ? launch_tile<true>(a, p.max_tiles, st)
                     : launch_small<true>(a, p.max_tiles, st))
    return rc;
  a.w0 = g->off[PMOE_DOWN_W], a.s0 = g->off[PMOE_DOWN_S];
  a.features = g->hidden;
  a.cols = g->inter;
  a.pair = p.hpair, a.third = nullptr, a.ascale = p.hscale, a.asteps = nullptr;
  a.y = p.y;
  return large ? launch_tile<false>(a, p.max_tiles, st) : launch_small<false>(a, p.max_tiles, st);
}

}  // namespace pmoe
