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
#include "mx_pieces.h"
#include "mx_experts.h"
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
      for (int f = 0; f < NF; ++f) mx_mma(acc[f], w[f][i], sw[f][i], b1, sa - 4);
      if constexpr (DUAL) {
        const uint4* s3 = reinterpret_cast<const uint4*>(third + size_t(gc) * kMxThirdBytes);
        const uint4 d0 = s3[0], d1 = s3[1];
        const uint32_t b2[6] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y};
#pragma unroll
        for (int f = 0; f < NF; ++f) mx_mma(acc[f], w[f][i], sw[f][i], b2, sa - 8);
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

}  // namespace

int mx_tile_rows(int, int, int) { return kSmallRows; }
int mx_min_tile_rows() { return kSmallRows; }

int mx_experts(const MxPlan& p, hipStream_t st) {
  const pmoe_geom* g = p.geom;
  {
    ProfScope prof_scope(K_MX_SPLIT, st);
    mx_split_kernel<<<p.n, 256, 0, st>>>(p.x, p.n, g->hidden / kMxGroup, p.xpair, p.xthird,
                                         p.xscale, p.xsteps);
    PMOE_LAUNCH_CHECK("mx_split_kernel");
  }
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
  a.pair = p.xpair, a.third = p.xthird, a.ascale = p.xscale;
  a.hpair = p.hpair, a.hscale = p.hscale;
  if (int rc = launch_small<true>(a, p.max_tiles, st)) return rc;
  a.w0 = g->off[PMOE_DOWN_W], a.s0 = g->off[PMOE_DOWN_S];
  a.features = g->hidden;
  a.cols = g->inter;
  a.pair = p.hpair, a.third = nullptr, a.ascale = p.hscale;
  a.y = p.y;
  return launch_small<false>(a, p.max_tiles, st);
}

}  // namespace pmoe
