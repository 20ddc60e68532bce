// The RMS norm of a residual stream before a MoE block, and what follows the
// block in one pass over its outputs.
//
//   norm   h = w * x / sqrt(mean(x^2) + eps)
//   join   y   = sum over slots of weight_k * y_k (+ s * shared)   [slots given]
//          y   = w_post * y / sqrt(mean(y^2) + eps)                [post norm]
//          y   = gate * y, or sigmoid(gate) * y                    [gate]
//          out = residual_scale * residual + branch_scale * y
//          h   = w_next * out / sqrt(mean(out^2) + eps)            [next norm]
//
// All of it in fp32 from what the arrays hold, each result rounded once to its
// array's type: the next norm takes out as it was before its rounding.
//
// Both are bound by HBM: a row's elements stay in registers between the
// sums, so every array is read or written once.  A block a row; a thread
// holds 8 consecutive elements (16 or 32 bytes a load) of up to 8
// stretches; the two sums of a row go through a wave's lanes and then LDS.  Rows
// that are no multiple of 8 long or not on 16 bytes go element by element.
// Join of 16384 x 4096 bf16 with a gate per element and both norms: 671 MB in 113
// us, 5.9 TB/s; of 1000 rows with 10 slots of 2048: 53 MB in 10.9.  Few rows are
// bound by latency: norm of one row of 4096 2.4 us, join of 5 rows of 7168 fp32 4.4
// (rounds of loads between two sums; asking for everything before the first sum made
// 64 rows no faster and 16384 bf16 rows 111 -> 131, by its registers).
#include <type_traits>

#include "pmoe_internal.h"
#include "pmoe_kernels.h"

namespace pmoe {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxHidden = 16384;  // 256 threads with 64 elements each
constexpr int kMaxRows = 1 << 23;  // a launch holds less than 2^32 threads

struct JoinArgs {
  const void* residual;
  const uint16_t* y;
  const float* weights;       // [n, k] or null (k = 1)
  const uint16_t* shared_y;   // [n, d] or null
  const float* shared_logit;  // [n] or null
  const void* post;           // [d] or null
  const void* gate;
  const void* next;           // [d] or null
  void* out;
  uint16_t* h;
  int k, d;
  int stream_f32, weight_f32, gate_kind, gate_f32, gate_sigmoid;
  float residual_scale, branch_scale, eps, offset;
};

// NT: past the caches (what they would not hold anyway).
template <bool NT>
__device__ __forceinline__ u32x4 get16(const void* at) {
  if constexpr (NT)
    return __builtin_nontemporal_load(static_cast<const u32x4*>(at));
  else
    return *static_cast<const u32x4*>(at);
}

// 8 elements from base[at], at a multiple of 8.
template <bool NT>
__device__ __forceinline__ void get8(const void* base, bool f32, size_t at, float (&v)[8]) {
  if (f32) {
    const float* p = static_cast<const float*>(base) + at;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const u32x4 u = get16<NT>(p + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i + j] = __uint_as_float(u[j]);
    }
  } else {
    const u32x4 u = get16<NT>(static_cast<const uint16_t*>(base) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = bf16lo(u[i]), v[2 * i + 1] = bf16hi(u[i]);
  }
}

template <bool NT>
__device__ __forceinline__ void put16(void* at, u32x4 v) {
  if constexpr (NT)
    __builtin_nontemporal_store(v, static_cast<u32x4*>(at));
  else
    *static_cast<u32x4*>(at) = v;
}

template <bool NT>
__device__ __forceinline__ void put8(void* base, bool f32, size_t at, const float (&v)[8]) {
  if (f32) {
    float* p = static_cast<float*>(base) + at;
#pragma unroll
    for (int i = 0; i < 8; i += 4)
      put16<NT>(p + i, u32x4{__float_as_uint(v[i]), __float_as_uint(v[i + 1]),
                             __float_as_uint(v[i + 2]), __float_as_uint(v[i + 3])});
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = uint32_t(f2bf(v[2 * i])) | uint32_t(f2bf(v[2 * i + 1])) << 16;
    put16<NT>(static_cast<uint16_t*>(base) + at, u32x4{w[0], w[1], w[2], w[3]});
  }
}

__device__ __forceinline__ float get1(const void* base, bool f32, size_t at) {
  return f32 ? static_cast<const float*>(base)[at] : bf16f(static_cast<const uint16_t*>(base)[at]);
}

__device__ __forceinline__ void put1(void* base, bool f32, size_t at, float v) {
  if (f32)
    static_cast<float*>(base)[at] = v;
  else
    static_cast<uint16_t*>(base)[at] = f2bf(v);
}

// a + the same of the lane 32 (16) away, for a and b at once: lanes of the lower
// half (of even rows of 16) end with a's sums, the others with b's.
__device__ __forceinline__ float fold32(float a, float b) {
  const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false,
                                                  false);
  return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}
__device__ __forceinline__ float fold16(float a, float b) {
  const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false,
                                                  false);
  return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}
__device__ __forceinline__ float sum16(float v) {  // over a row of 16 lanes
  v += xor_lane<8>(v);
  v += xor_lane<4>(v);
  v += xor_lane<2>(v);
  return v + xor_lane<1>(v);
}

// The block's sum of v, whose v[j] are of stretch j: the sums of 512 elements that
// a wave holds of a stretch, one after the other, so that it does not depend on how
// many threads hold the row.  A wave folds up to four stretches at once.
template <int T, int NV = 1>
__device__ __forceinline__ float block_sum(const float (&v)[NV], float* s) {
  constexpr int W = T / 64;
  const int lane = threadIdx.x & 63;
  float* to = s + (threadIdx.x >> 6);
  if constexpr (NV == 1) {
    const float u = fold32(v[0], v[0]);
    const float p = sum16(fold16(u, u));
    if constexpr (W == 1) return p;
    if (lane == 0) *to = p;
  } else if constexpr (NV == 2) {
    const float u = fold32(v[0], v[1]);
    const float p = sum16(fold16(u, u));
    if ((lane & 31) == 0) to[W * (lane >> 5)] = p;
  } else {
#pragma unroll
    for (int j = 0; j < NV; j += 4) {
      const float p = sum16(fold16(fold32(v[j], v[j + 1]), fold32(v[j + 2], v[j + 3])));
      if ((lane & 15) == 0) to[W * (j + (lane >> 5) + (lane >> 3 & 2))] = p;
    }
  }
  __syncthreads();
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < NV * W; ++i) sum += s[i];
  return sum;
}

// 1 / sqrt(mean + eps)
__device__ __forceinline__ float inv_rms(float sum, int d, float eps) {
  return 1.0f / __builtin_sqrtf(sum / float(d) + eps);
}

__device__ __forceinline__ float gate_act(float g, int sigmoid) { return sigmoid ? psigmoid(g) : g; }

template <int T, int NV, bool NT>
__global__ __launch_bounds__(T) void norm_kernel(const void* x, int x_f32, const void* weight,
                                                 int w_f32, int d, float eps, float offset,
                                                 uint16_t* h) {
  __shared__ float s[NV * T / 64];
  const size_t row = size_t(blockIdx.x) * d;
  float v[NV][8];
  float sum[NV] = {};
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * T + int(threadIdx.x)) * 8;
    if (c < d) get8<false>(x, x_f32, row + c, v[j]);
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * T + int(threadIdx.x)) * 8;
    if (c < d)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[j] = __builtin_fmaf(v[j][i], v[j][i], sum[j]);
  }
  const float r = inv_rms(block_sum<T>(sum, s), d, eps);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * T + int(threadIdx.x)) * 8;
    if (c >= d) continue;
    float w[8];
    get8<false>(weight, w_f32, c, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = v[j][i] * r * (w[i] + offset);
    put8<NT>(h, false, row + c, v[j]);
  }
}

template <int T, int NV, bool NT>
__global__ __launch_bounds__(T) void join_kernel(const JoinArgs a) {
  __shared__ float s[2][NV * T / 64];
  const int d = a.d;
  const size_t n = blockIdx.x;
  const size_t row = n * d;
  float y[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * T + int(threadIdx.x)) * 8;
    if (c >= d) continue;
    if (!a.weights) {
      get8<NT>(a.y, false, row + c, y[j]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[j][i] = 0.0f;
      for (int k = 0; k < a.k; ++k) {
        float t[8];
        get8<NT>(a.y, false, (n * a.k + k) * d + c, t);
        const float w = a.weights[n * a.k + k];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[j][i] = __builtin_fmaf(w, t[i], y[j][i]);
      }
    }
    if (a.shared_y) {
      float t[8];
      get8<NT>(a.shared_y, false, row + c, t);
      const float w = a.shared_logit ? psigmoid(a.shared_logit[n]) : 1.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[j][i] = __builtin_fmaf(w, t[i], y[j][i]);
    }
  }
  if (a.post) {
    float sum[NV] = {};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * T + int(threadIdx.x)) * 8;
      if (c < d)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[j] = __builtin_fmaf(y[j][i], y[j][i], sum[j]);
    }
    const float r = inv_rms(block_sum<T>(sum, s[0]), d, a.eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * T + int(threadIdx.x)) * 8;
      if (c >= d) continue;
      float w[8];
      get8<false>(a.post, a.weight_f32, c, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[j][i] = y[j][i] * r * (w[i] + a.offset);
    }
  }
  const float tg = a.gate_kind == PMOE_GATE_TOKEN
                       ? gate_act(get1(a.gate, a.gate_f32, n), a.gate_sigmoid)
                       : 1.0f;
  float sum[NV] = {};
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * T + int(threadIdx.x)) * 8;
    if (c >= d) continue;
    float res[8];
    get8<NT>(a.residual, a.stream_f32, row + c, res);
    if (a.gate_kind == PMOE_GATE_CHANNEL || a.gate_kind == PMOE_GATE_ELEMENT) {
      float g[8];
      get8<false>(a.gate, a.gate_f32, (a.gate_kind == PMOE_GATE_ELEMENT ? row : 0) + c, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[j][i] *= gate_act(g[i], a.gate_sigmoid);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[j][i] *= tg;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[j][i] = __builtin_fmaf(a.residual_scale, res[i], a.branch_scale * y[j][i]);
      sum[j] = __builtin_fmaf(y[j][i], y[j][i], sum[j]);
    }
    put8<NT>(a.out, a.stream_f32, row + c, y[j]);
  }
  if (!a.next) return;
  const float r = inv_rms(block_sum<T>(sum, s[1]), d, a.eps);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * T + int(threadIdx.x)) * 8;
    if (c >= d) continue;
    float w[8];
    get8<false>(a.next, a.weight_f32, c, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[j][i] = y[j][i] * r * (w[i] + a.offset);
    put8<NT>(a.h, false, row + c, y[j]);
  }
}

// Element by element, rows of any length and alignment.
__global__ __launch_bounds__(256) void norm_any_kernel(const void* x, int x_f32, const void* weight,
                                                       int w_f32, int d, float eps, float offset,
                                                       uint16_t* h) {
  __shared__ float s[4];
  const size_t row = size_t(blockIdx.x) * d;
  float sum[1] = {};
  for (int c = threadIdx.x; c < d; c += 256) {
    const float v = get1(x, x_f32, row + c);
    sum[0] = __builtin_fmaf(v, v, sum[0]);
  }
  const float r = inv_rms(block_sum<256>(sum, s), d, eps);
  for (int c = threadIdx.x; c < d; c += 256)
    h[row + c] = f2bf(get1(x, x_f32, row + c) * r * (get1(weight, w_f32, c) + offset));
}

__device__ __forceinline__ float branch(const JoinArgs& a, size_t n, int c) {
  float y;
  if (!a.weights) {
    y = bf16f(a.y[n * a.d + c]);
  } else {
    y = 0.0f;
    for (int k = 0; k < a.k; ++k)
      y = __builtin_fmaf(a.weights[n * a.k + k], bf16f(a.y[(n * a.k + k) * a.d + c]), y);
  }
  if (a.shared_y)
    y = __builtin_fmaf(a.shared_logit ? psigmoid(a.shared_logit[n]) : 1.0f,
                       bf16f(a.shared_y[n * a.d + c]), y);
  return y;
}

// keep: out's fp32 values between the passes, a thread's in its registers (what
// out holds is rounded, and may have replaced the residual).
__global__ __launch_bounds__(256) void join_any_kernel(const JoinArgs a) {
  __shared__ float s[2][4];
  constexpr int kEach = kMaxHidden / 256;
  float keep[kEach];
  const int d = a.d;
  const size_t n = blockIdx.x;
  const size_t row = n * d;
  float rp = 1.0f;
  if (a.post) {
    float sum[1] = {};
    for (int c = threadIdx.x; c < d; c += 256) {
      const float y = branch(a, n, c);
      sum[0] = __builtin_fmaf(y, y, sum[0]);
    }
    rp = inv_rms(block_sum<256>(sum, s[0]), d, a.eps);
  }
  float sum[1] = {};
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int c = j * 256 + int(threadIdx.x);
    if (c >= d) continue;
    float y = branch(a, n, c);
    if (a.post) y = y * rp * (get1(a.post, a.weight_f32, c) + a.offset);
    if (a.gate_kind != PMOE_GATE_NONE)
      y *= gate_act(get1(a.gate, a.gate_f32,
                         a.gate_kind == PMOE_GATE_CHANNEL ? c
                         : a.gate_kind == PMOE_GATE_TOKEN ? n
                                                          : row + c),
                    a.gate_sigmoid);
    y = __builtin_fmaf(a.residual_scale, get1(a.residual, a.stream_f32, row + c),
                       a.branch_scale * y);
    sum[0] = __builtin_fmaf(y, y, sum[0]);
    put1(a.out, a.stream_f32, row + c, y);
    keep[j] = y;
  }
  if (!a.next) return;
  const float r = inv_rms(block_sum<256>(sum, s[1]), d, a.eps);
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int c = j * 256 + int(threadIdx.x);
    if (c < d) a.h[row + c] = f2bf(keep[j] * r * (get1(a.next, a.weight_f32, c) + a.offset));
  }
}

bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Results of this many bytes and more, and a join's inputs beside them, go past the
// caches (join of 8192 x 4096 bf16 66 -> 60 us, 16384 123 -> 119; norm of 16384 x
// 4096 fp32 70.5 -> 68.5, which its input past them too makes 73); below, the
// next kernel finds them there.
constexpr int64_t kPastCaches = int64_t(64) << 20;

// Rows up to which a row gets more threads than it needs.  us, more / fewest, bf16
// with a gate per element and both norms:
//   4096    64 rows 4.0 / 5.2   512: 5.9 / 6.7   1024: 10.0 / 9.7   16384: 129 / 111
//   7168    64: 4.9 / 8.2   512: 9.4 / 11.6   1024: 16.6 / 16.5   2048: 29.5 / 28.9
//   12288   64: 6.1 / 12.2   512: 13.4 / 19   1024: 23 / 25   2048: 43 / 46
constexpr int kFewRows = 512;

// go(threads, stretches) for n rows of d: few rows get as many threads as pay, for
// the shortest way through them, many the fewest that hold a row (the same sums).
template <class Go>
void by_width(int n, int d, Go go) {
  const bool few = n <= kFewRows;
  const auto with = [&](auto narrow_stretches, auto threads, auto stretches) {
    if (few)
      go(threads, stretches);
    else
      go(std::integral_constant<int, 256>{}, narrow_stretches);
  };
  constexpr std::integral_constant<int, 1> one{};
  constexpr std::integral_constant<int, 2> two{};
  if (d <= 512)
    go(std::integral_constant<int, 64>{}, one);
  else if (d <= 2048)
    go(std::integral_constant<int, 256>{}, one);
  else if (d <= 4096)
    with(two, std::integral_constant<int, 512>{}, one);
  else if (d <= 8192)
    with(std::integral_constant<int, 4>{}, std::integral_constant<int, 1024>{}, one);
  else
    with(std::integral_constant<int, 8>{}, std::integral_constant<int, 1024>{}, two);
}

bool stream_dtype(int t) { return t == PMOE_F32 || t == PMOE_BF16; }

}  // namespace

}  // namespace pmoe

extern "C" int pmoe_block_norm(const void* x, int x_dtype, const void* weight, int weight_dtype,
                               int n, int hidden, float eps, int unit_offset, void* h,
                               void* stream) {
  using namespace pmoe;
  clear_error();
  PMOE_REQUIRE(x && weight && h, "block_norm: null pointer");
  PMOE_REQUIRE(stream_dtype(x_dtype) && stream_dtype(weight_dtype),
               "block_norm: arrays are fp32 or bf16");
  PMOE_REQUIRE(n >= 0 && hidden > 0 && hidden <= kMaxHidden,
               "block_norm: hidden must be 1..16384");
  PMOE_REQUIRE(n <= kMaxRows, "block_norm: more than 2^23 rows");
  PMOE_REQUIRE(eps >= 0.0f, "block_norm: eps must not be negative");
  if (n == 0) return PMOE_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  ProfScope prof_scope(K_BLOCK_NORM, st);
  const float off = unit_offset ? 1.0f : 0.0f;
  uint16_t* out = static_cast<uint16_t*>(h);
  const int xf = x_dtype == PMOE_F32, wf = weight_dtype == PMOE_F32;
  if (hidden % 8 == 0 && on16(x) && on16(weight) && on16(h))
    by_width(n, hidden, [&](auto t, auto nv) {
      constexpr int T = decltype(t)::value, NV = decltype(nv)::value;
      if (int64_t(n) * hidden * 2 >= kPastCaches)
        norm_kernel<T, NV, true><<<n, T, 0, st>>>(x, xf, weight, wf, hidden, eps, off, out);
      else
        norm_kernel<T, NV, false><<<n, T, 0, st>>>(x, xf, weight, wf, hidden, eps, off, out);
    });
  else
    norm_any_kernel<<<n, 256, 0, st>>>(x, xf, weight, wf, hidden, eps, off, out);
  PMOE_LAUNCH_CHECK("norm_kernel");
  return PMOE_OK;
}

extern "C" int pmoe_block_join(const pmoe_join* j, const void* residual, const void* y,
                               const float* weights, const void* shared_y,
                               const float* shared_logit, const void* post_weight,
                               const void* gate, const void* next_weight, int n, int k, int hidden,
                               void* out, void* h, void* stream) {
  using namespace pmoe;
  clear_error();
  PMOE_REQUIRE(j && residual && y && out, "block_join: null pointer");
  PMOE_REQUIRE(stream_dtype(j->stream_dtype) && stream_dtype(j->weight_dtype) &&
                   stream_dtype(j->gate_dtype),
               "block_join: arrays are fp32 or bf16");
  PMOE_REQUIRE(n >= 0 && k > 0 && hidden > 0 && hidden <= kMaxHidden,
               "block_join: bad shape (hidden must be 1..16384)");
  PMOE_REQUIRE(n <= kMaxRows, "block_join: more than 2^23 rows");
  PMOE_REQUIRE(weights || k == 1, "block_join: several slots need weights");
  PMOE_REQUIRE(!shared_logit || shared_y, "block_join: shared_logit without shared_y");
  PMOE_REQUIRE((j->gate_kind == PMOE_GATE_NONE) == (gate == nullptr) &&
                   j->gate_kind >= PMOE_GATE_NONE && j->gate_kind <= PMOE_GATE_ELEMENT,
               "block_join: gate and gate_kind do not agree");
  PMOE_REQUIRE((next_weight == nullptr) == (h == nullptr),
               "block_join: next_weight and h go together");
  PMOE_REQUIRE(j->eps >= 0.0f, "block_join: eps must not be negative");
  if (n == 0) return PMOE_OK;
  JoinArgs a{};
  a.residual = residual;
  a.y = static_cast<const uint16_t*>(y);
  a.weights = weights;
  a.shared_y = static_cast<const uint16_t*>(shared_y);
  a.shared_logit = shared_logit;
  a.post = post_weight;
  a.gate = gate;
  a.next = next_weight;
  a.out = out;
  a.h = static_cast<uint16_t*>(h);
  a.k = k, a.d = hidden;
  a.stream_f32 = j->stream_dtype == PMOE_F32;
  a.weight_f32 = j->weight_dtype == PMOE_F32;
  a.gate_kind = j->gate_kind;
  a.gate_f32 = j->gate_dtype == PMOE_F32;
  a.gate_sigmoid = j->gate_sigmoid;
  a.residual_scale = j->residual_scale, a.branch_scale = j->branch_scale;
  a.eps = j->eps;
  a.offset = j->unit_offset ? 1.0f : 0.0f;
  hipStream_t st = static_cast<hipStream_t>(stream);
  ProfScope prof_scope(K_BLOCK_NORM, st);
  const bool gate_ok = j->gate_kind == PMOE_GATE_TOKEN || on16(gate);
  if (hidden % 8 == 0 && on16(residual) && on16(y) && on16(shared_y) && on16(post_weight) &&
      on16(next_weight) && on16(out) && on16(h) && gate_ok)
    by_width(n, hidden, [&](auto t, auto nv) {
      constexpr int T = decltype(t)::value, NV = decltype(nv)::value;
      if (int64_t(n) * hidden * (a.stream_f32 ? 4 : 2) >= kPastCaches)
        join_kernel<T, NV, true><<<n, T, 0, st>>>(a);
      else
        join_kernel<T, NV, false><<<n, T, 0, st>>>(a);
    });
  else
    join_any_kernel<<<n, 256, 0, st>>>(a);
  PMOE_LAUNCH_CHECK("join_kernel");
  return PMOE_OK;
}
