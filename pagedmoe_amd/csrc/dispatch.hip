// Token -> expert dispatch: histogram, exclusive scan, stable scatter.
//
// Replaces the reference's host-side dispatch: order = np.argsort(flat,
// kind="stable"), rows = order // K, per-expert searchsorted
// (streaming.py:789-808) and the unsort inv[order] = arange (:833-836).
// Integer work, HBM/latency bound; no float anywhere, so every output is
// bit-exact.
//
// Stability: the position of flat row r inside expert e's segment is the
// number of earlier rows with the same expert.  Rows are cut into blocks of
// kChunk; a row's rank inside its block is its rank inside its wave plus the
// earlier waves' counts (block_rank), and the block's base per expert comes
// from an exclusive scan over blocks (block-major within each expert).
#include "dispatch_small.h"
#include "pmoe_internal.h"
#include "pmoe_kernels.h"

namespace pmoe {

namespace {

constexpr int kChunk = kDispatchChunk;

__global__ __launch_bounds__(1024) void dispatch_small_kernel(
    const IdSrc src, int rows, int n_experts, int32_t* __restrict__ order,
    int32_t* __restrict__ counts, int32_t* __restrict__ offsets, int32_t* __restrict__ inv,
    int32_t* __restrict__ active, int32_t* __restrict__ n_active, const TileSink ts) {
  __shared__ DispatchLds lds;
  dispatch_small(lds, src, rows, n_experts, order, counts, offsets, inv, active, n_active, ts);
}

// Multi-block path, phase 1: per-block histogram and in-block ranks.
__global__ __launch_bounds__(kChunk) void dispatch_count_kernel(
    const IdSrc src, int rows, int n_experts, int32_t* __restrict__ hist,
    int32_t* __restrict__ rank_out) {
  __shared__ __attribute__((aligned(16))) int s_e[kChunk];
  __shared__ __attribute__((aligned(16))) uint8_t s_wc[kMaxExperts * 4];
  const int tid = threadIdx.x;
  const int row = blockIdx.x * kChunk + tid;
  reinterpret_cast<uint4*>(s_wc)[tid] = make_uint4(0, 0, 0, 0);
  const int my_e = row < rows ? load_id(src, row) : -1;
  s_e[tid] = my_e;
  __syncthreads();
  const int rank = block_rank<4>(my_e, rows - int(blockIdx.x) * kChunk, s_e, s_wc);
  if (my_e >= 0) rank_out[row] = rank;
  for (int e = tid; e < n_experts; e += kChunk)
    hist[size_t(blockIdx.x) * n_experts + e] = block_count<4>(s_wc, e);
}

__global__ __launch_bounds__(1024) void dispatch_scan_kernel(
    int32_t* __restrict__ hist, int n_blocks, int n_experts, int32_t* __restrict__ counts,
    int32_t* __restrict__ offsets, int32_t* __restrict__ active, int32_t* __restrict__ n_active,
    const TileSink ts) {
  __shared__ ScanLds lds;
  dispatch_scan(lds, hist, n_blocks, n_experts, counts, offsets, active, n_active, ts);
}

// Phase 3: scatter rows to their positions.
__global__ __launch_bounds__(kChunk) void dispatch_scatter_kernel(
    const IdSrc src, int rows, int n_experts, const int32_t* __restrict__ hist,
    const int32_t* __restrict__ rank, int32_t* __restrict__ order, int32_t* __restrict__ inv) {
  const int row = blockIdx.x * kChunk + threadIdx.x;
  if (row >= rows) return;
  const int e = load_id(src, row);
  if (e < 0) {
    inv[row] = -1;
    return;
  }
  const int pos = hist[size_t(blockIdx.x) * n_experts + e] + rank[row];
  order[pos] = row;
  inv[row] = pos;
}

}  // namespace

size_t dispatch_workspace(int rows, int n_experts) {
  if (rows <= kSmallRows) return 256;
  const size_t blocks = (rows + kChunk - 1) / kChunk;
  return ((blocks * n_experts + rows) * sizeof(int32_t) + 255) / 256 * 256;
}

int dispatch_count(const IdSrc& src, int rows, int n_ids, int32_t* hist, int32_t* rank,
                   hipStream_t st) {
  const int blocks = (rows + kChunk - 1) / kChunk;
  dispatch_count_kernel<<<blocks, kChunk, 0, st>>>(src, rows, n_ids, hist, rank);
  PMOE_LAUNCH_CHECK("dispatch_count_kernel");
  return PMOE_OK;
}

int dispatch_scatter(const IdSrc& src, int rows, int n_ids, const int32_t* hist,
                     const int32_t* rank, int32_t* order, int32_t* inv, hipStream_t st) {
  const int blocks = (rows + kChunk - 1) / kChunk;
  dispatch_scatter_kernel<<<blocks, kChunk, 0, st>>>(src, rows, n_ids, hist, rank, order, inv);
  PMOE_LAUNCH_CHECK("dispatch_scatter_kernel");
  return PMOE_OK;
}

// Internal entry: also builds the prefill tile list when tile_m > 0 (slots
// from table, the shared pseudo-id's from shared_slot).  Ids outside their
// range are dropped: counted nowhere, inv = -1.
int dispatch_ext(const int32_t* inds, int rows, int k_routed, int kk, int n_ids, int32_t* order,
                 int32_t* counts, int32_t* offsets, int32_t* inv, int32_t* active,
                 int32_t* n_active, int tile_m, int4* tiles, int32_t* n_tiles,
                 const int32_t* table, int shared_slot, void* ws, size_t ws_bytes,
                 hipStream_t st) {
  PMOE_REQUIRE(n_ids > 0 && n_ids <= kMaxExperts, "dispatch: experts must be 1..1024");
  PMOE_REQUIRE(rows >= 0, "dispatch: negative rows");
  PMOE_REQUIRE(k_routed >= 1 && kk >= k_routed && kk <= k_routed + 1, "dispatch: bad columns");
  PMOE_REQUIRE(rows % kk == 0, "dispatch: rows must be a multiple of the columns");
  const IdSrc src{inds, k_routed, kk, kk > k_routed ? n_ids - 1 : n_ids};
  PMOE_REQUIRE(tile_m == 0 || (tiles && n_tiles && table), "dispatch: tile list needs the slot table");
  const TileSink ts{tiles, n_tiles, tile_m, table, src.n_routed, shared_slot};
  ProfScope prof_scope(K_DISPATCH, st);
  if (rows <= kSmallRows) {
    dispatch_small_kernel<<<1, 1024, 0, st>>>(src, rows, n_ids, order, counts, offsets, inv,
                                              active, n_active, ts);
    PMOE_LAUNCH_CHECK("dispatch_small_kernel");
    return PMOE_OK;
  }
  PMOE_REQUIRE(ws != nullptr && ws_bytes >= dispatch_workspace(rows, n_ids),
               "dispatch: workspace too small");
  const int blocks = (rows + kChunk - 1) / kChunk;
  int32_t* hist = static_cast<int32_t*>(ws);
  int32_t* rank = hist + size_t(blocks) * n_ids;
  if (int rc = dispatch_count(src, rows, n_ids, hist, rank, st)) return rc;
  dispatch_scan_kernel<<<1, 1024, 0, st>>>(hist, blocks, n_ids, counts, offsets, active,
                                           n_active, ts);
  PMOE_LAUNCH_CHECK("dispatch_scan_kernel");
  return dispatch_scatter(src, rows, n_ids, hist, rank, order, inv, st);
}

}  // namespace pmoe

extern "C" size_t pmoe_dispatch_workspace(int rows, int n_experts) {
  return pmoe::dispatch_workspace(rows, n_experts);
}

extern "C" int pmoe_dispatch(const int32_t* inds, int rows, int n_experts, int32_t* order,
                             int32_t* counts, int32_t* offsets, int32_t* inv, int32_t* active,
                             int32_t* n_active, void* ws, size_t ws_bytes, void* stream) {
  pmoe::clear_error();
  return pmoe::dispatch_ext(inds, rows, 1, 1, n_experts, order, counts, offsets, inv, active,
                            n_active, 0, nullptr, nullptr, nullptr, -1, ws, ws_bytes,
                            static_cast<hipStream_t>(stream));
}
