// Launch interface of the microscaled 4-bit experts (mx_experts.hip).
#pragma once

#include "pmoe_internal.h"

namespace pmoe {

// Whether a geometry's experts are microscaled 4-bit (include/pmoe.h).
inline bool is_mx(const pmoe_geom* g) { return g->group == 32; }

// One grouped product over an expert's rows: features [features, cols] of the
// slot times activation pieces.
struct MxArgs {
  const uint8_t* slab;
  int64_t expert_bytes;
  int64_t w0, s0, w1, s1;  // component offsets; 1: the up projection
  const int4* tiles;       // {slot, first row, rows, offset}
  const int32_t* n_tiles;
  const int32_t* order;    // sorted position -> flat row
  int kk, features, cols;
  const uint8_t* pair;     // rows of pieces (mx_pieces.h)
  const uint8_t* third;
  const uint8_t* ascale;   // their scales
  const uint16_t* asteps;  // [rows, 4]: bit s: step s of 128 has a third piece
  uint8_t* hpair;          // gate/up out, by sorted row
  uint8_t* hscale;
  uint16_t* y;             // down out: [flat row, features], bf16 or fp16 under yscale
  uint8_t* yscale;         // [flat row, features / 32]
  bool past_caches;        // y's stores
};

struct MxPlan {
  const pmoe_geom* geom;
  const uint8_t* slab;
  const int32_t* table;
  int n_experts, shared_slot;
  const uint16_t* x;   // bf16 [n, hidden]
  const int32_t* ids;  // [n, k]
  int n, k, kk;
  const uint16_t* shared_gate;  // or null; shared_logit[n] receives x . shared_gate
  float* shared_logit;
  // scratch: the dispatch's (pmoe_kernels.h) ...
  int32_t *order, *counts, *offsets, *inv, *active, *n_active;
  int tile_rows;  // of the tile list
  int4* tiles;
  int32_t* n_tiles;
  int max_tiles;
  void* dws;
  size_t dws_bytes;
  // ... the tokens' pieces, the sorted rows' intermediate
  uint8_t *xpair, *xthird, *xscale;
  uint16_t* xsteps;  // [n, 4]
  uint8_t *hpair, *hscale;
  // [n * kk, hidden]: fp16 under yscale, for mx_combine, or (yscale null) the seam's
  // bf16 rows, those of dropped ids zero
  uint16_t* y;
  uint8_t* yscale;  // [n * kk, hidden / 32]
};

// Rows of the dispatch's tiles for such a call, and the fewest that any has.
int mx_tile_rows(const pmoe_geom* g, int n, int kk, int n_experts);
int mx_min_tile_rows();
// Dispatch, split, gate/up, down; rows whose expert is not resident come out zero.
int mx_experts(const MxPlan& p, hipStream_t st);
// Tokens one by one in two launches, without a dispatch: out bf16 [n, hidden]
// combined (wts given) or [n, k, hidden].  slots [n, k + 1], h fp32 [n, k + 1, inter]:
// scratch.  mx_one_tokens: how many of n tokens may go this way (all of them or none do;
// the scratch serves shorter calls too).
int mx_one_tokens(const pmoe_geom* g, int n, int k, int shared, int n_experts, bool combined);
bool mx_one_wanted(const pmoe_geom* g, int n, int k, int shared, int n_experts, bool combined);
int mx_one(const pmoe_geom* g, const uint8_t* slab, const int32_t* table, int n_experts,
           const uint16_t* x, const int32_t* ids, const float* wts, int n, int k, int shared_slot,
           const uint16_t* shared_gate, float* shared_logit, int32_t* slots, float* h,
           uint16_t* out, hipStream_t st);
// out[n] = sum over columns in order of weight * y (+ the shared column's).
int mx_combine(const uint16_t* y, const uint8_t* yscale, const float* w, const int32_t* inv,
               const float* shared_logit, int n, int k, int kk, int d, uint16_t* out,
               hipStream_t st);

}  // namespace pmoe
