// Launchers of the paged-cache operators (C++ linkage, library-private). The C
// ABI in paged.cpp validates arguments; these configure and launch.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mlq.h"

namespace mlq {

// paged_ops.hip
struct PlanArgs {
  int n_seqs, max_pages, max_rows, page_shift, n_pages;
  const int32_t* lengths;
  const int32_t* n_new;
  const int32_t* n_free;
  int32_t* free_pages;
  int32_t* n_free_out;
  int32_t* block_table;
  int32_t* lengths_out;
  int32_t* row_start;
  int32_t* positions;
  int64_t* slots;
  int32_t* status;
};
hipError_t launch_paged_plan(const PlanArgs& a, hipStream_t stream);

struct RotaryArgs {
  int rows, n_heads, n_kv, hd, rot, neox;
  float magnitude, eps;
  const double* freqs;
  const float* q_norm;
  const float* k_norm;
  const int32_t* positions;
  const float* q;
  const float* k;
  const float* v;
  float* q_out;
  float* k_out;  // may be null
  int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
  void* keys;    // of the layer; null: no cache
  void* values;
  int type, page_shift;
  int64_t n_slots;
  const int64_t* slots;
  int stream;    // set by the launcher: q_out written past the caches
};
hipError_t launch_qk_norm_rope(const RotaryArgs& a, hipStream_t stream);

// paged_attention.hip
struct PagedAttnArgs {
  const void* keys;    // of the layer
  const void* values;
  int type, n_pages, page_shift, n_kv, hd, group;
  int n_seqs, max_pages, max_rows, max_len;
  const int32_t* block_table;
  const int32_t* lengths;
  const int32_t* row_start;
  const float* q;
  float* out;
  int64_t q_stride, out_stride;
  float scale, softcap;
  int window;
  const float* slopes;
  // decode: launches of launch_seqs sequences, at most `ranges` workgroups;
  // `part`: the workspace, null when every sequence is one piece, of `whole`
  // key tiles
  int launch_seqs, ranges, whole;
  // prefill: workgroups that share a tile's keys
  int splits;
  void* part;
};
// Sets launch_seqs and ranges for lengths up to a.max_len; the workspace.
size_t plan_paged_decode(PagedAttnArgs& a);
hipError_t launch_paged_decode(const PagedAttnArgs& a, hipStream_t stream);
// Workgroups of a launch, without the splits'.
int64_t prefill_groups(const PagedAttnArgs& a);
// Sets splits for a.max_rows rows and lengths up to a.max_len; the workspace.
size_t plan_paged_prefill(PagedAttnArgs& a);
hipError_t launch_paged_prefill(const PagedAttnArgs& a, hipStream_t stream);

}  // namespace mlq
