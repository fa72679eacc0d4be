// ifx_drafts_impl.h -- what the kernels of drafted tokens (draft_plan.hip,
// verify_drafts.hip, keep_path.hip) and their entry points (drafts_api.hip)
// share.
#pragma once

#include "ifx_attn.h"
#include "ifx_drafts.h"
#include "ifx_qgemm.h"

namespace ifx {

constexpr int kMaxNodes = IFX_TREE_MAX_NODES;  // a wave's lanes
// The workspace of the attention entries: counters first, at one place for all
// calls, as only they have to be zero between calls.
constexpr int kSplitUnits = 8192;
constexpr int64_t kSplitCntBytes = kSplitUnits * 4;

struct TreeArgs {
  const int32_t *parents, *cu, *kv_len;
  int32_t *positions;
  uint64_t *masks;
  int B, T;
};
hipError_t launch_plan_tree(const TreeArgs &a, hipStream_t s);

struct KeptArgs {
  const int32_t *cu, *kv_len, *accepted, *table;
  int32_t *free_pages;
  const int32_t *free_count;
  int32_t *ctx_len, *free_left, *status;
  int table_width, free_capacity, page_shift, B;
};
hipError_t launch_plan_kept(const KeptArgs &a, hipStream_t s);

struct VerifyArgs {
  const int32_t *tokens, *parents, *cu;
  const void *target, *drafter;
  int64_t target_stride, drafter_stride;  // elements
  const float *accept_u, *sample_u;
  int32_t *accepted, *path, *emitted;
  uint32_t *cnt;
  double *part;  // [request][chunk]{sum of the weights, of the target's row}
  int B, T, V, max_q, chunks, chunk;  // chunk: values of one
};
hipError_t launch_verify(const VerifyArgs &a, int prob_dtype, hipStream_t s);
void verify_split(int B, int V, int *chunks, int *chunk);

struct KeepArgs {
  void *k, *v, *scales;
  const int32_t *table, *cu, *kv_len, *path, *accepted;
  int64_t num_pages;
  int page_shift, Hkv, D, table_width, B, T, max_q;
};
hipError_t launch_keep_path(const KeepArgs &a, int elem_bytes, hipStream_t s);

// Of the entry points: what a launch's result is to the caller, and log2 of a page
// size that the cache can have, else -1.
inline int status_of(hipError_t e) { return e == hipSuccess ? IFX_OK : -static_cast<int>(e); }
inline int page_shift_of(int page_size) {
  for (int sh = 4; sh <= 8; ++sh)
    if (page_size == 1 << sh) return sh;
  return -1;
}

}  // namespace ifx
