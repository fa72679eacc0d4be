// drafts_api.hip -- the C entry points of include/ifx_drafts.h but the
// attention's (attention_api.hip): validation and the launches.
#include <climits>

#include "ifx_drafts_impl.h"
#include "ifx_qgemm.h"

namespace {

using namespace ifx;

bool batch_ok(int B, int T) { return B >= 1 && B <= IFX_ATTN_MAX_BATCH && T >= 0 && T < (1 << 30); }
bool nodes_ok(int max_q) { return max_q >= 1 && max_q <= IFX_TREE_MAX_NODES; }

// Whether an output is in the place of an input or another output.
bool overlap(std::initializer_list<const void *> out, std::initializer_list<const void *> in) {
  for (auto o = out.begin(); o != out.end(); ++o) {
    for (const void *i : in)
      if (*o == i) return true;
    for (auto p = out.begin(); p != o; ++p)
      if (*o == *p) return true;
  }
  return false;
}

}  // namespace

extern "C" {

int ifx_plan_tree(const int32_t *parents, const int32_t *cu_q, const int32_t *kv_len, int B, int T,
                  int32_t *positions, uint64_t *masks, void *stream) {
  if (!batch_ok(B, T)) return IFX_BAD_GEOMETRY;
  if (T == 0) return IFX_OK;
  if (!parents || !cu_q || !kv_len || !positions || !masks) return IFX_NULL_POINTER;
  if (overlap({positions, masks}, {parents, cu_q, kv_len})) return IFX_BAD_GEOMETRY;
  const TreeArgs a{parents, cu_q, kv_len, positions, masks, B, T};
  return status_of(launch_plan_tree(a, static_cast<hipStream_t>(stream)));
}

int64_t ifx_verify_workspace_bytes(int B, int V) {
  if (!batch_ok(B, 0) || V < 1 || V > (1 << 30)) return 0;
  int chunks, chunk;
  verify_split(B, V, &chunks, &chunk);
  return kSplitCntBytes + static_cast<int64_t>(B) * chunks * 16;
}

int ifx_verify(const int32_t *tokens, const int32_t *parents, const int32_t *cu_q, int B, int T,
               int max_q, const void *target, int64_t target_stride, const void *drafter,
               int64_t drafter_stride, int prob_dtype, int V, const float *accept_u,
               const float *sample_u, int32_t *accepted, int32_t *path, int32_t *emitted,
               void *workspace, int64_t workspace_bytes, void *stream) {
  if (prob_dtype != IFX_ATTN_F32 && prob_dtype != IFX_ATTN_F16 && prob_dtype != IFX_ATTN_BF16)
    return IFX_UNSUPPORTED_TYPE;
  if (!batch_ok(B, T) || !nodes_ok(max_q) || V < 1 || V > (1 << 30) || target_stride < V ||
      (drafter && (drafter_stride < V || parents)))
    return IFX_BAD_GEOMETRY;
  if (!cu_q || !sample_u || !accepted || !workspace ||
      (T && (!tokens || !target || !accept_u || !path || !emitted)))
    return IFX_NULL_POINTER;
  if (overlap({accepted}, {tokens, parents, cu_q, accept_u, sample_u}) ||
      (T && overlap({accepted, path, emitted}, {tokens, parents, cu_q, accept_u, sample_u})))
    return IFX_BAD_GEOMETRY;
  if (workspace_bytes < ifx_verify_workspace_bytes(B, V) ||
      (reinterpret_cast<uintptr_t>(workspace) & 255))
    return IFX_BAD_GEOMETRY;
  VerifyArgs a{};
  a.tokens = tokens, a.parents = parents, a.cu = cu_q;
  a.target = target, a.drafter = drafter;
  a.target_stride = target_stride, a.drafter_stride = drafter_stride;
  a.accept_u = accept_u, a.sample_u = sample_u;
  a.accepted = accepted, a.path = path, a.emitted = emitted;
  a.cnt = static_cast<uint32_t *>(workspace);
  a.part = reinterpret_cast<double *>(static_cast<char *>(workspace) + kSplitCntBytes);
  a.B = B, a.T = T, a.V = V, a.max_q = max_q;
  verify_split(B, V, &a.chunks, &a.chunk);
  return status_of(launch_verify(a, prob_dtype, static_cast<hipStream_t>(stream)));
}

int ifx_keep_path(void *k_cache, void *v_cache, void *scales, int elem_bytes, int64_t num_pages,
                  int page_size, int Hkv, int D, const int32_t *block_table, int table_width,
                  const int32_t *cu_q, const int32_t *kv_len, const int32_t *path,
                  const int32_t *accepted, int B, int T, int max_q, void *stream) {
  if (elem_bytes != 1 && elem_bytes != 2) return IFX_UNSUPPORTED_TYPE;
  const int sh = page_shift_of(page_size);
  if (sh < 0 || num_pages < 1 || num_pages > (INT_MAX >> sh) || table_width < 1 ||
      table_width > ((1 << 30) >> sh))
    return IFX_BAD_GEOMETRY;
  if (!batch_ok(B, T) || !nodes_ok(max_q) || Hkv < 1 || Hkv > 65536 || D < 8 || D > 256 ||
      D % (16 / elem_bytes))
    return IFX_BAD_GEOMETRY;
  if (T == 0) return IFX_OK;
  if (!k_cache || !v_cache || (elem_bytes == 1 && !scales) || !block_table || !cu_q || !kv_len ||
      !path || !accepted)
    return IFX_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
       reinterpret_cast<uintptr_t>(scales)) & 15)
    return IFX_BAD_GEOMETRY;
  const KeepArgs a{k_cache, v_cache, scales, block_table, cu_q, kv_len, path, accepted,
                   num_pages, sh, Hkv, D, table_width, B, T, max_q};
  return status_of(launch_keep_path(a, elem_bytes, static_cast<hipStream_t>(stream)));
}

int ifx_plan_kept(const int32_t *cu_q, const int32_t *kv_len, const int32_t *accepted,
                  const int32_t *block_table, int table_width, int32_t *free_pages,
                  int free_capacity, const int32_t *free_count, int page_size, int B,
                  int32_t *ctx_len, int32_t *free_left, int32_t *status, void *stream) {
  const int sh = page_shift_of(page_size);
  if (sh < 0 || !batch_ok(B, 0) || table_width < 1 || table_width > ((1 << 30) >> sh) ||
      free_capacity < 0)
    return IFX_BAD_GEOMETRY;
  if (!cu_q || !kv_len || !accepted || !block_table || !free_count || !ctx_len || !free_left ||
      !status || (free_capacity && !free_pages))
    return IFX_NULL_POINTER;
  if (overlap({ctx_len, free_left, status}, {cu_q, kv_len, accepted, block_table, free_count, free_pages}))
    return IFX_BAD_GEOMETRY;
  const KeptArgs a{cu_q, kv_len, accepted, block_table, free_pages, free_count, ctx_len, free_left,
                   status, table_width, free_capacity, sh, B};
  return status_of(launch_plan_kept(a, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
