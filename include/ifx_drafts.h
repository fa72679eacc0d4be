/*
 * ifx_drafts.h -- C ABI of what a serving step does with drafted tokens on
 * MI355X (gfx950): positions and masks of trees of drafts, the attention of
 * their nodes over the paged cache, which drafts the target's probabilities
 * accept, and what the batch keeps of them.  Conventions are those of
 * ifx_attention.h, whose paged cache, plan and workspace these entries share.
 *
 * A request brings the nodes of one tree as its new tokens, at most
 * IFX_TREE_MAX_NODES: row i of it is node i, and parents[i] is the node before
 * it, one of its earlier rows (any other number: none).  Node 0 is the root,
 * the last token that was accepted or sampled, which the cache does not hold
 * yet; a request that only decodes is a tree of its root.  The nodes' K and V
 * are written to the slots that ifx_plan_batch gives them (token ctx + i for
 * node i), rotated by the positions that ifx_plan_tree gives them.
 */
#ifndef IFX_DRAFTS_H
#define IFX_DRAFTS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define IFX_TREE_MAX_NODES 64

/* Bits of ifx_plan_kept's status word. */
enum ifx_kept_status {
  IFX_KEPT_NO_SPACE = 1  /* the pages given back do not fit free_pages */
};

/* Positions and masks of the nodes of B trees, rows as cu_q [B + 1] has them:
 *   positions [T]  kv_len - n + depth of the node (n: the request's rows; the
 *                  root's depth is 0, as that of every node without a parent)
 *   masks [T]      bit j: node j is the node itself or on its way to the root
 * Rows past a request's first IFX_TREE_MAX_NODES and rows from cu_q[B] on get
 * position 0 and an empty mask.  1 <= B <= IFX_ATTN_MAX_BATCH, T < 2^30. */
int ifx_plan_tree(const int32_t *parents, const int32_t *cu_q, const int32_t *kv_len, int B, int T,
                  int32_t *positions, uint64_t *masks, void *stream);

/* Attention of the nodes over the paged cache, which holds them already: as
 * ifx_attn_paged without a window, but that row i of a request of n sees the
 * keys before its n new ones, and of these token kv_len - n + j where bit j of
 * masks[row] is set (j < n; the node itself too only where its bit is).
 * 1 <= max_q <= IFX_TREE_MAX_NODES.  workspace: as ifx_attn_paged's, of
 * ifx_attn_tree_workspace_bytes; one may serve both. */
int64_t ifx_attn_tree_workspace_bytes(int B, int T, int Hq, int Hkv, int D, int max_q,
                                      int max_kv);
int ifx_attn_tree(const void *q, int64_t q_stride, int dtype, const void *k_cache,
                  const void *v_cache, int64_t num_pages, int page_size,
                  const int32_t *block_table, int table_width, const int32_t *cu_q,
                  const int32_t *kv_len, const uint64_t *masks, int B, int T, int Hq, int Hkv,
                  int D, int max_q, int max_kv, float scale, void *out, int64_t out_stride,
                  int out_dtype, void *workspace, int64_t workspace_bytes, void *stream);

/* Which drafted nodes the target's probabilities accept, and the token behind
 * them.  tokens [T]: the nodes' tokens.  Row t of target [T][V] (type
 * prob_dtype, rows target_stride elements apart) holds the target's
 * probabilities of what follows node t.  Negative and NaN ones count as 0.
 *
 * drafter NULL: the drafts are the drafter's choices.  From node i, with
 * u = accept_u[row of i], the walk goes on to its first child c with
 * u < p_i(token of c) + those of the children before c, and stops if there is
 * none.  A child whose token an earlier one has, or one outside [0, V), is
 * never gone to.  The next token is drawn from p_i without the children's
 * tokens.  parents NULL: a chain, node i + 1 the child of node i.
 *
 * drafter [T][V] (same type): the drafts are a chain and were drawn from it,
 * node i + 1 from row i; parents must be NULL.  The walk goes on where
 * u drafter_i(x) < p_i(x), x the token of node i + 1.  The next token is drawn
 * from max(p_i - drafter_i, 0), behind the last node from its p_i.
 *
 * Drawn: the smallest v with w_0 + ... + w_v > sample_u[b] sum(w), in 64 bits;
 * from p_i whole where no weight is left, and -1 if p_i is all 0 too.
 *
 * Outputs, all int32, of request b with rows cu_q[b] .. cu_q[b + 1] - 1:
 *   accepted [B]  accepted drafts, -1 of a request without rows
 *   path [T]      the nodes walked, the root first; then -1
 *   emitted [T]   the tokens of the accepted drafts and the one drawn; then -1
 * Rows from cu_q[B] on are left as they were.  Nodes past the first max_q of a
 * request (1 <= max_q <= IFX_TREE_MAX_NODES) are not considered.
 *
 * workspace: ifx_verify_workspace_bytes bytes (at most IFX_ATTN_WORKSPACE_BYTES),
 * kept as that of ifx_attn_paged, which serves here too.  1 <= V <= 2^30. */
int64_t ifx_verify_workspace_bytes(int B, int V);
int ifx_verify(const int32_t *tokens, const int32_t *parents, const int32_t *cu_q, int B, int T,
               int max_q, const void *target, int64_t target_stride, const void *drafter,
               int64_t drafter_stride, int prob_dtype, int V, const float *accept_u,
               const float *sample_u, int32_t *accepted, int32_t *path, int32_t *emitted,
               void *workspace, int64_t workspace_bytes, void *stream);

/* Moves the K and V of the nodes that a request keeps behind the tokens that
 * were in the cache: token kv_len - n + i takes those of node path[i], for
 * 0 < i <= accepted[b].  Caches of elem_bytes 2 (ifx_attention.h; scales NULL)
 * or 1 (ifx_attention_q8.h).  path increases, as ifx_verify's does; what it
 * does not keep stays as it is.  accepted is held to [0, max_q - 1]. */
int ifx_keep_path(void *k_cache, void *v_cache, void *scales, int elem_bytes, int64_t num_pages,
                  int page_size, int Hkv, int D, const int32_t *block_table, int table_width,
                  const int32_t *cu_q, const int32_t *kv_len, const int32_t *path,
                  const int32_t *accepted, int B, int T, int max_q, void *stream);

/* What a batch keeps of a step's new tokens, on the device: request b goes on
 * with ctx_len[b] = kv_len - n + accepted + 1 tokens (kv_len where n is 0;
 * accepted held to [-1, n - 1]).  Pages of its table row that hold none of them
 * are given back, put behind free_pages[0 .. free_count[0]) so that
 * ifx_plan_batch, which takes them from the end, takes them in the order in
 * which it gave them out; their entries stay.  free_left [1]: pages free then.
 * status [1]: 0 or bits of ifx_kept_status; then no page is given back.
 * Outputs must not overlap inputs (free_pages apart). */
int ifx_plan_kept(const int32_t *cu_q, const int32_t *kv_len, const int32_t *accepted,
                  const int32_t *block_table, int table_width, int32_t *free_pages,
                  int free_capacity, const int32_t *free_count, int page_size, int B,
                  int32_t *ctx_len, int32_t *free_left, int32_t *status, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* IFX_DRAFTS_H */
