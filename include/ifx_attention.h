/*
 * ifx_attention.h -- C ABI of the MI355X (gfx950) attention of a serving
 * step: what lies between a layer's Q/K/V projections and its O projection
 * (ifx_qgemm.h).  Conventions are those of ifx_qgemm.h: plain pointers and
 * sizes, caller-owned device memory, every call enqueued on the caller's HIP
 * stream, no allocation and no host synchronisation.  Status codes: 0 =
 * launched; > 0 = not handled (ifx_status of ifx_qgemm.h); < 0 = -hipError_t.
 * All device buffers of a call are on the current device, and `stream` is one
 * of its streams.  Calls may be captured into HIP graphs.
 *
 * The paged cache.  A cache of one layer is num_pages pages of page_size
 * tokens (16, 32, 64, 128 or 256), 16-bit (fp16 or bf16), in the order in
 * which the MFMA instructions take their operands, so that a lane reads 16
 * contiguous bytes and half a wave half a kilobyte (of K at pages of 16 tokens
 * two pages' 256 bytes):
 *   K  [page][kv head][D / 8][token in page][8]
 *   V  [page][kv head][token in page / 8][D][8]
 * Token i of a request lives in slot page * page_size + i % page_size, where
 * page = block_table[request][i / page_size].
 */
#ifndef IFX_ATTENTION_H
#define IFX_ATTENTION_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of rows and caches (the values of ifx_out_dtype and
 * IFX_IN_BF16 in ifx_qgemm.h). */
enum ifx_attn_dtype { IFX_ATTN_F32 = 0, IFX_ATTN_F16 = 1, IFX_ATTN_BF16 = 2 };

/* Bits of ifx_plan_batch's status word. */
enum ifx_plan_status {
  IFX_PLAN_NO_PAGES = 1,    /* the new tokens need more pages than are free       */
  IFX_PLAN_NARROW = 2,      /* a request needs more pages than the table is wide  */
  IFX_PLAN_NO_ROOM = 4,     /* more new tokens than max_tokens                    */
  IFX_PLAN_BAD_LENGTH = 8   /* a negative length, or one past 2^31 - 1            */
};

/* Largest batch of ifx_plan_batch and of the attention entries. */
#define IFX_ATTN_MAX_BATCH 4096

/* Plans one step of B requests on the device: request b has ctx_len[b] tokens
 * in the cache and brings new_len[b] >= 0 more.  Its table row holds the
 * ceil(ctx_len / page_size) pages it has; the pages that its new tokens need
 * besides are taken from the end of free_pages[0 .. free_count[0]), request
 * by request, and written into its row.  Outputs, all int32:
 *   cu_q [B + 1]   first row of each request among the new tokens
 *   kv_len [B]     ctx_len + new_len
 *   positions, slots [max_tokens]  per new token, request by request; rows
 *                  behind the last token get position 0 and slot -1, so that
 *                  a captured step of max_tokens rows can be replayed
 *   free_left [1]  free_count less the pages taken
 *   status [1]     0, or bits of ifx_plan_status: then nothing is taken, the
 *                  table is as it was, kv_len = ctx_len, cu_q is all 0 and
 *                  every slot -1
 * Outputs must not overlap inputs (block_table apart, which is updated in
 * place).  Calling again with the same inputs gives the same results.
 * 1 <= B <= IFX_ATTN_MAX_BATCH, 1 <= table_width, 0 <= max_tokens <= 2^30. */
int ifx_plan_batch(const int32_t *ctx_len, const int32_t *new_len, int32_t *block_table,
                   int table_width, const int32_t *free_pages, int free_capacity,
                   const int32_t *free_count, int page_size, int B, int max_tokens, int32_t *cu_q,
                   int32_t *kv_len, int32_t *positions, int32_t *slots, int32_t *free_left,
                   int32_t *status, void *stream);

/* Rotates the new tokens' Q and K by their positions and writes K and V into
 * the paged cache.  q [T][Hq][D], k and v [T][Hkv][D] as the projections
 * wrote them (src_dtype), rows q_stride / k_stride / v_stride elements apart,
 * heads D apart.  Each of the first rot_dim values of a head is rotated with
 * its partner: (i, i + rot_dim / 2), or (2i, 2i + 1) where interleaved, by the
 * angle positions[t] * inv_freq[i], which is formed and reduced in 64 bits
 * (inv_freq: fp64 [rot_dim / 2] on the device; rot_dim = 0: no rotation).
 * Computed in fp32 and rounded once to cache_dtype (fp16 or bf16).  q_out
 * [T][Hq][D] rows q_out_stride elements apart.  A token whose slot is outside
 * [0, num_pages * page_size) is left out: nothing of it is written, q_out's
 * row neither.  Slots of one call must differ.  D: a multiple of 8 up to 256;
 * rot_dim a multiple of 16 up to D; num_pages * page_size < 2^31; T up to
 * 2^27 - 8, as many as a launch has workgroups for. */
int ifx_rope_append(const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                    const void *v, int64_t v_stride, int src_dtype, const int32_t *positions,
                    const int32_t *slots, const double *inv_freq, int rot_dim, int interleaved,
                    int T, int Hq, int Hkv, int D, void *q_out, int64_t q_out_stride,
                    void *k_cache, void *v_cache, int cache_dtype, int64_t num_pages,
                    int page_size, void *stream);

/* Attention of the new tokens over the paged cache, which holds them already.
 * Row t of q [T][Hq][D] (dtype as the cache; rows q_stride elements apart)
 * belongs to request b with cu_q[b] <= t < cu_q[b + 1]; as the i-th of its n
 * rows it stands at position p = kv_len[b] - n + i and sees the keys
 *   j <= p, and j > p - window where window > 0,
 * so out = sum_j softmax_j(scale q . k_j) v_j, query head h reading key/value
 * head h / (Hq / Hkv).  A row that sees nothing (kv_len[b] < n) is 0.  What a
 * row does not see has no influence on it, infinities and NaN included.  Rows
 * from cu_q[B] on are left as they were.  Scores, their maximum and their sum
 * are fp32; the probabilities are rounded to the cache's type for the product
 * with V; the result is rounded once to out_dtype (fp32, fp16 or bf16; rows
 * out_stride elements apart, which must not overlap the keys and values).
 *
 * max_q and max_kv bound the requests' new rows and kv_len, and plan the
 * launch: which kernel takes it, how many workgroups there are and what
 * workspace they need.  Of a request with more than max_q rows only the first
 * max_q are sure to be computed; one with more than max_kv keys is computed
 * whole, if not as fast.  Lengths outside [0, table_width * page_size] and page
 * numbers outside [0, num_pages) are clamped, so that no memory outside the
 * cache is touched.
 *
 * workspace: ifx_attn_paged_workspace_bytes bytes (at most
 * IFX_ATTN_WORKSPACE_BYTES for any shape), 256-byte aligned, zeroed once
 * before its first use; every call leaves it ready for the next one.  Split
 * sums are added in order: the same bits on every call.  Calls that share a
 * workspace must not overlap.  May be NULL with 0 bytes where none is needed.
 *
 * D: 64, 96, 128 or 256.  Hq a multiple of Hkv, Hkv * D < 2^22.  scale > 0,
 * and scale log2 e finite.
 * table_width * page_size <= 2^30. */
#define IFX_ATTN_WORKSPACE_BYTES (64 << 20)
int64_t ifx_attn_paged_workspace_bytes(int B, int T, int Hq, int Hkv, int D, int max_q,
                                       int max_kv);
int ifx_attn_paged(const void *q, int64_t q_stride, int dtype, const void *k_cache,
                   const void *v_cache, int64_t num_pages, int page_size,
                   const int32_t *block_table, int table_width, const int32_t *cu_q,
                   const int32_t *kv_len, int B, int T, int Hq, int Hkv, int D, int max_q,
                   int max_kv, float scale, int window, void *out, int64_t out_stride,
                   int out_dtype, void *workspace, int64_t workspace_bytes, void *stream);

/* Attention over B whole prompts packed one after the other, without a cache:
 * q [T][Hq][D], k and v [T][Hkv][D], rows cu_len[b] .. cu_len[b + 1] - 1 are
 * prompt b.  Row i of a prompt of n sees its rows j < n, and j <= i where
 * causal, and j > i - window where causal and window > 0.  Otherwise as
 * ifx_attn_paged; k_stride, v_stride < 2^23.  max_len > 0 is a bound of the
 * prompts' lengths; it is checked to be positive and plans nothing: prompts of
 * any length up to T are computed whole. */
int ifx_attn_prompt(const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                    const void *v, int64_t v_stride, int dtype, const int32_t *cu_len, int B,
                    int T, int Hq, int Hkv, int D, int max_len, int causal, int window,
                    float scale, void *out, int64_t out_stride, int out_dtype, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* IFX_ATTENTION_H */
