/*
 * ifx_attention_q8.h -- C ABI of the 8-bit paged cache on MI355X (gfx950):
 * quantising K and V as they are written, the attention over them, and reading
 * them back.  Conventions are those of ifx_attention.h, whose plans, tables,
 * slots and workspace these entries share.
 *
 * The cache.  Of every token and key/value head K and V are each D codes, int8
 * from -127 to 127, and a bf16 scale: a value is code * scale.  num_pages pages
 * of page_size tokens (16, 32, 64, 128 or 256), in the order in which the
 * attention's lanes take their operands:
 *   K       [page][kv head][D / 16][token in page][16]
 *   V       [page][kv head][token in page / 16][D][16]
 *   scales  [page][kv head][token in page][2]   bf16: K's, V's
 * 2 D + 4 bytes a token and head, where the 16-bit cache takes 4 D.
 */
#ifndef IFX_ATTENTION_Q8_H
#define IFX_ATTENTION_Q8_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* As ifx_rope_append, into the 8-bit cache.  Q is rotated in fp32 and rounded
 * once to q_dtype (fp16 or bf16).  K is rotated in fp64; of the rotated K and of
 * V, for each token and head, the scale is the smallest bf16 that is no less
 * than max |x| / 127, and a code is x / scale rounded to nearest, ties to even:
 * a value is off by at most half a scale.  A head's row of zeros has scale 0;
 * one that holds an infinity or NaN, or a rotated K past fp32's range, has scale
 * NaN and codes 0, so that all of it reads back as NaN.  Slots within the cache
 * must differ: what two tokens write to one is codes and scales of either.
 * D: a multiple of 32 up to 256; scales 16-byte aligned. */
int ifx_rope_append_q8(const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                       const void *v, int64_t v_stride, int src_dtype, const int32_t *positions,
                       const int32_t *slots, const double *inv_freq, int rot_dim, int interleaved,
                       int T, int Hq, int Hkv, int D, void *q_out, int64_t q_out_stride,
                       int q_dtype, void *k_cache, void *v_cache, void *scales, int64_t num_pages,
                       int page_size, void *stream);

/* Reads tokens back: row i of k_out and v_out [N][Hkv][D] (rows k_stride and
 * v_stride elements apart) is what slot slots[i] holds, code * scale rounded
 * once to out_dtype (fp32, fp16 or bf16); 0 for a slot outside the cache.  D: a
 * multiple of 32 up to 256; N < 2^27. */
int ifx_read_rows_q8(const void *k_cache, const void *v_cache, const void *scales,
                     int64_t num_pages, int page_size, const int32_t *slots, int N, int Hkv, int D,
                     void *k_out, int64_t k_stride, void *v_out, int64_t v_stride, int out_dtype,
                     void *stream);

/* Attention of the new tokens over the 8-bit cache: as ifx_attn_paged on the
 * values that the cache stands for, q of q_dtype (fp16 or bf16).  With masks
 * [T], those of ifx_plan_tree (ifx_drafts.h), as ifx_attn_tree instead; window
 * must be 0 and max_q at most IFX_TREE_MAX_NODES then.  workspace: as
 * ifx_attn_paged's, of ifx_attn_paged_q8_workspace_bytes; one may serve both.
 *
 * Codes are exact in the products, which are summed in fp32.  Q of bf16 is
 * taken to fp16 with a power of two for each row, which loses nothing of what is
 * at least 2^-28 of the row's largest value, if that is 2^-63 or more.
 * Probabilities times V's scales are rounded to fp16, relative to the largest
 * scale among the keys that the row has met: what weighs 2^-20 of that and less
 * loses bits.  Scales of V count as 2^-80 at least in this; where they pass 2^108,
 * keys whose weight is less than 2^-132 of them count as nothing. */
int64_t ifx_attn_paged_q8_workspace_bytes(int B, int T, int Hq, int Hkv, int D, int max_q,
                                          int max_kv);
int ifx_attn_paged_q8(const void *q, int64_t q_stride, int q_dtype, const void *k_cache,
                      const void *v_cache, const void *scales, int64_t num_pages, int page_size,
                      const int32_t *block_table, int table_width, const int32_t *cu_q,
                      const int32_t *kv_len, const uint64_t *masks, int B, int T, int Hq, int Hkv,
                      int D, int max_q, int max_kv, float scale, int window, void *out,
                      int64_t out_stride, int out_dtype, void *workspace, int64_t workspace_bytes,
                      void *stream);

#ifdef __cplusplus
}
#endif

#endif /* IFX_ATTENTION_Q8_H */
