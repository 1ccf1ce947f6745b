/*
 * cie_kv_q8.h -- a KV pool held in 8 bits: pages quantised as they are written,
 * read back, and attended to by decode rows. In libcie_attention.so; same
 * conventions and status codes as cie_attention.h (device pointers, element
 * strides, asynchronous on `stream`, no allocation, no host synchronisation,
 * graph-capturable). No counterpart in the reference, whose KVStorage
 * (kv_cache/storage.py:32-48) holds fp16 pages; these take half the bytes.
 *
 * Layouts:
 *   k / v pool  (n_pages, num_kv_heads, page_size, head_dim) int8 codes, row
 *               stride head_dim, unit inner stride, 16-byte aligned, strides
 *               multiples of 16
 *   kv_scales   (n_pages, 2, num_kv_heads) fp32, contiguous: the scale of a
 *               page's K (index 0) and V (index 1) rows per kv head; a value is
 *               code * scale
 *   block_table, lens, slot_ids, cu_seqlens, kv_lens: as in cie_attention.h; the
 *               *_bt32 variants take the table as int32 page ids
 *               (a row holds min(bt_stride, n_pages) pages: longer lengths set
 *               CIE_DEVERR_BAD_LENGTH, also where rows of a wider table lie further apart)
 * head_dim 64, page_size 16.
 *
 * What the update calls store: the scale of (page, K or V, kv head) is
 *   max(scale of the rows already in the page, 2^e),
 *   e = the smallest integer in [-24, 9] with max |x| <= 127 * 2^e over the new rows,
 * and a code is x / scale rounded to nearest even, clamped to +-127. A page
 * counts as empty when its first new row is row 0: its old scale and codes are
 * then ignored. When a page's scale grows, the codes of its older rows are
 * brought to the new scale (rounded to nearest even). Powers of two keep that
 * exact but for the bits shifted out: a value is off by at most one step of its
 * page's final scale however often the page grew, and by half a step when its
 * page was written at once; code * scale is exact in fp16. Pages that another program
 * filled may have any scale >= 0: it stays while the new rows fit, and then holds for
 * these too. A stored scale that is negative, infinite or NaN holds no values: the update
 * makes the older rows 0 and sets CIE_DEVERR_BAD_SCALE. Rows a call does
 * not write, and their codes, stay as they were unless the scale grew.
 * Values beyond +-65024 saturate; an infinity is stored saturated and a NaN as
 * 0, and both set CIE_DEVERR_NONFINITE. Pages may be shared by slots that read
 * them; the sequences of one update call must write different pages.
 * The kernels are programmatic dependents of the preceding kernel in `stream` and
 * touch nothing of the caller's before it is done. Inside a call the later kernels start
 * early: the merge of several splits reads slots and lengths beside the split
 * kernel, and the attention of cie_rope_kv_q8_decode_attention reads slots, lengths, block
 * table and older pages beside the update, none of which the earlier kernel writes.
 */
#ifndef CIE_KV_Q8_H_
#define CIE_KV_Q8_H_

#include <stddef.h>
#include <stdint.h>

#include "cie_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- writes ---------------------------------------------------------------- */

/*
 * One decode token per sequence (cie_kv_decode_update's addressing): row i goes
 * to slot s = slot_ids[i] at position lens[s], the slot's length before it.
 * When a slot appears more than once (padding rows on slot 0) its last row is
 * the one written.
 */
int cie_kv_q8_decode_update(void* k_cache, void* v_cache, float* kv_scales, const int64_t* lens,
                            const int64_t* slot_ids, const int64_t* block_table,
                            const void* k_new, const void* v_new, int batch, int num_kv_heads,
                            int head_dim, int page_size, int64_t n_pages, int64_t n_slots,
                            int64_t bt_stride, int64_t cache_page_stride,
                            int64_t cache_head_stride, int64_t k_tok_stride,
                            int64_t k_head_stride, int64_t v_tok_stride, int64_t v_head_stride,
                            cie_stream_t stream);
int cie_kv_q8_decode_update_bt32(void* k_cache, void* v_cache, float* kv_scales,
                                 const int64_t* lens, const int64_t* slot_ids,
                                 const int32_t* block_table, const void* k_new,
                                 const void* v_new, int batch, int num_kv_heads, int head_dim,
                                 int page_size, int64_t n_pages, int64_t n_slots,
                                 int64_t bt_stride, int64_t cache_page_stride,
                                 int64_t cache_head_stride, int64_t k_tok_stride,
                                 int64_t k_head_stride, int64_t v_tok_stride,
                                 int64_t v_head_stride, cie_stream_t stream);

/*
 * The chunks of a mixed pass: sequence b owns rows [cu_seqlens[b], cu_seqlens[b+1])
 * of k_new / v_new (num_tokens rows in all; rows outside every sequence are not
 * written) and they go to slot slot_ids[b] at positions kv_lens[b] onward. The
 * pass is given by sequence and not by (page, offset) per row because a page's
 * rows are quantised together. When a slot appears in more than one sequence
 * with rows, the last one's are written.
 */
int cie_kv_q8_mixed_update(void* k_cache, void* v_cache, float* kv_scales,
                           const int64_t* cu_seqlens, const int64_t* kv_lens,
                           const int64_t* slot_ids, const int64_t* block_table,
                           const void* k_new, const void* v_new, int batch, int64_t num_tokens,
                           int num_kv_heads, int head_dim, int page_size, int64_t n_pages,
                           int64_t n_slots, int64_t bt_stride, int64_t cache_page_stride,
                           int64_t cache_head_stride, int64_t k_tok_stride,
                           int64_t k_head_stride, int64_t v_tok_stride, int64_t v_head_stride,
                           cie_stream_t stream);
int cie_kv_q8_mixed_update_bt32(void* k_cache, void* v_cache, float* kv_scales,
                                const int64_t* cu_seqlens, const int64_t* kv_lens,
                                const int64_t* slot_ids, const int32_t* block_table,
                                const void* k_new, const void* v_new, int batch,
                                int64_t num_tokens, int num_kv_heads, int head_dim,
                                int page_size, int64_t n_pages, int64_t n_slots,
                                int64_t bt_stride, int64_t cache_page_stride,
                                int64_t cache_head_stride, int64_t k_tok_stride,
                                int64_t k_head_stride, int64_t v_tok_stride,
                                int64_t v_head_stride, cie_stream_t stream);

/*
 * The same with the rotary embedding of q and k in the call (the arguments of
 * cie_rope_kv_decode_update / cie_rope_kv_mixed_update): q_out gets rotated q of
 * every row, rotated k and plain v are quantised into their pages. The rotation
 * x * cos + rotate_half(x) * sin is computed in fp32 and rounded once (q to fp16,
 * k to its code) -- the fp16 entry points round every operation to fp16, as
 * transformers does, so q may differ from theirs in the last bit.
 */
int cie_rope_kv_q8_decode_update(const void* qkv, int64_t qkv_tok_stride, const void* cos,
                                 const void* sin, int64_t cs_tok_stride, void* q_out,
                                 void* k_cache, void* v_cache, float* kv_scales,
                                 const int64_t* lens, const int64_t* slot_ids,
                                 const int64_t* block_table, int batch, int num_q_heads,
                                 int num_kv_heads, int head_dim, int page_size, int64_t n_pages,
                                 int64_t n_slots, int64_t bt_stride, int64_t cache_page_stride,
                                 int64_t cache_head_stride, cie_stream_t stream);
int cie_rope_kv_q8_decode_update_bt32(const void* qkv, int64_t qkv_tok_stride, const void* cos,
                                      const void* sin, int64_t cs_tok_stride, void* q_out,
                                      void* k_cache, void* v_cache, float* kv_scales,
                                      const int64_t* lens, const int64_t* slot_ids,
                                      const int32_t* block_table, int batch, int num_q_heads,
                                      int num_kv_heads, int head_dim, int page_size,
                                      int64_t n_pages, int64_t n_slots, int64_t bt_stride,
                                      int64_t cache_page_stride, int64_t cache_head_stride,
                                      cie_stream_t stream);

int cie_rope_kv_q8_mixed_update(const void* qkv, int64_t qkv_tok_stride, const void* cos,
                                const void* sin, int64_t cs_tok_stride, void* q_out,
                                void* k_cache, void* v_cache, float* kv_scales,
                                const int64_t* cu_seqlens, const int64_t* kv_lens,
                                const int64_t* slot_ids, const int64_t* block_table, int batch,
                                int64_t num_tokens, int num_q_heads, int num_kv_heads,
                                int head_dim, int page_size, int64_t n_pages, int64_t n_slots,
                                int64_t bt_stride, int64_t cache_page_stride,
                                int64_t cache_head_stride, cie_stream_t stream);
int cie_rope_kv_q8_mixed_update_bt32(const void* qkv, int64_t qkv_tok_stride, const void* cos,
                                     const void* sin, int64_t cs_tok_stride, void* q_out,
                                     void* k_cache, void* v_cache, float* kv_scales,
                                     const int64_t* cu_seqlens, const int64_t* kv_lens,
                                     const int64_t* slot_ids, const int32_t* block_table,
                                     int batch, int64_t num_tokens, int num_q_heads,
                                     int num_kv_heads, int head_dim, int page_size,
                                     int64_t n_pages, int64_t n_slots, int64_t bt_stride,
                                     int64_t cache_page_stride, int64_t cache_head_stride,
                                     cie_stream_t stream);

/* ---- read back --------------------------------------------------------------- */

/*
 * Positions [starts[b], lens[b]) of slot slot_ids[b], dequantised into a fp16
 * pool of the same page ids: out[page, h, row] = fp16(code * scale) (a scale that is no
 * fp16 number: by way of fp32). Everything
 * else in the fp16 pool stays as it was, so a pass that attends to fp16 pages
 * (cie_mixed_attention) reads the result through the same block table. k_out /
 * v_out: (n_pages, num_kv_heads, page_size, head_dim) fp16 with their own page
 * and head strides (elements). starts may be NULL (all 0). batch <= 65535.
 */
int cie_kv_q8_read(const void* k_cache, const void* v_cache, const float* kv_scales,
                   const int64_t* starts, const int64_t* lens, const int64_t* slot_ids,
                   const int64_t* block_table, void* k_out, void* v_out, int batch,
                   int num_kv_heads, int head_dim, int page_size, int64_t n_pages,
                   int64_t n_slots, int64_t bt_stride, int64_t cache_page_stride,
                   int64_t cache_head_stride, int64_t out_page_stride, int64_t out_head_stride,
                   cie_stream_t stream);
int cie_kv_q8_read_bt32(const void* k_cache, const void* v_cache, const float* kv_scales,
                        const int64_t* starts, const int64_t* lens, const int64_t* slot_ids,
                        const int32_t* block_table, void* k_out, void* v_out, int batch,
                        int num_kv_heads, int head_dim, int page_size, int64_t n_pages,
                        int64_t n_slots, int64_t bt_stride, int64_t cache_page_stride,
                        int64_t cache_head_stride, int64_t out_page_stride,
                        int64_t out_head_stride, cie_stream_t stream);

/* ---- split-KV decode attention over 8-bit pages ------------------------------- */

/*
 * cie_decode_attention over the 8-bit pool: one query token per sequence, sequence
 * b sees rows [0, lens[b]) of slot slot_ids[b], lens[b] == 0 gives a zero row.
 * q / o (1, batch, num_q_heads, head_dim) fp16 contiguous, 16-byte aligned.
 * num_kv_heads 1, 2 or 4; num_q_heads / num_kv_heads 1 to 8; batch <= 65535. num_splits <= 0:
 * cie_decode_q8_default_splits; workspace: cie_decode_workspace_bytes(batch,
 * num_q_heads, head_dim, splits) bytes, 16-byte aligned (NULL when one split).
 * Any scales whose scores fit fp32 and whose values fit fp16 give softmax(q k^T / 8) v
 * of k = code * scale, v = code * scale; the products are taken with the codes (exact in
 * fp16) and scaled in fp32, probabilities are rounded to fp16 as cie_decode_attention
 * rounds them.
 */
int cie_decode_q8_default_splits(int batch, int device);

int cie_decode_attention_q8(const void* q, const void* k, const void* v, const float* kv_scales,
                            const int64_t* lens, const int64_t* slot_ids,
                            const int64_t* block_table, void* o, void* workspace,
                            size_t workspace_bytes, int batch, int num_q_heads,
                            int num_kv_heads, int head_dim, int page_size, int64_t n_pages,
                            int64_t n_slots, int64_t bt_stride, int64_t kv_page_stride,
                            int64_t kv_head_stride, int num_splits, cie_stream_t stream);
int cie_decode_attention_q8_bt32(const void* q, const void* k, const void* v,
                                 const float* kv_scales, const int64_t* lens,
                                 const int64_t* slot_ids, const int32_t* block_table, void* o,
                                 void* workspace, size_t workspace_bytes, int batch,
                                 int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                                 int64_t n_pages, int64_t n_slots, int64_t bt_stride,
                                 int64_t kv_page_stride, int64_t kv_head_stride, int num_splits,
                                 cie_stream_t stream);

/*
 * The attention step of a decode pass in one call (cie_rope_kv_decode_attention over
 * the 8-bit pool): cie_rope_kv_q8_decode_update, then cie_decode_attention_q8 over the
 * lens[s] + 1 rows of every sequence's slot s, bit for bit; `lens` is per slot, the
 * length before the new row, and is not advanced. The attention starts while the
 * update runs: a page that the call writes must be the last page of every sequence
 * that reads it (of padding rows that share one page the result is unspecified).
 * `workspace`: cie_rope_kv_q8_decode_workspace_bytes(batch, num_q_heads,
 * head_dim, splits) bytes, 16-byte aligned, for the rotated q and the splits.
 */
size_t cie_rope_kv_q8_decode_workspace_bytes(int batch, int num_q_heads, int head_dim,
                                             int num_splits);
int cie_rope_kv_q8_decode_attention(
    const void* qkv, int64_t qkv_tok_stride, const void* cos, const void* sin,
    int64_t cs_tok_stride, void* k_cache, void* v_cache, float* kv_scales, const int64_t* lens,
    const int64_t* slot_ids, const int64_t* block_table, void* o, void* workspace,
    size_t workspace_bytes, int batch, int num_q_heads, int num_kv_heads, int head_dim,
    int page_size, int64_t n_pages, int64_t n_slots, int64_t bt_stride,
    int64_t cache_page_stride, int64_t cache_head_stride, int num_splits, cie_stream_t stream);
int cie_rope_kv_q8_decode_attention_bt32(
    const void* qkv, int64_t qkv_tok_stride, const void* cos, const void* sin,
    int64_t cs_tok_stride, void* k_cache, void* v_cache, float* kv_scales, const int64_t* lens,
    const int64_t* slot_ids, const int32_t* block_table, void* o, void* workspace,
    size_t workspace_bytes, int batch, int num_q_heads, int num_kv_heads, int head_dim,
    int page_size, int64_t n_pages, int64_t n_slots, int64_t bt_stride,
    int64_t cache_page_stride, int64_t cache_head_stride, int num_splits, cie_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* CIE_KV_Q8_H_ */
