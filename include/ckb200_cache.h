/*
 * ckb200_cache.h - a KV cache held in 4 bits, in pages that sequences share.
 *
 * The other caches of this library are one slab of fp32 or fp16 rows a sequence (kv_cache_store, kv_cache_store_f16:
 * src/kernels/kv_cache_kernels.c:111-163 of the reference).  Here a row of head_dim values is head_dim / 32 blocks block_q4_1
 * (include/ckernel_quant.h: fp16 d, fp16 m, 16 bytes of nibbles, 20 bytes per 32 values; value = d * code + m, the element order of
 * dequant_q4_1_row, src/kernels/dequant_kernels.c:119-139), 0.31 of the fp16 cache's bytes, and rows lie in pages:
 *
 *   pool         k_pages, v_pages  [num_pages][num_kv_heads][page_tokens][head_dim / 32] blocks, one pair for each layer
 *   page table   page_table        [batch][table_stride] int32: pages of a sequence's tokens 0 .., page_tokens tokens each
 *   lengths      kv_lens           [batch] int32: tokens of each sequence
 *   references   page_refs         [num_pages] int32: how many table entries name the page (0: free)
 *
 * A table serves all layers.  Everything is DEVICE memory; calls enqueue on `stream` (NULL: the library's own) without synchronising,
 * may be captured in graphs, and may run at once on several streams as long as what they write (pages, tables, workspaces) is apart.
 * They return 0 or a CKB_ERR_* code.  The current device must be the one that the library was initialised on.
 *
 * A call's `num_tokens` T new tokens are the LAST T of every sequence, kv_lens counting them: row t of sequence b (row b * T + t of q, k, v, out)
 * is position kv_lens[b] - T + t.  Rows of negative position (sequences shorter than T) are padding: nothing is stored for them and their
 * results are zeros.  A table entry outside 0 .. num_pages - 1 (-1 by convention) means that there is no page: its tokens are neither stored nor seen.
 * kv_lens outside 0 .. table_stride * page_tokens is taken as the nearer end.
 *
 * head_dim 64, 96, 128, 192 or 256; page_tokens a multiple of 16; pools aligned to 16 bytes.
 */
#ifndef CKB200_CACHE_H
#define CKB200_CACHE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of one page of K or of V: num_kv_heads * page_tokens * head_dim / 32 * 20; 0 for sizes that are not supported. */
size_t ckb200_kv_q4_page_bytes(int num_kv_heads, int page_tokens, int head_dim);
/* Where the row of kv head `head` at position `pos` lies in a pool, in bytes, given its sequence's row of a page table in HOST memory (the kernels
 * use the same arithmetic on the device's table); -1: the position has no page. */
long long ckb200_kv_q4_row_offset(const int *table_row, int table_stride, int num_pages, int page_tokens, int num_kv_heads, int head_dim, int head, int pos);

/* New rows of K and V go into the cache: the counterpart of kv_cache_store_f16 (src/kernels/kv_cache_kernels.c:131-163).  Row b * T + t of k is at
 * k + (b * T + t) * k_stride floats, [num_kv_heads][head_dim].  Of each 32 values x: m = fp16(min x), d = fp16((max x - min x) / 15),
 * code = floor((x - m) * (1 / d) + 0.5) held in 0 .. 15 (0 where d = 0), each step rounded to fp32.  A block with a NaN or an infinity, or whose
 * d or m is beyond fp16, is stored with d = m = NaN. */
int ckb200_dev_kv_cache_store_q4(void *k_pages, void *v_pages, const float *k, const float *v, long long k_stride, long long v_stride, const int *page_table,
                                 int table_stride, const int *kv_lens, int batch, int num_tokens, int num_pages, int page_tokens, int num_kv_heads, int head_dim,
                                 void *stream);
/* The way back: the last T rows of every sequence as fp32 (what the prefill attention of a prompt's own tokens is given, so that it sees the values that
 * later tokens will see). */
int ckb200_dev_kv_cache_load_q4(float *k, float *v, long long k_stride, long long v_stride, const void *k_pages, const void *v_pages, const int *page_table,
                                int table_stride, const int *kv_lens, int batch, int num_tokens, int num_pages, int page_tokens, int num_kv_heads, int head_dim,
                                void *stream);

/* A decode step's turn: one new token of each sequence, at position kv_lens[b] - 1.  q [batch][num_heads][head_dim] is rotated in place, k [batch][num_kv_heads][head_dim]
 * rotated and stored, v stored: rope_forward_qk (src/kernels/rope_kernels.c:806-819) and the store above, as ckb200_dev_rope_kv_store_f16.  Tables of rope_positions rows of
 * head_dim / 2 values; a sequence whose position lies outside them is left as it is. */
int ckb200_dev_rope_kv_store_q4(float *q, const float *k, const float *v, void *k_pages, void *v_pages, const float *cos_cache, const float *sin_cache, int rope_positions,
                                const int *page_table, int table_stride, const int *kv_lens, int batch, int num_pages, int page_tokens, int num_heads, int num_kv_heads,
                                int head_dim, void *stream);

/* Causal attention of the T new tokens (one for a decode step, several for drafted tokens or a portion of a prompt) of every sequence over its cache, the new
 * tokens' own rows among it: attention_forward_decode_head_major_gqa_flash_f16cache (src/kernels/attention_kernels.c:3450-3557) over Q4_1 rows.
 * q, out: rows of [num_heads][head_dim] floats, q_stride and out_stride floats apart; scale 1 / sqrt(head_dim).  The token at position p sees keys
 * max(0, p - sliding_window + 1) .. p (sliding_window 0: 0 .. p); one that sees none gets zeros.  num_heads is a multiple of num_kv_heads.
 * Queries, weights, steps and middles (m + 8 d) enter products as two fp16 pieces, 22 bits, sums are fp32.  Pieces end at 2^-35 of its row's largest for a weight, at 2^-39 of it for a query's
 * channel and at 2^-33 of it for the sum of 32 channels that goes with m.
 * `workspace`: ckb200_attention_q4cache_workspace_bytes() bytes of any content, aligned to 16; not shared by calls that may run at once. */
size_t ckb200_attention_q4cache_workspace_bytes(int batch, int num_tokens, int num_heads, int num_kv_heads, int head_dim);
int ckb200_dev_attention_q4cache(const float *q, long long q_stride, const void *k_pages, const void *v_pages, float *out, long long out_stride, const int *page_table,
                                 int table_stride, const int *kv_lens, int batch, int num_tokens, int num_pages, int page_tokens, int num_heads, int num_kv_heads,
                                 int head_dim, int sliding_window, void *workspace, size_t workspace_bytes, void *stream);

/* ------------------------------------------------------------------ pages
 * The pool of all layers, for the calls that move page contents: `planes` planes (K and V of every layer), plane i at pages + i * plane_stride bytes, page p
 * of it page_bytes * p further on (all multiples of 16).  planes = 0: only the tables are kept.
 * These calls keep page_refs: a page's references are the entries of the first ceil(kv_lens / page_tokens) columns that name it; entries behind are -1.
 * Entries there outside 0 .. num_pages - 1 are passed over.
 * `workspace`: ckb200_kv_pages_workspace_bytes() bytes of any content, aligned to 16; not shared by calls that may run at once. */
size_t ckb200_kv_pages_workspace_bytes(int batch, int table_stride, int num_pages);

/* Page dst[i] becomes a copy of page src[i] in every plane, i < count (src, dst: device int32).  A pair with an index outside 0 .. num_pages - 1, or
 * with src = dst, is passed over.  No dst may appear twice or also as a src. */
int ckb200_dev_kv_pages_copy(void *pages, int planes, long long plane_stride, long long page_bytes, const int *src, const int *dst, int count, int num_pages, void *stream);

/* Sequences become new_lens[b] tokens long (negative: stay as they are): 0 frees a sequence, a smaller number takes back its last tokens (drafts that were
 * refused), a larger one makes room for rows to be stored.  First all that shrink give back their pages; then those that grow, in the order of b, get theirs:
 * each the free pages of lowest number, for its new columns in their order.  A growing sequence whose last page has room but is named by others too gets a
 * copy of that page first (the last one that names it keeps it).  Where the free pages do not suffice or the table has too few columns, the sequence
 * stays as it is and status[b] is 1, else 0; later ones may still grow.
 * This call and the two below: batch at most 4096, batch * table_stride below 2^31. */
int ckb200_dev_kv_pages_resize(int *page_table, int table_stride, int *kv_lens, int *page_refs, const int *new_lens, int batch, int num_pages, int page_tokens,
                               void *pages, int planes, long long plane_stride, long long page_bytes, int *status, void *workspace, size_t workspace_bytes, void *stream);
/* Sequence b becomes what sequence parent[b] was before the call (a parent outside 0 .. batch - 1, or b itself: it stays as it is): its own pages are
 * given back, the parent's are shared, nothing is copied.  One call branches a prompt, reorders beams or swaps sequences. */
int ckb200_dev_kv_pages_fork(int *page_table, int table_stride, int *kv_lens, int *page_refs, const int *parent, int batch, int num_pages, int page_tokens,
                             void *workspace, size_t workspace_bytes, void *stream);
/* With L pages in use, the pages numbered L and above that are in use move, in their order, to the free ones below L; tables and references follow.
 * *live (may be NULL) becomes L: the pool's pages from L on hold nothing.  With batch 0 nothing is done, as in every call here: *live stays as it is. */
int ckb200_dev_kv_pages_compact(int *page_table, int table_stride, const int *kv_lens, int *page_refs, int batch, int num_pages, int page_tokens, void *pages,
                                int planes, long long plane_stride, long long page_bytes, int *live, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* CKB200_CACHE_H */
