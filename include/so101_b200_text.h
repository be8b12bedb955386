/*
 * so101_b200_text.h — C ABI of the text tower's serving kernels (libso101_b200.so): causal
 * attention over packed prompts, and a paged K/V cache in 8 bits with the attention that reads it.
 *
 * The conventions are those of so101_b200.h: device pointers, element strides, sizes and a
 * cudaStream_t; asynchronous on that stream; nothing is allocated; an int status. Index arrays
 * (starts, seqs, tables, lengths) live on the device, so the host cannot check their values: the
 * kernels do, skip what is out of range and record SO101_ERR_PAGES in the device status word
 * (so101_device_status). The reference (so101-smolvla-edge) has no counterpart of any of these: it
 * keeps one fixed-size bf16 K/V buffer per engine (its model/smolvla_triton.py:9-17).
 */
#ifndef SO101_B200_TEXT_H
#define SO101_B200_TEXT_H

#include "so101_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SO101_ERR_PAGES 6 /* an index out of range, or too few free pages (so101_device_status) */

/* Causal grouped-query attention over whole prompts packed end to end, bf16 in and out, fp32
 * softmax (exp2), P rounded to bf16 for P V. q: (rows, >= nq*hd) with head h at columns
 * [h*hd, (h+1)*hd); k, v: (rows, >= nkv*hd). Sequence i is rows [starts[i], starts[i+1]) of all
 * three (starts: n_seqs + 1 int32, non-decreasing, starts[n_seqs] <= rows; empty sequences are
 * fine); its row r sees its rows 0..r and nothing else, whatever the other rows hold (infinities
 * and NaN included). max_len: 0 where all of them are empty (nothing is launched); else without
 * effect, the lengths are read from starts. cos / sin (rows, hd/2 fp32) rotate q
 * on load in fp32 (NULL: none), kept as two bf16 parts; k comes rotated. scale multiplies q.k. hd 64
 * or 128; 16-byte aligned bases (cos and sin too) and row strides. Rows outside every sequence are
 * not written. */
SO101_API int so101_attention_packed(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
                                     int64_t ldv, void* o, int64_t ldo, int64_t rows, const int* starts,
                                     int n_seqs, int64_t max_len, int nq, int nkv, int hd, float scale,
                                     const float* cos, const float* sin, cudaStream_t stream);

/* A paged K/V cache. Token t of sequence s lies in page table[s * max_pages + t / page] at slot
 * t % page; a page number serves every layer. Codes: k / v [layer][page][kv head][slot][dim] int8;
 * scales: k_scale / v_scale [layer][page][kv head] fp32, one power of two per page and head, the
 * value being code * scale. refs[p] counts the sequences that hold page p (0: free). table rows
 * hold -1 past a sequence's pages. page 16, 32 or 64; hd 64 or 128; k, v, k_scale, v_scale
 * 16-byte aligned. scratch: so101_kv_scratch ints, zero before the first call, used by
 * reserve, free, append, fork and compact, which must be ordered on one stream. */
typedef struct so101_kv_pages {
  int8_t* k;
  int8_t* v;
  float* k_scale;
  float* v_scale;
  int* table;
  int* lengths;
  int* refs;
  int* scratch;
  int n_layers, n_pages, n_kv, page, hd, max_seqs, max_pages;
} so101_kv_pages;

/* The ints of so101_kv_pages.scratch for these sizes. */
SO101_API int so101_kv_scratch(const so101_kv_pages* c, int64_t* ints);

/* Quantise new tokens into the pages of one layer. k, v: (rows, >= n_kv*hd) bf16, rows
 * [starts[i], starts[i+1]) being the LAST tokens of sequence seqs[i] (lengths already count them:
 * so101_kv_reserve; starts NULL: one row per sequence; seqs NULL: sequence i), which are distinct. max_new: at least
 * the most rows of a sequence. cos / sin (rows, hd/2 fp32) rotate the keys first, in fp32, as
 * so101_rope_kv does but without its rounding to bf16 (NULL: none). k, v, cos, sin 16-byte aligned, ldk and
 * ldv multiples of 8. The rule, per page and head:
 * scale = 2^e, e = ceil(log2(max |x| / 127)) clamped to [-126, 121]; code = rint(x / scale) clamped
 * to +-127. New tokens in a part-filled page: scale' = max(scale, theirs), older codes become
 * rint(code * scale / scale'). A value that is not finite makes the page's scale NaN for good.
 * A sequence whose last so101_kv_reserve was refused takes no rows (its length does not count them:
 * they would replace older tokens) until one is met or it is freed; SO101_ERR_PAGES is recorded. */
SO101_API int so101_kv_append(const so101_kv_pages* c, int layer, const void* k, int64_t ldk, const void* v,
                              int64_t ldv, int64_t rows, const int* starts, const int* seqs, int n_seqs,
                              int64_t max_new, const float* cos, const float* sin, cudaStream_t stream);

/* Cached tokens back as bf16 rows (exact: a code times a power of two): row starts[i] + r of k_out /
 * v_out (rows, n_kv*hd) is token first[i] + r of sequence seqs[i] (first NULL: 0, seqs NULL:
 * sequence i), as so101_rope_kv's cache rows. */
SO101_API int so101_kv_read(const so101_kv_pages* c, int layer, const int* starts, const int* seqs,
                            const int* first, int n_seqs, int64_t rows, void* k_out, int64_t ldk, void* v_out,
                            int64_t ldv, cudaStream_t stream);

/* Attention of each sequence's last tokens over its cached ones. q: (rows, >= nq*hd) bf16, rows
 * [starts[i], starts[i+1]) being the last n_i tokens of sequence seqs[i] (starts NULL: one row
 * per sequence), n_i <= max_q. causal: row r sees tokens <= lengths - n_i + r; otherwise all
 * lengths of them. A row that sees none is 0. o: (rows, nq*hd) bf16. cos / sin rotate q. q, cos and
 * sin are 16-byte aligned, o 8-byte; ldq is a multiple of 8, ldo of 4. Probabilities
 * are rounded to fp16, sums are fp32. workspace (fp32 partials) and tickets (zero before the first
 * call, left zero) join the parts of a sequence that several CTAs read: 40 MB and 1184 tickets let every
 * shape use the whole GPU, with less it uses fewer CTAs. Calls that may run at the same time (other
 * streams, other graphs) need a workspace and tickets each; after SO101_ERR_TIMEOUT zero the tickets. */
SO101_API int so101_attention_pages(const void* q, int64_t ldq, void* o, int64_t ldo, int64_t rows,
                                    const so101_kv_pages* c, int layer, int nq, const int* starts,
                                    const int* seqs, int n_seqs, int64_t max_q, int causal, float scale,
                                    const float* cos, const float* sin, void* workspace,
                                    int64_t workspace_bytes, int* tickets, int64_t n_tickets,
                                    cudaStream_t stream);

/* lengths[seqs[i]] += tokens[i], taking the lowest free pages in the order of the list. If any
 * sequence would pass max_pages * page tokens, is named twice, or the pages do not suffice, nothing
 * changes, so101_kv_append takes no rows of these sequences until a call for them is met, and
 * SO101_ERR_PAGES is recorded. */
SO101_API int so101_kv_reserve(const so101_kv_pages* c, const int* seqs, const int* tokens, int n,
                               cudaStream_t stream);

/* Sequences give their pages back: counts go down, lengths become 0, table rows -1. */
SO101_API int so101_kv_free(const so101_kv_pages* c, const int* seqs, int n, cudaStream_t stream);

/* Each child becomes its parent's continuation: whole pages are shared (counts go up), a part-filled
 * last page is copied, in every layer, into the lowest free pages in the order of the list, so that
 * parent and child may both append. Children are distinct and empty (length 0). If a child is not
 * empty or the pages do not suffice, nothing changes and SO101_ERR_PAGES is recorded. */
SO101_API int so101_kv_fork(const so101_kv_pages* c, const int* parents, const int* children, int n,
                            cudaStream_t stream);

/* Page src[i]'s codes and scales into page dst[i], every layer. No destination is a source or
 * another destination. Counts and tables stay. */
SO101_API int so101_kv_copy(const so101_kv_pages* c, const int* src, const int* dst, int n, cudaStream_t stream);

/* Move the L live pages into page numbers 0 .. L-1: the k-th live page past L goes to the k-th free
 * one below it; counts and tables follow. */
SO101_API int so101_kv_compact(const so101_kv_pages* c, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* SO101_B200_TEXT_H */
