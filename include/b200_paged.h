/*
 * b200_paged.h — C ABI of the paged key/value cache and of attention for
 * drafted tokens over it: the answering half of inference (one token at a
 * time, or a tree of drafted tokens at a time), next to the attention forward
 * of b200_attn.h, which serves whole prompts.
 *
 * Cache.  Two pools of pages, K and V, of element type `dtype`; element
 * (layer, page, head, row, 0..head_dim) is contiguous in its last dimension
 * and lies at the strides given.  page_table[b][s] is the page in slot s of
 * sequence b (-1: none); token i of sequence b lies in row i % page_size of
 * the page in slot i / page_size.  seq_lens[b] counts the committed tokens of
 * sequence b; drafted tokens lie directly behind them.  page_refs[p] counts
 * the sequences that hold page p (0: free).  All bookkeeping is in device
 * memory: no operation synchronises with the host, and a whole decode step can
 * be captured in a CUDA graph.
 *
 * Entry points validate on the host what the host can see (pointers, sizes,
 * strides, types) and return the B200_ATTN_* codes.  What lies in device memory
 * (page numbers, sequence numbers, lengths) is bounds-checked by the kernels: a
 * bad value skips its access and sets B200_ATTN_DEVERR_BOUNDS in the error
 * word (b200_attn.h, "Error word"); it never reaches memory outside the
 * tensors given.
 *
 * Results do not depend on the order in which the device runs the work: free
 * pages are given out lowest number first, in (sequence, slot) order, and
 * counts are integer sums.
 */
#ifndef B200_PAGED_H_
#define B200_PAGED_H_

#include "b200_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Most sequences of one page table. */
#define B200_CACHE_MAX_BATCH 8192

/* Bits of the status b200_cache_reserve writes; 0: done.  With any bit set
 * nothing was changed. */
enum {
  B200_CACHE_NO_PAGES = 1, /* fewer free pages than needed */
  B200_CACHE_ROW_FULL = 2, /* a sequence does not fit its slots */
  B200_CACHE_BAD_ENTRY = 4 /* a page number or length out of range */
};

typedef struct b200_cache {
  void* k; /* pools; NULL both for b200_cache_fork and b200_cache_free */
  void* v;
  int64_t layers;
  int64_t pages;
  int64_t kv_heads;
  int64_t page_size;
  int64_t head_dim;     /* multiple of 8, up to 128 */
  int64_t k_stride[4];  /* layer, page, head, row: elements */
  int64_t v_stride[4];
  int32_t* page_table;  /* [batch, slots], rows table_stride apart */
  int64_t batch;        /* 1..B200_CACHE_MAX_BATCH */
  int64_t slots;
  int64_t table_stride; /* elements */
  int32_t* seq_lens;    /* [batch]; compact does not need it */
  int32_t* page_refs;   /* [pages]; needed by reserve, fork, free and compact */
  int32_t dtype;        /* B200_ATTN_DTYPE_* */
  int32_t reserved;     /* 0 */
  int32_t* error_word;  /* optional, as in b200_attn_fwd_params */
} b200_cache;

/* Rows to write into the cache: element (layer, sequence, head, token, 0..D). */
typedef struct b200_cache_rows {
  const void* k;
  const void* v;
  int64_t tokens;        /* rows given for each sequence */
  int64_t k_stride[4];   /* layer, sequence, head, token: elements */
  int64_t v_stride[4];
  const int32_t* counts; /* optional [batch]: rows of each sequence that are written, 0..tokens
                            (a sequence with another number is skipped and reported) */
} b200_cache_rows;

/* Host-only validation of the cache description.  Makes no CUDA call. */
B200_ATTN_API int32_t b200_cache_check(const b200_cache* c);

/* Bytes of device scratch that reserve and compact need (16-byte aligned). */
B200_ATTN_API int64_t b200_cache_workspace_bytes(const b200_cache* c);

/* Write row j of `rows` as token seq_lens[b] + j of every sequence b.  The
 * slots must hold pages of the sequence's own (b200_cache_reserve with status 0:
 * a page that is still shared is written for all that hold it).  Tokens without
 * a page, past the slots or of a negative length are skipped and reported. */
B200_ATTN_API int32_t b200_cache_append(const b200_cache* c, const b200_cache_rows* rows,
                                        void* stream);

/* Keep counts[b] of the drafted tokens of sequence b: token seq_lens[b] + j
 * becomes the drafted token paths[b][j] (strictly increasing in j), in all
 * layers; new_lens[b] = seq_lens[b] + counts[b] (new_lens overlaps neither
 * seq_lens nor the table, paths or counts).  A sequence whose count is not in
 * 0..width, or would not fit its slots, keeps its length and is reported. */
B200_ATTN_API int32_t b200_cache_accept(const b200_cache* c, const int32_t* paths, int64_t width,
                                        int64_t path_stride, const int32_t* counts,
                                        int32_t* new_lens, void* stream);

/* Give every sequence b pages of its own for tokens seq_lens[b] ..
 * seq_lens[b] + n - 1, n = tokens ? tokens[b] : uniform: empty slots get a free
 * page, and so do slots whose page other sequences hold too; committed rows of
 * such a page are copied (copy on write).  status: one int32 in device memory. */
B200_ATTN_API int32_t b200_cache_reserve(const b200_cache* c, const int32_t* tokens,
                                         int64_t uniform, int32_t* status, void* workspace,
                                         int64_t workspace_bytes, void* stream);

/* Sequence dst[i] lets go of its pages and shares those of src[i] that cover its
 * committed tokens.  No dst may be another's dst or any src (such an entry is
 * skipped and reported, as is one whose src has a length that does not fit its slots). */
B200_ATTN_API int32_t b200_cache_fork(const b200_cache* c, const int32_t* src, const int32_t* dst,
                                      int64_t n, void* stream);

/* Sequences rows[0..n) let go of their pages; their length becomes 0. */
B200_ATTN_API int32_t b200_cache_free(const b200_cache* c, const int32_t* rows, int64_t n,
                                      void* stream);

/* Close the gaps: with n pages held, the i-th held page at or past n moves to
 * the i-th free page before n, and the table and counts follow.  *live = n. */
B200_ATTN_API int32_t b200_cache_compact(const b200_cache* c, int32_t* live, void* workspace,
                                         int64_t workspace_bytes, void* stream);

/*
 * Attention for drafted tokens.  Query i of sequence b stands at position
 * seq_lens[b] + i and sees every committed token and the drafted tokens j <
 * n_b (n_b = draft_lens ? draft_lens[b] : tokens) whose mask byte (b, i, j) is
 * set; without a mask, those with j <= i.  A tree is given by its ancestor
 * mask (each token sees its ancestors and itself).
 *   o_i = sum_p softmax_p(scale * q_i . k_p) v_p.
 * Scores, maxima, sums of weights and sums of values are fp32, and the output is
 * rounded once.  With 16-bit caches the weights, relative to the largest so far,
 * are rounded to the element type for the product with the values, as the tensor
 * cores take them, and their sum is taken of the rounded ones; with fp32 caches
 * they are not rounded.
 * Rows that see nothing, rows i >= n_b, and all rows of a sequence whose length or
 * draft does not fit its slots or the call (which is reported) are zero.  Head h reads key head
 * h / (heads / kv_heads).  `cache` describes one layer (layers = 1).
 */
typedef struct b200_tree_attn_params {
  b200_cache cache;
  const void* q; /* [batch, heads, tokens, head_dim] */
  void* o;       /* may be q, element for element; overlaps no other input */
  int64_t heads;
  int64_t tokens;
  int64_t q_stride[3]; /* batch, head, token: elements; head_dim contiguous */
  int64_t o_stride[3];
  const uint8_t* mask; /* optional bool [batch, tokens, tokens] */
  int64_t mask_stride[3]; /* bytes; batch stride 0: one mask for all */
  const int32_t* draft_lens; /* optional [batch], 0..tokens */
  float scale;            /* > 0 */
  int32_t reserved;       /* 0 */
  void* workspace;        /* b200_tree_attn_workspace_bytes(p) bytes, 16-byte aligned */
  int64_t workspace_bytes;
  /* Optional B200_TREE_ATTN_COUNTERS int32 in device memory, zero before the first
   * call and left zero by every call, for calls that do not overlap in time (one
   * stream's): most calls of few rows then join their partial results in the same
   * kernel instead of a second one. */
  int32_t* counters;
} b200_tree_attn_params;

#define B200_TREE_ATTN_COUNTERS 1024

B200_ATTN_API int32_t b200_tree_attn_check(const b200_tree_attn_params* p);
B200_ATTN_API int64_t b200_tree_attn_workspace_bytes(const b200_tree_attn_params* p);
B200_ATTN_API int32_t b200_tree_attn_fwd(const b200_tree_attn_params* p, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* B200_PAGED_H_ */
