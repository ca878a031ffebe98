/*
 * b200_cache4.h — C ABI of the paged cache held in 4 bits: append, read back, and
 * attention for drafted tokens over it (b200_paged.h has the cache of 16 and 32 bits,
 * and the page operations of both).
 *
 * Format.  A row holds one head's vector of head_dim numbers (a multiple of 8, up to
 * 128), padded to P = 64 or 128, in four groups of P / 4.  With the group's largest and
 * smallest number,
 *   low  = the bf16 number at or below the smallest,
 *   step = the bf16 number at or above (largest - low) / 15, and 2^-100 at least
 *          where it is not 0,
 *   code = (x - low) / step rounded to the nearest whole number, ties to even, 0..15,
 * and the row stands for low + step * code: nothing is clipped, and a number is off by half
 * a step at most.  A group that holds an infinity or NaN stands for NaN (step and low NaN,
 * codes 0), and so does one whose largest - low is past the largest fp32 number: fifteen of
 * its steps would be no fp32 number, in which the attention adds them to low.  A group past
 * head_dim has step, low and codes 0.  The row is P / 2 bytes of codes, four bf16 steps, four bf16 lows: 48 or 80
 * bytes.  Half bytes are counted from the low half of byte 0.  Number e of group g of a row
 * of keys lies in half byte
 *   P = 128:  32 (e / 8) + 8 g       + 2 (e % 8 / 4) + e % 4 / 2 + 4 (e % 2)
 *   P = 64:   16 (e / 4) + 8 (g / 2) + 2 (g % 2)     + e % 4 / 2 + 4 (e % 2)
 * and that of a row of values, with n = P / 32, in half byte
 *   (e / n) P / 8 + n g + e % n.
 * These are the orders in which the lanes of the matrix instruction take them.
 *
 * Pools.  A pool of such rows is described by the b200_cache that the page operations
 * take for it: dtype B200_ATTN_DTYPE_BF16, head_dim = b200_cache4_row_bytes(head_dim) / 2,
 * and strides in 16-bit elements; b200_cache_accept, _reserve, _fork, _free and _compact move
 * the rows as they are.  The entry points here take the vectors' head_dim and type beside it.
 */
#ifndef B200_CACHE4_H_
#define B200_CACHE4_H_

#include "b200_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of a row: 48 (head_dim up to 64) or 80; 0 for a head_dim that is not supported. */
B200_ATTN_API int32_t b200_cache4_row_bytes(int64_t head_dim);

/* b200_cache_append into a 4-bit cache: rows of `dtype` (bf16, fp16 or fp32). */
B200_ATTN_API int32_t b200_cache4_append(const b200_cache* c, int64_t head_dim, int32_t dtype,
                                         const b200_cache_rows* rows, void* stream);

/* Writes token seq_lens[b] + j of every sequence b to row j of `rows` (k and v are
 * outputs here, no element of theirs twice), each number rounded once to `dtype`; rows j >=
 * counts[b], and rows whose token has no page (which is reported), are zero. */
B200_ATTN_API int32_t b200_cache4_read(const b200_cache* c, int64_t head_dim, int32_t dtype,
                                       const b200_cache_rows* rows, void* stream);

/*
 * b200_tree_attn_fwd over a 4-bit cache (p->cache as above); queries and output of `dtype`
 * (bf16 or fp16).  The queries are taken as fp16 numbers times a power of two of their row,
 * which loses nothing of a bf16 or fp16 number that is no smaller than 2^-23 of the row's
 * largest.  Scores, maxima, sums of weights and output sums are fp32 (scores keep their bits where
 * the row's largest number times the scale lies between 2^-113 and 2^116), and the output is
 * rounded once.  Up to 16 rows (tokens * heads / kv_heads), and all calls but those below:
 * products with the codes are exact in the tensor cores' fp32 sums; steps and lows are applied
 * in fp32; a weight times the step of its value is rounded to fp16 for the product (with fp16
 * queries, for codes less 8), relative to the largest step that the row sees (what is below 2^-34
 * of it is lost); weights times lows, and the sum of weights, are fp32.
 * More rows with bf16 queries, heads / kv_heads up to 128, and no mask or up to 64 tokens: keys
 * are rounded to fp16 numbers times a power of two of the 32 committed keys that they are among
 * (what is below 2^-38 of their largest number is lost), or of a key alone where drafted ones
 * are near, and values to bf16; a weight is the sum of two bf16 numbers.
 */
B200_ATTN_API int32_t b200_cache4_attn_check(const b200_tree_attn_params* p, int64_t head_dim,
                                             int32_t dtype);
B200_ATTN_API int64_t b200_cache4_attn_workspace_bytes(const b200_tree_attn_params* p,
                                                       int64_t head_dim, int32_t dtype);
B200_ATTN_API int32_t b200_cache4_attn_fwd(const b200_tree_attn_params* p, int64_t head_dim,
                                           int32_t dtype, void* stream);

/* Self-test of failure detection.  Launches the attention kernel of more than 16 rows like
 * b200_cache4_attn_fwd (without the join of the units that were cut), except that in every CTA a copy
 * of key tile number `skipped_tile` (0: its first) is announced to its barrier but never issued.
 * The wait on it runs out after a second: the kernel ORs B200_ATTN_DEVERR_WAIT_TIMEOUT into the
 * error word, waits (bounded) for its own copies and products, frees its tensor memory and returns,
 * leaving the CUDA context usable.  For bf16, head_dim over 64, calls that take that kernel, and a
 * non-null error_word (B200_ATTN_ERR_UNSUPPORTED otherwise).  The output is undefined. */
B200_ATTN_API int32_t b200_cache4_selftest_stall(const b200_tree_attn_params* p, int64_t head_dim,
                                                 int32_t dtype, int32_t skipped_tile, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* B200_CACHE4_H_ */
