/*
 * b200_verify.h — C ABI of the check of drafted tokens against the target's
 * probabilities, with given random numbers: the end of a speculative decoding step.
 * What it writes goes into b200_cache_accept (b200_paged.h).
 *
 * Sequence b has n_b = draft_lens ? draft_lens[b] : nodes drafted nodes.  Node 0 is the root
 * (the last token that is already decided; its id is not read); node i > 0 has the token
 * tokens[b][i] and the parent parents[b][i] < i (a chain without `parents`: i - 1).  A node
 * whose parent is -1 is not looked at.  Row logits[b][i] is the target's after node i, and
 * p_i = softmax(logits[b][i] / temperature); temperature 0: all weight on the largest
 * logit, the first of equal ones.  Row draft_probs[b][i] is the distribution q_i that the
 * children of node i were drawn from, independently; without draft_probs, and at
 * temperature 0, every draft counts as certain: q is 1 at its token and 0 elsewhere.
 *
 * The path starts at the root.  At node i with p = p_i its children c are asked in order:
 *   uniforms[b][c] * q(x_c) < p(x_c), x_c = tokens[b][c]:  c is kept and the path goes on
 *       from it (its siblings behind it are not looked at);
 *   else  p <- max(p - q, 0) / sum of it  (as it was where nothing is left).
 * Where no child is kept the path ends, and the next token is the first v with
 *   p(0) + ... + p(v) > uniforms[b][0] * sum of p   and   p(v) > 0.
 * With uniforms in [0, 1) the tokens so found are distributed as the target's own.
 *
 * paths[b]: the nodes of the path in order, the root first, then -1.  counts[b]: how many;
 * 0 where n_b = 0.  next[b]: the next token; -1 where n_b = 0 and where the path ends at a row
 * without a distribution (a NaN or +infinity, or nothing above -infinity), whose children
 * are not kept.  Draft probabilities below 0 and NaN count as 0.
 *
 * Exponentials and sums are 64-bit.
 * Results do not depend on execution order.  A token id out of range, a parent that
 * does not come before its child and a draft length out of range are reported in the error
 * word (B200_ATTN_DEVERR_BOUNDS): such a node is not kept, such a sequence counts as empty.
 */
#ifndef B200_VERIFY_H_
#define B200_VERIFY_H_

#include "b200_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define B200_VERIFY_MAX_NODES 1024
#define B200_VERIFY_MAX_VOCAB (1 << 24)

typedef struct b200_verify_params {
  const void* logits;       /* [batch, nodes, vocab], vocab contiguous */
  int64_t logits_stride[2]; /* batch, node: elements */
  const void* draft_probs;  /* optional [batch, nodes - 1, vocab] */
  int64_t draft_stride[2];
  const void* tokens;       /* [batch, nodes] int32, or int64 with wide_tokens */
  int64_t token_stride;     /* of a sequence, elements; nodes are contiguous */
  const float* uniforms;    /* [batch, nodes] */
  int64_t uniform_stride;
  const int32_t* parents;   /* optional [batch, nodes]; stride 0: one tree for all */
  int64_t parent_stride;
  const int32_t* draft_lens; /* optional [batch], 0..nodes */
  int32_t* paths;           /* [batch, nodes], contiguous */
  int32_t* counts;          /* [batch] */
  int64_t* next;            /* [batch] */
  int64_t batch;            /* 1.. */
  int64_t nodes;            /* 1..B200_VERIFY_MAX_NODES */
  int64_t vocab;            /* 1..B200_VERIFY_MAX_VOCAB */
  double temperature;       /* 0, or positive with a finite reciprocal */
  int32_t dtype;            /* of the logits: B200_ATTN_DTYPE_* */
  int32_t draft_dtype;      /* of draft_probs */
  int32_t wide_tokens;      /* 1: tokens are int64 */
  int32_t reserved;         /* 0 */
  int32_t* error_word;      /* optional, as in b200_attn_fwd_params */
} b200_verify_params;

/* Host-only validation.  Makes no CUDA call. */
B200_ATTN_API int32_t b200_verify_check(const b200_verify_params* p);
B200_ATTN_API int32_t b200_verify_drafts(const b200_verify_params* p, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* B200_VERIFY_H_ */
