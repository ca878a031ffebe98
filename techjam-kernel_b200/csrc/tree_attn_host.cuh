// tree_attn_host.cuh — host-side pieces shared by the drafted-token attention of 16- and
// 32-bit caches and that of 4-bit ones.
#pragma once

#include <cstdint>
#include <mutex>

#include "byte_range.h"
#include "paged_host.h"
#include "tree_attn.cuh"

namespace b200tree {

inline int64_t round16(int64_t n) { return (n + 15) & ~static_cast<int64_t>(15); }

// Whether the output can share bytes with what the call reads, or with itself.  In the place
// of the queries, element for element, it may: a unit's rows are written when all its CTAs have
// read its queries.
// `head_dim` elements of `eb` bytes a row of the queries and the output; the pools' are the
// cache's own.
inline bool output_collides(const b200_tree_attn_params* p, int64_t head_dim, int64_t eb) {
  using b200attn::may_overlap;
  using b200attn::stretches_of;
  const b200_cache& c = p->cache;
  const int64_t pool_eb = b200paged::elem_bytes(c.dtype);
  const int64_t rows[3] = {c.batch, p->heads, p->tokens};
  const int64_t pool[3] = {c.pages, c.kv_heads, c.page_size};
  bool in_place = p->q == p->o;
  for (int d = 0; d < 3; ++d) {
    if (rows[d] <= 1) continue;
    if (p->o_stride[d] == 0) return true;
    in_place = in_place && p->o_stride[d] == p->q_stride[d];
  }
  const auto o = stretches_of(p->o, p->o_stride, rows, 3, head_dim, eb);
  if (!in_place && may_overlap(o, stretches_of(p->q, p->q_stride, rows, 3, head_dim, eb)))
    return true;
  if (may_overlap(o, stretches_of(c.k, c.k_stride + 1, pool, 3, c.head_dim, pool_eb)) ||
      may_overlap(o, stretches_of(c.v, c.v_stride + 1, pool, 3, c.head_dim, pool_eb)) ||
      may_overlap(o, stretches_of(c.page_table, &c.table_stride, &c.batch, 1, c.slots, 4)) ||
      may_overlap(o, stretches_of(c.seq_lens, nullptr, nullptr, 0, c.batch, 4)))
    return true;
  const int64_t marks[3] = {c.batch, p->tokens, p->tokens};
  return (p->mask && may_overlap(o, stretches_of(p->mask, p->mask_stride, marks, 3, 1, 1))) ||
         (p->draft_lens && may_overlap(o, stretches_of(p->draft_lens, nullptr, nullptr, 0, c.batch, 4)));
}

// Most SMs that a call runs on.  Workspaces are sized on the host for as many, without asking
// a device: more than the 148 of a B200, and every one counts (256 rows of 128 columns: 42.6 MB
// for 160 SMs).
constexpr int64_t kMaxSms = 160;

// What the kernels take from the call as it is.  `pool_eb`, `eb`: bytes of an element of the
// pools and of the queries.
inline void fill_args(const b200_tree_attn_params* p, int64_t pool_eb, int64_t eb, int64_t head_dim,
                      Args* a) {
  const b200_cache& c = p->cache;
  a->k = static_cast<const uint8_t*>(c.k);
  a->v = static_cast<const uint8_t*>(c.v);
  a->k_page = c.k_stride[1] * pool_eb;
  a->k_head = c.k_stride[2] * pool_eb;
  a->k_row = c.k_stride[3] * pool_eb;
  a->v_page = c.v_stride[1] * pool_eb;
  a->v_head = c.v_stride[2] * pool_eb;
  a->v_row = c.v_stride[3] * pool_eb;
  a->table = c.page_table;
  a->table_stride = c.table_stride;
  a->lens = c.seq_lens;
  a->drafts = p->draft_lens;
  a->q = static_cast<const uint8_t*>(p->q);
  a->o = static_cast<uint8_t*>(p->o);
  a->q_seq = p->q_stride[0] * eb;
  a->q_head = p->q_stride[1] * eb;
  a->q_tok = p->q_stride[2] * eb;
  a->o_seq = p->o_stride[0] * eb;
  a->o_head = p->o_stride[1] * eb;
  a->o_tok = p->o_stride[2] * eb;
  a->mask = p->mask;
  a->m_seq = p->mask_stride[0];
  a->m_row = p->mask_stride[1];
  a->m_col = p->mask_stride[2];
  a->batch = static_cast<int32_t>(c.batch);
  a->kv_heads = static_cast<int32_t>(c.kv_heads);
  a->group = static_cast<int32_t>(p->heads / c.kv_heads);
  a->tokens = static_cast<int32_t>(p->tokens);
  a->head_dim = static_cast<int32_t>(head_dim);
  a->slots = static_cast<int32_t>(c.slots);
  a->pages = static_cast<int32_t>(c.pages);
  a->page_size = static_cast<int32_t>(c.page_size);
}

// Launches an attention kernel on `runs` CTAs.
template <void (*kKernel)(Args)>
int32_t run_one(int threads, int smem, const Args& a, int runs, int device, cudaStream_t s) {
  static std::once_flag once[b200paged::kMaxDevices];
  static cudaError_t err[b200paged::kMaxDevices];
  std::call_once(once[device], [&] {
    err[device] = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  if (err[device] != cudaSuccess) {
    b200paged::set_error(cudaGetErrorString(err[device]));
    return B200_ATTN_ERR_LAUNCH;
  }
  return b200paged::launch(kKernel, dim3(runs), dim3(threads), smem, s, a);
}

template <int RM, int DP, int DT, int WARPS>
int32_t run_join_rows(const Args& a, int64_t units, bool spread, cudaStream_t s) {
  if (spread)
    return b200paged::launch(join_spread_kernel<RM, DP, DT>,
                             dim3(static_cast<unsigned>(units), RM / 4), dim3(32 * kJoinWarps), 0,
                             s, a);
  return b200paged::launch(join_rows_kernel<RM, DP, DT, WARPS>, dim3(static_cast<unsigned>(units)),
                           dim3(32 * WARPS), 0, s, a);
}

template <int RM, int DP, int DT>
int32_t run_join_columns(const Args& a, int64_t units, cudaStream_t s) {
  // few units: the blocks that share a unit's rows share its columns too
  const bool spread = units * (RM / 32) < 300;
  return b200paged::launch(spread ? join_columns_kernel<RM, DP, DT, true> : join_columns_kernel<RM, DP, DT, false>,
                dim3(static_cast<unsigned>(units), RM / 32, spread ? DP / kJoinCols : 1),
                dim3(32 * kJoinWarps), 0, s, a);
}

}  // namespace b200tree
