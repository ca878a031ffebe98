// tree_attn4.cuh — what the drafted-token attention kernels over 4-bit caches share.
#pragma once

#include <cstdint>

#include "tree_attn.cuh"

namespace b200tree {
namespace {

// Adds NaN to the numbers of a finished row (`out`) or its partial sums (`part`, columns
// `pitch` apart) whose group is NaN in a drafted token that the row's token sees: such steps and
// lows were left out of the products, where a weight of zero would not hide them.
template <int DP, int DT>
__device__ __noinline__ void add_odd4(const Args& a, int b, int h, Seq s, int tok, int d0, int d1,
                                      int col0, int col1, uint16_t* out, float* part,
                                      int pitch) {
  using E = Elem<DT>;
  const uint32_t size = static_cast<uint32_t>(a.page_size);
  for (int d = max(0, d0); d < min(s.drafts, d1); ++d) {
    if (!sees(a, b, tok, d)) continue;
    const uint32_t key = s.len + d, slot = key / size;
    const int pg = a.table[b * a.table_stride + slot];
    if (pg < 0 || pg >= a.pages) continue;
    const uint16_t* meta = reinterpret_cast<const uint16_t*>(
        a.v + pg * a.v_page + h * a.v_head + static_cast<int64_t>(key - slot * size) * a.v_row +
        DP / 2);
    for (int c = col0; c < col1; ++c) {
      const int g = c / (DP / 4);
      const float x = __uint_as_float(static_cast<uint32_t>(meta[g]) << 16) +
                      __uint_as_float(static_cast<uint32_t>(meta[4 + g]) << 16);
      if (isfinite(x)) continue;
      if (out) reinterpret_cast<typename E::T*>(out)[c] = E::round(x - x);
      else part[c * pitch] += x - x;
    }
  }
}

// `bytes` (a multiple of 16) of global memory to shared memory; counted by barrier `bar`.
__device__ __forceinline__ void bulk_copy(uint32_t dst, const uint8_t* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

}  // namespace

// Host side of tree_attn4_sm100.cu: row tiles of 128 or 256 rows, bf16 queries.
int32_t launch_coded(int rm, int dp, const Args& a, int runs, int device, cudaStream_t s);
// The same for the stall self-test, head dims over 64.
int32_t launch_coded_stall(int rm, const Args& a, int runs, int device, cudaStream_t s, int32_t skip);

}  // namespace b200tree
