// tree_attn.cuh — what the drafted-token attention kernels share: the view of
// the call, the division of its work over the CTAs, and the partial results.
//
// Work.  The rows of one (sequence, key head) are its drafted tokens times the
// query heads of the key head, row r = token * group + head in group.  They are
// cut into row tiles of RM rows; a unit is one row tile of one (sequence, key
// head), and reads the sequence's keys in tiles of TN.  All tiles of all units,
// in the order (sequence, key head, row tile, key tile), form one line that is
// cut into equal runs, one for each CTA, whatever the lengths of the
// sequences are: one long sequence fills the GPU and a ragged batch has no
// tail.  A unit that lies inside one run is finished there; one that is cut
// leaves partial results (unnormalised sums, row maximum, row sum) that a second
// kernel joins in the order of the runs, so the result does not depend on timing.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "b200_paged.h"
#include "error_word.cuh"
#include "sm100_ptx.cuh"

namespace b200tree {

using b200attn::report_error;

struct Args {
  const uint8_t* k;
  const uint8_t* v;
  int64_t k_page, k_head, k_row;  // bytes
  int64_t v_page, v_head, v_row;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  const int32_t* drafts;  // null: every sequence has `tokens`
  const uint8_t* q;
  uint8_t* o;
  int64_t q_seq, q_head, q_tok;  // bytes
  int64_t o_seq, o_head, o_tok;
  const uint8_t* mask;
  int64_t m_seq, m_row, m_col;
  int32_t batch, kv_heads, group, tokens, head_dim;
  int32_t slots, pages, page_size;
  int32_t row_tiles;  // of a full draft: the stride of unit numbers
  float scale_log2;
  int2* desc;       // [batch * kv_heads * row_tiles] first and last run of a unit
  float* partial;   // [2 * runs] x {sums [RM][DP], maximum [RM], sum [RM]}
  int32_t* err;
};

// Sequence b's committed and drafted tokens, forced into range.
struct Seq {
  int32_t len, drafts;
};

__device__ __forceinline__ Seq seq_of(const Args& a, int b) {
  Seq s;
  s.len = a.lens[b];
  s.drafts = a.drafts ? a.drafts[b] : a.tokens;
  const int64_t room = static_cast<int64_t>(a.slots) * a.page_size;
  if (s.len < 0 || s.drafts < 0 || s.drafts > a.tokens ||
      (s.drafts > 0 && static_cast<int64_t>(s.len) + s.drafts > room)) {
    report_error(a.err, B200_ATTN_DEVERR_BOUNDS);
    s.len = 0;
    s.drafts = 0;
  }
  return s;
}

template <int RM, int TN>
struct Shape {
  __device__ static int key_tiles(const Seq& s) {
    return s.drafts > 0 ? (s.len + s.drafts + TN - 1) / TN : 0;
  }
  __device__ static int row_tiles(const Args& a, const Seq& s) {
    return (s.drafts * a.group + RM - 1) / RM;
  }
};

// A place in the line of tiles: a key tile of a unit.
struct Place {
  int b, h, rt, t;     // sequence, key head, row tile, key tile
  int tiles, rts;      // key tiles and row tiles of the sequence
  Seq s;
};

template <int RM, int TN>
__device__ __forceinline__ void enter_seq(const Args& a, Place& p) {
  // the first sequence from p.b on with work; p.b == batch at the end
  p.tiles = 0;
  while (p.b < a.batch) {
    p.s = seq_of(a, p.b);
    p.tiles = Shape<RM, TN>::key_tiles(p.s);
    p.rts = Shape<RM, TN>::row_tiles(a, p.s);
    if (p.tiles > 0) break;
    ++p.b;
  }
}

// One unit further.
template <int RM, int TN>
__device__ __forceinline__ void next_unit(const Args& a, Place& p) {
  p.t = 0;
  if (++p.rt < p.rts) return;
  p.rt = 0;
  if (++p.h < a.kv_heads) return;
  p.h = 0;
  ++p.b;
  enter_seq<RM, TN>(a, p);
}

__device__ __forceinline__ int unit_of(const Args& a, const Place& p) {
  return (p.b * a.kv_heads + p.h) * a.row_tiles + p.rt;
}

// The line of tiles: `total` of them over the CTAs, run c has tiles
// [begin(c), begin(c + 1)).  No run is empty: with fewer tiles than CTAs the last
// CTAs have none.
struct Line {
  int64_t total;
  int64_t runs;
  __device__ Line(int64_t tiles, int64_t ctas) : total(tiles), runs(min(tiles, ctas)) {}
  __device__ int64_t begin(int64_t c) const { return c * total / runs; }
  // the run that tile t lies in: the last c with begin(c) <= t
  __device__ int owner(int64_t t) const { return static_cast<int>(((t + 1) * runs - 1) / total); }
};

// Start of this CTA's run.  Every thread sums the tiles of its share of the
// sequences, a scan finds the total, and the thread whose share holds the run's
// first tile walks to it.  `sums` is scratch for blockDim.x / 32 + 1 values;
// `out` receives the place.  Ends with a barrier.
struct Start {
  Place p;
  int64_t total;
};

template <int RM, int TN>
__device__ __forceinline__ void find_start(const Args& a, int64_t run, int64_t runs, int64_t* sums,
                                           Start* out) {
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int each = (a.batch + nt - 1) / nt;
  const int b0 = min(a.batch, tid * each), b1 = min(a.batch, b0 + each);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) {
    const Seq s = seq_of(a, b);
    mine += static_cast<int64_t>(Shape<RM, TN>::key_tiles(s)) * Shape<RM, TN>::row_tiles(a, s) *
            a.kv_heads;
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  int64_t before = incl - mine, total = 0;
  for (int w = 0; w < nt >> 5; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  const Line line(total, runs);
  if (tid == 0) out->total = total;
  const int64_t first = run < line.runs ? line.begin(run) : total;
  if (mine > 0 && first >= before && first < before + mine) {
    int64_t left = first - before;
    Place p{};
    for (int b = b0; b < b1; ++b) {
      p.b = b;
      p.s = seq_of(a, b);
      p.tiles = Shape<RM, TN>::key_tiles(p.s);
      p.rts = Shape<RM, TN>::row_tiles(a, p.s);
      const int64_t all = static_cast<int64_t>(p.tiles) * p.rts * a.kv_heads;
      if (left < all) break;
      left -= all;
    }
    p.t = static_cast<int>(left % p.tiles);
    const int u = static_cast<int>(left / p.tiles);
    p.rt = u % p.rts;
    p.h = u / p.rts;
    out->p = p;
  }
  __syncthreads();
}

// The drafted tokens i >= n_b of the sequences that this CTA looks after get
// zero rows (sequences without drafted tokens have no unit at all).
// `threads`: the first threads of the CTA, which call this.
__device__ __forceinline__ void zero_unused_rows(const Args& a, int elem_bytes, int threads) {
  const int heads = a.kv_heads * a.group;
  const int pieces = a.head_dim * elem_bytes / 16;
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    const Seq s = seq_of(a, b);
    const int n = (a.tokens - s.drafts) * heads * pieces;
    for (int x = threadIdx.x; x < n; x += threads) {
      const int row = x / pieces;
      const int i = s.drafts + row / heads;
      uint8_t* dst = a.o + b * a.o_seq + (row % heads) * a.o_head + i * a.o_tok;
      reinterpret_cast<uint4*>(dst)[x - row * pieces] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
}

// Whether drafted token i of sequence b sees drafted token j.
__device__ __forceinline__ bool sees(const Args& a, int b, int i, int j) {
  return a.mask ? a.mask[b * a.m_seq + i * a.m_row + j * a.m_col] != 0 : j <= i;
}

// Bit x: whether drafted token i of sequence b (of `drafts`) sees place d0 + x of the
// draft.  Places before the draft are committed tokens, which it sees.  A row of
// mask bytes is read as the aligned words that hold it, all at once: a byte at a
// time, each waiting for its load, these reads took longer than the tile's products.
__device__ __forceinline__ uint32_t seen_word(const Args& a, int b, int i, int d0, int drafts) {
  uint32_t word = 0u;
  int n = drafts - d0;  // bits of the word that lie in the draft or before it
  if (!a.mask) {
    n = min(n, i + 1 - d0);
    word = ~0u;
  } else {
    const uint8_t* row = a.mask + b * a.m_seq + i * a.m_row;
    if (a.m_col == 1) {
      const uintptr_t lo = reinterpret_cast<uintptr_t>(row), hi = lo + drafts;
      const uintptr_t at = lo + d0, base = at & ~static_cast<uintptr_t>(3);
      const uint32_t shift = 8u * static_cast<uint32_t>(at & 3u);
      uint32_t w[9];
#pragma unroll
      for (int x = 0; x < 9; ++x) {
        const uintptr_t p = base + 4 * x;
        w[x] = p + 4 > lo && p < hi ? __ldg(reinterpret_cast<const uint32_t*>(p)) : 0u;
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const uint32_t v = __vcmpne4(__funnelshift_r(w[x], w[x + 1], shift), 0u) & 0x01010101u;
        word |= ((v * 0x10204080u) >> 28) << (4 * x);  // the four bytes' low bits side by side
      }
    } else {
#pragma unroll 8
      for (int x = 0; x < 32; ++x)
        if (d0 + x >= 0 && x < n && row[(d0 + x) * a.m_col]) word |= 1u << x;
    }
    if (d0 < 0) word |= d0 <= -32 ? ~0u : (1u << -d0) - 1u;
  }
  return n >= 32 ? word : (n <= 0 ? 0u : word & ((1u << n) - 1u));
}

template <int DT>
struct Elem;
template <>
struct Elem<B200_ATTN_DTYPE_BF16> {
  static constexpr int kBytes = 2;
  using T = __nv_bfloat16;
  __device__ static float widen(T x) { return __bfloat162float(x); }
  __device__ static T round(float x) { return __float2bfloat16_rn(x); }
};
template <>
struct Elem<B200_ATTN_DTYPE_FP16> {
  static constexpr int kBytes = 2;
  using T = __half;
  __device__ static float widen(T x) { return __half2float(x); }
  __device__ static T round(float x) { return __float2half_rn(x); }
};
template <>
struct Elem<B200_ATTN_DTYPE_FP32> {
  static constexpr int kBytes = 4;
  using T = float;
  __device__ static float widen(T x) { return x; }
  __device__ static T round(float x) { return x; }
};

// Joins the partial results of cut units: a warp takes one row, its lanes the
// columns, and adds the runs' sums in order, weighted by 2^(m - top).
constexpr int kJoinWarps = 8;

template <int RM, int DP, int DT>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const __grid_constant__ Args a) {
  using E = Elem<DT>;
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  const int unit = blockIdx.x;
  const int rt = unit % a.row_tiles, bh = unit / a.row_tiles;
  const int b = bh / a.kv_heads, h = bh % a.kv_heads;
  const int drafts = a.drafts ? a.drafts[b] : a.tokens;
  const int rows = min(RM, drafts * a.group - rt * RM);
  const int r = blockIdx.y * kJoinWarps + (threadIdx.x >> 5);
  if (r >= rows || drafts > a.tokens) return;
  const int2 d = a.desc[unit];
  if (d.x >= d.y) return;
  const int lane = threadIdx.x & 31;
  constexpr int kSlot = RM * (DP + 2);
  // the first run holds the unit's first tile (second slot of the run), the
  // others begin inside the unit (first slot)
  auto slot = [&](int c) { return a.partial + static_cast<int64_t>(2 * c + (c == d.x)) * kSlot; };
  float top = -INFINITY;
  for (int c = d.x + lane; c <= d.y; c += 32) top = fmaxf(top, slot(c)[RM * DP + r]);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float base = top == -INFINITY ? 0.f : top;
  constexpr int kCols = DP / 32;
  float acc[kCols] = {};
  float total = 0.f;
#pragma unroll 4
  for (int c = d.x; c <= d.y; ++c) {
    const float* p = slot(c);
    const float w = exp2f(p[RM * DP + r] - base);
    total += w * p[RM * DP + RM + r];
#pragma unroll
    for (int x = 0; x < kCols; ++x) acc[x] += w * p[r * DP + lane + 32 * x];
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const int row = rt * RM + r;
  typename E::T* dst = reinterpret_cast<typename E::T*>(
      a.o + b * a.o_seq + (h * a.group + row % a.group) * a.o_head + (row / a.group) * a.o_tok);
#pragma unroll
  for (int x = 0; x < kCols; ++x)
    if (lane + 32 * x < a.head_dim) dst[lane + 32 * x] = E::round(acc[x] * inv);
}

// Host side of tree_attn_sm100.cu: the row tiles of 128 or 256, and the largest
// power of two up to 128 that divides a page (the kernel takes 8 and more).
int32_t launch_tiles(int rm, int dp, int dtype, const Args& a, int runs, int device,
                     cudaStream_t s);
int box_rows_of(int64_t page_size);

}  // namespace b200tree
