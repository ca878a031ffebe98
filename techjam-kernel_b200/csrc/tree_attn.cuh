// tree_attn.cuh — what the drafted-token attention kernels share: the view of
// the call, the division of its work over the CTAs, and the partial results.
//
// Work.  The rows of one (sequence, key head) are its drafted tokens times the
// query heads of the key head, row r = token * group + head in group.  They are
// cut into row tiles of up to RM rows; a unit is one row tile of one (sequence, key
// head), and reads the sequence's keys in tiles of TN.  All tiles of all units,
// in the order (sequence, key head, row tile, key tile), form one line that is
// cut into equal runs, one for each CTA, whatever the lengths of the
// sequences are: one long sequence fills the GPU and a ragged batch has no
// tail.  What a unit costs beside its tiles (queries in, results out) is counted as
// EX tiles ahead of its first.  A unit that lies inside one run is finished there; one that is cut
// leaves partial results (unnormalised sums, row maximum, row sum), which are joined in
// the order of the runs, so the result does not depend on timing: by the last of its
// runs to arrive where the kernel of few rows has counters, else by a second kernel.
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
  int32_t unit_rows;  // rows of a row tile (whole tokens for the kernel of many rows)
  int32_t row_tiles;  // of a full draft: the stride of unit numbers
  float scale_log2;
  int2* desc;       // [batch * kv_heads * row_tiles] first and last run of a unit
  int32_t runs;     // CTAs of the attention kernel
  int32_t* counters;  // null, or one a unit, zero between calls
  float* partial;   // [2 * runs] x {sums [RM][DP], maximum [RM], sum [RM]}
  int32_t* err;
};

// Sequence b's committed and drafted tokens, forced into range.
struct Seq {
  int32_t len, drafts;
};

// Without a report; false: out of range, and the sequence has no unit.
__device__ __forceinline__ bool read_seq(const Args& a, int b, Seq* s) {
  s->len = a.lens[b];
  s->drafts = a.drafts ? a.drafts[b] : a.tokens;
  const int64_t room = static_cast<int64_t>(a.slots) * a.page_size;
  if (s->len >= 0 && s->drafts >= 0 && s->drafts <= a.tokens &&
      (s->drafts == 0 || static_cast<int64_t>(s->len) + s->drafts <= room))
    return true;
  s->len = 0;
  s->drafts = 0;
  return false;
}

__device__ __forceinline__ Seq seq_of(const Args& a, int b) {
  Seq s;
  if (!read_seq(a, b, &s)) report_error(a.err, B200_ATTN_DEVERR_BOUNDS);
  return s;
}

// RM rows and TN keys a tile, EX tiles' worth of work beside a unit's tiles.
template <int RM_, int TN_, uint32_t EX_>
struct Grid {
  static constexpr int RM = RM_, TN = TN_;
  static constexpr uint32_t EX = EX_;
  __device__ static int key_tiles(const Seq& s) {
    return s.drafts > 0 ? (s.len + s.drafts + TN - 1) / TN : 0;
  }
  __device__ static int row_tiles(const Args& a, const Seq& s) {
    return (s.drafts * a.group + a.unit_rows - 1) / a.unit_rows;
  }
  // places of a sequence in the line (all sequences' together fit 31 bits)
  __device__ static uint32_t places(const Args& a, const Seq& s) {
    const int t = key_tiles(s);
    return t == 0 ? 0u : (t + EX) * row_tiles(a, s) * a.kv_heads;
  }
};

// A key tile of a unit.
struct Place {
  int b, h, rt, t;     // sequence, key head, row tile, key tile
  int tiles, rts;      // key tiles and row tiles of the sequence
  Seq s;
};

template <class G>
__device__ __forceinline__ void enter_seq(const Args& a, Place& p) {
  // the first sequence from p.b on with work; p.b == batch at the end
#pragma unroll 1
  while (p.b < a.batch) {
    p.s = seq_of(a, p.b);
    p.tiles = G::key_tiles(p.s);
    p.rts = G::row_tiles(a, p.s);
    if (p.tiles > 0) break;
    ++p.b;
  }
}

// The first tile of the unit after p's.  Not inlined, like the other parts that run
// once a unit: with them in line at each use the kernels were up to 188 KB of code, and
// fetching the instructions of what runs seldom took longer than its work.
template <class G>
__device__ __noinline__ Place next_unit(const Args& a, Place p) {
  p.t = 0;
  if (++p.rt < p.rts) return p;
  p.rt = 0;
  if (++p.h < a.kv_heads) return p;
  p.h = 0;
  ++p.b;
  enter_seq<G>(a, p);
  return p;
}

__device__ __forceinline__ int unit_of(const Args& a, const Place& p) {
  return (p.b * a.kv_heads + p.h) * a.row_tiles + p.rt;
}

// A CTA's run: from place `p` up to, not including, tile et of unit (eb, eh, ert).
// first_run: the run that holds the first tile of p's unit; end_first, end_last: the
// runs that hold the first and the last tile of the unit that the run ends in.
struct Run {
  Place p;
  int eb, eh, ert, et;
  int first_run, end_first, end_last;

  __device__ __forceinline__ bool ends_in(const Place& x) const {
    return x.b == eb && x.h == eh && x.rt == ert;
  }
  __device__ __forceinline__ bool done(const Place& x) const { return ends_in(x) && x.t >= et; }
  // tiles of the run from x on in x's unit
  __device__ __forceinline__ int tiles(const Place& x) const {
    return (ends_in(x) ? et : x.tiles) - x.t;
  }
};

// Run boundaries: `more` runs of q + 1 places, then runs of q; none is empty of places.
struct Cuts {
  uint32_t total, runs, q, more;
  __device__ Cuts(uint32_t places, uint32_t ctas) : total(places), runs(min(places, ctas)) {
    q = runs ? total / runs : 0u;
    more = total - q * runs;
  }
  __device__ uint32_t begin(uint32_t c) const { return c < runs ? c * q + min(c, more) : total; }
  __device__ int owner(uint32_t place) const {
    const uint32_t head = more * (q + 1);
    return static_cast<int>(place < head ? place / (q + 1) : more + (place - head) / q);
  }
};

// Writes the run's first (end = false) or one-past-last place `at`, which lies `left`
// places into the work of sequence b.
template <class G>
__device__ __forceinline__ void put_place(const Args& a, const Cuts& cuts, bool end, int b,
                                          const Seq& s, uint32_t at, uint32_t left, Run* out) {
  Place p{b, 0, 0, 0, 0, 0, s};
  int first_run = 0, last_run = 0;
  if (b < a.batch) {
    p.tiles = G::key_tiles(s);
    p.rts = G::row_tiles(a, s);
    const uint32_t span = p.tiles + G::EX, u = left / span, x = left - u * span;
    p.t = x > G::EX ? static_cast<int>(x - G::EX) : 0;
    p.h = static_cast<int>(u) / p.rts;
    p.rt = static_cast<int>(u) - p.h * p.rts;
    // the runs that the unit's first and last tile lie in
    first_run = cuts.owner(at - x + G::EX);
    last_run = cuts.owner(at - x + span - 1);
  }
  if (!end) {
    out->p = p;
    out->first_run = first_run;
  } else {
    out->eb = p.b;
    out->eh = p.h;
    out->ert = p.rt;
    out->et = p.t;
    out->end_first = first_run;
    out->end_last = last_run;
  }
}

// find_run: this CTA's run.  Every thread counts the places of its share of the
// sequences, a scan finds the total, and the threads whose shares hold the run's
// first place and the next run's walk to them.  `sums`: scratch of one value a warp.
// Ends with a barrier; *out is in shared memory.
template <class G>
__device__ __noinline__ void find_run(const Args& a, uint32_t run, uint32_t ctas, uint32_t* sums,
                                      Run* out) {
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const bool one = a.batch <= 32;  // a lane a sequence: one warp finds the run by itself
  if (one && warp > 0) {
    __syncthreads();
    return;
  }
  const int each = one ? 1 : (a.batch + nt - 1) / nt;
  const int b0 = min(a.batch, tid * each), b1 = min(a.batch, b0 + each);
  uint32_t mine = 0;
  Seq s{0, 0};
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    s = seq_of(a, b);
    mine += G::places(a, s);
  }
  uint32_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  uint32_t before = incl - mine, total = __shfl_sync(0xffffffffu, incl, 31);
  if (!one) {
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    total = 0;
#pragma unroll 1
    for (int w = 0; w < nt >> 5; ++w) {
      if (w < warp) before += sums[w];
      total += sums[w];
    }
  }
  const Cuts cuts(total, ctas);
#pragma unroll 1
  for (uint32_t end = 0; end < 2; ++end) {
    const uint32_t at = cuts.begin(run + end);
    if (at == total) {
      if (tid == 0) put_place<G>(a, cuts, end, a.batch, Seq{0, 0}, 0, 0, out);
    } else if (at >= before && at < before + mine) {
      uint32_t left = at - before;
      int b = b0;
      if (each > 1) {
#pragma unroll 1
        for (; b < b1; ++b) {
          s = seq_of(a, b);
          const uint32_t all = G::places(a, s);
          if (left < all) break;
          left -= all;
        }
      }
      put_place<G>(a, cuts, end, b, s, at, left, out);
    }
  }
  __syncthreads();
}

// The drafted tokens i >= n_b of the sequences that this CTA looks after get
// zero rows (sequences without drafted tokens have no unit at all).
// `threads`: the first threads of the CTA, which call this.
static __device__ __noinline__ void zero_unused_rows(const Args& a, int elem_bytes, int threads) {
  const int heads = a.kv_heads * a.group;
  const int pieces = a.head_dim * elem_bytes / 16;
#pragma unroll 1
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    const Seq s = seq_of(a, b);
    const int n = (a.tokens - s.drafts) * heads * pieces;
#pragma unroll 1
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
static __device__ __noinline__ uint32_t seen_word(const Args& a, int b, int i, int d0, int drafts) {
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

// Adds to a finished row (`out`) or its partial sums (`part`, columns `pitch` apart) the
// values of drafted tokens d0..d1 that are not finite and that the row's token sees.
// They were left out of the product, where a weight of zero would not hide them.
template <int DT>
__device__ __noinline__ void add_odd(const Args& a, int b, int h, Seq s, int tok, int d0, int d1,
                                     int col0, int col1, uint16_t* out, float* part, int pitch) {
  using E = Elem<DT>;
  const uint32_t size = static_cast<uint32_t>(a.page_size);
  for (int d = max(0, d0); d < min(s.drafts, d1); ++d) {
    if (!sees(a, b, tok, d)) continue;
    const uint32_t key = s.len + d, slot = key / size;
    const int pg = a.table[b * a.table_stride + slot];
    if (pg < 0 || pg >= a.pages) continue;
    const typename E::T* v = reinterpret_cast<const typename E::T*>(
        a.v + pg * a.v_page + h * a.v_head + static_cast<int64_t>(key - slot * size) * a.v_row);
    for (int c = col0; c < col1; ++c) {
      const float x = E::widen(v[c]);
      if (isfinite(x)) continue;
      if (out) {
        typename E::T* o = reinterpret_cast<typename E::T*>(out) + c;
        *o = E::round(E::widen(*o) + x);
      } else {
        part[c * pitch] += x;
      }
    }
  }
}

// Joins the partial results of cut units.  The warps of a block share the runs of a
// unit, so that all of them are read at once, each with its own maximum and sums;
// then they join in shared memory.  The runs of a warp and the warps are taken in
// order: the result does not depend on timing.
constexpr int kJoinWarps = 8;

struct Joint {
  int2 runs;   // first and last run of the unit
  int row0;    // first row of the block in the unit
  int rows;    // rows of the unit
  int b, h, rt;
};

// False: nothing to join.  Units of sequences that were left out have no entry, and a CTA
// whose wait ran out leaves its units without one: what the workspace held before is not
// taken for a range of runs.
__device__ __forceinline__ bool joint_of(const Args& a, int row0, Joint* j) {
  const int unit = blockIdx.x, bh = unit / a.row_tiles;
  j->rt = unit % a.row_tiles;
  j->b = bh / a.kv_heads;
  j->h = bh % a.kv_heads;
  j->row0 = row0;
  j->runs = a.desc[unit];
  Seq s;
  read_seq(a, j->b, &s);
  j->rows = min(a.unit_rows, s.drafts * a.group - j->rt * a.unit_rows);
  return row0 < j->rows && j->runs.x >= 0 && j->runs.x < j->runs.y && j->runs.y < a.runs;
}

// The partial result of run c: the unit's first run kept it in its second place (the
// unit began there), the others in their first.
template <int RM, int DP>
__device__ __forceinline__ const float* part_of(const Args& a, const Joint& j, int c) {
  return a.partial + static_cast<int64_t>(2 * c + (c == j.runs.x)) * (RM * (DP + 2));
}

__device__ __forceinline__ uint8_t* out_row(const Args& a, const Joint& j, int r) {
  const int row = j.rt * a.unit_rows + r, tok = row / a.group;
  return a.o + j.b * a.o_seq + (j.h * a.group + row - tok * a.group) * a.o_head + tok * a.o_tok;
}

// Row by row, partial sums [RM][DP], a lane taking DP / 32 columns.  Up to 4 rows: the WARPS
// warps of a block share the runs and join in shared memory.  Reads past L1: other CTAs of this kernel may have
// written the partial results.
template <int DP, int WARPS>
struct JoinSmem {
  float sums[WARPS][4][DP];
  float tops[WARPS][4], totals[WARPS][4];
};

template <int RM, int DP, int DT, int WARPS>
__device__ __noinline__ void join_four(const Args& a, Joint j, JoinSmem<DP, WARPS>* sm) {
  using E = Elem<DT>;
  constexpr int kCols = DP / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float top[4], total[4], acc[4][kCols];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    top[r] = -INFINITY;
    total[r] = 0.f;
#pragma unroll
    for (int x = 0; x < kCols; ++x) acc[r][x] = 0.f;
  }
#pragma unroll 3
  for (int c = j.runs.x + warp; c <= j.runs.y; c += WARPS) {
    const float* p = part_of<RM, DP>(a, j, c);
    float v[4][kCols], m[4], l[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = min(j.row0 + r, j.rows - 1);
#pragma unroll
      for (int x = 0; x < kCols; ++x) v[r][x] = __ldcg(p + row * DP + lane + 32 * x);
      m[r] = __ldcg(p + RM * DP + row);
      l[r] = __ldcg(p + RM * DP + RM + row);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float now = fmaxf(top[r], m[r]), base = now == -INFINITY ? 0.f : now;
      const float keep = exp2f(top[r] - base), w = exp2f(m[r] - base);
      top[r] = now;
      total[r] = total[r] * keep + w * l[r];
#pragma unroll
      for (int x = 0; x < kCols; ++x) acc[r][x] = acc[r][x] * keep + w * v[r][x];
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (lane == 0) {
      sm->tops[warp][r] = top[r];
      sm->totals[warp][r] = total[r];
    }
#pragma unroll
    for (int x = 0; x < kCols; ++x) sm->sums[warp][r][lane + 32 * x] = acc[r][x];
  }
  __syncthreads();
#pragma unroll 1
  for (int y = threadIdx.x; y < 4 * DP; y += 32 * WARPS) {
    const int r = y / DP, col = y % DP;
    if (j.row0 + r >= j.rows || col >= a.head_dim) continue;
    float best = -INFINITY, sum = 0.f, all = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) best = fmaxf(best, sm->tops[w][r]);
    const float base = best == -INFINITY ? 0.f : best;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = exp2f(sm->tops[w][r] - base);
      sum += f * sm->sums[w][r][col];
      all += f * sm->totals[w][r];
    }
    reinterpret_cast<typename E::T*>(out_row(a, j, j.row0 + r))[col] =
        E::round(all == 0.f ? 0.f * sum : sum / all);
  }
  __syncthreads();
}

// More rows: each warp takes RM / WARPS of them over all runs, without shared memory.
template <int RM, int DP, int DT, int WARPS>
__device__ __noinline__ void join_many(const Args& a, Joint j) {
  using E = Elem<DT>;
  constexpr int kCols = DP / 32, kN = RM / WARPS;
  const int lane = threadIdx.x & 31, r0 = (threadIdx.x >> 5) * kN;
  if (r0 >= j.rows) return;
  float top[kN], total[kN], acc[kN][kCols];
#pragma unroll
  for (int r = 0; r < kN; ++r) {
    top[r] = -INFINITY;
    total[r] = 0.f;
#pragma unroll
    for (int x = 0; x < kCols; ++x) acc[r][x] = 0.f;
  }
#pragma unroll 4
  for (int c = j.runs.x; c <= j.runs.y; ++c) {
    const float* p = part_of<RM, DP>(a, j, c);
    float v[kN][kCols], m[kN], l[kN];
#pragma unroll
    for (int r = 0; r < kN; ++r) {
#pragma unroll
      for (int x = 0; x < kCols; ++x) v[r][x] = __ldcg(p + (r0 + r) * DP + lane + 32 * x);
      m[r] = __ldcg(p + RM * DP + r0 + r);
      l[r] = __ldcg(p + RM * DP + RM + r0 + r);
    }
#pragma unroll
    for (int r = 0; r < kN; ++r) {
      const float now = fmaxf(top[r], m[r]), base = now == -INFINITY ? 0.f : now;
      const float keep = exp2f(top[r] - base), w = exp2f(m[r] - base);
      top[r] = now;
      total[r] = total[r] * keep + w * l[r];
#pragma unroll
      for (int x = 0; x < kCols; ++x) acc[r][x] = acc[r][x] * keep + w * v[r][x];
    }
  }
#pragma unroll
  for (int r = 0; r < kN; ++r) {
    if (r0 + r >= j.rows) break;
    typename E::T* out = reinterpret_cast<typename E::T*>(out_row(a, j, r0 + r));
#pragma unroll
    for (int x = 0; x < kCols; ++x)
      if (lane + 32 * x < a.head_dim)
        out[lane + 32 * x] =
            E::round(total[r] == 0.f ? 0.f * acc[r][x] : acc[r][x] / total[r]);
  }
}

template <int RM, int DP, int DT, int WARPS>
__device__ __forceinline__ void join_unit(const Args& a, const Joint& j, JoinSmem<DP, WARPS>* sm) {
  if (j.rows <= 4) join_four<RM, DP, DT, WARPS>(a, j, sm);
  else join_many<RM, DP, DT, WARPS>(a, j);
}

// A block a unit.  WARPS as in the kernel that left the partial results: the same sums in
// the same order, wherever they are joined.
template <int RM, int DP, int DT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) join_rows_kernel(const __grid_constant__ Args a) {
  __shared__ JoinSmem<DP, WARPS> sm;
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  Joint j;
  if (joint_of(a, 0, &j)) join_unit<RM, DP, DT, WARPS>(a, j, &sm);
}

// Few units of many runs and more than 4 rows: four rows a block, whose warps share the runs.
// (One CTA joining 37 runs of 16 rows took 20 us, half a sequence's worth of reads.)
template <int RM, int DP, int DT>
__global__ void __launch_bounds__(32 * kJoinWarps)
    join_spread_kernel(const __grid_constant__ Args a) {
  __shared__ JoinSmem<DP, kJoinWarps> sm;
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  Joint j;
  if (joint_of(a, 4 * blockIdx.y, &j)) join_four<RM, DP, DT, kJoinWarps>(a, j, &sm);
}

// The same within the kernel that left the partial results: the last of a unit's runs to
// arrive joins them all.  By all threads of a CTA, after it has written its own.
template <int RM, int DP, int DT, int WARPS>
__device__ __noinline__ void join_if_last(const Args& a, int b, int h, int rt, int rows, int first,
                                          int last, JoinSmem<DP, WARPS>* sm) {
  __threadfence();
  __syncthreads();
  int32_t* counter = &a.counters[(b * a.kv_heads + h) * a.row_tiles + rt];
  bool mine = false;
  if (threadIdx.x == 0) {
    mine = atomicAdd(counter, 1) == last - first;
    if (mine) *counter = 0;
  }
  if (!__syncthreads_or(mine)) return;
  __threadfence();
  join_unit<RM, DP, DT, WARPS>(a, Joint{make_int2(first, last), 0, rows, b, h, rt}, sm);
}

// Column by column: partial sums [DP][RM], a block takes 32 rows, a lane one of them.
// A unit of up to kFewRuns runs, as in batches: each warp joins DP / 8 columns over all
// runs by itself.  Longer ones: the warps share the runs and join kJoinCols columns at a time
// in shared memory; gridDim.z blocks share the columns.  Few units: SPREAD, with more reads
// in flight in a warp; many units: fewer registers, and so more warps.  Bound by latency
// (27 MB out of L2 for 32 sequences, 256 rows).  The warps sharing every unit's runs, however
// few: 198 us against 183 us for attention and join there; one warp a column group for up
// to 4 runs only: 58 us against 53 us with 12 (3 sequences of 10000 tokens).
constexpr int kFewRuns = 12, kJoinCols = 16;

// Folds the runs c, c + step ... into the columns from c0 on of a row; U runs are read at once.
template <int RM, int DP, int U, int N>
__device__ __forceinline__ void fold_runs(const Args& a, const Joint& j, int c, int step, int c0,
                                          int row, float& top, float& total, float (&acc)[N]) {
  top = -INFINITY;
  total = 0.f;
#pragma unroll
  for (int x = 0; x < N; ++x) acc[x] = 0.f;
#pragma unroll 1
  for (; c <= j.runs.y; c += U * step) {
    float v[U][N], m[U], l[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c + u * step > j.runs.y) continue;
      const float* p = part_of<RM, DP>(a, j, c + u * step) + row;
#pragma unroll
      for (int x = 0; x < N; ++x) v[u][x] = p[(c0 + x) * RM];
      m[u] = p[RM * DP];
      l[u] = p[RM * DP + RM];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c + u * step > j.runs.y) continue;
      const float now = fmaxf(top, m[u]), base = now == -INFINITY ? 0.f : now;
      const float keep = exp2f(top - base), w = exp2f(m[u] - base);
      top = now;
      total = total * keep + w * l[u];
#pragma unroll
      for (int x = 0; x < N; ++x) acc[x] = acc[x] * keep + w * v[u][x];
    }
  }
}

template <int RM, int DP, int DT, bool SPREAD>
__global__ void __launch_bounds__(32 * kJoinWarps)
    join_columns_kernel(const __grid_constant__ Args a) {
  using E = Elem<DT>;
  using T = typename E::T;
  __shared__ float sums[kJoinWarps][32][kJoinCols + 1];
  __shared__ float tops[kJoinWarps][32], totals[kJoinWarps][32];
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  Joint j;
  if (!joint_of(a, 32 * blockIdx.y, &j)) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = min(j.row0 + lane, j.rows - 1);
  float top, total;
  if (j.runs.y - j.runs.x < kFewRuns) {
    constexpr int kN = DP / kJoinWarps;
    const int c0 = kN * warp;
    if (blockIdx.z > 0 || c0 >= a.head_dim) return;
    float acc[kN];
    fold_runs<RM, DP, SPREAD ? 2 : 1>(a, j, j.runs.x, 1, c0, row, top, total, acc);
    if (j.row0 + lane >= j.rows) return;
    const float inv = total == 0.f ? 0.f : 1.f / total;
    T* dst = reinterpret_cast<T*>(out_row(a, j, row)) + c0;
#pragma unroll
    for (int x = 0; x < kN; x += 8) {
      if (c0 + x >= a.head_dim) break;
      union {
        T e[8];
        uint4 w;
      } o;
#pragma unroll
      for (int y = 0; y < 8; ++y) o.e[y] = E::round(acc[x + y] * inv);
      *reinterpret_cast<uint4*>(dst + x) = o.w;
    }
    return;
  }
  for (int c0 = kJoinCols * blockIdx.z; c0 < a.head_dim; c0 += kJoinCols * gridDim.z) {
    float acc[kJoinCols];
    fold_runs<RM, DP, SPREAD ? 3 : 1>(a, j, j.runs.x + warp, kJoinWarps, c0, row, top, total, acc);
    tops[warp][lane] = top;
    totals[warp][lane] = total;
#pragma unroll
    for (int x = 0; x < kJoinCols; ++x) sums[warp][lane][x] = acc[x];
    __syncthreads();
    // a thread finishes 2 columns of a row
    const int r = threadIdx.x >> 3, x0 = 2 * (threadIdx.x & 7);
    if (j.row0 + r < j.rows && c0 + x0 < a.head_dim) {
      float best = -INFINITY, all = 0.f, sum[2] = {};
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) best = fmaxf(best, tops[w][r]);
      const float base = best == -INFINITY ? 0.f : best;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) {
        const float f = exp2f(tops[w][r] - base);
        all += f * totals[w][r];
#pragma unroll
        for (int x = 0; x < 2; ++x) sum[x] += f * sums[w][r][x0 + x];
      }
      const float inv = all == 0.f ? 0.f : 1.f / all;
      T* dst = reinterpret_cast<T*>(out_row(a, j, j.row0 + r)) + c0 + x0;
#pragma unroll
      for (int x = 0; x < 2; ++x) dst[x] = E::round(sum[x] * inv);
    }
    __syncthreads();
  }
}

// Host side of tree_attn_sm100.cu: the row tiles of 128 or 256, and the largest
// power of two up to 128 that divides a page (the kernel takes 8 and more).
int32_t launch_tiles(int rm, int dp, int dtype, const Args& a, int heads, int runs, int device,
                     cudaStream_t s);
int box_rows_of(int64_t page_size);

}  // namespace b200tree
