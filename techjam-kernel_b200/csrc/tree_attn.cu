// tree_attn.cu — attention for drafted tokens over a paged key/value cache:
// entry points, and the kernel for 32-bit caches.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "b200_paged.h"
#include "byte_range.h"
#include "error_word.cuh"
#include "paged_host.h"
#include "tree_attn.cuh"
#include "tree_attn_rows.cuh"

namespace b200tree {

namespace {

// ------------------------------------------------------------ plain kernel
// 16 rows by 64 keys a tile, fp32 multiply-adds: scores from shared memory, one
// pass over the keys with the running maximum and sum, the products' sums in
// registers.  fp32 caches are for checking a model, not for serving it: the products stay
// exact fp32 and each tile's loads, scores and sums follow one another.  Trees of up to 5
// tokens over 3 sequences of up to 700 keys, 4 key heads of 3, D 40, take 15.6 us, most of it
// the launch and the chain of loads; their 0.56 MB would take 0.09 us.
constexpr int kRows = 16, kKeys = 64, kThreads = 256;
constexpr int kScoreRows = kRows * kKeys / kThreads;  // rows of a thread's key
constexpr int kWarpRows = kRows * 32 / kThreads;      // rows of a warp in the softmax step
using PlainGrid = Grid<kRows, kKeys, 1>;

template <int DP>
struct PlainSmem {
  float q[kRows][DP + 4];
  float k[kKeys][DP + 4];
  float v[kKeys][DP];
  float p[kRows][kKeys + 1];
  float m[kRows], l[kRows], alpha[kRows];
  bool live[kKeys];  // the key is there
  uint32_t sums[kThreads / 32];
  Run run;
};

template <int DP, int DT>
__global__ void __launch_bounds__(kThreads) plain_kernel(const __grid_constant__ Args a) {
  using E = Elem<DT>;
  constexpr int kPer16 = 16 / E::kBytes;
  extern __shared__ __align__(16) uint8_t raw[];
  PlainSmem<DP>& sm = *reinterpret_cast<PlainSmem<DP>*>(raw);
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  const int tid = threadIdx.x;
  find_run<PlainGrid>(a, blockIdx.x, gridDim.x, sm.sums, &sm.run);
  zero_unused_rows(a, E::kBytes, kThreads);
  const Run& run = sm.run;
  Place pl = run.p;

  constexpr int kColGroups = kThreads / DP;         // row groups of the second product
  constexpr int kRowsPer = kRows / (kColGroups > 0 ? kColGroups : 1);
  const int col = tid % DP, rg = tid / DP;
  const int pieces = a.head_dim / kPer16;
#pragma unroll 1
  while (!run.done(pl)) {
    // ---- one unit, from key tile pl.t on
    const int rows = min(kRows, pl.s.drafts * a.group - pl.rt * kRows);
    const int t0 = pl.t;
    const int n = run.tiles(pl);
    const int keys = pl.s.len + pl.s.drafts;
    auto row_ptr = [&](const uint8_t* base, int64_t seq, int64_t head, int64_t tok, int r) {
      const int row = pl.rt * kRows + r;
      return base + pl.b * seq + (pl.h * a.group + row % a.group) * head + (row / a.group) * tok;
    };
#pragma unroll 4
    for (int x = tid; x < kRows * (DP / kPer16); x += kThreads) {
      const int r = x / (DP / kPer16), c = x % (DP / kPer16);
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows && c < pieces)
        w = __ldg(reinterpret_cast<const uint4*>(row_ptr(a.q, a.q_seq, a.q_head, a.q_tok, r)) + c);
#pragma unroll
      for (int e = 0; e < kPer16; ++e)
        sm.q[r][c * kPer16 + e] =
            E::widen(reinterpret_cast<const typename E::T*>(&w)[e]) * a.scale_log2;
    }
    if (tid < kRows) {
      sm.m[tid] = -INFINITY;
      sm.l[tid] = 0.f;
    }
    float acc[kRowsPer] = {};
#pragma unroll 1
    for (int t = t0; t < t0 + n; ++t) {
      const int k0 = t * kKeys;
      __syncthreads();
      // keys and values, a thread 4 pieces of 16 bytes of each at a time: page numbers,
      // then rows, are all read before any is used
      constexpr int kRowPieces = DP / kPer16, kBatch = 4;
#pragma unroll 1
      for (int x0 = tid; x0 < kKeys * kRowPieces; x0 += kBatch * kThreads) {
        int page[kBatch];
        uint4 kw[kBatch], vw[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int key = (x0 + u * kThreads) / kRowPieces;
          page[u] = -1;
          if (k0 + key < keys) {
            page[u] = __ldg(a.table + pl.b * a.table_stride + (k0 + key) / a.page_size);
            if (page[u] < 0 || page[u] >= a.pages) {
              report_error(a.err, B200_ATTN_DEVERR_BOUNDS);
              page[u] = -1;
            }
          }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int x = x0 + u * kThreads, key = x / kRowPieces, c = x % kRowPieces;
          kw[u] = vw[u] = make_uint4(0u, 0u, 0u, 0u);
          if (page[u] >= 0 && c < pieces) {
            const int64_t row = (k0 + key) % a.page_size;
            kw[u] = *reinterpret_cast<const uint4*>(a.k + page[u] * a.k_page + pl.h * a.k_head +
                                                    row * a.k_row + 16 * c);
            vw[u] = *reinterpret_cast<const uint4*>(a.v + page[u] * a.v_page + pl.h * a.v_head +
                                                    row * a.v_row + 16 * c);
          }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int x = x0 + u * kThreads, key = x / kRowPieces, c = x % kRowPieces;
          if (c == 0) sm.live[key] = page[u] >= 0;
#pragma unroll
          for (int e = 0; e < kPer16; ++e) {
            sm.k[key][c * kPer16 + e] = E::widen(reinterpret_cast<const typename E::T*>(&kw[u])[e]);
            sm.v[key][c * kPer16 + e] = E::widen(reinterpret_cast<const typename E::T*>(&vw[u])[e]);
          }
        }
      }
      __syncthreads();
      {  // scores: this thread's key, some rows
        const int key = tid & (kKeys - 1), r0 = (tid / kKeys) * kScoreRows;
        float s[kScoreRows] = {};
        for (int c = 0; c < DP; c += 4) {
          const float4 kk = *reinterpret_cast<const float4*>(&sm.k[key][c]);
#pragma unroll
          for (int r = 0; r < kScoreRows; ++r) {
            const float4 qq = *reinterpret_cast<const float4*>(&sm.q[r0 + r][c]);
            s[r] = fmaf(qq.x, kk.x, fmaf(qq.y, kk.y, fmaf(qq.z, kk.z, fmaf(qq.w, kk.w, s[r]))));
          }
        }
        const int j = k0 + key - pl.s.len;  // place in the draft
#pragma unroll
        for (int r = 0; r < kScoreRows; ++r) {
          const int i = (pl.rt * kRows + r0 + r) / a.group;
          const bool shown = r0 + r < rows && sm.live[key] &&
                             (j < 0 || (j < pl.s.drafts && sees(a, pl.b, i, j)));
          sm.p[r0 + r][key] = shown ? s[r] : -INFINITY;
        }
      }
      __syncthreads();
      {  // softmax step
        const int lane = tid & 31, warp = tid >> 5;
#pragma unroll
        for (int r = warp * kWarpRows; r < warp * kWarpRows + kWarpRows; ++r) {
          const float x0 = sm.p[r][lane], x1 = sm.p[r][lane + 32];
          float top = fmaxf(x0, x1);
#pragma unroll
          for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const float old = sm.m[r], now = fmaxf(old, top);
          const float base = now == -INFINITY ? 0.f : now;
          const float p0 = exp2f(x0 - base), p1 = exp2f(x1 - base);
          float sum = p0 + p1;
#pragma unroll
          for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          __syncwarp();
          sm.p[r][lane] = p0;
          sm.p[r][lane + 32] = p1;
          if (lane == 0) {
            const float alpha = exp2f(old - base);
            sm.alpha[r] = alpha;
            sm.m[r] = now;
            sm.l[r] = sm.l[r] * alpha + sum;
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < kRowsPer; ++r) acc[r] *= sm.alpha[rg * kRowsPer + r];
#pragma unroll 8
      for (int key = 0; key < kKeys; ++key) {
        const float vv = sm.v[key][col];
#pragma unroll
        for (int r = 0; r < kRowsPer; ++r) {
          // a weight of zero leaves out its row, whatever it holds
          const float p = sm.p[rg * kRowsPer + r][key];
          acc[r] = fmaf(p, p == 0.f ? 0.f : vv, acc[r]);
        }
      }
    }
    __syncthreads();
    // ---- finished, or a partial result
    if (t0 == 0 && n == pl.tiles) {
      if (col < a.head_dim) {
#pragma unroll
        for (int r = 0; r < kRowsPer; ++r) {
          const int rr = rg * kRowsPer + r;
          if (rr < rows) {
            const float l = sm.l[rr];
            uint8_t* dst = const_cast<uint8_t*>(row_ptr(a.o, a.o_seq, a.o_head, a.o_tok, rr));
            reinterpret_cast<typename E::T*>(dst)[col] = E::round(l == 0.f ? 0.f : acc[r] / l);
          }
        }
      }
    } else {
      float* part = a.partial + static_cast<int64_t>(2 * blockIdx.x + (t0 == 0 ? 1 : 0)) *
                                    (kRows * (DP + 2));
#pragma unroll
      for (int r = 0; r < kRowsPer; ++r) part[(rg * kRowsPer + r) * DP + col] = acc[r];
      if (tid < kRows) {
        part[kRows * DP + tid] = sm.m[tid];
        part[kRows * DP + kRows + tid] = sm.l[tid];
      }
    }
    const bool first = t0 == 0, last = t0 + n == pl.tiles;
    if (!(first && last)) {
      const int from = run.ends_in(pl) ? run.end_first : (first ? blockIdx.x : run.first_run);
      const int to = run.ends_in(pl) ? run.end_last : blockIdx.x;
      if (a.counters) {
        static_assert(sizeof(JoinSmem<DP, kThreads / 32>) <= sizeof(sm.k), "joins in place");
        join_if_last<kRows, DP, DT, kThreads / 32>(
            a, pl.b, pl.h, pl.rt, rows, from, to,
            reinterpret_cast<JoinSmem<DP, kThreads / 32>*>(&sm.k[0][0]));
      } else if (tid == 0 && last) {
        a.desc[unit_of(a, pl)] = make_int2(from, to);
      }
    } else if (tid == 0 && !a.counters) {
      a.desc[unit_of(a, pl)] = make_int2(0, 0);
    }
    pl.t += n;
    if (pl.t == pl.tiles) pl = next_unit<PlainGrid>(a, pl);
    __syncthreads();
  }
}

// -------------------------------------------------------------------- host
using namespace b200paged;

int64_t round16(int64_t n) { return (n + 15) & ~static_cast<int64_t>(15); }

// The kernel a call takes, its row tile (`rm` places, `rows` of them used), key tile and
// padded head dim, and the most CTAs it may run on an SM.
enum Kernel { kPlain, kFewRows, kManyRows };
struct Choice {
  Kernel kernel;
  int rm, rows, tn, dp;
  int ctas_per_sm;
};

// Queries and pools can be read through tensor maps: page boxes of `box_rows` or more (8 at
// least), and strides that move.
bool by_tensor_maps(const b200_tree_attn_params* p, int box_rows) {
  const b200_cache& c = p->cache;
  if (box_rows_of(c.page_size) < box_rows) return false;
  const int64_t extent[4] = {1, c.pages, c.kv_heads, c.page_size};
  for (int d = 1; d < 4; ++d)
    if (extent[d] > 1 && (c.k_stride[d] <= 0 || c.v_stride[d] <= 0)) return false;
  const int64_t q_extent[3] = {c.batch, p->heads, p->tokens};
  for (int d = 0; d < 3; ++d)
    if (q_extent[d] > 1 && p->q_stride[d] <= 0) return false;
  return true;
}

Choice choose(const b200_tree_attn_params* p) {
  const int dp = p->cache.head_dim <= 64 ? 64 : 128;
  if (p->cache.dtype == B200_ATTN_DTYPE_FP32) return Choice{kPlain, kRows, kRows, kKeys, dp, dp == 64 ? 4 : 2};
  const int64_t rows = p->tokens * (p->heads / p->cache.kv_heads);
  const int64_t group = p->heads / p->cache.kv_heads;
  // More than 16 rows: the tcgen05 kernel, unless its boxes would be so small that issuing
  // them takes longer than their bytes.  Up to 32 rows, D 128: ahead of the few-row kernel
  // with boxes of 8 keys already (131001 keys: 143 us against 166 us; 64 sequences of 3000 to
  // 8000 keys: 333 against 444; of up to 400: 51 against 64).  D 64: behind with boxes of
  // 16 (64 sequences of 3000 to 8000: 258 us against 222 us), but not where the slots hold
  // short contexts only, whose ends of units weigh more (64 of up to 400: 45 us against 46
  // us with boxes of 8).
  // Up to 16 rows the few-row kernel reads near the rate of memory (16 rows: 103 us, 4
  // rows: 97 us).
  const bool eight = rows > 32 || dp == 128 || p->cache.slots * p->cache.page_size <= 2048;
  const int least = eight ? 8 : 32;
  if (rows > 16 && group <= 128 && by_tensor_maps(p, least)) {
    // whole tokens to a tile of 128 places
    const int tile = static_cast<int>(128 / group * group);
    if (rows <= tile) return Choice{kManyRows, 128, tile, 128, dp, 1};
    return Choice{kManyRows, 256, 2 * tile, 128, dp, 1};
  }
  // (the shapes do not depend on the head dim)
  if (rows <= 16) return Choice{kFewRows, 16, 16, RowShape<1, false, 64>::kTile, dp, RowShape<1, false, 64>::kCtas};
  return Choice{kFewRows, 32, 32, RowShape<2, false, 64>::kTile, dp, 1};
}

// Whether the output can share bytes with what the call reads, or with itself.  In the place
// of the queries, element for element, it may: a unit's rows are written when all its CTAs have
// read its queries.
bool output_collides(const b200_tree_attn_params* p) {
  using b200attn::may_overlap;
  using b200attn::stretches_of;
  const b200_cache& c = p->cache;
  const int64_t eb = elem_bytes(c.dtype);
  const int64_t rows[3] = {c.batch, p->heads, p->tokens};
  const int64_t pool[3] = {c.pages, c.kv_heads, c.page_size};
  bool in_place = p->q == p->o;
  for (int d = 0; d < 3; ++d) {
    if (rows[d] <= 1) continue;
    if (p->o_stride[d] == 0) return true;
    in_place = in_place && p->o_stride[d] == p->q_stride[d];
  }
  const auto o = stretches_of(p->o, p->o_stride, rows, 3, c.head_dim, eb);
  if (!in_place && may_overlap(o, stretches_of(p->q, p->q_stride, rows, 3, c.head_dim, eb)))
    return true;
  if (may_overlap(o, stretches_of(c.k, c.k_stride + 1, pool, 3, c.head_dim, eb)) ||
      may_overlap(o, stretches_of(c.v, c.v_stride + 1, pool, 3, c.head_dim, eb)) ||
      may_overlap(o, stretches_of(c.page_table, &c.table_stride, &c.batch, 1, c.slots, 4)) ||
      may_overlap(o, stretches_of(c.seq_lens, nullptr, nullptr, 0, c.batch, 4)))
    return true;
  const int64_t marks[3] = {c.batch, p->tokens, p->tokens};
  return (p->mask && may_overlap(o, stretches_of(p->mask, p->mask_stride, marks, 3, 1, 1))) ||
         (p->draft_lens && may_overlap(o, stretches_of(p->draft_lens, nullptr, nullptr, 0, c.batch, 4)));
}

int64_t row_tiles(const b200_tree_attn_params* p, const Choice& c) {
  return (p->tokens * (p->heads / p->cache.kv_heads) + c.rows - 1) / c.rows;
}

int64_t units_of(const b200_tree_attn_params* p, const Choice& c) {
  return p->cache.batch * p->cache.kv_heads * row_tiles(p, c);
}

// Most SMs that a call runs on.  Workspaces are sized on the host for as many, without asking
// a device: more than the 148 of a B200, and every one counts (256 rows of 128 columns: 42.6 MB
// for 160 SMs).
constexpr int64_t kMaxSms = 160;

// Whether the cut units of few rows get a join kernel of their own although the attention
// kernel could join them: a long context of several rows leaves many partial results to the one
// CTA that would (one sequence, 16 rows: 33.8 us against 23.4 us at 4000 keys, 19.6 against 18.6
// at 1000, 112 against 103 at 131001; 4 sequences of 4000: 26.4 against 24.2).  For short contexts the second launch costs
// more (500 keys, 8 rows: 15.0 us against 17.0 us).
bool join_apart(const b200_tree_attn_params* p, const Choice& c, int64_t runs, int64_t units) {
  return c.kernel != kManyRows && p->tokens * (p->heads / p->cache.kv_heads) > 4 &&
         p->cache.slots * p->cache.page_size >= 12 * c.tn && runs >= 8 * units;
}

// CTAs of a call on a GPU of `sms` SMs: no more than there can be key tiles.
int64_t runs_of(const b200_tree_attn_params* p, const Choice& c, int64_t sms) {
  const int64_t keys = p->cache.slots * p->cache.page_size;
  const double tiles = static_cast<double>(p->cache.batch * p->cache.kv_heads) *
                       static_cast<double>(row_tiles(p, c)) *
                       static_cast<double>((keys + c.tn - 1) / c.tn);
  const int64_t most = (sms < kMaxSms ? sms : kMaxSms) * c.ctas_per_sm;
  return tiles < static_cast<double>(most) ? static_cast<int64_t>(tiles) : most;
}

int64_t desc_bytes(const b200_tree_attn_params* p, const Choice& c) {
  return round16(8 * p->cache.batch * p->cache.kv_heads * row_tiles(p, c));
}


template <int RM, int DP, int DT, int WARPS>
int32_t run_join_rows(const Args& a, int64_t units, bool spread, cudaStream_t s) {
  if (spread)
    return launch(join_spread_kernel<RM, DP, DT>, dim3(static_cast<unsigned>(units), RM / 4),
                  dim3(32 * kJoinWarps), 0, s, a);
  return launch(join_rows_kernel<RM, DP, DT, WARPS>, dim3(static_cast<unsigned>(units)),
                dim3(32 * WARPS), 0, s, a);
}

template <int RM, int DP, int DT>
int32_t run_join_columns(const Args& a, int64_t units, cudaStream_t s) {
  // few units: the blocks that share a unit's rows share its columns too
  const bool spread = units * (RM / 32) < 300;
  return launch(spread ? join_columns_kernel<RM, DP, DT, true> : join_columns_kernel<RM, DP, DT, false>,
                dim3(static_cast<unsigned>(units), RM / 32, spread ? DP / kJoinCols : 1),
                dim3(32 * kJoinWarps), 0, s, a);
}

template <int RM, int DP, int DT>
int32_t run_one(void (*kernel)(Args), int threads, int smem, const Args& a, int runs, int device,
                cudaStream_t s) {
  static std::once_flag once[kMaxDevices];
  static cudaError_t err[kMaxDevices];
  std::call_once(once[device], [&] {
    err[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  if (err[device] != cudaSuccess) {
    set_error(cudaGetErrorString(err[device]));
    return B200_ATTN_ERR_LAUNCH;
  }
  return launch(kernel, dim3(runs), dim3(threads), smem, s, a);
}

// One kernel over the runs, and where it does not join the units that were cut, one that
// does.
template <int DP, int DT>
int32_t run_width(const Choice& c, const Args& a, int runs, int64_t units, bool spread, int device,
                  cudaStream_t s) {
  int32_t rc;
  if constexpr (DT == B200_ATTN_DTYPE_FP32) {
    rc = run_one<16, DP, DT>(plain_kernel<DP, DT>, kThreads, sizeof(PlainSmem<DP>), a, runs, device,
                             s);
    return rc != B200_ATTN_OK || a.counters ? rc : run_join_rows<kRows, DP, DT, kThreads / 32>(a, units, spread, s);
  } else {
    using Few = RowShape<1, true, DP>;
    using One = RowShape<1, false, DP>;
    using Two = RowShape<2, false, DP>;
    if (c.kernel == kManyRows)
      rc = launch_tiles(c.rm, c.dp, DT, a, a.kv_heads * a.group, runs, device, s);
    else if (a.tokens * a.group <= 8)
      rc = run_one<8, DP, DT>(rows_kernel<Few, DT>, Few::kThreads, Few::kSmemBytes, a, runs, device, s);
    else if (c.rm == 16)
      rc = run_one<16, DP, DT>(rows_kernel<One, DT>, One::kThreads, One::kSmemBytes, a, runs, device,
                               s);
    else
      rc = run_one<32, DP, DT>(rows_kernel<Two, DT>, Two::kThreads, Two::kSmemBytes, a, runs, device,
                               s);
    if (rc != B200_ATTN_OK || a.counters) return rc;
    switch (c.rm) {
      case 16: return run_join_rows<16, DP, DT, One::kWarps>(a, units, spread, s);
      case 32: return run_join_rows<32, DP, DT, Two::kWarps>(a, units, spread, s);
      case 128: return run_join_columns<128, DP, DT>(a, units, s);
      default: return run_join_columns<256, DP, DT>(a, units, s);
    }
  }
}

template <int DT>
int32_t run_type(const Choice& c, const Args& a, int runs, int64_t units, bool spread, int device,
                 cudaStream_t s) {
  return c.dp == 64 ? run_width<64, DT>(c, a, runs, units, spread, device, s)
                    : run_width<128, DT>(c, a, runs, units, spread, device, s);
}

}  // namespace
}  // namespace b200tree

using namespace b200tree;

extern "C" int32_t b200_tree_attn_check(const b200_tree_attn_params* p) {
  if (!p) return B200_ATTN_ERR_INVALID_ARGUMENT;
  const b200_cache& c = p->cache;
  const int32_t rc = b200_cache_check(&c);
  if (rc != B200_ATTN_OK) return rc;
  if (!c.seq_lens || !p->q || !p->o || c.layers != 1 || p->tokens < 1 || p->heads < 1 || p->heads % c.kv_heads ||
      p->reserved != 0)
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (!(p->scale > 0.f) || !std::isfinite(p->scale)) return B200_ATTN_ERR_INVALID_ARGUMENT;
  // rows, units and row pieces of a call are numbered in 32 bits
  if (p->tokens > (1 << 24) || p->heads > (1 << 16) || p->tokens * p->heads > (1ll << 25) ||
      c.batch * p->heads * p->tokens > 0x7fffffffll)
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  const int64_t extent[3] = {c.batch, p->heads, p->tokens};
  const int64_t eb = b200paged::elem_bytes(c.dtype);
  if (!b200paged::vectors_aligned(p->q, p->q_stride, extent, 3, eb) ||
      !b200paged::vectors_aligned(p->o, p->o_stride, extent, 3, eb) ||
      ((reinterpret_cast<uintptr_t>(p->draft_lens) | reinterpret_cast<uintptr_t>(p->counters)) & 3u))
    return B200_ATTN_ERR_ALIGNMENT;
  // so are all key tiles of a call
  const Choice ch = choose(p);
  if (static_cast<double>(c.batch * c.kv_heads * row_tiles(p, ch)) *
          static_cast<double>(c.slots * c.page_size / ch.tn + 4) > 2e9)
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (p->mask && (p->mask_stride[0] < 0 || p->mask_stride[1] < 0 || p->mask_stride[2] < 0))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (output_collides(p)) return B200_ATTN_ERR_INVALID_ARGUMENT;
  return B200_ATTN_OK;
}

extern "C" int64_t b200_tree_attn_workspace_bytes(const b200_tree_attn_params* p) {
  if (b200_tree_attn_check(p) != B200_ATTN_OK) return 0;
  const Choice c = choose(p);
  return desc_bytes(p, c) + 2 * runs_of(p, c, kMaxSms) * 4 * c.rm * (c.dp + 2);
}

extern "C" int32_t b200_tree_attn_fwd(const b200_tree_attn_params* p, void* stream) {
  int32_t rc = b200_tree_attn_check(p);
  if (rc != B200_ATTN_OK) return rc;
  if (!p->workspace || p->workspace_bytes < b200_tree_attn_workspace_bytes(p))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(p->workspace) & 15u) return B200_ATTN_ERR_ALIGNMENT;
  const b200_cache& c = p->cache;
  b200paged::DeviceScope scope;
  if ((rc = scope.enter(p->q, "q is not a device pointer")) != B200_ATTN_OK) return rc;
  const Choice ch = choose(p);
  const int64_t eb = b200paged::elem_bytes(c.dtype);
  Args a{};
  if ((rc = b200attn::resolve_error_word(c.error_word, &a.err)) != B200_ATTN_OK) return rc;
  a.k = static_cast<const uint8_t*>(c.k);
  a.v = static_cast<const uint8_t*>(c.v);
  a.k_page = c.k_stride[1] * eb;
  a.k_head = c.k_stride[2] * eb;
  a.k_row = c.k_stride[3] * eb;
  a.v_page = c.v_stride[1] * eb;
  a.v_head = c.v_stride[2] * eb;
  a.v_row = c.v_stride[3] * eb;
  a.table = c.page_table;
  a.table_stride = c.table_stride;
  a.lens = c.seq_lens;
  a.drafts = p->draft_lens;
  a.q = static_cast<const uint8_t*>(p->q);
  a.o = static_cast<uint8_t*>(p->o);
  a.q_seq = p->q_stride[0] * eb;
  a.q_head = p->q_stride[1] * eb;
  a.q_tok = p->q_stride[2] * eb;
  a.o_seq = p->o_stride[0] * eb;
  a.o_head = p->o_stride[1] * eb;
  a.o_tok = p->o_stride[2] * eb;
  a.mask = p->mask;
  a.m_seq = p->mask_stride[0];
  a.m_row = p->mask_stride[1];
  a.m_col = p->mask_stride[2];
  a.batch = static_cast<int32_t>(c.batch);
  a.kv_heads = static_cast<int32_t>(c.kv_heads);
  a.group = static_cast<int32_t>(p->heads / c.kv_heads);
  a.tokens = static_cast<int32_t>(p->tokens);
  a.head_dim = static_cast<int32_t>(c.head_dim);
  a.slots = static_cast<int32_t>(c.slots);
  a.pages = static_cast<int32_t>(c.pages);
  a.page_size = static_cast<int32_t>(c.page_size);
  a.unit_rows = ch.rows;
  a.row_tiles = static_cast<int32_t>(row_tiles(p, ch));
  a.scale_log2 = p->scale * 1.4426950408889634f;
  a.desc = static_cast<int2*>(p->workspace);
  a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(p->workspace) + desc_bytes(p, ch));
  const int runs = static_cast<int>(runs_of(p, ch, b200paged::sm_count(scope.device)));
  a.runs = runs;
  const int64_t units = units_of(p, ch);
  const bool spread = join_apart(p, ch, runs, units);
  if (ch.kernel != kManyRows && !spread && units <= B200_TREE_ATTN_COUNTERS) a.counters = p->counters;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (c.dtype) {
    case B200_ATTN_DTYPE_BF16:
      return run_type<B200_ATTN_DTYPE_BF16>(ch, a, runs, units, spread, scope.device, s);
    case B200_ATTN_DTYPE_FP16:
      return run_type<B200_ATTN_DTYPE_FP16>(ch, a, runs, units, spread, scope.device, s);
    default:
      return run_type<B200_ATTN_DTYPE_FP32>(ch, a, runs, units, spread, scope.device, s);
  }
}
