// paged_cache.cu — page operations of the paged key/value cache on B200:
// append, accept, reserve (with copy on write), fork, free, compact.
//
// They move rows and integers; what bounds them is HBM for large calls (each
// moved byte is read once and written once) and launches for small ones.  Rows
// move 16 bytes per thread with several loads in flight before the first store;
// the bookkeeping (free pages in ascending order, all-or-nothing) is planned by
// one CTA with block scans, so its result does not depend on any execution
// order, and a second kernel moves the planned rows.
#include <cuda_runtime.h>

#include <cstdint>

#include "b200_paged.h"
#include "byte_range.h"
#include "error_word.cuh"
#include "paged_host.h"
#include "sm100_ptx.cuh"

namespace b200paged {

using b200attn::ByteRange;
using b200attn::rows_range;
using b200attn::report_error;

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;

// The cache as the kernels see it.
struct Pool {
  uint8_t* k;
  uint8_t* v;
  int64_t k_layer, k_page, k_head, k_row;  // bytes
  int64_t v_layer, v_page, v_head, v_row;
  int32_t* table;
  int64_t table_stride;
  int32_t* lens;
  int32_t* refs;
  int32_t batch, slots, pages, page_size, layers, heads;
  int32_t chunks;  // 16-byte pieces of a row
  int32_t* err;
};

// Page of slot `s` of sequence `b`, or -1 (reported) when there is none.
__device__ __forceinline__ int page_at(const Pool& c, int b, uint32_t s) {
  int p = -1;
  if (s < static_cast<uint32_t>(c.slots))
    p = c.table[static_cast<int64_t>(b) * c.table_stride + s];
  if (p < 0 || p >= c.pages) {
    report_error(c.err, B200_ATTN_DEVERR_BOUNDS);
    return -1;
  }
  return p;
}

// ------------------------------------------------------------------ append
struct Rows {
  const uint8_t* k;
  const uint8_t* v;
  int64_t k_layer, k_seq, k_head, k_tok;  // bytes
  int64_t v_layer, v_seq, v_head, v_tok;
  const int32_t* counts;
  int32_t tokens;
};

// One thread moves one 16-byte piece of one token's key and value row in up to
// kLayerGroup layers: the page is looked up once, and up to 2 x kLayerGroup
// loads are in flight before the stores.  Bound by HBM: 64 sequences of 16 tokens in
// 32 layers (268 MB read and written) take 45 us, the rate of a plain copy of as many
// bytes (44 us).  Groups of 2 or 8 layers, token-major order and streaming stores were
// all within 3 % or slower.
constexpr int kLayerGroup = 4;

__global__ void __launch_bounds__(kCopyThreads) append_kernel(const Pool c, const Rows r) {
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * kCopyThreads + threadIdx.x;
  const int64_t per_seq = static_cast<int64_t>(r.tokens) * c.heads * c.chunks;
  if (idx >= per_seq * c.batch) return;
  const int b = static_cast<int>(idx / per_seq);
  uint32_t rest = static_cast<uint32_t>(idx - b * per_seq);
  const uint32_t per_tok = static_cast<uint32_t>(c.heads) * c.chunks;
  const int j = static_cast<int>(rest / per_tok);
  rest -= j * per_tok;
  const int h = static_cast<int>(rest / static_cast<uint32_t>(c.chunks));
  const int x = static_cast<int>(rest) - h * c.chunks;
  const int count = r.counts ? r.counts[b] : r.tokens;
  const int len = c.lens[b];
  const bool given = count >= 0 && count <= r.tokens;
  if (given && j >= count) return;
  if (!given || len < 0) {  // (len + j would wrap round to the first tokens)
    report_error(c.err, B200_ATTN_DEVERR_BOUNDS);
    return;
  }
  const uint32_t at = static_cast<uint32_t>(len) + j;
  const uint32_t slot = at / static_cast<uint32_t>(c.page_size);
  const int page = page_at(c, b, slot);
  if (page < 0) return;
  const int64_t row = at - slot * c.page_size;
  const uint8_t* ks = r.k + b * r.k_seq + h * r.k_head + j * r.k_tok + 16 * x;
  const uint8_t* vs = r.v + b * r.v_seq + h * r.v_head + j * r.v_tok + 16 * x;
  uint8_t* kd = c.k + page * c.k_page + h * c.k_head + row * c.k_row + 16 * x;
  uint8_t* vd = c.v + page * c.v_page + h * c.v_head + row * c.v_row + 16 * x;
  const int l0 = blockIdx.y * kLayerGroup;
  uint4 a[kLayerGroup], w[kLayerGroup];
#pragma unroll
  for (int l = 0; l < kLayerGroup; ++l) {
    if (l0 + l < c.layers) {
      a[l] = __ldcs(reinterpret_cast<const uint4*>(ks + (l0 + l) * r.k_layer));
      w[l] = __ldcs(reinterpret_cast<const uint4*>(vs + (l0 + l) * r.v_layer));
    }
  }
#pragma unroll
  for (int l = 0; l < kLayerGroup; ++l) {
    if (l0 + l < c.layers) {
      *reinterpret_cast<uint4*>(kd + (l0 + l) * c.k_layer) = a[l];
      *reinterpret_cast<uint4*>(vd + (l0 + l) * c.v_layer) = w[l];
    }
  }
}

// ------------------------------------------------------------------ accept
// One thread owns one 16-byte column of one (layer, K or V, sequence, head) and
// moves it along the path in order.  paths increases strictly, so paths[j] >= j:
// a row is overwritten only by the move of an earlier or the same step, whose
// batch of loads was complete before its stores.  Paths of up to 16 rows in 64 sequences
// and 32 layers: 16 us, of which the launch and the chain path -> page -> row are most.
constexpr int kPathBatch = 8;

__global__ void __launch_bounds__(kCopyThreads)
    accept_kernel(const Pool c, const int32_t* paths, int64_t path_stride, int32_t width,
                  const int32_t* counts, int32_t* new_lens) {
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * kCopyThreads + threadIdx.x;
  const uint32_t per_seq = static_cast<uint32_t>(c.heads) * c.chunks;
  if (idx >= static_cast<int64_t>(per_seq) * c.batch) return;
  const int b = static_cast<int>(idx / per_seq);
  const uint32_t rest = static_cast<uint32_t>(idx - static_cast<int64_t>(b) * per_seq);
  const int h = static_cast<int>(rest / static_cast<uint32_t>(c.chunks));
  const int x = static_cast<int>(rest) - h * c.chunks;
  const int len = c.lens[b];
  int n = counts[b];
  const int64_t room = static_cast<int64_t>(c.slots) * c.page_size;
  if (n < 0 || n > width || len < 0 || (n > 0 && static_cast<int64_t>(len) + n > room)) {
    report_error(c.err, B200_ATTN_DEVERR_BOUNDS);
    n = 0;
  }
  if (rest == 0 && blockIdx.y == 0) new_lens[b] = len + n;
  const int layer = blockIdx.y >> 1;
  const bool value = blockIdx.y & 1;
  uint8_t* base = (value ? c.v + layer * c.v_layer + h * c.v_head
                         : c.k + layer * c.k_layer + h * c.k_head) + 16 * x;
  const int64_t page_bytes = value ? c.v_page : c.k_page;
  const int64_t row_bytes = value ? c.v_row : c.k_row;
  const int32_t* path = paths + b * path_stride;
  const uint32_t size = static_cast<uint32_t>(c.page_size);
  for (int j0 = 0; j0 < n; j0 += kPathBatch) {
    uint4 a[kPathBatch];
    int from[kPathBatch];
#pragma unroll
    for (int u = 0; u < kPathBatch; ++u) {
      from[u] = -1;
      const int j = j0 + u;
      if (j >= n) continue;
      const int p = path[j];
      if (p == j) continue;
      const uint32_t at = static_cast<uint32_t>(len) + static_cast<uint32_t>(max(p, 0));
      const uint32_t slot = at / size;
      const int page = page_at(c, b, p < 0 ? ~0u : slot);
      if (page < 0) continue;
      from[u] = p;
      a[u] = *reinterpret_cast<const uint4*>(
          base + page * page_bytes + static_cast<int64_t>(at - slot * size) * row_bytes);
    }
#pragma unroll
    for (int u = 0; u < kPathBatch; ++u) {
      if (from[u] < 0) continue;
      const uint32_t at = static_cast<uint32_t>(len) + j0 + u;
      const uint32_t slot = at / size;
      const int page = page_at(c, b, slot);
      if (page < 0) continue;
      *reinterpret_cast<uint4*>(base + page * page_bytes +
                                static_cast<int64_t>(at - slot * size) * row_bytes) = a[u];
    }
  }
}

// ------------------------------------------------------------- block scans
// Exclusive sum over the CTA's threads in thread order; *total gets the sum.
// `part` is a scratch of 33 ints.
__device__ __forceinline__ int block_scan(int v, int* part, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  __syncthreads();  // part may still be read from the scan before
  if (lane == 31) part[warp] = s;
  __syncthreads();
  if (warp == 0) {
    const int n = static_cast<int>(blockDim.x) >> 5;
    const int w = lane < n ? part[lane] : 0;
    int t = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += u;
    }
    if (lane < n) part[lane] = t - w;
    if (lane == 31) part[32] = t;
  }
  __syncthreads();
  *total = part[32];
  return part[warp] + s - v;
}

// One planned move of rows 0..rows-1 of page `src` to page `dst`.
struct Move {
  int32_t src, dst, rows, pad;
};

// Scratch of reserve and compact: the number of moves, the moves, the free
// pages (compact: the places of moved pages) and reserve's flags.
struct Scratch {
  int32_t* count;    // [4]
  Move* moves;       // [max(batch, pages)]
  int32_t* list;     // [pages]
  uint32_t* flags;   // [ceil(batch * slots / 32) + 32]
};

// ------------------------------------------------------------------- moves
// Warps take (move, layer, K or V, head) segments in turn; a segment's rows are
// contiguous pieces of 16 bytes, and a lane keeps kUnroll of them in flight.  Stored as
// streaming: nothing reads the rows soon (copies of 224 part-filled pages in 32 layers,
// 451 MB: 74 us = 6.1 TB/s against 87 us with plain stores; 8 pieces in flight 100 us, 2:
// 95 us).  Bound by HBM; compacting 186 whole pages of 32 layers, 780 MB, takes 112 us with
// its plan, part of it out of L2.
constexpr int kUnroll = 4;

// By warp `warp` of `warps`.
__device__ __forceinline__ void move_rows(const Pool& c, const Scratch& w, int count, int warp,
                                          int warps) {
  const int lane = threadIdx.x & 31;
  const int per_move = c.layers * 2 * c.heads;
  const int64_t items = static_cast<int64_t>(count) * per_move;
  for (int64_t it = warp; it < items; it += warps) {
    const int i = static_cast<int>(it / per_move);
    const int rest = static_cast<int>(it - static_cast<int64_t>(i) * per_move);
    const int h = rest % c.heads, lv = rest / c.heads;
    const int layer = lv >> 1;
    const bool value = lv & 1;
    const Move m = w.moves[i];
    uint8_t* base = value ? c.v + layer * c.v_layer + h * c.v_head
                          : c.k + layer * c.k_layer + h * c.k_head;
    const int64_t page_bytes = value ? c.v_page : c.k_page;
    const int64_t row_bytes = value ? c.v_row : c.k_row;
    const uint8_t* src = base + m.src * page_bytes;
    uint8_t* dst = base + m.dst * page_bytes;
    const int pieces = m.rows * c.chunks;
    for (int x0 = lane; x0 < pieces; x0 += 32 * kUnroll) {
      uint4 a[kUnroll];
      int64_t off[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int x = x0 + 32 * u;
        const int row = x / c.chunks;
        off[u] = row * row_bytes + 16 * (x - row * c.chunks);
        if (x < pieces) a[u] = __ldcs(reinterpret_cast<const uint4*>(src + off[u]));
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (x0 + 32 * u < pieces) __stcs(reinterpret_cast<uint4*>(dst + off[u]), a[u]);
    }
  }
}

// Table entries follow the moved pages.  By thread `at` of `threads`.
__device__ __forceinline__ void remap_table(const Pool& c, const Scratch& w, int held, int64_t at,
                                            int64_t threads) {
  const int64_t entries = static_cast<int64_t>(c.batch) * c.slots;
  for (int64_t e = at; e < entries; e += threads) {
    int32_t* t = &c.table[(e / c.slots) * c.table_stride + e % c.slots];
    const int p = *t;
    if (p >= c.pages) report_error(c.err, B200_ATTN_DEVERR_BOUNDS);
    else if (p >= held && c.refs[p] == 0) *t = w.list[p];
  }
}

template <bool kRemap>
__global__ void __launch_bounds__(kCopyThreads) move_kernel(const Pool c, const Scratch w) {
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  const int warps = kCopyThreads / 32;
  move_rows(c, w, w.count[0], blockIdx.x * warps + (threadIdx.x >> 5), gridDim.x * warps);
  if constexpr (kRemap)
    remap_table(c, w, w.count[1], static_cast<int64_t>(blockIdx.x) * kCopyThreads + threadIdx.x,
                static_cast<int64_t>(gridDim.x) * kCopyThreads);
}

// ----------------------------------------------------------------- reserve
// One CTA.  The slots that the batch writes are numbered in (sequence, slot)
// order; pass 1 flags those that need a page, pass 2 lists as many free pages,
// lowest first, pass 3 gives them out.  Nothing is written to the table or the
// counts before the whole request is known to fit.
__global__ void __launch_bounds__(kPlanThreads)
    reserve_plan_kernel(const Pool c, const int32_t* tokens, int64_t uniform, int32_t* status,
                        const Scratch w, const bool moves_here) {
  extern __shared__ int32_t first_of[];  // [batch + 1] slots wanted before sequence b
  __shared__ int part[33];
  __shared__ int bad, carry, copies;
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  const int tid = threadIdx.x;
  if (tid == 0) bad = carry = copies = 0;
  __syncthreads();

  // slots wanted by each sequence
  for (int b0 = 0; b0 < c.batch; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int n = 0;
    if (b < c.batch) {
      const int64_t more = tokens ? tokens[b] : uniform;
      const int64_t len = c.lens[b];
      if (len < 0 || more < 0) {
        atomicOr(&bad, B200_CACHE_BAD_ENTRY);
      } else if (more > 0) {
        const int64_t end = len + more;
        if (end > static_cast<int64_t>(c.slots) * c.page_size)
          atomicOr(&bad, B200_CACHE_ROW_FULL);
        else
          n = static_cast<int>((end - 1) / c.page_size - len / c.page_size + 1);
      }
    }
    int total;
    const int before = block_scan(n, part, &total);
    if (b < c.batch) first_of[b] = carry + before;
    __syncthreads();
    if (tid == 0) carry += total;
    __syncthreads();
  }
  const int wanted = carry;
  if (tid == 0) first_of[c.batch] = wanted;
  __syncthreads();

  // sequence and slot of wanted slot number i
  auto locate = [&](int i, int* b, int* slot, bool* leading) {
    int lo = 0, hi = c.batch;  // first_of[lo] <= i < first_of[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first_of[mid] <= i) lo = mid;
      else hi = mid;
    }
    *b = lo;
    *leading = i == first_of[lo];
    *slot = c.lens[lo] / c.page_size + (i - first_of[lo]);
  };

  // pass 1: which of them need a page
  int need_total = 0;
  for (int i0 = 0; i0 < wanted; i0 += kPlanThreads) {
    const int i = i0 + tid;
    bool need = false;
    if (i < wanted) {
      int b, slot;
      bool leading;
      locate(i, &b, &slot, &leading);
      const int e = c.table[static_cast<int64_t>(b) * c.table_stride + slot];
      if (e >= c.pages || (e < 0 && e != -1)) atomicOr(&bad, B200_CACHE_BAD_ENTRY);
      else need = e < 0 || c.refs[e] > 1;
      // committed rows without a page cannot be continued
      if (e < 0 && leading && c.lens[b] % c.page_size != 0) atomicOr(&bad, B200_CACHE_BAD_ENTRY);
    }
    const uint32_t word = __ballot_sync(0xffffffffu, need);
    if ((tid & 31) == 0) w.flags[(i0 + tid) >> 5] = word;
    need_total += __syncthreads_count(need);
  }

  // pass 2: the lowest need_total free pages
  int have = 0;
  for (int p0 = 0; p0 < c.pages && have < need_total; p0 += 4 * kPlanThreads) {
    const int p = p0 + 4 * tid;
    bool f[4];
    int n = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      f[u] = p + u < c.pages && c.refs[p + u] == 0;
      n += f[u];
    }
    int total;
    int at = have + block_scan(n, part, &total);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (f[u]) {
        if (at < need_total) w.list[at] = p + u;
        ++at;
      }
    have += total;
  }
  __syncthreads();
  const int code = bad | (have < need_total ? B200_CACHE_NO_PAGES : 0);
  if (tid == 0) *status = code;

  // pass 3: give them out
  if (code == 0) {
    int given = 0;
    for (int i0 = 0; i0 < wanted; i0 += kPlanThreads) {
      const int i = i0 + tid;
      const bool need = i < wanted && ((w.flags[i >> 5] >> (i & 31)) & 1u);
      int total;
      const int rank = given + block_scan(need ? 1 : 0, part, &total);
      if (need) {
        int b, slot;
        bool leading;
        locate(i, &b, &slot, &leading);
        int32_t* entry = &c.table[static_cast<int64_t>(b) * c.table_stride + slot];
        const int old = *entry, page = w.list[rank];
        if (old >= 0) {
          atomicSub(&c.refs[old], 1);
          const int rows = leading ? c.lens[b] % c.page_size : 0;
          if (rows > 0) w.moves[atomicAdd(&copies, 1)] = Move{old, page, rows, 0};
        }
        c.refs[page] = 1;
        *entry = page;
      }
      given += total;
    }
  }
  __syncthreads();
  if (moves_here) move_rows(c, w, copies, tid >> 5, kPlanThreads / 32);
  else if (tid == 0) w.count[0] = copies;
}

// ----------------------------------------------------------------- compact
// Small calls are bound by the launch and by the plan's chain of passes: with moves of up to
// 1 MiB done by the planning CTA itself a call is one launch (a pool of 38 pages: 3.4 us
// behind the call before it).
// One CTA plans: n pages are held; the free pages before n (ascending) receive
// the held pages at or past n (ascending), so sources and destinations never
// meet and every page moves at most once.
__global__ void __launch_bounds__(kPlanThreads)
    compact_plan_kernel(const Pool c, int32_t* live, const Scratch w, const bool moves_here) {
  __shared__ int part[33];
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  const int tid = threadIdx.x;
  int n = 0;
  for (int p = tid; p < c.pages; p += kPlanThreads) n += c.refs[p] > 0;
  int held;
  block_scan(n, part, &held);
  int holes = 0, movers = 0;
  for (int p0 = 0; p0 < c.pages; p0 += 4 * kPlanThreads) {
    const int p = p0 + 4 * tid;
    bool hole[4], mover[4];
    int packed = 0;  // holes and movers of a chunk are at most 4096: two 16-bit sums
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool used = p + u < c.pages && c.refs[p + u] > 0;
      hole[u] = p + u < held && !used;
      mover[u] = p + u >= held && used;
      packed += (hole[u] ? 1 : 0) + (mover[u] ? 0x10000 : 0);
    }
    int total;
    const int before = block_scan(packed, part, &total);
    int ha = holes + (before & 0xffff), ma = movers + (before >> 16);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (hole[u]) w.moves[ha++].dst = p + u;
      if (mover[u]) w.moves[ma++].src = p + u;
      else if (p + u >= held && p + u < c.pages) w.list[p + u] = p + u;  // not held: stays
    }
    holes += total & 0xffff;
    movers += total >> 16;
  }
  __syncthreads();
  for (int i = tid; i < holes; i += kPlanThreads) {
    Move m = w.moves[i];
    w.moves[i].rows = c.page_size;
    w.list[m.src] = m.dst;
    c.refs[m.dst] = c.refs[m.src];
    c.refs[m.src] = 0;
  }
  if (tid == 0) {
    w.count[0] = holes;
    w.count[1] = held;
    *live = held;
  }
  if (moves_here) {
    __syncthreads();
    move_rows(c, w, holes, tid >> 5, kPlanThreads / 32);
    remap_table(c, w, held, tid, kPlanThreads);
  }
}

// ------------------------------------------------------------ fork and free
// One CTA per row.  Counts are integer sums, so the order of the CTAs does not
// matter; sources are not destinations, so no CTA reads what another writes.
__global__ void __launch_bounds__(kCopyThreads)
    fork_kernel(const Pool c, const int32_t* src, const int32_t* dst, int32_t n) {
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  const int i = blockIdx.x;
  const int s = src[i], d = dst[i];
  bool ok = s >= 0 && s < c.batch && d >= 0 && d < c.batch;
  for (int j = threadIdx.x; j < n; j += kCopyThreads)
    if (src[j] == d || (dst[j] == d && j != i)) ok = false;
  const int len = ok ? c.lens[s] : 0;
  if (len < 0 || len > static_cast<int64_t>(c.slots) * c.page_size) ok = false;
  ok = __syncthreads_and(ok);
  if (!ok) {
    if (threadIdx.x == 0) report_error(c.err, B200_ATTN_DEVERR_BOUNDS);
    return;
  }
  for (int m = threadIdx.x; m < c.slots; m += kCopyThreads) {
    int32_t* to = &c.table[static_cast<int64_t>(d) * c.table_stride + m];
    const int old = *to;
    int page = static_cast<int64_t>(m) * c.page_size < len
                   ? c.table[static_cast<int64_t>(s) * c.table_stride + m] : -1;
    if (old >= c.pages || page >= c.pages) report_error(c.err, B200_ATTN_DEVERR_BOUNDS);
    if (page >= c.pages) page = -1;
    if (old == page) continue;
    if (old >= 0 && old < c.pages) atomicSub(&c.refs[old], 1);
    if (page >= 0) atomicAdd(&c.refs[page], 1);
    *to = page;
  }
  if (threadIdx.x == 0) c.lens[d] = len;
}

__global__ void __launch_bounds__(kCopyThreads)
    free_kernel(const Pool c, const int32_t* rows, int32_t n) {
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  const int i = blockIdx.x;
  const int r = rows[i];
  if (r < 0 || r >= c.batch) {
    if (threadIdx.x == 0) report_error(c.err, B200_ATTN_DEVERR_BOUNDS);
    return;
  }
  bool again = false;  // a row given twice is freed by its first mention
  for (int j = threadIdx.x; j < i; j += kCopyThreads) again |= rows[j] == r;
  if (__syncthreads_or(again)) return;
  for (int m = threadIdx.x; m < c.slots; m += kCopyThreads) {
    int32_t* e = &c.table[static_cast<int64_t>(r) * c.table_stride + m];
    const int old = *e;
    if (old >= c.pages) report_error(c.err, B200_ATTN_DEVERR_BOUNDS);
    else if (old >= 0) atomicSub(&c.refs[old], 1);
    *e = -1;
  }
  if (threadIdx.x == 0) c.lens[r] = 0;
}

// -------------------------------------------------------------------- host
int64_t round16(int64_t n) { return (n + 15) & ~static_cast<int64_t>(15); }

int64_t move_slots(const b200_cache* c) { return c->batch > c->pages ? c->batch : c->pages; }

int64_t flag_words(const b200_cache* c) { return (c->batch * c->slots + 31) / 32 + 32; }

Scratch scratch_of(const b200_cache* c, void* ws) {
  uint8_t* p = static_cast<uint8_t*>(ws);
  Scratch s;
  s.count = reinterpret_cast<int32_t*>(p);
  p += 16;
  s.moves = reinterpret_cast<Move*>(p);
  p += 16 * move_slots(c);
  s.list = reinterpret_cast<int32_t*>(p);
  p += round16(4 * c->pages);
  s.flags = reinterpret_cast<uint32_t*>(p);
  return s;
}

Pool pool_of(const b200_cache* c) {
  const int64_t eb = elem_bytes(c->dtype);
  Pool p;
  p.k = static_cast<uint8_t*>(c->k);
  p.v = static_cast<uint8_t*>(c->v);
  p.k_layer = c->k_stride[0] * eb;
  p.k_page = c->k_stride[1] * eb;
  p.k_head = c->k_stride[2] * eb;
  p.k_row = c->k_stride[3] * eb;
  p.v_layer = c->v_stride[0] * eb;
  p.v_page = c->v_stride[1] * eb;
  p.v_head = c->v_stride[2] * eb;
  p.v_row = c->v_stride[3] * eb;
  p.table = c->page_table;
  p.table_stride = c->table_stride;
  p.lens = c->seq_lens;
  p.refs = c->page_refs;
  p.batch = static_cast<int32_t>(c->batch);
  p.slots = static_cast<int32_t>(c->slots);
  p.pages = static_cast<int32_t>(c->pages);
  p.page_size = static_cast<int32_t>(c->page_size);
  p.layers = static_cast<int32_t>(c->layers);
  p.heads = static_cast<int32_t>(c->kv_heads);
  p.chunks = static_cast<int32_t>(c->head_dim * eb / 16);
  p.err = nullptr;
  return p;
}

// The part of the description that every operation uses.
int32_t check_table(const b200_cache* c) {
  if (!c || !c->page_table || c->reserved != 0)
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (c->batch < 1 || c->batch > B200_CACHE_MAX_BATCH || c->slots < 1 || c->slots > (1ll << 24) ||
      c->pages < 1 || c->pages > (1ll << 30) || c->page_size < 1 || c->page_size > (1ll << 20))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  // token positions and slot numbers fit 32 bits, the latter up to the end of the planning
  // CTA's last round over them
  if (c->slots * c->page_size > 0x3fffffffll || c->batch * c->slots > 0x7fffffffll - kPlanThreads)
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (c->batch > 1 && c->table_stride < c->slots) return B200_ATTN_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(c->page_table) | reinterpret_cast<uintptr_t>(c->seq_lens) |
       reinterpret_cast<uintptr_t>(c->page_refs)) & 3u)
    return B200_ATTN_ERR_ALIGNMENT;
  return B200_ATTN_OK;
}

// Bytes of one page's keys and values in all layers.
int64_t page_bytes(const b200_cache* c) {
  return 2 * c->layers * c->kv_heads * c->page_size * c->head_dim * elem_bytes(c->dtype);
}

int32_t check_scratch(const b200_cache* c, const void* ws, int64_t bytes) {
  if (!ws || bytes < b200_cache_workspace_bytes(c)) return B200_ATTN_ERR_INVALID_ARGUMENT;
  return (reinterpret_cast<uintptr_t>(ws) & 15u) ? B200_ATTN_ERR_ALIGNMENT : B200_ATTN_OK;
}

// Bytes spanned by a 4-D view with a contiguous last dimension.
ByteRange span(const void* base, const int64_t* stride, const int64_t* extent, int64_t cols,
               int64_t eb) {
  int64_t last = cols;
  for (int d = 0; d < 4; ++d) last += (extent[d] - 1) * stride[d];
  const uintptr_t lo = reinterpret_cast<uintptr_t>(base);
  return ByteRange{lo, lo + static_cast<uintptr_t>(last * eb)};
}

// Up to so many bytes are moved by the planning CTA itself: a second launch takes longer.
constexpr int64_t kMovesHere = 1 << 20;

unsigned move_grid(int device, int64_t items) {
  const int64_t most = 8ll * sm_count(device);
  const int64_t want = (items + kCopyThreads / 32 - 1) / (kCopyThreads / 32);
  return static_cast<unsigned>(want < 1 ? 1 : (want < most ? want : most));
}

}  // namespace
}  // namespace b200paged

using namespace b200paged;

extern "C" int32_t b200_cache_check(const b200_cache* c) {
  const int32_t rc = check_table(c);
  if (rc != B200_ATTN_OK) return rc;
  if (!c->k || !c->v || c->layers < 1 || c->layers > (1 << 15) || c->kv_heads < 1 ||
      c->kv_heads > (1 << 16))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  // so are the pieces of a page in all layers that a move is cut into
  if (2 * c->layers * c->kv_heads > 0x7fffffffll) return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (!known_dtype(c->dtype) || c->head_dim < 8 || c->head_dim > 128 || c->head_dim % 8)
    return B200_ATTN_ERR_UNSUPPORTED;
  const int64_t extent[4] = {c->layers, c->pages, c->kv_heads, c->page_size};
  if (!vectors_aligned(c->k, c->k_stride, extent, 4, elem_bytes(c->dtype)) ||
      !vectors_aligned(c->v, c->v_stride, extent, 4, elem_bytes(c->dtype)))
    return B200_ATTN_ERR_ALIGNMENT;
  return B200_ATTN_OK;
}

extern "C" int64_t b200_cache_workspace_bytes(const b200_cache* c) {
  if (check_table(c) != B200_ATTN_OK) return 0;
  return 16 + 16 * move_slots(c) + round16(4 * c->pages) + round16(4 * flag_words(c));
}

extern "C" int32_t b200_cache_append(const b200_cache* c, const b200_cache_rows* rows,
                                     void* stream) {
  int32_t rc = b200_cache_check(c);
  if (rc != B200_ATTN_OK) return rc;
  if (!c->seq_lens || !rows || !rows->k || !rows->v || rows->tokens < 1) return B200_ATTN_ERR_INVALID_ARGUMENT;
  const int64_t eb = elem_bytes(c->dtype);
  const int64_t extent[4] = {c->layers, c->batch, c->kv_heads, rows->tokens};
  if (!vectors_aligned(rows->k, rows->k_stride, extent, 4, eb) ||
      !vectors_aligned(rows->v, rows->v_stride, extent, 4, eb) ||
      (reinterpret_cast<uintptr_t>(rows->counts) & 3u))
    return B200_ATTN_ERR_ALIGNMENT;
  Pool p = pool_of(c);
  if (rows->tokens * c->kv_heads * p.chunks > 0x7fffffffll)
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  const int64_t threads = c->batch * rows->tokens * c->kv_heads * p.chunks;
  if (threads > (1ll << 38)) return B200_ATTN_ERR_INVALID_ARGUMENT;
  // the rows must not lie in the pools: a piece could be overwritten before it is read
  const int64_t pe[4] = {c->layers, c->pages, c->kv_heads, c->page_size};
  const ByteRange kp = span(c->k, c->k_stride, pe, c->head_dim, eb);
  const ByteRange vp = span(c->v, c->v_stride, pe, c->head_dim, eb);
  const ByteRange kr = span(rows->k, rows->k_stride, extent, c->head_dim, eb);
  const ByteRange vr = span(rows->v, rows->v_stride, extent, c->head_dim, eb);
  if (kr.overlaps(kp) || kr.overlaps(vp) || vr.overlaps(kp) || vr.overlaps(vp))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  DeviceScope scope;
  if ((rc = scope.enter(c->k, "the pools are not device memory")) != B200_ATTN_OK) return rc;
  if ((rc = resolve_error_word(c->error_word, &p.err)) != B200_ATTN_OK) return rc;
  Rows r;
  r.k = static_cast<const uint8_t*>(rows->k);
  r.v = static_cast<const uint8_t*>(rows->v);
  r.k_layer = rows->k_stride[0] * eb;
  r.k_seq = rows->k_stride[1] * eb;
  r.k_head = rows->k_stride[2] * eb;
  r.k_tok = rows->k_stride[3] * eb;
  r.v_layer = rows->v_stride[0] * eb;
  r.v_seq = rows->v_stride[1] * eb;
  r.v_head = rows->v_stride[2] * eb;
  r.v_tok = rows->v_stride[3] * eb;
  r.counts = rows->counts;
  r.tokens = static_cast<int32_t>(rows->tokens);
  const dim3 grid(static_cast<unsigned>((threads + kCopyThreads - 1) / kCopyThreads),
                  static_cast<unsigned>((c->layers + kLayerGroup - 1) / kLayerGroup));
  return launch(append_kernel, grid, dim3(kCopyThreads), 0, static_cast<cudaStream_t>(stream), p,
                r);
}

extern "C" int32_t b200_cache_accept(const b200_cache* c, const int32_t* paths, int64_t width,
                                     int64_t path_stride, const int32_t* counts,
                                     int32_t* new_lens, void* stream) {
  int32_t rc = b200_cache_check(c);
  if (rc != B200_ATTN_OK) return rc;
  if (!c->seq_lens || !paths || !counts || !new_lens || new_lens == c->seq_lens || width < 1 ||
      width > 0x3fffffff || (c->batch > 1 && path_stride < 0))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(paths) | reinterpret_cast<uintptr_t>(counts) |
       reinterpret_cast<uintptr_t>(new_lens)) & 3u)
    return B200_ATTN_ERR_ALIGNMENT;
  // the new lengths must not lie where other blocks of the kernel still read
  const ByteRange out = rows_range(new_lens, 1, c->batch, 0, 4);
  if (out.overlaps(rows_range(c->seq_lens, 1, c->batch, 0, 4)) ||
      out.overlaps(rows_range(counts, 1, c->batch, 0, 4)) ||
      out.overlaps(rows_range(paths, c->batch, width, path_stride, 4)) ||
      out.overlaps(rows_range(c->page_table, c->batch, c->slots, c->table_stride, 4)))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  DeviceScope scope;
  if ((rc = scope.enter(c->k, "the pools are not device memory")) != B200_ATTN_OK) return rc;
  Pool p = pool_of(c);
  if ((rc = resolve_error_word(c->error_word, &p.err)) != B200_ATTN_OK) return rc;
  const int64_t threads = c->batch * c->kv_heads * p.chunks;
  const dim3 grid(static_cast<unsigned>((threads + kCopyThreads - 1) / kCopyThreads),
                  static_cast<unsigned>(2 * c->layers));
  if (grid.y > 65535u) return B200_ATTN_ERR_INVALID_ARGUMENT;
  return launch(accept_kernel, grid, dim3(kCopyThreads), 0, static_cast<cudaStream_t>(stream), p,
                paths, path_stride, static_cast<int32_t>(width), counts, new_lens);
}

extern "C" int32_t b200_cache_reserve(const b200_cache* c, const int32_t* tokens, int64_t uniform,
                                      int32_t* status, void* workspace, int64_t workspace_bytes,
                                      void* stream) {
  int32_t rc = b200_cache_check(c);
  if (rc != B200_ATTN_OK) return rc;
  if (!c->seq_lens || !c->page_refs || !status || (!tokens && (uniform < 0 || uniform > 0x3fffffff)))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if ((rc = check_scratch(c, workspace, workspace_bytes)) != B200_ATTN_OK) return rc;
  if ((reinterpret_cast<uintptr_t>(tokens) | reinterpret_cast<uintptr_t>(status)) & 3u)
    return B200_ATTN_ERR_ALIGNMENT;
  DeviceScope scope;
  if ((rc = scope.enter(c->k, "the pools are not device memory")) != B200_ATTN_OK) return rc;
  Pool p = pool_of(c);
  if ((rc = resolve_error_word(c->error_word, &p.err)) != B200_ATTN_OK) return rc;
  const Scratch w = scratch_of(c, workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // at most one page of a sequence is copied
  const bool here = c->batch * page_bytes(c) <= kMovesHere;
  rc = launch(reserve_plan_kernel, dim3(1), dim3(kPlanThreads),
              sizeof(int32_t) * static_cast<size_t>(c->batch + 1), s, p, tokens, uniform, status, w,
              here);
  if (rc != B200_ATTN_OK || here) return rc;
  return launch(move_kernel<false>, dim3(move_grid(scope.device, c->batch * c->layers * 2 * c->kv_heads)),
                dim3(kCopyThreads), 0, s, p, w);
}

extern "C" int32_t b200_cache_fork(const b200_cache* c, const int32_t* src, const int32_t* dst,
                                   int64_t n, void* stream) {
  int32_t rc = check_table(c);
  if (rc != B200_ATTN_OK) return rc;
  if (!c->seq_lens || !c->page_refs || n < 0 || n > c->batch || (n > 0 && (!src || !dst)))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) & 3u)
    return B200_ATTN_ERR_ALIGNMENT;
  if (n == 0) return B200_ATTN_OK;
  DeviceScope scope;
  if ((rc = scope.enter(c->page_table, "the page table is not device memory")) != B200_ATTN_OK)
    return rc;
  Pool p = pool_of(c);
  if ((rc = resolve_error_word(c->error_word, &p.err)) != B200_ATTN_OK) return rc;
  return launch(fork_kernel, dim3(static_cast<unsigned>(n)), dim3(kCopyThreads), 0,
                static_cast<cudaStream_t>(stream), p, src, dst, static_cast<int32_t>(n));
}

extern "C" int32_t b200_cache_free(const b200_cache* c, const int32_t* rows, int64_t n,
                                   void* stream) {
  int32_t rc = check_table(c);
  if (rc != B200_ATTN_OK) return rc;
  if (!c->seq_lens || !c->page_refs || n < 0 || n > (1 << 24) || (n > 0 && !rows))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(rows) & 3u) return B200_ATTN_ERR_ALIGNMENT;
  if (n == 0) return B200_ATTN_OK;
  DeviceScope scope;
  if ((rc = scope.enter(c->page_table, "the page table is not device memory")) != B200_ATTN_OK)
    return rc;
  Pool p = pool_of(c);
  if ((rc = resolve_error_word(c->error_word, &p.err)) != B200_ATTN_OK) return rc;
  return launch(free_kernel, dim3(static_cast<unsigned>(n)), dim3(kCopyThreads), 0,
                static_cast<cudaStream_t>(stream), p, rows, static_cast<int32_t>(n));
}

extern "C" int32_t b200_cache_compact(const b200_cache* c, int32_t* live, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  int32_t rc = b200_cache_check(c);
  if (rc != B200_ATTN_OK) return rc;
  if (!c->page_refs || !live) return B200_ATTN_ERR_INVALID_ARGUMENT;
  if ((rc = check_scratch(c, workspace, workspace_bytes)) != B200_ATTN_OK) return rc;
  if (reinterpret_cast<uintptr_t>(live) & 3u) return B200_ATTN_ERR_ALIGNMENT;
  DeviceScope scope;
  if ((rc = scope.enter(c->k, "the pools are not device memory")) != B200_ATTN_OK) return rc;
  Pool p = pool_of(c);
  if ((rc = resolve_error_word(c->error_word, &p.err)) != B200_ATTN_OK) return rc;
  const Scratch w = scratch_of(c, workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // at most every second page moves
  const bool here = c->pages / 2 * page_bytes(c) <= kMovesHere;
  rc = launch(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p, live, w, here);
  if (rc != B200_ATTN_OK || here) return rc;
  return launch(move_kernel<true>, dim3(move_grid(scope.device, c->pages * c->layers * 2 * c->kv_heads)),
                dim3(kCopyThreads), 0, s, p, w);
}
