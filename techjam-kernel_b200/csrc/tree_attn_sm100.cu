// tree_attn_sm100.cu — drafted-token attention for many rows (more than 16 a
// key head where pages allow large boxes, else more than 32), 16-bit caches, on the
// fifth-generation tensor cores: wide trees, and pieces of prompts over a cache.
//
// The mathematics is that of the kernel for few rows: one pass over the keys with a
// running maximum and sum.  What bounds it: R rows do 4 R D operations for the 4 D
// bytes of a key and value, so from about 260 rows the tensor cores, below it
// HBM.  Measured (bf16, D 128): 32 sequences of 1 to 8 thousand keys, 8 key heads, 256
// rows, 638 MB and 153 GFLOP: 212 us in a stream of calls (718 TFLOP/s and 3.0 TB/s, 43 and
// 46 % of the measured rates), where the board's power limit lowers the clock, and 177 us in
// runs too short for that; DRAM reads are the cache's bytes exactly.  A key tile of 256 rows takes about 4000 cycles, in which a softmax
// group waits for its scores (570 cycles of products and 300 to be seen), copies them (400),
// exponentiates (128 a thread, 3000 cycles with its waits) and hands over the weights;
// tensor pipe and exponential unit are each active under half of the time.
// 64 rows over 131001 keys: 537 MB, 111 us in a stream of calls, 4.8 TB/s (96 us in short
// runs).  Short contexts (5 sequences of 601 to 5003 keys, 63 rows a head, fp16, pages of 48:
// 28 us against 6 us of bytes) are bound by the ends of a unit (queries in, results out) and by
// issuing boxes of 16 rows.
// Scores of half a tile (64 keys) in buffers of their own: 260 us against 228 us then.
//
// A CTA owns one run of the line of key tiles (tree_attn.cuh).  Twelve warps:
//   warps 0-3, 4-7  two softmax groups, one thread per row = one TMEM lane
//   warp 8          TMA producer: K and V tiles of 128 keys into a ring
//   warp 9          tcgen05 issuer of the scores, owner of the tensor memory
//   warp 10         tcgen05 issuer of the weighted values; it also makes the values of
//                   a unit's last tile fit for the product
//   warp 11         TMA producer of the queries, as soon as the scores of the unit
//                   before are complete, and packer of the tree masks
// A thread of a softmax group holds a row of 128 scores, which leaves few registers:
// what is needed of the unit only at its ends lies in shared memory.
// Tensor memory: S (128 columns, shared) | P0 P1 (64 each) | O0 O1 (DP each).  A
// group copies its scores to registers at once, so the next scores are formed
// while it exponentiates; weights that lie over their scores instead, which
// would leave S to each group, made every product wait for the one before it
// (measured 5400 cycles a tile of 256 rows).
// With up to 128 rows (kTwo false) both groups hold the same rows and take the
// key tiles in turn, each with its own maximum, sum and output sums, joined in
// tensor memory at the end of the unit: the tensor cores work for one group while
// the other exponentiates, although there is only one row tile.
// With up to 256 rows (kTwo) each group has its own 128 rows and every key tile
// serves both, so a key is read once for 256 rows.
// A key tile is gathered from its pages by boxes of gcd(page_size, 128) rows,
// one box a lane of the producer; a box past the last key reads page number
// `pages`, which is out of range and arrives as zeros.  The ring runs on over
// unit borders.
// Every wait is bounded (about a second); when one runs out, the CTA reports it in
// the error word, waits (bounded) for its own copies and products, frees its
// tensor memory and returns.
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <cstdint>
#include <mutex>

#include "paged_host.h"
#include "tree_attn.cuh"

namespace b200tree {
namespace {

namespace ptx = b200attn::ptx;

constexpr int kThreads = 384;
constexpr int kSoftmaxThreads = 256;
constexpr int kLoadWarp = 8, kQkWarp = 9, kPvWarp = 10, kQWarp = 11;
constexpr int kTile = 128;  // keys of a tile, rows of a row tile
constexpr uint32_t kTmemCols = 512;
constexpr uint64_t kWaitNs = 1000000000ull;
// Output sums are rescaled when the maximum grew by 2^1.  A larger step would rescale less
// often (2^8: 1 % faster), but then the weights of the largest scores are not 1, and their
// rounding shows: 0.0023 instead of 0.0019 off over 131001 keys in bf16, where rounding the
// output alone gives 0.0017.
constexpr float kRescale = 1.0f;
constexpr int kSeen = 64;  // tokens of a draft whose masks fit a word of 64 bits each
constexpr int kIssuerSpin = 4096;  // polls of an issuer before its suspending wait

template <int DP_, bool kTwo_>
struct TileShape {
  static constexpr int DP = DP_;
  static constexpr bool kTwo = kTwo_;
  static constexpr int RM = kTwo ? 256 : 128;
  static constexpr int kChunks = DP / 64;                  // 128-byte swizzle blocks of a row
  static constexpr int kChunkBytes = kTile * 128;
  static constexpr int kTileBytes = kChunks * kChunkBytes;  // a Q, K or V tile
  static constexpr int kPieces = DP / 8;                   // 16-byte pieces of a row
  static constexpr int kQTiles = kTwo ? 2 : 1;
  static constexpr int kSlots = DP == 128 ? (kTwo ? 5 : 6) : (kTwo ? 10 : 12);
  static constexpr int kOffQ = 0;
  static constexpr int kOffRing = kQTiles * kTileBytes;
  static constexpr int kOffSums = kOffRing + kSlots * kTileBytes;
  static constexpr int kOffRun = kOffSums + 8 * 12;  // one sum a warp
  static constexpr int kOffPlace = kOffRun + 64;  // one a softmax warp
  static constexpr int kOffSeen = kOffPlace + 8 * 32;  // [2][kSeen] masks of a unit's tokens
  static constexpr int kOffBar = kOffSeen + 2 * 8 * kSeen;
  static_assert(sizeof(Place) == 32, "eight numbers");
  static_assert(sizeof(Run) <= 64, "a run's place");
  using G = Grid<RM, kTile, 4>;
  static constexpr int kBarQ = 0, kBarQRead = 1, kBarSeen = 2, kBarFull = 3, kBarEmpty = kBarFull + kSlots,
                       kBarScores = kBarEmpty + kSlots, kBarRead = kBarScores + 2,
                       kBarWeights = kBarRead + 2, kBarSums = kBarWeights + 2,
                       kBarDrain = kBarSums + 2, kBars = kBarDrain + 1;
  static constexpr int kOffMisc = kOffBar + 8 * kBars;
  static constexpr int kSmemBytes = kOffMisc + 16 + 1024;
  static_assert(kSmemBytes <= 232448, "exceeds the shared memory of a block");
  static constexpr uint32_t kColP = 128, kColO = 256;
  // Numbers of the loads, in the order of their use: the scores lead the values by a
  // tile, K0 K1 V0 K2 V1 ... (the place of the key tile past the last stays empty).
  __device__ static uint32_t load_k(uint32_t t) { return t ? 2 * t - 1 : 0u; }
  __device__ static uint32_t load_v(uint32_t t) { return 2 * t + 2; }
  static_assert(kColO + 2 * DP <= kTmemCols, "exceeds the tensor memory");
};

__device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag,
                                       int32_t* err) {
  const uint64_t t0 = ptx::globaltimer_ns();
  while (true) {
#pragma unroll 1
    for (int k = 0; k < 32; ++k)
      if (ptx::mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (ptx::globaltimer_ns() - t0 > kWaitNs) {
      *abort_flag = 1u;
      report_error(err, B200_ATTN_DEVERR_WAIT_TIMEOUT);
      return false;
    }
  }
}

__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity,
                                         volatile uint32_t* abort_flag, int32_t* err) {
  return ptx::mbar_try_wait(bar, parity) || wait_slow(bar, parity, abort_flag, err);
}

// By every lane; the result is the same for the warp.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity,
                                          volatile uint32_t* abort_flag, int32_t* err) {
  const bool all = __all_sync(0xffffffffu, wait_bar(bar, parity, abort_flag, err));
  if (!all) *abort_flag = 1u;
  return all;
}

// The same, spinning at first: for the issuers, on whom all others wait.
__device__ __forceinline__ bool issuer_wait(uint32_t bar, uint32_t parity,
                                            volatile uint32_t* abort_flag, int32_t* err) {
#pragma unroll 1
  for (int k = 0; k < kIssuerSpin; ++k)
    if (__all_sync(0xffffffffu, ptx::mbar_test_wait(bar, parity))) return true;
  return warp_wait(bar, parity, abort_flag, err);
}

// The lane of a converged warp that issues.
__device__ __forceinline__ bool elect_one() {
  uint32_t mine;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(mine));
  return mine != 0;
}

__device__ __forceinline__ void warp_arrive(uint32_t bar, int lane) {
  ptx::tc_fence_before();
  __syncwarp();
  if (lane == 0) ptx::mbar_arrive(bar);
}

// 16 tensor-memory columns of this thread's lane.
__device__ __forceinline__ void st_x16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void ld_x16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
// Two tensor-memory columns of this thread's lane.
__device__ __forceinline__ void st_pair(uint32_t addr, uint32_t x, uint32_t y) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void ld_pair(uint32_t addr, uint32_t& x, uint32_t& y) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0, %1}, [%2];"
               : "=r"(x), "=r"(y)
               : "r"(addr));
}

// Waits (bounded) for a barrier without regard to the abort flag.
__device__ __forceinline__ void settle(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = ptx::globaltimer_ns();
  while (!ptx::mbar_try_wait(bar, parity) && ptx::globaltimer_ns() - t0 < kWaitNs) {
  }
}

// Largest of three; (x, y) = (a, b) * m + c; (x, y) += (a, b): two lanes an instruction.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float m, float c) {
  asm("{\n\t.reg .b64 p, q, r, s;\n\t"
      "mov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %4};\n\tmov.b64 r, {%5, %5};\n\t"
      "fma.rn.f32x2 s, p, q, r;\n\tmov.b64 {%0, %1}, s;\n\t}"
      : "=f"(x), "=f"(y)
      : "f"(a), "f"(b), "f"(m), "f"(c));
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
  asm("{\n\t.reg .b64 p, q, s;\n\t"
      "mov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\t"
      "add.rn.f32x2 s, p, q;\n\tmov.b64 {%0, %1}, s;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (DT == B200_ATTN_DTYPE_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <int DT>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (DT == B200_ATTN_DTYPE_BF16)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <int DT>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr uint32_t kExp = DT == B200_ATTN_DTYPE_BF16 ? 0x7f807f80u : 0x7c007c00u;
  return __vcmpeq2(w & kExp, kExp);
}

// Scores whose bit is not set become -inf.
__device__ __forceinline__ void hide(uint32_t (&s)[32], uint32_t word) {
#pragma unroll
  for (int k = 0; k < 32; ++k)
    if (!((word >> k) & 1u)) s[k] = __float_as_uint(-INFINITY);
}

// Bits 15 and 31: whether the halves of a word are not finite (adding one to an exponent
// of all ones carries into the sign's place).
template <int DT>
__device__ __forceinline__ uint32_t exponent_carry(uint32_t w) {
  return (w & 0x7fff7fffu) + (DT == B200_ATTN_DTYPE_BF16 ? 0x00800080u : 0x04000400u);
}

template <class S, int DT>
__global__ void __launch_bounds__(kThreads, 1)
    tiles_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v,
                 const __grid_constant__ Args a, const int32_t box_rows) {
  constexpr int DP = S::DP, NS = S::kSlots, RM = S::RM;
  constexpr bool kTwo = S::kTwo, kBF16 = DT == B200_ATTN_DTYPE_BF16;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = ptx::smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Run* found = reinterpret_cast<Run*>(smem + S::kOffRun);
  // misc[0] tensor memory base, [1] abort flag, [2] last segment with a value that is not finite
  uint64_t* seen = reinterpret_cast<uint64_t*>(smem + S::kOffSeen);
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(smem + S::kOffMisc);
  volatile uint32_t* abort_flag = misc + 1;
  auto bar = [&](int i) { return sbase + S::kOffBar + 8u * static_cast<uint32_t>(i); };

  ptx::launch_dependents();
  if (threadIdx.x == 0) {
    misc[1] = 0u;
    misc[2] = 0u;
    ptx::mbar_init(bar(S::kBarQ), 1);
    ptx::mbar_init(bar(S::kBarSeen), 1);
    ptx::mbar_init(bar(S::kBarQRead), 1);
    for (int s = 0; s < NS; ++s) {
      ptx::mbar_init(bar(S::kBarFull + s), 1);
      ptx::mbar_init(bar(S::kBarEmpty + s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(bar(S::kBarScores + i), 1);
      ptx::mbar_init(bar(S::kBarRead + i), 4);
      ptx::mbar_init(bar(S::kBarWeights + i), 4);
      ptx::mbar_init(bar(S::kBarSums + i), 1);
    }
    ptx::mbar_init(bar(S::kBarDrain), 2);
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
    ptx::tma_prefetch_desc(&tm_q);
    ptx::tma_prefetch_desc(&tm_k);
    ptx::tma_prefetch_desc(&tm_v);
  }
  ptx::grid_dependency_wait();
  find_run<typename S::G>(a, blockIdx.x, gridDim.x, reinterpret_cast<uint32_t*>(smem + S::kOffSums),
                          found);
  const Run& run = *found;
  Place pl = run.p;
  if (run.done(pl)) {
    zero_unused_rows(a, 2, kThreads);
    return;
  }
  if (warp == kQkWarp) {
    ptx::tmem_alloc(sbase + S::kOffMisc, kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = misc[0];
  // rows of a unit, and of those one group's share
  auto unit_rows = [&](const Place& p) {
    return min(a.unit_rows, p.s.drafts * a.group - p.rt * a.unit_rows);
  };
  const int share = kTwo ? a.unit_rows >> 1 : a.unit_rows;
  // group i takes tile j of a segment
  auto takes = [&](int i, int j, int rows) {
    return kTwo ? (i == 0 || rows > share) : (j & 1) == i;
  };

  auto next_segment = [&](Place& p) {
    p.t += run.tiles(p);
    if (p.t == p.tiles) p = next_unit<typename S::G>(a, p);
  };

  if (warp == kLoadWarp) {
    // ------------------------------------------------------ TMA producer
    const int boxes = kTile / box_rows;
    const int u = lane % boxes, chunk = lane / boxes;
    const bool mine = chunk < S::kChunks;
    const uint32_t part = chunk * S::kChunkBytes + u * box_rows * 128;
    const uint32_t size = static_cast<uint32_t>(a.page_size);
    struct Box {
      int page, row, head;
    };
    auto look_up = [&]() {
      const int key = pl.t * kTile + u * box_rows;
      Box x{a.pages, 0, pl.h};
      if (mine && key < pl.s.len + pl.s.drafts) {
        const uint32_t slot = static_cast<uint32_t>(key) / size;
        x.page = __ldg(a.table + pl.b * a.table_stride + slot);
        x.row = static_cast<int>(static_cast<uint32_t>(key) - slot * size);
        if (x.page >= a.pages) x.page = -1;
      }
      return x;
    };
    auto load = [&](uint32_t number, const CUtensorMap* map, Box x) {
      const uint32_t s = number % NS;
      if (!warp_wait(bar(S::kBarEmpty + s), ((number / NS) & 1u) ^ 1u, abort_flag, a.err))
        return false;
      if (x.page < 0) {
        report_error(a.err, B200_ATTN_DEVERR_BOUNDS);
        x.page = a.pages;
      }
      const uint32_t at = sbase + S::kOffRing + s * S::kTileBytes;
      const uint32_t full = bar(S::kBarFull + s);
      if (elect_one()) ptx::mbar_arrive_expect_tx(full, S::kTileBytes);
      __syncwarp();
      if (S::kChunks == 1 || boxes <= 2) {
        if (mine)
          ptx::tma_load_4d(at + part, map, full, 64 * chunk, x.row, x.head, x.page);
        return true;
      }
      // Many small boxes: one lane issues them all, four boxes of both halves of a row
      // at a time from uniform registers; with a lane each the producer, not the memory,
      // set the pace (64 rows over 131001 keys in pages of 16: 141 us against 116 us;
      // large boxes and D = 64: 1 to 3 % the other way).
      const int head = __shfl_sync(0xffffffffu, x.head, 0);
#pragma unroll 1
      for (int i = 0; i < boxes; i += 4) {
        int row[4], page[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          row[y] = __shfl_sync(0xffffffffu, x.row, i + y);
          page[y] = __shfl_sync(0xffffffffu, x.page, i + y);
        }
        if (elect_one()) {
#pragma unroll
          for (int y = 0; y < 4; ++y)
#pragma unroll
            for (int c = 0; c < S::kChunks; ++c)
              ptx::tma_load_4d(at + c * S::kChunkBytes + (i + y) * box_rows * 128, map, full, 64 * c,
                               row[y], head, page[y]);
        }
        __syncwarp();
      }
      return true;
    };
    // The page numbers of a tile are read while the loads before it are issued, and
    // serve its keys and, two loads later, its values.
    Box next = look_up(), before[2] = {next, next};  // of tiles t, and t - 2, t - 1
    uint32_t issued = 0;                             // one past the last load issued
    bool ok = true;
    int rest = 2;  // rounds after the last keys, for the last values
#pragma unroll 1
    for (uint32_t t = 0; ok && rest > 0; ++t) {
      const Box now = next;
      if (t >= 2) {
        ok = load(S::load_v(t - 2), &tm_v, before[0]);
        if (ok) issued = S::load_v(t - 2) + 1;
      }
      before[0] = before[1];
      before[1] = now;
      if (run.done(pl)) {
        --rest;
        continue;
      }
      ok = ok && load(S::load_k(t), &tm_k, now);
      if (ok) issued = S::load_k(t) + 1;
      if (++pl.t == pl.tiles) pl = next_unit<typename S::G>(a, pl);
      if (!run.done(pl)) next = look_up();
    }
    if (!ok) {
      // copies in flight land before the shared memory goes
      for (uint32_t x = issued > NS ? issued - NS : 0u; x < issued; ++x)
        settle(bar(S::kBarFull + x % NS), (x / NS) & 1u);
    }
    __syncwarp();
  } else if (warp == kQkWarp) {
    // -------------------------------------------------- scores S = Q K^T
    // By the whole warp, one lane of which issues: in control flow that is the same for the
    // warp the operands' descriptors stay in uniform registers.
    constexpr uint32_t id = ptx::idesc_f16(kBF16, kTile, kTile, false);
    uint32_t tile = 0, seg = 0;
    uint32_t made = 0u;  // bit i: parity of the number of scores made for group i
    int prev = -1;
    bool ok = true;
#pragma unroll 1
    for (; ok; ++seg) {
      const int n = __shfl_sync(0xffffffffu, run.tiles(pl), 0);
      if (n <= 0) break;
      const bool second = !kTwo || __shfl_sync(0xffffffffu, unit_rows(pl), 0) > share;
      // the first tile that needs the masks
      const int masked = __shfl_sync(0xffffffffu, min(n - 1, max(0, pl.s.len / kTile - pl.t)), 0);
      ok = warp_wait(bar(S::kBarQ), seg & 1u, abort_flag, a.err);
#pragma unroll 1
      for (int j = 0; ok && j < n; ++j, ++tile) {
        // the masks are there before the scores that need them
        if (j == masked) ok = warp_wait(bar(S::kBarSeen), seg & 1u, abort_flag, a.err);
        const uint32_t number = S::load_k(tile), s = number % NS;
        ok = ok && issuer_wait(bar(S::kBarFull + s), (number / NS) & 1u, abort_flag, a.err);
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          if (!ok || (kTwo ? (i == 1 && !second) : (j & 1) != i)) continue;
          // the scores before these have been copied to registers
          ok = prev < 0 ||
               issuer_wait(bar(S::kBarRead + prev), ((made >> prev) & 1u) ^ 1u, abort_flag, a.err);
          if (!ok) continue;
          ptx::tc_fence_after();
          const uint64_t qd = ptx::smem_desc_sw128(
              sbase + S::kOffQ + (kTwo ? i : 0) * S::kTileBytes, 16, 1024);
          const uint64_t kd =
              ptx::smem_desc_sw128(sbase + S::kOffRing + s * S::kTileBytes, 16, 1024);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
              const uint32_t off = ((kk >> 2) * S::kChunkBytes + (kk & 3) * 32) >> 4;
              ptx::tc_mma_ss(tmem, qd + off, kd + off, id, kk > 0 ? 1u : 0u);
            }
            ptx::tc_commit(bar(S::kBarScores + i));
          }
          __syncwarp();
          made ^= 1u << i;
          prev = i;
        }
        if (ok && elect_one()) ptx::tc_commit(bar(S::kBarEmpty + s));
        __syncwarp();
      }
      if (elect_one()) ptx::tc_commit(bar(S::kBarQRead));
      __syncwarp();
      next_segment(pl);
    }
    if (elect_one()) {
      ptx::tc_commit(bar(S::kBarDrain));
      settle(bar(S::kBarDrain), 0);
    }
    __syncwarp();
  } else if (warp == kQWarp) {
    // ------------------------------------------------------------- queries
    // Row r of a row tile is head r % group of token r / group: a box of whole tokens.
    const int tokens = share / a.group;
    const uint32_t bytes = static_cast<uint32_t>(share) * 128u * S::kChunks;
    uint32_t seg = 0;
    bool ok = true;
#pragma unroll 1
    for (; ok && !run.done(pl); ++seg) {
      ok = seg == 0 || warp_wait(bar(S::kBarQRead), (seg - 1u) & 1u, abort_flag, a.err);
      if (!ok) break;
      const int first = pl.rt * (a.unit_rows / a.group);  // token
      if (lane == 0) {
        const int tiles = kTwo && unit_rows(pl) > share ? 2 : 1;
        ptx::mbar_arrive_expect_tx(bar(S::kBarQ), tiles * bytes);
        for (int i = 0; i < tiles; ++i)
#pragma unroll
          for (int c = 0; c < S::kChunks; ++c)
            ptx::tma_load_4d(sbase + S::kOffQ + i * S::kTileBytes + c * S::kChunkBytes, &tm_q,
                             bar(S::kBarQ), 64 * c, pl.h * a.group, first + i * tokens, pl.b);
      }
      if (a.tokens <= kSeen) {
        // a bit for each drafted token that a token sees
#pragma unroll 1
        for (int tok = lane; tok < a.tokens; tok += 32) {
          const uint32_t lo = seen_word(a, pl.b, tok, 0, pl.s.drafts);
          const uint32_t hi = a.tokens > 32 ? seen_word(a, pl.b, tok, 32, pl.s.drafts) : 0u;
          seen[(seg & 1u) * kSeen + tok] = static_cast<uint64_t>(hi) << 32 | lo;
        }
        __syncwarp();
      }
      if (lane == 0) ptx::mbar_arrive(bar(S::kBarSeen));
      next_segment(pl);
    }
    if (!ok && seg > 0) settle(bar(S::kBarQ), (seg - 1u) & 1u);
    __syncwarp();
  } else if (warp == kPvWarp) {
    // ------------------------------------------------------- O_i += P_i V
    constexpr uint32_t id = ptx::idesc_f16(kBF16, kTile, DP, true);
    uint32_t tile = 0, seg = 0;
    uint32_t made = 0u;  // bit i: parity of the number of products made for group i
    bool ok = true;
#pragma unroll 1
    for (; ok; ++seg) {
      const int n = __shfl_sync(0xffffffffu, run.tiles(pl), 0);
      if (n <= 0) break;
      const int rows = __shfl_sync(0xffffffffu, unit_rows(pl), 0), len = pl.s.len;
      uint32_t begun = 0u;  // bit i: O_i holds a product of this segment
#pragma unroll 1
      for (int j = 0; ok && j < n; ++j, ++tile) {
        const uint32_t number = S::load_v(tile), s = number % NS;
        ok = warp_wait(bar(S::kBarFull + s), (number / NS) & 1u, abort_flag, a.err);
        const uint32_t va = sbase + S::kOffRing + s * S::kTileBytes;
        const int k0 = (pl.t + j) * kTile;
        if (ok && k0 + kTile > len) {
          // Values past the last key become 0 (their rows may hold anything, and 0 x
          // infinity would reach the sums), and so do elements of drafted values that
          // are not finite: the softmax groups add those to the rows that see them.
          const int r0 = max(0, len - k0), r1 = min(kTile, len + pl.s.drafts - k0);
          const int r2 = min(kTile, (r1 + box_rows - 1) & -box_rows);  // later boxes are zero
          auto piece = [&](int x) {  // shared-memory address of piece x of the tile's rows
            const int pc = x % S::kPieces;
            return va + (pc >> 3) * S::kChunkBytes + (x / S::kPieces) * 128 + ((pc & 7) << 4);
          };
          auto put = [&](int x, uint32_t (&w)[4]) {
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece(x)), "r"(w[0]),
                         "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
          };
          bool odd = false;
#pragma unroll 1
          for (int x0 = r0 * S::kPieces; x0 < r1 * S::kPieces; x0 += 32 * 8) {
            uint32_t w[8][4], any = 0u;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const int x = x0 + 32 * u + lane;
              w[u][0] = w[u][1] = w[u][2] = w[u][3] = 0u;
              if (x < r1 * S::kPieces)
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(w[u][0]), "=r"(w[u][1]), "=r"(w[u][2]), "=r"(w[u][3])
                             : "r"(piece(x)));
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
              for (int y = 0; y < 4; ++y) any |= exponent_carry<DT>(w[u][y]);
            if (any & 0x80008000u) {
              odd = true;
#pragma unroll
              for (int u = 0; u < 8; ++u) {
                const int x = x0 + 32 * u + lane;
#pragma unroll
                for (int y = 0; y < 4; ++y) w[u][y] &= ~not_finite<DT>(w[u][y]);
                if (x < r1 * S::kPieces) put(x, w[u]);
              }
            }
          }
          uint32_t zero[4] = {0u, 0u, 0u, 0u};
#pragma unroll 1
          for (int x = r1 * S::kPieces + lane; x < r2 * S::kPieces; x += 32) put(x, zero);
          if (odd) misc[2] = seg + 1u;
          ptx::fence_proxy_async_smem();
          __syncwarp();
        }
        const uint64_t vd = ptx::smem_desc_sw128(va, S::kChunkBytes, 1024);
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          if (!ok || !takes(i, j, rows)) continue;
          ok = issuer_wait(bar(S::kBarWeights + i), (made >> i) & 1u, abort_flag, a.err);
          if (!ok) continue;
          ptx::tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kTile / 16; ++kk)
              ptx::tc_mma_ts(tmem + S::kColO + DP * i, tmem + S::kColP + 64 * i + kk * 8,
                             vd + kk * (2048 >> 4), id, (((begun >> i) & 1u) || kk > 0) ? 1u : 0u);
            ptx::tc_commit(bar(S::kBarSums + i));
          }
          __syncwarp();
          begun |= 1u << i;
          made ^= 1u << i;
        }
        if (ok && elect_one()) ptx::tc_commit(bar(S::kBarEmpty + s));
        __syncwarp();
      }
      next_segment(pl);
    }
    if (elect_one()) {
      ptx::tc_commit(bar(S::kBarDrain));
      settle(bar(S::kBarDrain), 0);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax
    const int i = warp >> 2, quad = warp & 3, rl = quad * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t tS = tmem + lanes, tP = tS + S::kColP + 64 * i, tO = tS + S::kColO;
    const int row0 = i * (kTwo ? share : 0);  // first row of this group in the unit
    Place* where = reinterpret_cast<Place*>(smem + S::kOffPlace) + warp;
    if (lane == 0) *where = pl;
    __syncwarp();
    zero_unused_rows(a, 2, kSoftmaxThreads);

    uint32_t seg = 0, cnt = 0;  // segments of the run, tiles of this group
    bool ok = true;
#pragma unroll 1
    for (; ok && !run.done(*where); ++seg) {
      const int n = run.tiles(*where), rows = unit_rows(*where), t0 = where->t, len = where->s.len;
      const bool idle = row0 + quad * 32 >= rows || quad * 32 >= share;  // padding rows only
      float m_run = -INFINITY, l_run = 0.f;
      int done = 0;
#pragma unroll 1
      for (int j = 0; j < n; ++j) {
        if (!takes(i, j, rows)) continue;
        if (!warp_wait(bar(S::kBarScores + i), cnt & 1u, abort_flag, a.err)) {
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        const int k0 = (t0 + j) * kTile;
        const bool partly = k0 + kTile > len;  // drafted tokens, or places past the last key
        if (idle) {  // nothing to compute, but the barriers count this warp
          warp_arrive(bar(S::kBarRead + i), lane);
          ok = cnt == 0 || warp_wait(bar(S::kBarSums + i), (cnt - 1u) & 1u, abort_flag, a.err);
          if (!ok) break;
          warp_arrive(bar(S::kBarWeights + i), lane);
          ++cnt;
          continue;
        }
        // a bit for each key that this row sees
        uint32_t words[4] = {~0u, ~0u, ~0u, ~0u};
        if (partly) {
          const int tok = min((where->rt * a.unit_rows + row0 + rl) / a.group, a.tokens - 1);
          const uint64_t bits = a.tokens <= kSeen ? seen[(seg & 1u) * kSeen + tok] : 0u;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int d = k0 + 32 * q - len;
            if (d <= -32) continue;
            if (a.tokens <= kSeen)
              words[q] = d >= 64 ? 0u
                                 : static_cast<uint32_t>(d < 0 ? bits << -d | ((1u << -d) - 1u) : bits >> d);
            else
              words[q] = seen_word(a, where->b, tok, d, where->s.drafts);
          }
        }
        uint32_t sr[kTile];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          ptx::tmem_ld_32x32b_x32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&sr[32 * c]));
        ptx::tmem_wait_ld();
        warp_arrive(bar(S::kBarRead + i), lane);
        if (partly) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            hide(*reinterpret_cast<uint32_t(*)[32]>(&sr[32 * q]), words[q]);
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < kTile; k += 2)
          top[(k >> 1) & 3] =
              max3(top[(k >> 1) & 3], __uint_as_float(sr[k]), __uint_as_float(sr[k + 1]));
        const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * a.scale_log2;
        const bool resc = mx > m_run + kRescale || (m_run == -INFINITY && mx > m_run);
        const float m_new = resc ? mx : m_run;
        const float alpha = resc ? ptx::ex2_approx(m_run - m_new) : 1.f;
        m_run = m_new;
        l_run *= alpha;
        // P_i was last read by the product before this one, which also left O_i at rest
        if (cnt > 0) {
          if (!warp_wait(bar(S::kBarSums + i), (cnt - 1u) & 1u, abort_flag, a.err)) {
            ok = false;
            break;
          }
          ptx::tc_fence_after();
        }
        if (done > 0 && __any_sync(0xffffffffu, resc)) {
#pragma unroll 1
          for (int c = 0; c < DP / 16; ++c) {
            uint32_t o[16];
            ld_x16(tO + DP * i + 16 * c, o);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            st_x16(tO + DP * i + 16 * c, o);
          }
        }
        const float neg = m_run == -INFINITY ? 0.f : -m_run;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {  // pieces of 32 keys, so that few registers are new
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int k = 32 * c + 2 * e;
            float x, y;
            fma2(x, y, __uint_as_float(sr[k]), __uint_as_float(sr[k + 1]), a.scale_log2, neg);
            x = ptx::ex2_approx(x);
            y = ptx::ex2_approx(y);
            pk[e] = pack2<DT>(x, y);
            // the sum is taken of the rounded weights, which the product uses
            const float2 r = unpack2<DT>(pk[e]);
            add2(sum[2 * (e & 1)], sum[2 * (e & 1) + 1], r.x, r.y);
          }
          st_x16(tP + 16 * c, pk);
        }
        l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        ptx::tmem_wait_st();
        warp_arrive(bar(S::kBarWeights + i), lane);
        ++cnt;
        ++done;
      }
      // while the last product runs: where the row's results go
      const Place unit = *where;
      const bool first = t0 == 0, last = t0 + n == unit.tiles, finish = first && last;
      const bool mine = rl < share && row0 + rl < rows;
      const int row = unit.rt * a.unit_rows + row0 + rl, tok = min(row / a.group, a.tokens - 1);
      uint8_t* out = a.o + unit.b * a.o_seq + (unit.h * a.group + row % a.group) * a.o_head +
                     tok * a.o_tok;
      float* part = a.partial +
                    static_cast<int64_t>(2 * blockIdx.x + (first ? 1 : 0)) * (RM * (DP + 2));
      __syncwarp();
      if (lane == 0) {
        Place next = unit;
        next_segment(next);
        *where = next;
      }
      if (ok && cnt > 0) ok = warp_wait(bar(S::kBarSums + i), (cnt - 1u) & 1u, abort_flag, a.err);
      __syncwarp();
      // ---------------------------------------------------- end of a segment
      if (!kTwo && ok) {
        // the other group reads this row's maximum and sum where P_i was
        ptx::tc_fence_after();
        st_pair(tP, __float_as_uint(m_run), __float_as_uint(l_run));
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
      }
      if constexpr (!kTwo) ok = ptx::named_barrier_and(1, kSoftmaxThreads, ok);
      if (!ok) break;
      ptx::tc_fence_after();
      // (a later segment's may have been noted already: then add_odd looks, and finds none)
      const bool any_odd = misc[2] > seg;
      // weights of the groups' sums in this thread's row
      float top = m_run, total = l_run, w[2] = {1.f, 1.f};
      if constexpr (!kTwo) {
        uint32_t om, ol;
        ld_pair(tS + S::kColP + 64 * (1 - i), om, ol);
        ptx::tmem_wait_ld();
        const float m_other = __uint_as_float(om);
        top = fmaxf(m_run, m_other);
        const float mine_w = m_run == -INFINITY ? 0.f : ptx::ex2_approx(m_run - top);
        const float other_w = m_other == -INFINITY ? 0.f : ptx::ex2_approx(m_other - top);
        total = mine_w * l_run + other_w * __uint_as_float(ol);
        w[0] = i == 0 ? mine_w : other_w;
        w[1] = i == 0 ? other_w : mine_w;
      }
      const float inv = total == 0.f ? 0.f : 1.f / total;
      if (!idle) {
        // kTwo: all columns of the own rows; else half the columns of the shared ones
        constexpr int kSpan = kTwo ? DP : DP / 2;
#pragma unroll 1
        for (int c = 0; c < kSpan / 32; ++c) {
          const int col = (kTwo ? 0 : i * kSpan) + 32 * c;
          uint32_t o[32];
          float acc[32];
          if constexpr (kTwo) {
            ptx::tmem_ld_32x32b_x32(tO + DP * i + col, o);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) acc[e] = __uint_as_float(o[e]);
          } else {
            ptx::tmem_ld_32x32b_x32(tO + col, o);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) acc[e] = w[0] * __uint_as_float(o[e]);
            if (n > 1) {
              ptx::tmem_ld_32x32b_x32(tO + DP + col, o);
              ptx::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) acc[e] += w[1] * __uint_as_float(o[e]);
            }
          }
          if (finish) {
            if (mine) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (col + 8 * e < a.head_dim)
                  *reinterpret_cast<uint4*>(out + 2 * (col + 8 * e)) = make_uint4(
                      pack2<DT>(acc[8 * e] * inv, acc[8 * e + 1] * inv),
                      pack2<DT>(acc[8 * e + 2] * inv, acc[8 * e + 3] * inv),
                      pack2<DT>(acc[8 * e + 4] * inv, acc[8 * e + 5] * inv),
                      pack2<DT>(acc[8 * e + 6] * inv, acc[8 * e + 7] * inv));
            }
          } else if (mine) {
            // A column of rows at a time.  Own rows only: where the head group does not divide
            // 128 a group's share is less than its 128 lanes, and the places of the lanes past
            // it are the other group's first rows.
#pragma unroll
            for (int e = 0; e < 32; ++e) part[(col + e) * RM + row0 + rl] = acc[e];
          }
        }
      }
      if (!finish && mine && (kTwo || i == 0)) {
        part[RM * DP + row0 + rl] = top;
        part[RM * DP + RM + row0 + rl] = total;
      }
      if (any_odd && mine) {
        const int col0 = kTwo ? 0 : i * (DP / 2), col1 = min(a.head_dim, kTwo ? DP : col0 + DP / 2);
        add_odd<DT>(a, unit.b, unit.h, unit.s, tok, t0 * kTile - len, (t0 + n) * kTile - len, col0, col1,
                    finish ? reinterpret_cast<uint16_t*>(out) : nullptr, part + row0 + rl, RM);
      }
      if (threadIdx.x == 0 && last)
        a.desc[unit_of(a, unit)] =
            make_int2(first ? static_cast<int>(blockIdx.x) : run.first_run,
                      static_cast<int>(blockIdx.x));
      // both groups' sums have been read by both
      ptx::tc_fence_before();
      if constexpr (!kTwo) ptx::named_barrier_sync(1, kSoftmaxThreads);
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == kQkWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, kTmemCols);
  }
}

// -------------------------------------------------------------------- host
using namespace b200paged;

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// Map {head_dim, page_size, kv_heads, pages} of a pool, boxes of {64, box_rows, 1, 1}.
int32_t encode_pool(CUtensorMap* map, const uint8_t* base, int64_t row, int64_t head, int64_t page,
                    const Args& a, int dtype, int box_rows) {
  auto fn = encode_fn();
  if (!fn) {
    set_error("cuTensorMapEncodeTiled entry point unavailable");
    return B200_ATTN_ERR_LAUNCH;
  }
  // strides of dimensions with one entry never move the address
  const int64_t any = a.head_dim * 16;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(a.page_size),
                        static_cast<cuuint64_t>(a.kv_heads), static_cast<cuuint64_t>(a.pages)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(a.page_size > 1 ? row : any),
                           static_cast<cuuint64_t>(a.kv_heads > 1 ? head : any),
                           static_cast<cuuint64_t>(a.pages > 1 ? page : any)};
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r =
      fn(map, dtype == B200_ATTN_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                            : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
         4, const_cast<uint8_t*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed");
    return B200_ATTN_ERR_LAUNCH;
  }
  return B200_ATTN_OK;
}

// Map {head_dim, heads, tokens, batch} of the queries, boxes of {64, group, tokens, 1}.
int32_t encode_q(CUtensorMap* map, const Args& a, int heads, int tokens, int dtype) {
  auto fn = encode_fn();
  if (!fn) {
    set_error("cuTensorMapEncodeTiled entry point unavailable");
    return B200_ATTN_ERR_LAUNCH;
  }
  const int64_t any = a.head_dim * 16;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(heads),
                        static_cast<cuuint64_t>(a.tokens), static_cast<cuuint64_t>(a.batch)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(heads > 1 ? a.q_head : any),
                           static_cast<cuuint64_t>(a.tokens > 1 ? a.q_tok : any),
                           static_cast<cuuint64_t>(a.batch > 1 ? a.q_seq : any)};
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(tokens), 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r =
      fn(map, dtype == B200_ATTN_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                            : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
         4, const_cast<uint8_t*>(a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed");
    return B200_ATTN_ERR_LAUNCH;
  }
  return B200_ATTN_OK;
}

struct Maps {
  CUtensorMap q, k, v;
};

template <class S, int DT>
int32_t launch_shape(const Maps& m, const Args& a, int box_rows, int runs, int device, cudaStream_t s) {
  static std::once_flag once[kMaxDevices];
  static cudaError_t err[kMaxDevices];
  auto kernel = tiles_kernel<S, DT>;
  std::call_once(once[device], [&] {
    err[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       S::kSmemBytes);
  });
  if (err[device] != cudaSuccess) {
    set_error(cudaGetErrorString(err[device]));
    return B200_ATTN_ERR_LAUNCH;
  }
  return launch(kernel, dim3(runs), dim3(kThreads), S::kSmemBytes, s, m.q, m.k, m.v, a, box_rows);
}

template <int DP, int DT>
int32_t launch_rows(bool two, const Maps& m, const Args& a, int box_rows, int runs, int device,
                    cudaStream_t s) {
  return two ? launch_shape<TileShape<DP, true>, DT>(m, a, box_rows, runs, device, s)
             : launch_shape<TileShape<DP, false>, DT>(m, a, box_rows, runs, device, s);
}

}  // namespace

int box_rows_of(int64_t page_size) {
  int g = 1;
  while (g < kTile && page_size % (2 * g) == 0) g *= 2;
  return g;
}

int32_t launch_tiles(int rm, int dp, int dtype, const Args& a, int heads, int runs, int device,
                     cudaStream_t s) {
  const int g = box_rows_of(a.page_size);
  const bool two = rm == 256;
  Maps m;
  int32_t rc = encode_q(&m.q, a, heads, a.unit_rows / a.group / (two ? 2 : 1), dtype);
  if (rc == B200_ATTN_OK)
    rc = encode_pool(&m.k, a.k, a.k_row, a.k_head, a.k_page, a, dtype, g);
  if (rc == B200_ATTN_OK)
    rc = encode_pool(&m.v, a.v, a.v_row, a.v_head, a.v_page, a, dtype, g);
  if (rc != B200_ATTN_OK) return rc;
  if (dtype == B200_ATTN_DTYPE_BF16)
    return dp == 64 ? launch_rows<64, B200_ATTN_DTYPE_BF16>(two, m, a, g, runs, device, s)
                    : launch_rows<128, B200_ATTN_DTYPE_BF16>(two, m, a, g, runs, device, s);
  return dp == 64 ? launch_rows<64, B200_ATTN_DTYPE_FP16>(two, m, a, g, runs, device, s)
                  : launch_rows<128, B200_ATTN_DTYPE_FP16>(two, m, a, g, runs, device, s);
}

}  // namespace b200tree
