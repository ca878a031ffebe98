// tree_attn4_sm100.cu — drafted-token attention of many rows over a paged cache held in 4
// bits, on the fifth-generation tensor cores: wide trees, and pieces of prompts.
//
// The kernel of 16-bit caches (tree_attn_sm100.cu has the roles, the tensor memory and the
// order of the loads) with another producer: one warp copies coded rows to shared memory
// in bulk, and of eight warps, a thread a row, four turn keys and four values into the operands of
// the products in the swizzled layout that the tensor cores read, each through a ring of its
// own.  The matrix instruction kernel (tree_attn4.cu) would decode a row again for every 16 rows of
// queries; here it is once for up to 256.
// Keys become fp16 numbers, as the queries do, each times a power of two, of the row of the
// queries and of 32 keys (of a key alone in tiles that hold drafted ones, which a row may not see),
// that the scores are rid of again: rounded to 11 bits, they cost a weight less than the values'
// rounding does.  Values are bf16: whatever the size of one, it fits.  A weight is two bf16 numbers, the
// second what rounding left, over the scores of its keys: one alone made the error against 64 bits 1.48
// times that of a rounded output instead of 1.36, for 4 % of the time.
// Each softmax group has scores of its own, over which its weights come to lie, and reads them
// twice, 32 at a time: with a row of 128 scores in registers there were none for a second
// warp of decoders on each scheduler, and code of four times the size kept all roles waiting
// for instructions (16 sequences, 128 rows: 188 us where this form took 140).
//
// Bound by latency along the chain codes -> operands -> scores -> weights -> sums, at half of the
// issue rate and a third of the tensor pipe: 16 sequences of 1001 to 8100 keys, 128 rows, 8 key heads, D
// 128: 99 us, 131001 keys and 64 rows 140 us (23 and 26 us of bytes).  Slower, with one
// number a weight, where this form took 95 and 133: one pass over the scores with the maximum followed a
// quarter at a time (108 and 145), 16 scores at a time with the next 16 on their way (109 and
// 154), a load warp more (80 registers a thread: 105 and 146), decoding loops unrolled twice (104 and
// 141), keys and values decoded on two schedulers each (101 and 139).
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>

#include "b200_cache4.h"
#include "paged_host.h"
#include "tree_attn.cuh"
#include "tree_attn4.cuh"
#include "tree_attn_tiles.cuh"

namespace b200tree {
namespace {

constexpr int kThreads = 640;
constexpr int kSoftmaxThreads = 256;
constexpr int kLoadWarp = 8, kQkWarp = 9, kPvWarp = 10, kPlanWarp = 11;
constexpr int kCodeWarp = 12, kCodeWarps = 8;
constexpr float kGrowth = 8.f;   // a maximum is followed when a score is over 2^8 times its weight
constexpr int kAhead = 4;        // segments that are planned ahead
constexpr int kReaders = 19;     // warps that go through the segments

// What is left of a unit in the CTA's run; tiles 0: the run's end.
struct Segment {
  int b, h, rt, t;  // sequence, key head, row tile, first key tile
  int n, tiles;     // key tiles of the segment and of the unit
  int len, drafts;
};
template <int DP_, bool kTwo_>
struct CodedShape {
  static constexpr int DP = DP_;
  static constexpr bool kTwo = kTwo_;
  static constexpr int RM = kTwo ? 256 : 128;
  static constexpr int kChunks = DP / 64;                  // 128-byte swizzle blocks of a row
  static constexpr int kChunkBytes = kTile * 128;
  static constexpr int kTileBytes = kChunks * kChunkBytes;  // a Q, K or V tile
  static constexpr int kQTiles = kTwo ? 2 : 1;
  static constexpr int kSlots = DP == 128 ? 2 : 3;  // of K and of V
  static constexpr int kRawRow = DP / 2 + 16, kRawBytes = kTile * kRawRow;  // coded
  static constexpr int kRawK = DP == 64 ? 4 : (kTwo ? 1 : 3), kRawV = DP == 64 ? 4 : (kTwo ? 1 : 2);
  static constexpr int kOffQ = 0;
  static constexpr int kOffRing = kQTiles * kTileBytes;
  static constexpr int kOffV = kOffRing + kSlots * kTileBytes;
  static constexpr int kOffRaw = kOffV + kSlots * kTileBytes;
  static constexpr int kOffRawV = kOffRaw + kRawK * kRawBytes;
  static constexpr int kOffSums = kOffRawV + kRawV * kRawBytes;
  static constexpr int kOffRun = kOffSums + 8 * 24;  // one sum a warp
  static constexpr int kOffPlan = kOffRun + 64;  // [kAhead]
  static constexpr int kOffSeen = kOffPlan + kAhead * 32;  // [kAhead][kSeen] masks of a unit's tokens
  static constexpr int kOffRowScale = kOffSeen + kAhead * 8 * kSeen;  // [kAhead][RM]
  static constexpr int kOffKeyScale = kOffRowScale + kAhead * 4 * RM;
  static constexpr int kOffOwnScale = kOffKeyScale + 8 * 4 * 4;  // [8 tiles][128 keys]
  static constexpr int kOffTold = kOffOwnScale + 8 * 4 * kTile;  // [2][128] maximum and sum of a row
  static constexpr int kOffBar = kOffTold + (kTwo ? 0 : 2 * 8 * kTile);
  static_assert(sizeof(Segment) == 32, "eight numbers");
  static_assert(sizeof(Run) <= 64, "a run's place");
  using G = Grid<RM, kTile, 4>;
  // (those of the values lie kSlots, kRawK or kRawV behind those of the keys)
  static constexpr int kBarQ = 0, kBarQRead = 1, kBarFull = 2, kBarEmpty = kBarFull + 2 * kSlots,
                       kBarScores = kBarEmpty + 2 * kSlots, kBarWeights = kBarScores + 2,
                       kBarSums = kBarWeights + 2, kBarDrain = kBarSums + 2,
                       kBarRawFull = kBarDrain + 1, kBarRawEmpty = kBarRawFull + kRawK + kRawV,
                       kBarPlan = kBarRawEmpty + kRawK + kRawV, kBarDone = kBarPlan + kAhead,
                       kBars = kBarDone + kAhead;
  static constexpr int kOffMisc = kOffBar + 8 * kBars;
  static constexpr int kSmemBytes = kOffMisc + 16 + 1024;
  static_assert(kSmemBytes <= 232448, "exceeds the shared memory of a block");
  static constexpr uint32_t kColO = 256;
  static_assert(kColO + 2 * DP <= kTmemCols, "exceeds the tensor memory");
};

// So many bytes more are to come before the barrier's phase ends.
__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}

// (x, y) times (a, b) m, two lanes an instruction.
__device__ __forceinline__ void scale2(uint32_t& x, uint32_t& y, float a, float b, float m) {
  asm("{\n\t.reg .b64 p, q, r;\n\t"
      "mov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %4};\n\tmov.b64 r, {%0, %1};\n\t"
      "mul.rn.f32x2 p, p, q;\n\tmul.rn.f32x2 r, r, p;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "+r"(x), "+r"(y)
      : "f"(a), "f"(b), "f"(m));
}

// The lowest n bits.
__device__ __forceinline__ uint32_t first_bits(int n) {
  return n >= 32 ? ~0u : (n <= 0 ? 0u : (1u << n) - 1u);
}

__device__ __forceinline__ float half_of(uint32_t w, int high) {
  return __uint_as_float(high ? w & 0xffff0000u : w << 16);
}
__device__ __forceinline__ uint32_t bits_of(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }
__device__ __forceinline__ uint32_t bits_of(__nv_bfloat162 x) { return *reinterpret_cast<uint32_t*>(&x); }

// Half bytes n and n + 4 of w as fp16 numbers: under the exponent of 1024, less 1024.
__device__ __forceinline__ __half2 codes_fp16(uint32_t w, int n) {
  const uint32_t x = (w >> (4 * n) & 0x000f000fu) | 0x64006400u;
  return __hsub2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(1024.f));
}
// The same as bf16 numbers.
__device__ __forceinline__ __nv_bfloat162 codes_bf16(uint32_t w, int n) {
  const uint32_t x = (w >> (4 * n) & 0x000f000fu) | 0x43004300u;
  return __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), __float2bfloat162_rn(128.f));
}

// A row of codes as operands, quarter q of them (16 or 8 bytes) at a time, so that the code is
// small: put(piece of 8 numbers, its bits).  Keys as fp16 numbers; step, low: of the groups.
template <int DP, class Put>
__device__ __forceinline__ void keys(const uint8_t* row, const __half2 (&step)[4],
                                     const __half2 (&low)[4], Put put) {
#pragma unroll 1
  for (int q = 0; q < DP / 32; ++q) {
    const uint4 v = *reinterpret_cast<const uint4*>(row + 16 * q);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      auto pair = [&](uint32_t x, int n) { return bits_of(__hfma2(codes_fp16(x, n), step[g], low[g])); };
      if constexpr (DP == 128) {  // lane q's word of the group
        put(4 * g + q, make_uint4(pair(w[g], 0), pair(w[g], 1), pair(w[g], 2), pair(w[g], 3)));
      } else {  // words g / 2 of lanes 2 q and 2 q + 1
        const uint32_t x = w[g / 2], y = w[2 + g / 2];
        const int n = 2 * (g % 2);
        put(2 * g + q, make_uint4(pair(x, n), pair(x, n + 1), pair(y, n), pair(y, n + 1)));
      }
    }
  }
}

// Values as bf16 numbers; step, low: of the two groups that share a word's halves.
template <int DP, class Put>
__device__ __forceinline__ void values(const uint8_t* row, const __nv_bfloat162 (&step)[2],
                                       const __nv_bfloat162 (&low)[2], Put put) {
#pragma unroll 1
  for (int q = 0; q < DP / 32; ++q) {
    const uint4 v = *reinterpret_cast<const uint4*>(row + 16 * q);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      auto pair = [&](uint32_t x, int n) { return bits_of(__hfma2(codes_bf16(x, n), step[y], low[y])); };
      uint32_t lo[4], hi[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        uint32_t a, b;
        if constexpr (DP == 128) {  // columns 2 q and 2 q + 1 of the row, groups 2 y and 2 y + 1
          const uint32_t word = w[2 * (x / 2) + y];
          a = pair(word, 2 * (x % 2)), b = pair(word, 2 * (x % 2) + 1);
        } else {  // column 4 q + x of the row, groups y and y + 2
          a = pair(w[x], 2 * y), b = pair(w[x], 2 * y + 1);
        }
        lo[x] = __byte_perm(a, b, 0x5410);
        hi[x] = __byte_perm(a, b, 0x7632);
      }
      put(DP == 128 ? 8 * y + q : 2 * y + q, make_uint4(lo[0], lo[1], lo[2], lo[3]));
      put(DP == 128 ? 8 * y + 4 + q : 2 * (y + 2) + q, make_uint4(hi[0], hi[1], hi[2], hi[3]));
    }
  }
}

// kStall: the stall self-test's instance, which leaves out a copy of tile number `skip` of each CTA.
template <class S, bool kStall>
__global__ void __launch_bounds__(kThreads, 1)
    coded_kernel(const __grid_constant__ Args a, const int32_t box_rows, const int32_t skip) {
  constexpr int DP = S::DP, NS = S::kSlots, RM = S::RM, DT = B200_ATTN_DTYPE_BF16;
  constexpr bool kTwo = S::kTwo;
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
    ptx::mbar_init(bar(S::kBarQ), kCodeWarps / 2);
    ptx::mbar_init(bar(S::kBarQRead), 1);
    for (int s = 0; s < 2 * NS; ++s) {
      ptx::mbar_init(bar(S::kBarFull + s), kCodeWarps / 2);
      ptx::mbar_init(bar(S::kBarEmpty + s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(bar(S::kBarScores + i), 1);
      ptx::mbar_init(bar(S::kBarWeights + i), 4);
      ptx::mbar_init(bar(S::kBarSums + i), 1);
    }
    for (int s = 0; s < kAhead; ++s) {
      ptx::mbar_init(bar(S::kBarPlan + s), 1);
      ptx::mbar_init(bar(S::kBarDone + s), kReaders);
    }
    for (int s = 0; s < S::kRawK + S::kRawV; ++s) {
      ptx::mbar_init(bar(S::kBarRawFull + s), 1);
      ptx::mbar_init(bar(S::kBarRawEmpty + s), kCodeWarps / 2);
    }
    ptx::mbar_init(bar(S::kBarDrain), 2);
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
  }
  ptx::grid_dependency_wait();
  if (threadIdx.x < kSoftmaxThreads) zero_unused_rows(a, 2, kSoftmaxThreads);
  find_run<typename S::G>(a, blockIdx.x, gridDim.x, reinterpret_cast<uint32_t*>(smem + S::kOffSums),
                          found);
  const Run& run = *found;
  if (run.done(run.p)) return;
  if (warp == kQkWarp) {
    ptx::tmem_alloc(sbase + S::kOffMisc, kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = misc[0];
  // rows of a unit, and of those one group's share
  auto unit_rows = [&](const Segment& p) {
    return min(a.unit_rows, p.drafts * a.group - p.rt * a.unit_rows);
  };
  const int share = kTwo ? a.unit_rows >> 1 : a.unit_rows;
  // group i takes tile j of a segment
  auto takes = [&](int i, int j, int rows) {
    return kTwo ? (i == 0 || rows > share) : (j & 1) == i;
  };
  // Segment `seg` of the run, by every reading warp; false: there is none, or a wait ran out.  A warp
  // that is done with a segment says so.
  volatile int* plan = reinterpret_cast<volatile int*>(smem + S::kOffPlan);
  auto segment = [&](uint32_t seg, Segment* p) {
    if (!warp_wait(bar(S::kBarPlan + seg % kAhead), (seg / kAhead) & 1u, abort_flag, a.err)) {
      p->n = 0;
      return false;
    }
    volatile int* x = plan + 8 * (seg % kAhead);
    *p = Segment{x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]};
    return p->n > 0;
  };
  auto segment_done = [&](uint32_t seg) {
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(bar(S::kBarDone + seg % kAhead));
  };
  float* row_scale = reinterpret_cast<float*>(smem + S::kOffRowScale);  // [kAhead][RM]
  float* key_scale = reinterpret_cast<float*>(smem + S::kOffKeyScale);  // [8 tiles][4 warps]
  float* own_scale = reinterpret_cast<float*>(smem + S::kOffOwnScale);  // [8 tiles][128 keys]

  if (warp == kLoadWarp) {
    // ------------------------------------------------ producer of coded rows
    // A box of rows that lie side by side is one copy; a lane a box.  The page numbers of a
    // tile are read while the tile before is copied.
    const int boxes = kTile / box_rows;
    const uint32_t size = static_cast<uint32_t>(a.page_size), inv_size = 0xffffffffu / size + 1u;
    auto slot_of = [&](uint32_t key) {  // key / size: the product is it or one more
      if (size == 1u) return key;
      const uint32_t q = __umulhi(key, inv_size);
      return q * size > key ? q - 1u : q;
    };
    uint32_t tiles = 0, seg = 0;
    uint32_t rk = 0, rv = 0, pk = 1u, pv = 1u;  // raw slots, and parities of their release
    Segment p;
    bool ok = true, more = segment(0, &p);
    int j = 0, next = -1;
    auto look_up = [&]() {
      const int key = (p.t + j) * kTile + lane * box_rows;
      next = lane < boxes && key < p.len + p.drafts ? __ldg(a.table + p.b * a.table_stride + slot_of(key))
                                                    : -1;
    };
    if (more) look_up();
#pragma unroll 1
    for (; ok && more; ++tiles) {
      const int k0 = (p.t + j) * kTile, valid = min(kTile, p.len + p.drafts - k0);
      const int32_t* table = a.table + p.b * a.table_stride;
      const uint8_t* kb = a.k + p.h * a.k_head;
      const uint8_t* vb = a.v + p.h * a.v_head;
      const int now = next;
      if (++j == p.n) {
        segment_done(seg);
        more = segment(++seg, &p);
        j = 0;
      }
      if (more) look_up();
      const uint32_t fk = bar(S::kBarRawFull + rk), fv = bar(S::kBarRawFull + S::kRawK + rv);
      ok = warp_wait(bar(S::kBarRawEmpty + rk), pk, abort_flag, a.err) &&
           warp_wait(bar(S::kBarRawEmpty + S::kRawK + rv), pv, abort_flag, a.err);
      if (!ok) break;
      const uint32_t at_k = S::kOffRaw + rk * S::kRawBytes, at_v = S::kOffRawV + rv * S::kRawBytes;
#pragma unroll 1
      for (int u = lane; u < boxes; u += 32) {
        const int key = u * box_rows, n = min(box_rows, valid - key);
        if (n <= 0) break;
        const uint32_t slot = slot_of(k0 + key), in = k0 + key - slot * size;
        const int page = u == lane ? now : __ldg(table + slot);
        if (page < 0 || page >= a.pages) {
          report_error(a.err, B200_ATTN_DEVERR_BOUNDS);
          for (int x = 0; x < n * S::kRawRow; x += 16) {  // rows without a page are zero
            *reinterpret_cast<uint4*>(smem + at_k + key * S::kRawRow + x) = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(smem + at_v + key * S::kRawRow + x) = make_uint4(0u, 0u, 0u, 0u);
          }
          ptx::fence_proxy_async_smem();
          continue;
        }
        const uint32_t bytes = n * S::kRawRow;
        expect_tx(fk, bytes);
        expect_tx(fv, bytes);
        if (!(kStall && u == 0 && static_cast<int>(tiles) == skip))
          bulk_copy(sbase + at_k + key * S::kRawRow, kb + page * a.k_page + in * a.k_row, bytes, fk);
        bulk_copy(sbase + at_v + key * S::kRawRow, vb + page * a.v_page + in * a.v_row, bytes, fv);
      }
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive(fk);
        ptx::mbar_arrive(fv);
      }
      if (++rk == S::kRawK) rk = 0, pk ^= 1u;
      if (++rv == S::kRawV) rv = 0, pv ^= 1u;
    }
    // Copies in flight land before the shared memory goes, also where this warp had issued its last
    // when another's wait ran out, or found no further segment because of it.
    for (uint32_t x = tiles > S::kRawK ? tiles - S::kRawK : 0u; x < tiles; ++x)
      settle(bar(S::kBarRawFull + x % S::kRawK), (x / S::kRawK) & 1u);
    for (uint32_t x = tiles > S::kRawV ? tiles - S::kRawV : 0u; x < tiles; ++x)
      settle(bar(S::kBarRawFull + S::kRawK + x % S::kRawV), (x / S::kRawV) & 1u);
    __syncwarp();
  } else if (warp == kQkWarp) {
    // -------------------------------------------------- scores S = Q K^T
    // By the whole warp, one lane of which issues: in control flow that is the same for the
    // warp the operands' descriptors stay in uniform registers.
    constexpr uint32_t id = ptx::idesc_f16(false, kTile, kTile, false);
    uint32_t tile = 0, seg = 0;
    uint32_t made = 0u, any = 0u;  // bit i: parity of the number of scores made for group i, and any
    bool ok = true;
    Segment p;
#pragma unroll 1
    for (; ok && segment(seg, &p); ++seg) {
      const int n = __shfl_sync(0xffffffffu, p.n, 0);
      const bool second = !kTwo || __shfl_sync(0xffffffffu, unit_rows(p), 0) > share;
      ok = warp_wait(bar(S::kBarQ), seg & 1u, abort_flag, a.err);
#pragma unroll 1
      for (int j = 0; ok && j < n; ++j, ++tile) {
        const uint32_t s = tile % NS;
        ok = warp_wait(bar(S::kBarFull + s), (tile / NS) & 1u, abort_flag, a.err);
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          if (!ok || (kTwo ? (i == 1 && !second) : (j & 1) != i)) continue;
          // the weights that lie over the group's last scores have been used
          ok = !((any >> i) & 1u) ||
               warp_wait(bar(S::kBarSums + i), ((made >> i) & 1u) ^ 1u, abort_flag, a.err);
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
              ptx::tc_mma_ss(tmem + kTile * i, qd + off, kd + off, id, kk > 0 ? 1u : 0u);
            }
            ptx::tc_commit(bar(S::kBarScores + i));
          }
          __syncwarp();
          made ^= 1u << i;
          any |= 1u << i;
        }
        if (ok && elect_one()) ptx::tc_commit(bar(S::kBarEmpty + s));
        __syncwarp();
      }
      if (elect_one()) ptx::tc_commit(bar(S::kBarQRead));
      segment_done(seg);
    }
    if (elect_one()) {
      ptx::tc_commit(bar(S::kBarDrain));
      settle(bar(S::kBarDrain), 0);
    }
    __syncwarp();
  } else if (warp == kPlanWarp) {
    // ------------------------------------------------- segments and their masks
    Place pl = run.p;
    bool ok = true, more = true;
#pragma unroll 1
    for (uint32_t seg = 0; ok && more; ++seg) {
      const uint32_t at = seg % kAhead;
      ok = warp_wait(bar(S::kBarDone + at), ((seg / kAhead) & 1u) ^ 1u, abort_flag, a.err);
      if (!ok) break;
      more = !run.done(pl);
      const int n = more ? run.tiles(pl) : 0;
      if (more && a.tokens <= kSeen) {
        // a bit for each drafted token that a token sees
#pragma unroll 1
        for (int x = lane; x < 2 * a.tokens; x += 32)
          reinterpret_cast<uint32_t*>(seen)[at * 2 * kSeen + x] =
              (x & 1) && a.tokens <= 32 ? 0u : seen_word(a, pl.b, x >> 1, 32 * (x & 1), pl.s.drafts);
      }
      if (lane == 0) {
        volatile int* x = plan + 8 * at;
        x[0] = pl.b, x[1] = pl.h, x[2] = pl.rt, x[3] = pl.t, x[4] = n, x[5] = pl.tiles;
        x[6] = pl.s.len, x[7] = pl.s.drafts;
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(S::kBarPlan + at));
      pl.t += n;
      if (more && pl.t == pl.tiles) pl = next_unit<typename S::G>(a, pl);
    }
    __syncwarp();
  } else if (warp == kPvWarp) {
    // ------------------------------------------------------- O_i += P_i V
    constexpr uint32_t id = ptx::idesc_f16(true, kTile, DP, true);
    uint32_t tile = 0, seg = 0;
    uint32_t made = 0u;  // bit i: parity of the number of products made for group i
    bool ok = true;
    Segment p;
#pragma unroll 1
    for (; ok && segment(seg, &p); ++seg) {
      const int n = __shfl_sync(0xffffffffu, p.n, 0);
      const int rows = __shfl_sync(0xffffffffu, unit_rows(p), 0);
      uint32_t begun = 0u;  // bit i: O_i holds a product of this segment
#pragma unroll 1
      for (int j = 0; ok && j < n; ++j, ++tile) {
        const uint32_t s = tile % NS;
        ok = warp_wait(bar(S::kBarFull + NS + s), (tile / NS) & 1u, abort_flag, a.err);
        const uint32_t va = sbase + S::kOffV + s * S::kTileBytes;
        const uint64_t vd = ptx::smem_desc_sw128(va, S::kChunkBytes, 1024);
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          if (!ok || !takes(i, j, rows)) continue;
          ok = warp_wait(bar(S::kBarWeights + i), (made >> i) & 1u, abort_flag, a.err);
          if (!ok) continue;
          ptx::tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kTile / 16; ++kk) {
              // 32 keys' weights lie over their scores: 16 columns rounded, 16 of what that left
              const uint32_t w = tmem + kTile * i + 32 * (kk >> 1) + 8 * (kk & 1);
              ptx::tc_mma_ts(tmem + S::kColO + DP * i, w, vd + kk * (2048 >> 4), id,
                             (((begun >> i) & 1u) || kk > 0) ? 1u : 0u);
              ptx::tc_mma_ts(tmem + S::kColO + DP * i, w + 16, vd + kk * (2048 >> 4), id, 1u);
            }
            ptx::tc_commit(bar(S::kBarSums + i));
          }
          __syncwarp();
          begun |= 1u << i;
          made ^= 1u << i;
        }
        if (ok && elect_one()) ptx::tc_commit(bar(S::kBarEmpty + NS + s));
        __syncwarp();
      }
      segment_done(seg);
    }
    if (elect_one()) {
      ptx::tc_commit(bar(S::kBarDrain));
      settle(bar(S::kBarDrain), 0);
    }
    __syncwarp();
  } else if (warp >= kCodeWarp) {
    // ------------------------------------------- operands from queries and codes
    // Four warps for the keys, four for the queries and the values, a thread a row of a tile.
    const int wq = (warp - kCodeWarp) & 3, row = 32 * wq + lane;
    const bool value = warp >= kCodeWarp + 4;
    auto put = [&](uint32_t at, int piece, uint4 v) {
      *reinterpret_cast<uint4*>(smem + at + (piece >> 3) * S::kChunkBytes + row * 128 +
                                (((piece & 7) ^ (row & 7)) << 4)) = v;
    };
    auto hand_over = [&](int b) {  // what the warp wrote, to the tensor cores
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(b));
    };
    // The queries of a segment: fp16, times the power of two that brings the row's largest
    // number to 2^13..2^14.
    auto queries = [&](const Segment& p, uint32_t seg) {
      const int rows = unit_rows(p);
#pragma unroll 1
      for (int i = 0; i < (kTwo ? 2 : 1); ++i) {
        if (row >= share || i * share + row >= rows) continue;
        const int r = p.rt * a.unit_rows + i * share + row, tok = r / a.group;
        const uint8_t* src = a.q + p.b * a.q_seq + (p.h * a.group + r - tok * a.group) * a.q_head +
                             tok * a.q_tok;
        float big = 0.f;
#pragma unroll 4
        for (int x = 0; x < a.head_dim / 8; ++x) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + x);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float2 f = unpack2<DT>(w[y]);
            big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        const int e = max(static_cast<int>(__float_as_uint(big) >> 23), 20);
        const float up = __uint_as_float(static_cast<uint32_t>(267 - e) << 23);
#pragma unroll 4
        for (int x = 0; x < DP / 8; ++x) {
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (8 * x < a.head_dim) v = __ldg(reinterpret_cast<const uint4*>(src) + x);
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float2 f = unpack2<DT>(w[y]);
            w[y] = pack2<B200_ATTN_DTYPE_FP16>(f.x * up, f.y * up);
          }
          put(S::kOffQ + i * S::kTileBytes, x, make_uint4(w[0], w[1], w[2], w[3]));
        }
        row_scale[(seg % kAhead) * RM + i * kTile + row] =
            __uint_as_float(static_cast<uint32_t>(e - 13) << 23);
      }
      hand_over(S::kBarQ);
    };
    uint32_t r = 0, rp = 0;  // raw slot and parity of its filling
    uint32_t e0 = 0, ep = 1u;  // slot of the operand and parity of its release
    const uint32_t raw_slots = value ? S::kRawV : S::kRawK;
    auto tile_of = [&](int k0, int len, int total, uint32_t seg, uint32_t t) {
      const uint32_t raw_bar = value ? S::kRawK + r : r, s = value ? NS + e0 : e0;
      if (!warp_wait(bar(S::kBarRawFull + raw_bar), rp, abort_flag, a.err)) return false;
      const uint8_t* codes = smem + S::kOffRaw + raw_bar * S::kRawBytes + row * S::kRawRow;
      const int key = k0 + row;
      uint4 meta = make_uint4(0u, 0u, 0u, 0u);  // what lies past the last key counts as 0
      if (key < total) meta = *reinterpret_cast<const uint4*>(codes + DP / 2);
      uint32_t m[4] = {meta.x, meta.y, meta.z, meta.w};
      const uint32_t at = S::kOffRing + s * S::kTileBytes;
      auto put_here = [&](int piece, uint4 v) { put(at, piece, v); };
      if (value) {
        if (key >= len) {
          // a hidden value must not reach a row as 0 x NaN: added by the softmax groups
          bool odd = false;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t f = not_finite<DT>(m[x]);
            odd |= f != 0u;
            m[x] &= ~f;
          }
          // (a warp that is ahead may have noted a later segment)
          if (odd) atomicMax(const_cast<uint32_t*>(&misc[2]), seg + 1u);
        }
        auto as = [](uint32_t x) { return *reinterpret_cast<const __nv_bfloat162*>(&x); };
        __nv_bfloat162 step[2], low[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int from = y ? 0x7632 : 0x5410;
          step[y] = as(DP == 128 ? m[y] : __byte_perm(m[0], m[1], from));
          low[y] = as(DP == 128 ? m[2 + y] : __byte_perm(m[2], m[3], from));
        }
        if (!warp_wait(bar(S::kBarEmpty + s), ep, abort_flag, a.err)) return false;
        values<DP>(codes, step, low, put_here);
      } else {
        // fp16, times the power of two that brings the warp's largest number below 2^14
        uint32_t e = 20u;
        float steps[4], lows[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          steps[g] = half_of(m[g / 2], g & 1), lows[g] = half_of(m[2 + g / 2], g & 1);
          const float most = fmaxf(fabsf(lows[g]), fabsf(fmaf(15.f, steps[g], lows[g])));
          if (isfinite(steps[g]) && isfinite(lows[g]))
            e = max(e, __float_as_uint(fminf(most, 0x1.fffffep127f)) >> 23);
        }
        // Of drafted tokens each key's own power of two: one that a row does not see is not to cost it
        // bits of the others.
        const bool own = k0 + kTile > len;
        if (!own) e = __reduce_max_sync(0xffffffffu, e);
        const float down = __uint_as_float((e - 13u) << 23);
        if (own) own_scale[(t & 7u) * kTile + row] = down;
        if (lane == 0) key_scale[(t & 7u) * 4 + wq] = own ? 1.f : down;
        const float up = __uint_as_float((267u - e) << 23);
        __half2 step[4], low[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          step[g] = __float2half2_rn(steps[g] * up);
          low[g] = __float2half2_rn(lows[g] * up);
        }
        if (!warp_wait(bar(S::kBarEmpty + s), ep, abort_flag, a.err)) return false;
        keys<DP>(codes, step, low, put_here);
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(S::kBarRawEmpty + raw_bar));
      hand_over(S::kBarFull + s);
      if (++r == raw_slots) r = 0, rp ^= 1u;
      if (++e0 == NS) e0 = 0, ep ^= 1u;
      return true;
    };
    uint32_t t = 0;
    bool ok = true;
    Segment p;
#pragma unroll 1
    for (uint32_t seg = 0; ok && segment(seg, &p); ++seg) {
      if (value) {
        ok = seg == 0 || warp_wait(bar(S::kBarQRead), (seg - 1u) & 1u, abort_flag, a.err);
        if (ok) queries(p, seg);
      }
#pragma unroll 1
      for (int j = 0; ok && j < p.n; ++j, ++t)
        ok = tile_of((p.t + j) * kTile, p.len, p.len + p.drafts, seg, t);
      segment_done(seg);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax
    const int i = warp >> 2, quad = warp & 3, rl = quad * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    // the weights take the place of the scores that have been read
    const uint32_t tS = tmem + lanes + kTile * i, tO = tmem + lanes + S::kColO;
    const int row0 = i * (kTwo ? share : 0);  // first row of this group in the unit
    uint32_t seg = 0, cnt = 0;  // segments of the run, tiles of this group
    uint32_t tile0 = 0;         // tiles of both groups before the segment
    bool ok = true;
    // what is needed of the segment only at its ends stays in shared memory
    volatile int* unit = plan;
    Segment begin;
#pragma unroll 1
    for (;; ++seg) {
      if (!segment(seg, &begin)) {
        // Where a wait ran out some of the warps can have the segment and others not: each comes to the
        // barrier below once a segment, the one that none has included, or those that have it would wait
        // for the others for good.
        if constexpr (!kTwo) ptx::named_barrier_and(1, kSoftmaxThreads, false);
        break;
      }
      unit = plan + 8 * (seg % kAhead);
      const int n = begin.n, rows = unit_rows(begin), t0 = begin.t, len = begin.len;
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
          warp_arrive(bar(S::kBarWeights + i), lane);
          ++cnt;
          continue;
        }
        // from the products' unit to that of the exponents, for the keys of each of four warps
        const float* ks = key_scale + ((tile0 + j) & 7u) * 4;
        const float* pow_r = row_scale + (seg % kAhead) * RM + (kTwo ? i * kTile : 0) + rl;
        float rs = a.scale_log2 * *pow_r;
        // a bit for each of 32 keys that this row sees
        uint64_t bits = 0u;
        int tok = 0;
        if (partly) {
          tok = min((unit[2] * a.unit_rows + row0 + rl) / a.group, a.tokens - 1);
          if (a.tokens <= kSeen) bits = seen[(seg % kAhead) * kSeen + tok];
          rs = a.scale_log2 * fmaxf(*pow_r * 0x1p-13f, 1.f);
        }
        auto visible = [&](int c) {
          const int d = k0 + 32 * c - len;
          if (d <= -32) return ~0u;
          if (a.tokens > kSeen) return first_bits(min(unit[7], tok + 1) - d);  // a chain
          return d >= 64 ? 0u
                         : static_cast<uint32_t>(d < 0 ? bits << -d | ((1u << -d) - 1u) : bits >> d);
        };
        // A key's own power of two (up to 2^114) and the row's act as one factor: a score times the
        // key's alone would pass the range where the row's numbers are next to nothing.  What of the
        // row's is over 2^13 waits for the scale, so that the factor is finite.
        auto drafted = [&](uint32_t (&sr)[32], int c) {
          const float near = fminf(*pow_r, 0x1p13f);
          const float4* f = reinterpret_cast<const float4*>(own_scale + ((tile0 + j) & 7u) * kTile + 32 * c);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float4 x = f[k];
            scale2(sr[4 * k], sr[4 * k + 1], x.x, x.y, near);
            scale2(sr[4 * k + 2], sr[4 * k + 3], x.z, x.w, near);
          }
          hide(sr, visible(c));
        };
        // neither 0, as a hidden score is -inf, nor infinite, as a score may be 0
        auto to_log2 = [&](int c) { return fminf(fmaxf(rs * ks[c], 0x1p-149f), 0x1.fffffep127f); };
        // Twice over the scores, 32 at a time: little code, few registers.
        float mx = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t sr[32];
          ptx::tmem_ld_32x32b_x32(tS + 32 * c, sr);
          ptx::tmem_wait_ld();
          if (partly) drafted(sr, c);
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int k = 0; k < 32; k += 2)
            top[(k >> 1) & 1] =
                max3(top[(k >> 1) & 1], __uint_as_float(sr[k]), __uint_as_float(sr[k + 1]));
          mx = fmaxf(mx, fmaxf(top[0], top[1]) * to_log2(c));
        }
        const bool resc = mx > m_run + kGrowth || (m_run == -INFINITY && mx > m_run);
        const float m_new = resc ? mx : m_run;
        const float alpha = resc ? ptx::ex2_approx(m_run - m_new) : 1.f;
        m_run = m_new;
        l_run *= alpha;
        // (the scores were formed after the last product of the group, so O_i is at rest)
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
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t sr[32], hi[16], lo[16];
          ptx::tmem_ld_32x32b_x32(tS + 32 * c, sr);
          ptx::tmem_wait_ld();
          if (partly) drafted(sr, c);
          const float up = to_log2(c);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x, y;
            fma2(x, y, __uint_as_float(sr[2 * e]), __uint_as_float(sr[2 * e + 1]), up, neg);
            x = ptx::ex2_approx(x);
            y = ptx::ex2_approx(y);
            add2(sum[2 * (e & 1)], sum[2 * (e & 1) + 1], x, y);
            hi[e] = pack2<DT>(x, y);
            const float2 r = unpack2<DT>(hi[e]);
            lo[e] = pack2<DT>(x - r.x, y - r.y);
          }
          st_x16(tS + 32 * c, hi);
          st_x16(tS + 32 * c + 16, lo);
        }
        l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        ptx::tmem_wait_st();
        warp_arrive(bar(S::kBarWeights + i), lane);
        ++cnt;
        ++done;
      }
      // while the last product runs: where the row's results go
      const int ub = unit[0], uh = unit[1], urt = unit[2], tiles = unit[5];
      const bool first = t0 == 0, last = t0 + n == tiles, finish = first && last;
      const bool mine = rl < share && row0 + rl < rows;
      const int row = urt * a.unit_rows + row0 + rl, tok = min(row / a.group, a.tokens - 1);
      uint8_t* out = a.o + ub * a.o_seq + (uh * a.group + row % a.group) * a.o_head + tok * a.o_tok;
      float* part = a.partial +
                    static_cast<int64_t>(2 * blockIdx.x + (first ? 1 : 0)) * (RM * (DP + 2));
      tile0 += n;
      __syncwarp();
      if (ok && cnt > 0) ok = warp_wait(bar(S::kBarSums + i), (cnt - 1u) & 1u, abort_flag, a.err);
      __syncwarp();
      // ---------------------------------------------------- end of a segment
      float2* told = reinterpret_cast<float2*>(smem + S::kOffTold);  // for the other group
      if (!kTwo) told[kTile * i + rl] = make_float2(m_run, l_run);
      if constexpr (!kTwo) ok = ptx::named_barrier_and(1, kSoftmaxThreads, ok);
      if (!ok) break;
      ptx::tc_fence_after();
      // (a later segment's may have been noted already: then add_odd looks, and finds none)
      const bool any_odd = misc[2] > seg;
      // weights of the groups' sums in this thread's row
      float top = m_run, total = l_run, w[2] = {1.f, 1.f};
      if constexpr (!kTwo) {
        const float2 other = told[kTile * (1 - i) + rl];
        const float m_other = other.x;
        top = fmaxf(m_run, m_other);
        const float mine_w = m_run == -INFINITY ? 0.f : ptx::ex2_approx(m_run - top);
        const float other_w = m_other == -INFINITY ? 0.f : ptx::ex2_approx(m_other - top);
        total = mine_w * l_run + other_w * other.y;
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
        add_odd4<DP, DT>(a, ub, uh, Seq{len, unit[7]}, tok, t0 * kTile - len, (t0 + n) * kTile - len,
                         col0, col1, finish ? reinterpret_cast<uint16_t*>(out) : nullptr,
                         part + row0 + rl, RM);
      }
      if (threadIdx.x == 0 && last)
        a.desc[(ub * a.kv_heads + uh) * a.row_tiles + urt] =
            make_int2(first ? static_cast<int>(blockIdx.x) : run.first_run,
                      static_cast<int>(blockIdx.x));
      // both groups' sums have been read by both
      ptx::tc_fence_before();
      if constexpr (!kTwo) ptx::named_barrier_sync(1, kSoftmaxThreads);
      segment_done(seg);
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
template <class S, bool kStall = false>
int32_t launch_coded_shape(const Args& a, int box_rows, int runs, int device, cudaStream_t s,
                           int32_t skip = -1) {
  using namespace b200paged;
  static std::once_flag once[kMaxDevices];
  static cudaError_t err[kMaxDevices];
  std::call_once(once[device], [&] {
    err[device] = cudaFuncSetAttribute(coded_kernel<S, kStall>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmemBytes);
  });
  if (err[device] != cudaSuccess) {
    set_error(cudaGetErrorString(err[device]));
    return B200_ATTN_ERR_LAUNCH;
  }
  return launch(coded_kernel<S, kStall>, dim3(runs), dim3(kThreads), S::kSmemBytes, s, a, box_rows, skip);
}

// Rows that lie side by side and in one page, whatever the place of the first.
int box_of(int dp, const Args& a) {
  const int row = dp / 2 + 16;
  int box = 1;
  if (a.k_row == row && a.v_row == row)
    while (box < kTile && a.page_size % (2 * box) == 0) box *= 2;
  return box;
}

}  // namespace

int32_t launch_coded(int rm, int dp, const Args& a, int runs, int device, cudaStream_t s) {
  const int box = box_of(dp, a);
  if (rm == 256)
    return dp == 64 ? launch_coded_shape<CodedShape<64, true>>(a, box, runs, device, s)
                    : launch_coded_shape<CodedShape<128, true>>(a, box, runs, device, s);
  return dp == 64 ? launch_coded_shape<CodedShape<64, false>>(a, box, runs, device, s)
                  : launch_coded_shape<CodedShape<128, false>>(a, box, runs, device, s);
}

int32_t launch_coded_stall(int rm, const Args& a, int runs, int device, cudaStream_t s, int32_t skip) {
  const int box = box_of(128, a);
  return rm == 256 ? launch_coded_shape<CodedShape<128, true>, true>(a, box, runs, device, s, skip)
                   : launch_coded_shape<CodedShape<128, false>, true>(a, box, runs, device, s, skip);
}

}  // namespace b200tree
