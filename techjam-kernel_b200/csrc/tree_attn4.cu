// tree_attn4.cu — drafted-token attention over a paged cache held in 4 bits
// (format: b200_cache4.h; division of the work and joins: tree_attn.cuh).
//
// Mathematics.  With k = low + step code in each of four groups g of numbers,
//   q.k = sum_g step_g (q.code)_g + low_g (sum of q)_g,
// so the products are of queries and whole numbers 0..15, exact in the tensor cores' fp32
// sums, and steps are applied to the four partial products of a row and key in fp32; the lows
// are one more product, of the queries' group sums split into three bf16 numbers.  With
// weights w = 2^(s - m),
//   sum w v = sum_g (w step_g) code + w low_g:
// w step_g is rounded to fp16 (relative to a power of two that follows the largest step that the row
// sees), w low_g
// and sum w are fp32.  For results of fp16 the codes of values are taken less 8 and the lows plus
// 8 steps: of numbers on both sides of zero low and step code are each a multiple of the
// sum, and so was the error of the rounded w step_g (24 sequences of 7 rows, head dim 64: 1.45
// times that of weights and values rounded to fp16, now 1.1 times; 45.6 us without, 47.3 with).
//
// A half byte becomes an fp16 operand by one AND: bits 0..3 of a half word are the subnormal
// number code 2^-24, bits 4..7 the number 16 code 2^-24 (the factors go into the queries and
// the result).  The rows of keys and values are laid out so that a lane's operands of a product
// lie in its words: 8 numbers take 4 ANDs and a shift, and for values, whose pairs come
// from two rows, two byte permutes.
//
// As in the kernel of 16-bit caches (tree_attn_rows.cuh) the warps of a CTA share a key tile,
// 32 keys each, and fetch them into rings of their own, in bulk copies: one a block where its rows
// lie in one page.  Bound by the issue of instructions and their latency, with HBM at half of its
// rate: a block of 32 keys of 8 rows takes 690 instructions of a warp, of them 170 for the
// scores, 260 for the values and 60 for its copies (64 sequences of up to 8191 keys, 8 key heads x 4, D
// 128: 104 us, 51 us of bytes).  Four CTAs an SM where up to 8 rows leave the registers for it (64
// sequences of 250 keys: 22.3 us, with two 25.5).
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "b200_cache4.h"
#include "error_word.cuh"
#include "paged_host.h"
#include "tree_attn.cuh"
#include "tree_attn4.cuh"
#include "tree_attn_host.cuh"
#include "tree_attn_rows.cuh"

namespace b200tree {

namespace {

// Up to 16 rows a unit (FEW: up to 8, whose other half is left out of the softmax), head dim
// padded to DP.
template <bool FEW_, int DP_>
struct Shape4 {
  static constexpr bool FEW = FEW_;
  static constexpr int DP = DP_, RM = 16;
  static constexpr int kWarps = 4, kThreads = 32 * kWarps, kCtas = !FEW ? 2 : 4;  // CTAs of an SM
  static constexpr int kParts = 2, kKeys = kParts * kRowKeys;  // keys of a warp's block
  static constexpr int kTile = kWarps * kKeys;
  static constexpr int kHalves = FEW ? 1 : 2;
  static constexpr int kCodes = DP / 2, kRowBytes = kCodes + 16;
  static constexpr int kPieces = kRowBytes / 16;
  static constexpr int kPartBytes = kRowKeys * kRowBytes;  // 16 keys, or values
  static constexpr int kBlockBytes = kParts * 2 * kPartBytes;
  static constexpr int kStages = DP == 128 ? (FEW ? 2 : 4) : (FEW ? 3 : 5);
  static constexpr int kRingBytes = kWarps * kStages * kBlockBytes;
  static constexpr int kJoinRows = FEW ? 8 : 16;
  static constexpr int kJoinCols = 512 / kJoinRows;
  static constexpr int kEach = kJoinRows * kJoinCols / kThreads;  // columns of a thread in a join
  static constexpr int kJoinPitch = kJoinCols + 4;
  static constexpr int kOffJoin = kRingBytes;
  static constexpr int kJoinBytes = 4 * kWarps * kJoinRows * kJoinPitch;
  static constexpr int kOffStat = kOffJoin + kJoinBytes;
  static constexpr int kOffPlaces = kOffStat + 4 * 2 * kWarps * RM;  // of the warps' loads, and two units
  static constexpr int kOffBars = kOffPlaces + (kWarps + 2) * sizeof(Place);  // a barrier a block
  static constexpr int kOffMisc = kOffBars + 8 * kWarps * kStages;
  static constexpr int kSmemBytes = kOffMisc + 256;
  static_assert(kCtas * (kSmemBytes + 1024) <= 233472, "exceeds the shared memory of an SM");
  using G = Grid<RM, kTile, 1>;
  static_assert(sizeof(JoinSmem<DP, kWarps>) <= kJoinBytes, "joins in place");
};

// Products m16n8k16 without side effects, which the compiler may move: d = a b + c.
template <int DT>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                    float c0, float c1, float c2, float c3) {
  if constexpr (DT == B200_ATTN_DTYPE_BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2),
          "f"(c3));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2),
          "f"(c3));
}
template <class T>
__device__ __forceinline__ T lds(const uint8_t* at) {
  return *reinterpret_cast<const T*>(at);
}
__device__ __forceinline__ float low_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// A 16-bit number of shared memory in both halves.
__device__ __forceinline__ uint32_t twice16(const uint8_t* at) {
  return __byte_perm(lds<uint16_t>(at), 0u, 0x1010);
}
// The transpose of an 8 x 8 matrix of 16-bit numbers, of which each lane has two of a row.
__device__ __forceinline__ uint32_t turned(uint32_t w) {
  uint32_t v;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(v) : "r"(w));
  return v;
}
// The larger bf16 of each half; a NaN counts as nothing.
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Waits for a block's copies, a second at most; false (reported) when they did not come.  By
// whole warps.
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, int32_t* err) {
  const uint64_t t0 = b200attn::ptx::globaltimer_ns();
  bool ok;
  do {
    ok = b200attn::ptx::mbar_try_wait(bar, parity);
  } while (!ok && b200attn::ptx::globaltimer_ns() - t0 < 1000000000ull);
  ok = __all_sync(0xffffffffu, ok);
  if (!ok) report_error(err, B200_ATTN_DEVERR_WAIT_TIMEOUT);
  return ok;
}

constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;

// Pairs of fp16 numbers, x - y: of codes exact.
__device__ __forceinline__ uint32_t less(uint32_t x, uint32_t y) {
  const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y));
  return *reinterpret_cast<const uint32_t*>(&d);
}

template <class S, int DT>
__global__ void __launch_bounds__(S::kThreads, S::kCtas)
    rows4_kernel(const __grid_constant__ Args a) {
  constexpr int RM = S::RM, DP = S::DP, NS = S::kStages, NG = DP / 32, NT = S::kHalves;
  constexpr bool kCentred = DT == B200_ATTN_DTYPE_FP16;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sbase = b200attn::ptx::smem_u32(smem);
  float* join = reinterpret_cast<float*>(smem + S::kOffJoin);
  float* stat = reinterpret_cast<float*>(smem + S::kOffStat);  // [warp][{max, sum}][RM]
  uint32_t* sums = reinterpret_cast<uint32_t*>(smem + S::kOffMisc);
  Run* found = reinterpret_cast<Run*>(smem + S::kOffMisc + 80);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r8 = lane >> 2, c4 = lane & 3;  // row, and half the column, of this lane in a product
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  find_run<typename S::G>(a, blockIdx.x, gridDim.x, sums, found);
  const Run& run = *found;

  uint8_t* blocks = smem + warp * (NS * S::kBlockBytes);  // this warp's ring
  const uint32_t ring = sbase + warp * (NS * S::kBlockBytes);
  const uint32_t bars = sbase + S::kOffBars + 8 * NS * warp;
  const uint32_t size = static_cast<uint32_t>(a.page_size);
  const bool whole = a.page_size % kRowKeys == 0;  // 16 keys lie in one page

  // ------------------------------------------------------------- loads
  // The warp's next block to load: its first key and the blocks left in the unit, which itself is in
  // shared memory (`at`): registers are what limits the warps on an SM.  Page numbers are read
  // one block ahead.
  Place* at = reinterpret_cast<Place*>(smem + S::kOffPlaces) + warp;
  int ld_key = 0, ld_left = 0;
  auto enter = [&](const Place& p) {
    __syncwarp();
    if (lane == 0) *at = p;
    __syncwarp();
    ld_left = run.done(p) ? 0 : run.tiles(p);
    ld_key = p.t * S::kTile + warp * S::kKeys;
  };
  enter(run.p);
  int page = -1, page_row = 0;
  const uint32_t inv_size = 0xffffffffu / size + 1u;  // 0 for size 1
  auto look_up = [&]() {  // a lane a key, or where 16 keys share a page, the first of them
    const int key = ld_key + (whole ? lane & 16 : lane);
    page = -1;
    page_row = 0;
    if (key < at->s.len + at->s.drafts) {
      // key / size or one more: key is below 2^30
      uint32_t slot = size == 1u ? key : __umulhi(key, inv_size);
      page_row = key - static_cast<int>(slot * size);
      if (page_row < 0) {
        --slot;
        page_row += static_cast<int>(size);
      }
      page = __ldg(a.table + at->b * a.table_stride + slot);
    }
  };
  if (ld_left > 0) look_up();
  int stage = 0;  // stage the next loads go to
  bool dead = false;  // a wait ran out
  const bool tight = whole && a.k_row == S::kRowBytes && a.v_row == S::kRowBytes;
  auto issue = [&]() {
    if (ld_left > 0 && !dead) {
      const int ld_keys = at->s.len + at->s.drafts - ld_key;
      const uint8_t* ld_k = a.k + at->h * a.k_head;
      const uint8_t* ld_v = a.v + at->h * a.v_head;
      const uint32_t bar = bars + 8 * stage;
      const uint32_t dst = ring + stage * S::kBlockBytes + (lane / 16) * (2 * S::kPartBytes);
      if (tight && __all_sync(0xffffffffu, ld_keys >= S::kKeys && static_cast<uint32_t>(page) <
                                                                      static_cast<uint32_t>(a.pages))) {
        // 16 keys that lie side by side, and their values, in one copy each
        if (lane == 0) b200attn::ptx::mbar_arrive_expect_tx(bar, S::kBlockBytes);
        if ((lane & 15) == 0) {
          const int in = page_row * S::kRowBytes;
          bulk_copy(dst, ld_k + page * a.k_page + in, S::kPartBytes, bar);
          bulk_copy(dst + S::kPartBytes, ld_v + page * a.v_page + in, S::kPartBytes, bar);
        }
      } else {
        // a lane a key
        bool there = lane < ld_keys;
        if (there && (page < 0 || page >= a.pages)) {
          report_error(a.err, B200_ATTN_DEVERR_BOUNDS);
          there = false;
          for (int x = 0; x < 2 * S::kPieces; ++x)  // a row without a page is zero
            *reinterpret_cast<uint4*>(blocks + stage * S::kBlockBytes + (lane / 16) * (2 * S::kPartBytes) +
                                      (x / S::kPieces) * S::kPartBytes + (lane & 15) * S::kRowBytes +
                                      16 * (x % S::kPieces)) = make_uint4(0u, 0u, 0u, 0u);
          b200attn::ptx::fence_proxy_async_smem();
        }
        const uint32_t rows = __popc(__ballot_sync(0xffffffffu, there));
        if (lane == 0) b200attn::ptx::mbar_arrive_expect_tx(bar, rows * 2 * S::kRowBytes);
        if (there) {
          const int64_t in = page_row + (whole ? lane & 15 : 0);
          const uint32_t to = dst + (lane & 15) * S::kRowBytes;
          bulk_copy(to, ld_k + page * a.k_page + in * a.k_row, S::kRowBytes, bar);
          bulk_copy(to + S::kPartBytes, ld_v + page * a.v_page + in * a.v_row, S::kRowBytes, bar);
        }
      }
      ld_key += S::kTile;
      if (--ld_left == 0) {
        Place p = *at;
        p.t += run.tiles(p);
        if (p.t == p.tiles) p = next_unit<typename S::G>(a, p);
        enter(p);
      }
      if (ld_left > 0) look_up();
      stage = stage + 1 == NS ? 0 : stage + 1;
    }
  };
  if (lane == 0)
    for (int x = 0; x < NS; ++x) b200attn::ptx::mbar_init(bars + 8 * x, 1);
  b200attn::ptx::fence_mbar_init();
  __syncwarp();
#pragma unroll 1
  for (int x = 0; x < NS - 1; ++x) issue();

  // the CTA's unit, and the one after it
  Place* units = reinterpret_cast<Place*>(smem + S::kOffPlaces) + S::kWarps;
  if (tid == 0) units[0] = run.p;
  __syncthreads();
  int flip = 0;
  int use = 0;          // stage of the block at hand
  uint32_t parity = 0;  // of its barrier

#pragma unroll 1
  while (!run.done(units[flip])) {
    const Place& pl = units[flip];
    const int t0 = pl.t;
    const int n = run.tiles(pl);
    const int len = pl.s.len, keys = len + pl.s.drafts;
    const int rows = min(RM, pl.s.drafts * a.group - pl.rt * RM);

    // ----------------------------------------------------------- queries
    // Row r8 (and r8 + 8) as fp16 operands, times the power of two that brings the row's
    // largest number to 2^13..2^14; the pairs that meet the codes' high half bytes, by 1/16 more.
    uint32_t qf[NT][DP / 16][2];
    uint32_t qs[NT][2];   // the sums of the four groups, in three bf16 numbers
    float to_log2[NT][2];  // from the products' unit to that of the exponents: rows 2 c4, 2 c4 + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[DP / 16][4];
      const int r = r8 + 8 * nt;
      const int row = pl.rt * RM + r, tok = row / a.group;
      const uint8_t* src = a.q + pl.b * a.q_seq +
                           (pl.h * a.group + row - tok * a.group) * a.q_head + tok * a.q_tok;
      float big = 0.f, sum[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = DP / 4 * g + NG * 2 * c4;  // 8 or 4 numbers of the group
        uint32_t w[NG];
#pragma unroll
        for (int i = 0; i < NG; ++i) w[i] = 0u;
        if (r < rows && d < a.head_dim) {
          if constexpr (NG == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(src + 2 * d);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(src + 2 * d);
            w[0] = v.x, w[1] = v.y;
          }
        }
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          const float2 f = unpack_pair<DT>(w[i]);
          big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
          float* dst = x[NG == 4 ? 2 * g + i / 2 : g];
          dst[2 * (i & 1)] = f.x;
          dst[2 * (i & 1) + 1] = f.y;
        }
      }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      const int e = max(static_cast<int>(__float_as_uint(big) >> 23), 20);
      const float up = __uint_as_float(static_cast<uint32_t>(267 - e) << 23);  // 2^(13 - exponent)
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        qf[nt][i][0] = pack_pair<B200_ATTN_DTYPE_FP16>(x[i][0] * up, x[i][1] * up);
        qf[nt][i][1] =
            pack_pair<B200_ATTN_DTYPE_FP16>(x[i][2] * up * 0.0625f, x[i][3] * up * 0.0625f);
      }
      float mine = 0.f;  // the sum of group c4, in the unit of the products
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        sum[g] = 0.f;
#pragma unroll
        for (int i = DP / 64 * g; i < DP / 64 * (g + 1); ++i)
          sum[g] += (x[i][0] * up + x[i][1] * up) + (x[i][2] * up + x[i][3] * up);
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
        if (g == c4) mine = sum[g] * 0x1p-24f;
      }
      const uint32_t hi = pack_pair<B200_ATTN_DTYPE_BF16>(mine, 0.f);
      const float rest = mine - low_half(hi);
      const uint32_t mid = pack_pair<B200_ATTN_DTYPE_BF16>(rest, 0.f);
      qs[nt][0] = hi | mid << 16;
      qs[nt][1] = pack_pair<B200_ATTN_DTYPE_BF16>(rest - low_half(mid), 0.f);
      // (neither 0, as a hidden score is -inf, nor infinite, as a score may be 0)
      const float f = fminf(
          fmaxf(a.scale_log2 * 0x1p24f * __uint_as_float(static_cast<uint32_t>(e - 13) << 23), 0x1p-149f),
          0x1.fffffep127f);
      to_log2[nt][0] = __shfl_sync(0xffffffffu, f, 8 * c4);
      to_log2[nt][1] = __shfl_sync(0xffffffffu, f, 8 * c4 + 4);
    }

    // All products have keys, or the numbers of a value, as their rows and the unit's rows as their
    // columns: a lane has rows 2 c4 and 2 c4 + 1 of each eight (the second index, or two of
    // four).  o: sums of the step products, of places i and i + 1 of group g and column r8 of the
    // value's row; ol: this lane's keys' sums of weight times low; m, l: maximum and sum.
    float o[NT][2 * NG][4];
    float2 ol[NT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int x = 0; x < 2 * NG; ++x)
        o[nt][x][0] = o[nt][x][1] = o[nt][x][2] = o[nt][x][3] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int g = 0; g < 4; ++g) ol[nt][g] = make_float2(0.f, 0.f);
    }
    // Steps are multiplied by 2^(137 - top), which keeps them below 2^11, and weights, up to 2^4,
    // times them below 2^15; top is the exponent of the largest so far (2^-100 at least).
    uint32_t most_step = 27u << 7 | 0x7fu;  // steps up to which need no look, as bf16 bits
    float step_up[NT][2];                   // 2^137 over the power of two of a row's largest step
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) step_up[nt][0] = step_up[nt][1] = __uint_as_float((264u - 27u) << 23);
    bool odd = false;  // a drafted token's step or low was not finite

#pragma unroll 1
    for (int t = t0; t < t0 + n; ++t) {
      issue();
      if (!dead && !__all_sync(0xffffffffu, b200attn::ptx::mbar_try_wait(bars + 8 * use, parity)))
        dead = !wait_long(bars + 8 * use, parity, a.err);
      if (dead) break;
      uint8_t* block = blocks + use * S::kBlockBytes;
      if (++use == NS) {
        use = 0;
        parity ^= 1u;
      }
      const int k0 = t * S::kTile + warp * S::kKeys;
      if (k0 < keys) {
        // ------------------------------------------------------- scores
        // keys r8 (elements 0, 1) and r8 + 8 (2, 3) of each 16
        float s[S::kParts][NT][4];
#pragma unroll
        for (int h = 0; h < S::kParts; ++h) {
          const uint8_t* row0 = block + h * (2 * S::kPartBytes) + r8 * S::kRowBytes;
          const uint8_t* row1 = row0 + 8 * S::kRowBytes;
          uint32_t w0[NG], w1[NG];
          if constexpr (NG == 4) {
            const uint4 u = lds<uint4>(row0 + c4 * (S::kCodes / 4));
            const uint4 v = lds<uint4>(row1 + c4 * (S::kCodes / 4));
            w0[0] = u.x, w0[1] = u.y, w0[2] = u.z, w0[3] = u.w;
            w1[0] = v.x, w1[1] = v.y, w1[2] = v.z, w1[3] = v.w;
          } else {
            const uint2 u = lds<uint2>(row0 + c4 * (S::kCodes / 4)), v = lds<uint2>(row1 + c4 * (S::kCodes / 4));
            w0[0] = u.x, w0[1] = u.y;
            w1[0] = v.x, w1[1] = v.y;
          }
          const uint2 s0 = lds<uint2>(row0 + S::kCodes), s1 = lds<uint2>(row1 + S::kCodes);
          const uint32_t low0 = twice16(row0 + S::kCodes + 8 + 2 * c4);
          const uint32_t low1 = twice16(row1 + S::kCodes + 8 + 2 * c4);
          const uint32_t lows[4] = {low0, low1, low0, low1};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma<B200_ATTN_DTYPE_BF16>(s[h][nt], lows, qs[nt][0], qs[nt][1], 0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float p[NT][4];
#pragma unroll
            for (int y = 0; y < NG / 2; ++y) {
              const int step = NG / 2 * g + y, word = step / 2, shift = 8 * (step & 1);
              const uint32_t u = w0[word] >> shift, v = w1[word] >> shift;
              const uint32_t kf[4] = {u & kLow, v & kLow, u & kHigh, v & kHigh};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const bool on = y > 0;
                mma<B200_ATTN_DTYPE_FP16>(p[nt], kf, qf[nt][step][0], qf[nt][step][1],
                                          on ? p[nt][0] : 0.f, on ? p[nt][1] : 0.f,
                                          on ? p[nt][2] : 0.f, on ? p[nt][3] : 0.f);
              }
            }
            const uint32_t a0 = g < 2 ? s0.x : s0.y, a1 = g < 2 ? s1.x : s1.y;
            const float f0 = g & 1 ? high_half(a0) : low_half(a0);
            const float f1 = g & 1 ? high_half(a1) : low_half(a1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              s[h][nt][0] = fmaf(f0, p[nt][0], s[h][nt][0]);
              s[h][nt][1] = fmaf(f0, p[nt][1], s[h][nt][1]);
              s[h][nt][2] = fmaf(f1, p[nt][2], s[h][nt][2]);
              s[h][nt][3] = fmaf(f1, p[nt][3], s[h][nt][3]);
            }
          }
        }
        if (k0 + S::kKeys > len) {  // drafted tokens, or past the last key
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int row = pl.rt * RM + 8 * nt + 2 * c4 + e;
              const int tok = min(row / a.group, a.tokens - 1);
#pragma unroll
              for (int h = 0; h < S::kParts; ++h)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                  const int j = k0 + 16 * h + 8 * y + r8 - len;
                  if (j >= 0 && (j >= pl.s.drafts || !sees(a, pl.b, tok, j)))
                    s[h][nt][2 * y + e] = -INFINITY;
                }
            }
          // A hidden value must not reach a row as 0 x NaN: steps and lows that are not finite become 0
          // here, and are added below to the rows that see them.  A lane a key.  Behind the last
          // key lies what an earlier block left, which counts as 0 too.
          if (k0 + lane >= len) {
            uint8_t* at = block + (lane / 16) * (2 * S::kPartBytes) + S::kPartBytes +
                                (lane & 15) * S::kRowBytes + S::kCodes;
            uint4 v = lds<uint4>(at);
            uint32_t* w = reinterpret_cast<uint32_t*>(&v);
            uint32_t any = 0u;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t f =
                  k0 + lane < keys ? non_finite<B200_ATTN_DTYPE_BF16>(w[y]) : 0xffffffffu;
              any |= f;
              w[y] &= ~f;
            }
            if (any) {
              odd |= k0 + lane < keys;
              *reinterpret_cast<uint4*>(at) = v;
              b200attn::ptx::fence_proxy_async_smem();  // the next copy lands here
            }
          }
          __syncwarp();
        }
        // ------------------------------------------------------ softmax
        // The maximum and the largest step that weights and steps are taken relative to, a row's own, follow
        // the true ones only where a weight would pass 2^4, or a step is above the least of the rows'
        // largest: of 18 blocks of random keys about two, where every new maximum would rescale the sums in
        // ten.
        uint32_t big;  // steps of two keys' values
        bool grew = false;
        {
          uint8_t* at = block + S::kPartBytes + (lane & 15) * S::kRowBytes + S::kCodes;
          const uint2 u = lds<uint2>(at), v = lds<uint2>(at + 2 * S::kPartBytes);
          big = max_bf16x2(max_bf16x2(u.x, u.y), max_bf16x2(v.x, v.y));
          grew = (big >> 16) > most_step || (big & 0xffffu) > most_step;
        }
        float top[NT][2];  // of the lane's keys
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
#pragma unroll
            for (int h = 1; h < S::kParts; ++h) x = fmaxf(x, fmaxf(s[h][nt][e], s[h][nt][2 + e]));
            top[nt][e] = x * to_log2[nt][e];
            grew |= top[nt][e] > m[nt][e] + 4.f;
          }
        if (__any_sync(0xffffffffu, grew)) {
          // Largest steps among the lane's keys (16 h + 8 y + r8) that each of its rows sees: a value
          // that a row does not see is not to cost it bits.  A NaN counts as nothing.
          uint32_t step[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) step[nt][e] = 264u - (__float_as_uint(step_up[nt][e]) >> 23);
#pragma unroll
          for (int h = 0; h < S::kParts; ++h)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const uint2 u = lds<uint2>(block + h * (2 * S::kPartBytes) + S::kPartBytes +
                                         (8 * y + r8) * S::kRowBytes + S::kCodes);
              uint32_t most = 0u;
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const uint32_t one = (x < 2 ? u.x : u.y) >> 16 * (x & 1) & 0xffffu;
                most = max(most, (one & 0x7fffu) > 0x7f80u ? 0u : one >> 7);
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (s[h][nt][2 * y + e] > -INFINITY) step[nt][e] = max(step[nt][e], most);
            }
          uint32_t least = 255u;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float f[2], d[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
              for (int z = 4; z < 32; z <<= 1)
                step[nt][e] = max(step[nt][e], __shfl_xor_sync(0xffffffffu, step[nt][e], z));
              // 2^(the step before - this one): by 2^-126 nothing is left of a sum either
              const uint32_t less_by = step[nt][e] - (264u - (__float_as_uint(step_up[nt][e]) >> 23));
              d[e] = __uint_as_float((127u - min(less_by, 126u)) << 23);
              step_up[nt][e] = __uint_as_float((264u - step[nt][e]) << 23);
              float x = top[nt][e];
#pragma unroll
              for (int z = 4; z < 32; z <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, z));
              const float now = fmaxf(m[nt][e], x);
              f[e] = now == -INFINITY ? 1.f : b200attn::ptx::ex2_approx(m[nt][e] - now);
              m[nt][e] = now;
              l[nt][e] *= f[e];
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              ol[nt][g].x *= f[0];
              ol[nt][g].y *= f[1];
            }
            f[0] *= d[0];
            f[1] *= d[1];
#pragma unroll
            for (int x = 0; x < 2 * NG; ++x)
#pragma unroll
              for (int y = 0; y < 4; ++y) o[nt][x][y] *= f[y & 1];
#pragma unroll
            for (int e = 0; e < 2; ++e)  // a row that has seen no key takes its first later
              if (m[nt][e] > -INFINITY) least = min(least, step[nt][e]);
          }
          most_step = __reduce_min_sync(0xffffffffu, least) << 7 | 0x7fu;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float base = m[nt][e] == -INFINITY ? 0.f : m[nt][e];
#pragma unroll
            for (int h = 0; h < S::kParts; ++h)
#pragma unroll
              for (int y = 0; y < 4; y += 2) {
                s[h][nt][y + e] =
                    b200attn::ptx::ex2_approx(fmaf(s[h][nt][y + e], to_log2[nt][e], -base));
                l[nt][e] += s[h][nt][y + e];
              }
          }
        // ------------------------------------------------------- values
#pragma unroll
        for (int h = 0; h < S::kParts; ++h) {
          const uint8_t* vb = block + h * (2 * S::kPartBytes) + S::kPartBytes;
          // codes of keys 2 c4, 2 c4 + 1, and 8 further; steps and lows of keys r8 and r8 + 8
          uint32_t w[4][NG / 2];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint8_t* at = vb + (8 * (i >> 1) + 2 * c4 + (i & 1)) * S::kRowBytes + r8 * (S::kCodes / 8);
            if constexpr (NG == 4) {
              const uint2 v = lds<uint2>(at);
              w[i][0] = v.x, w[i][1] = v.y;
            } else {
              w[i][0] = lds<uint32_t>(at);
            }
          }
          const uint4 m0 = lds<uint4>(vb + r8 * S::kRowBytes + S::kCodes);
          const uint4 m1 = lds<uint4>(vb + (r8 + 8) * S::kRowBytes + S::kCodes);
          float pu[NT][4];  // weights times the steps' factor
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int y = 0; y < 4; ++y) pu[nt][y] = s[h][nt][y] * step_up[nt][y & 1];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint32_t sw0 = g < 2 ? m0.x : m0.y, sw1 = g < 2 ? m1.x : m1.y;
            const uint32_t lw0 = g < 2 ? m0.z : m0.w, lw1 = g < 2 ? m1.z : m1.w;
            const float st0 = g & 1 ? high_half(sw0) : low_half(sw0);
            const float st1 = g & 1 ? high_half(sw1) : low_half(sw1);
            float lo0 = g & 1 ? high_half(lw0) : low_half(lw0);
            float lo1 = g & 1 ? high_half(lw1) : low_half(lw1);
            if constexpr (kCentred) lo0 = fmaf(8.f, st0, lo0), lo1 = fmaf(8.f, st1, lo1);
            uint32_t pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              pf[nt][0] = turned(pack_pair<B200_ATTN_DTYPE_FP16>(pu[nt][0] * st0, pu[nt][1] * st0));
              pf[nt][1] = turned(pack_pair<B200_ATTN_DTYPE_FP16>(pu[nt][2] * st1, pu[nt][3] * st1));
              ol[nt][g].x = fmaf(s[h][nt][0], lo0, fmaf(s[h][nt][2], lo1, ol[nt][g].x));
              ol[nt][g].y = fmaf(s[h][nt][1], lo0, fmaf(s[h][nt][3], lo1, ol[nt][g].y));
            }
            // the half words of the group, of two keys each
            const int word = NG == 4 ? g / 2 : 0, half = NG == 4 ? g & 1 : g / 2;
            uint32_t v0 = __byte_perm(w[0][word], w[1][word], half ? 0x7632 : 0x5410);
            uint32_t v1 = __byte_perm(w[2][word], w[3][word], half ? 0x7632 : 0x5410);
            if (NG == 2 && (g & 1)) {
              v0 >>= 8;
              v1 >>= 8;
            }
#pragma unroll
            for (int y = 0; y < NG / 2; ++y) {
              uint32_t vf[4] = {(v0 >> 8 * y) & kLow, (v0 >> 8 * y) & kHigh,
                                (v1 >> 8 * y) & kLow, (v1 >> 8 * y) & kHigh};
              if constexpr (kCentred) {
                vf[0] = less(vf[0], 0x00080008u), vf[1] = less(vf[1], 0x00800080u);
                vf[2] = less(vf[2], 0x00080008u), vf[3] = less(vf[3], 0x00800080u);
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float(&d)[4] = o[nt][NG / 2 * g + y];
                mma<B200_ATTN_DTYPE_FP16>(d, vf, pf[nt][0], pf[nt][1], d[0], d[1], d[2], d[3]);
              }
            }
          }
        }
      }
      __syncwarp();  // the stage is free once every lane has read it
    }

    // ------------------------------------------- join the warps' results
    const Place& done = pl;
    const bool first = t0 == 0, last = t0 + n == pl.tiles;
    flip ^= 1;
    if (tid == 0) {
      Place p = pl;
      p.t += n;
      if (p.t == p.tiles) p = next_unit<typename S::G>(a, p);
      units[flip] = p;
    }
    // the steps' factor and the codes' 2^-24 leave the sums (in two factors)
    float unit0[NT][2], unit1[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t step = 264u - (__float_as_uint(step_up[nt][e]) >> 23);
        unit0[nt][e] = __uint_as_float((127u + step / 2) << 23);
        unit1[nt][e] = __uint_as_float((127u + (step + 1) / 2 - 137u + 24u) << 23);
      }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
#pragma unroll
        for (int e = 0; e < 2; ++e) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          ol[nt][g].x += __shfl_xor_sync(0xffffffffu, ol[nt][g].x, x);
          ol[nt][g].y += __shfl_xor_sync(0xffffffffu, ol[nt][g].y, x);
        }
      }
      if (r8 == 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          stat[(2 * warp) * RM + 8 * nt + 2 * c4 + e] = m[nt][e];
          stat[(2 * warp + 1) * RM + 8 * nt + 2 * c4 + e] = l[nt][e];
        }
      }
    }
    const bool any_odd = __syncthreads_or(odd);
    float scale[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < S::kWarps; ++w) top = fmaxf(top, stat[2 * w * RM + 8 * nt + 2 * c4 + e]);
        scale[nt][e] = top == -INFINITY ? 0.f : b200attn::ptx::ex2_approx(m[nt][e] - top);
      }
    float* part = a.partial + static_cast<int64_t>(2 * blockIdx.x + (first ? 1 : 0)) * (RM * (DP + 2));
    const bool finish = first && last;
    constexpr int kC = S::kJoinCols, kPitch = S::kJoinPitch, kEach = S::kEach;
    const int r = tid / (kC / kEach), c = (tid % (kC / kEach)) * kEach;
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < S::kWarps; ++w) top = fmaxf(top, stat[2 * w * RM + r]);
#pragma unroll
    for (int w = 0; w < S::kWarps; ++w) {
      const float mw = stat[2 * w * RM + r];
      if (mw != -INFINITY) total += stat[(2 * w + 1) * RM + r] * b200attn::ptx::ex2_approx(mw - top);
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int row = done.rt * RM + r, tok = row / a.group;
    uint8_t* out = a.o + done.b * a.o_seq + (done.h * a.group + row - tok * a.group) * a.o_head +
                   tok * a.o_tok;
#pragma unroll
    for (int c0 = 0; c0 < DP; c0 += kC) {
      if (c0) __syncthreads();
      // numbers DP / 4 g + NG r8 + i of rows 2 c4 and 2 c4 + 1
#pragma unroll
      for (int g = c0 / (DP / 4); g < (c0 + kC) / (DP / 4); ++g)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float* d = join + (warp * S::kJoinRows + 8 * nt + 2 * c4 + e) * kPitch + DP / 4 * g - c0 + NG * r8;
            const float low = (e ? ol[nt][g].y : ol[nt][g].x) * scale[nt][e];
            float v[NG];
#pragma unroll
            for (int i = 0; i < NG; ++i)
              v[i] = fmaf(o[nt][NG / 2 * g + i / 2][2 * (i & 1) + e] * (scale[nt][e] * unit0[nt][e]),
                          i & 1 ? unit1[nt][e] * 0.0625f : unit1[nt][e], low);
            if constexpr (NG == 4)
              *reinterpret_cast<float4*>(d) = make_float4(v[0], v[1], v[2], v[3]);
            else
              *reinterpret_cast<float2*>(d) = make_float2(v[0], v[1]);
          }
      __syncthreads();
      float acc[kEach];
#pragma unroll
      for (int e = 0; e < kEach; ++e) acc[e] = 0.f;
#pragma unroll
      for (int w = 0; w < S::kWarps; ++w)
#pragma unroll
        for (int e = 0; e < kEach; e += 4) {
          const float4 v = *reinterpret_cast<const float4*>(join + (w * S::kJoinRows + r) * kPitch + c + e);
          acc[e] += v.x;
          acc[e + 1] += v.y;
          acc[e + 2] += v.z;
          acc[e + 3] += v.w;
        }
      if (!finish) {
#pragma unroll
        for (int e = 0; e < kEach; e += 2)
          *reinterpret_cast<float2*>(part + r * DP + c0 + c + e) = make_float2(acc[e], acc[e + 1]);
      } else if (r < rows && c0 + c < a.head_dim) {
#pragma unroll
        for (int e = 0; e < kEach; e += 4)
          *reinterpret_cast<uint2*>(out + 2 * (c0 + c + e)) =
              make_uint2(pack_pair<DT>(acc[e] * inv, acc[e + 1] * inv),
                         pack_pair<DT>(acc[e + 2] * inv, acc[e + 3] * inv));
      }
    }
    if (any_odd && r < rows)
      for (int c0 = c; c0 < DP; c0 += kC)
        add_odd4<DP, DT>(a, done.b, done.h, done.s, tok, t0 * S::kTile - done.s.len,
                         (t0 + n) * S::kTile - done.s.len, c0, min(a.head_dim, c0 + kEach),
                         finish ? reinterpret_cast<uint16_t*>(out) : nullptr, part + r * DP, 1);
    if (!finish && c == 0) {
      part[RM * DP + r] = top;
      part[RM * DP + RM + r] = total;
    }
    if (!finish) {
      const int from = run.ends_in(done) ? run.end_first : (first ? blockIdx.x : run.first_run);
      const int to = run.ends_in(done) ? run.end_last : blockIdx.x;
      if (a.counters)
        join_if_last<RM, DP, DT, S::kWarps>(a, done.b, done.h, done.rt, rows, from, to,
                                            reinterpret_cast<JoinSmem<DP, S::kWarps>*>(join));
      else if (tid == 0 && last)
        a.desc[unit_of(a, done)] = make_int2(from, to);
    } else if (tid == 0 && !a.counters) {
      a.desc[unit_of(a, done)] = make_int2(0, 0);
    }
    __syncthreads();
  }
  zero_unused_rows(a, 2, S::kThreads);
  if (dead)  // its copies may be on their way still
    for (int x = 0; x < NS; ++x) wait_long(bars + 8 * x, (x >= use) == (parity != 0u), nullptr);
}

// -------------------------------------------------------------------- host
using namespace b200paged;

using AnyShape = Shape4<false, 128>;  // row and key tiles do not depend on the instance
static_assert(AnyShape::kTile == Shape4<true, 64>::kTile && AnyShape::RM == Shape4<true, 64>::RM,
              "one division of the work");

// Up to so many rows a key head the kernel of matrix instructions of a warp, whose time grows
// with each 16 rows; the tcgen05 kernel takes as long for 16 as for 128.  Measured, this kernel
// and that one (8 key heads x 4, D 128, pages of 64, us): 131001 keys, 16 rows 82 and 136, 32 rows 130 and
// 139, 64 rows 233 and 140; 16 sequences of 1001 to 8100 keys 63 and 95, 100 and 97, 175 and 97; 64
// sequences of 500 to 2000 keys 79 and 118, 139 and 120, 261 and 124.  (32 rows over one long context
// would be 7 % faster here; the rule goes by the rows alone.)  fp16 queries of more rows, and masks of
// more than 64 tokens, take this kernel all the same: the other has neither.
constexpr int64_t kFewRows4 = 16;

int64_t rows_of(const b200_tree_attn_params* p) { return p->tokens * (p->heads / p->cache.kv_heads); }

// The kernel a call takes: its row tile (`rm` places, `rows` of them used), its key tile and the
// CTAs of an SM.
struct Choice4 {
  bool many;  // the tcgen05 kernel
  int rm, rows, tn, ctas;
};

Choice4 choose(const b200_tree_attn_params* p, int32_t dtype) {
  const int64_t rows = rows_of(p), group = p->heads / p->cache.kv_heads;
  // The tcgen05 kernel has bf16 values and weights, too few bits for fp16 results, and masks of up
  // to 64 tokens.
  if (rows > kFewRows4 && dtype == B200_ATTN_DTYPE_BF16 && group <= 128 && (p->tokens <= 64 || !p->mask)) {
    const int tile = static_cast<int>(128 / group * group);  // whole tokens to 128 places
    if (rows <= tile) return Choice4{true, 128, tile, 128, 1};
    return Choice4{true, 256, 2 * tile, 128, 1};
  }
  const bool narrow = p->cache.head_dim == 24;  // rows of 48 bytes
  return Choice4{false, AnyShape::RM, AnyShape::RM, AnyShape::kTile,
                 rows > 8 ? AnyShape::kCtas : narrow ? Shape4<true, 64>::kCtas : Shape4<true, 128>::kCtas};
}

int64_t row_tiles(const b200_tree_attn_params* p, const Choice4& c) {
  return (rows_of(p) + c.rows - 1) / c.rows;
}

int64_t units_of(const b200_tree_attn_params* p, const Choice4& c) {
  return p->cache.batch * p->cache.kv_heads * row_tiles(p, c);
}

int64_t runs_of(const b200_tree_attn_params* p, const Choice4& c, int64_t sms) {
  const int64_t keys = p->cache.slots * p->cache.page_size;
  const double tiles =
      static_cast<double>(units_of(p, c)) * static_cast<double>((keys + c.tn - 1) / c.tn);
  const int64_t most = (sms < kMaxSms ? sms : kMaxSms) * c.ctas;
  return tiles < static_cast<double>(most) ? static_cast<int64_t>(tiles) : most;
}

template <int DP, int DT>
int32_t run_width(const Choice4& c, const Args& a, int runs, int64_t units, bool spread, int device,
                  cudaStream_t s) {
  using Few = Shape4<true, DP>;
  using One = Shape4<false, DP>;
  if constexpr (DT == B200_ATTN_DTYPE_BF16) {
    if (c.many) {
      const int32_t rc = launch_coded(c.rm, DP, a, runs, device, s);
      if (rc != B200_ATTN_OK) return rc;
      return c.rm == 128 ? run_join_columns<128, DP, DT>(a, units, s)
                         : run_join_columns<256, DP, DT>(a, units, s);
    }
  }
  const int32_t rc =
      a.tokens * a.group <= 8
          ? run_one<rows4_kernel<Few, DT>>(Few::kThreads, Few::kSmemBytes, a, runs, device, s)
          : run_one<rows4_kernel<One, DT>>(One::kThreads, One::kSmemBytes, a, runs, device, s);
  return rc != B200_ATTN_OK || a.counters
             ? rc
             : run_join_rows<One::RM, DP, DT, One::kWarps>(a, units, spread, s);
}

}  // namespace
}  // namespace b200tree

using namespace b200tree;

extern "C" int32_t b200_cache4_attn_check(const b200_tree_attn_params* p, int64_t head_dim,
                                          int32_t dtype) {
  if (!p) return B200_ATTN_ERR_INVALID_ARGUMENT;
  const b200_cache& c = p->cache;
  const int32_t rc = b200_cache_check(&c);
  if (rc != B200_ATTN_OK) return rc;
  const int32_t bytes = b200_cache4_row_bytes(head_dim);
  if (bytes == 0 || (dtype != B200_ATTN_DTYPE_BF16 && dtype != B200_ATTN_DTYPE_FP16))
    return B200_ATTN_ERR_UNSUPPORTED;
  if (c.dtype != B200_ATTN_DTYPE_BF16 || 2 * c.head_dim != bytes || !c.seq_lens || !p->q || !p->o ||
      c.layers != 1 || p->tokens < 1 || p->heads < 1 || p->heads % c.kv_heads || p->reserved != 0)
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (!(p->scale > 0.f) || !std::isfinite(p->scale)) return B200_ATTN_ERR_INVALID_ARGUMENT;
  // rows, units and row pieces of a call are numbered in 32 bits
  if (p->tokens > (1 << 24) || p->heads > (1 << 16) || p->tokens * p->heads > (1ll << 25) ||
      c.batch * p->heads * p->tokens > 0x7fffffffll)
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  const int64_t extent[3] = {c.batch, p->heads, p->tokens};
  if (!b200paged::vectors_aligned(p->q, p->q_stride, extent, 3, 2) ||
      !b200paged::vectors_aligned(p->o, p->o_stride, extent, 3, 2) ||
      ((reinterpret_cast<uintptr_t>(p->draft_lens) | reinterpret_cast<uintptr_t>(p->counters)) & 3u))
    return B200_ATTN_ERR_ALIGNMENT;
  // so are all key tiles of a call
  const Choice4 ch = choose(p, dtype);
  if (static_cast<double>(units_of(p, ch)) *
          static_cast<double>(c.slots * c.page_size / ch.tn + 5) > 2e9)
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (p->mask && (p->mask_stride[0] < 0 || p->mask_stride[1] < 0 || p->mask_stride[2] < 0))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (output_collides(p, head_dim, 2)) return B200_ATTN_ERR_INVALID_ARGUMENT;
  return B200_ATTN_OK;
}

extern "C" int64_t b200_cache4_attn_workspace_bytes(const b200_tree_attn_params* p,
                                                    int64_t head_dim, int32_t dtype) {
  if (b200_cache4_attn_check(p, head_dim, dtype) != B200_ATTN_OK) return 0;
  const int dp = head_dim <= 64 ? 64 : 128;
  const Choice4 ch = choose(p, dtype);
  return round16(8 * units_of(p, ch)) + 2 * runs_of(p, ch, kMaxSms) * 4 * ch.rm * (dp + 2);
}

namespace {

// What both entry points do: checks, and the arguments of the kernels.
struct Prepared {
  b200paged::DeviceScope scope;
  Args a{};
  Choice4 ch{};
  int64_t units = 0;
  int runs = 0;
  bool spread = false;
};

int32_t prepare(const b200_tree_attn_params* p, int64_t head_dim, int32_t dtype, Prepared* r) {
  int32_t rc = b200_cache4_attn_check(p, head_dim, dtype);
  if (rc != B200_ATTN_OK) return rc;
  if (!p->workspace || p->workspace_bytes < b200_cache4_attn_workspace_bytes(p, head_dim, dtype))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(p->workspace) & 15u) return B200_ATTN_ERR_ALIGNMENT;
  if ((rc = r->scope.enter(p->q, "q is not a device pointer")) != B200_ATTN_OK) return rc;
  Args& a = r->a;
  if ((rc = b200attn::resolve_error_word(p->cache.error_word, &a.err)) != B200_ATTN_OK) return rc;
  fill_args(p, 2, 2, head_dim, &a);
  const Choice4 ch = r->ch = choose(p, dtype);
  a.unit_rows = ch.rows;
  a.row_tiles = static_cast<int32_t>(row_tiles(p, ch));
  a.scale_log2 = p->scale * 1.4426950408889634f;
  r->units = units_of(p, ch);
  a.desc = static_cast<int2*>(p->workspace);
  a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(p->workspace) + round16(8 * r->units));
  r->runs = static_cast<int>(runs_of(p, ch, b200paged::sm_count(r->scope.device)));
  a.runs = r->runs;
  // as for caches of 16 bits: long contexts of several rows are joined by a kernel of their own
  r->spread = rows_of(p) > 4 && p->cache.slots * p->cache.page_size >= 12 * ch.tn &&
              r->runs >= 8 * r->units;
  if (!ch.many && !r->spread && r->units <= B200_TREE_ATTN_COUNTERS) a.counters = p->counters;
  return B200_ATTN_OK;
}

}  // namespace

extern "C" int32_t b200_cache4_attn_fwd(const b200_tree_attn_params* p, int64_t head_dim,
                                        int32_t dtype, void* stream) {
  Prepared r;
  const int32_t rc = prepare(p, head_dim, dtype, &r);
  if (rc != B200_ATTN_OK) return rc;
  const int device = r.scope.device;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = head_dim > 64;
  if (dtype == B200_ATTN_DTYPE_BF16)
    return wide ? run_width<128, B200_ATTN_DTYPE_BF16>(r.ch, r.a, r.runs, r.units, r.spread, device, s)
                : run_width<64, B200_ATTN_DTYPE_BF16>(r.ch, r.a, r.runs, r.units, r.spread, device, s);
  return wide ? run_width<128, B200_ATTN_DTYPE_FP16>(r.ch, r.a, r.runs, r.units, r.spread, device, s)
              : run_width<64, B200_ATTN_DTYPE_FP16>(r.ch, r.a, r.runs, r.units, r.spread, device, s);
}

extern "C" int32_t b200_cache4_selftest_stall(const b200_tree_attn_params* p, int64_t head_dim,
                                              int32_t dtype, int32_t skipped_tile, void* stream) {
  if (!p || dtype != B200_ATTN_DTYPE_BF16 || head_dim <= 64 || head_dim > 128 ||
      !p->cache.error_word || skipped_tile < 0)
    return B200_ATTN_ERR_UNSUPPORTED;
  Prepared r;
  const int32_t rc = prepare(p, head_dim, dtype, &r);
  if (rc != B200_ATTN_OK) return rc;
  if (!r.ch.many) return B200_ATTN_ERR_UNSUPPORTED;
  return launch_coded_stall(r.ch.rm, r.a, r.runs, r.scope.device, static_cast<cudaStream_t>(stream),
                            skipped_tile);
}
