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
// w step_g is rounded to fp16 (relative to a power of two that follows the largest step), w low_g
// and sum w are fp32.
//
// A half byte becomes an fp16 operand by one AND: bits 0..3 of a half word are the subnormal
// number code 2^-24, bits 4..7 the number 16 code 2^-24 (the factors go into the queries and
// the result).  The rows of keys and values are laid out so that a lane's operands of a product
// lie in its words: 8 numbers take 4 ANDs and a shift, and for values, whose pairs come
// from two rows, two byte permutes.
//
// As in the kernel of 16-bit caches (tree_attn_rows.cuh) the warps of a CTA share a key tile,
// 16 keys each, and fetch them into rings of their own.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "b200_cache4.h"
#include "error_word.cuh"
#include "paged_host.h"
#include "tree_attn.cuh"
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
  static constexpr int kWarps = 4, kThreads = 32 * kWarps, kCtas = 3;
  static constexpr int kTile = kWarps * kRowKeys;
  static constexpr int kHalves = FEW ? 1 : 2;
  static constexpr int kCodes = DP / 2, kRowBytes = kCodes + 16;
  static constexpr int kPieces = kRowBytes / 16;
  static constexpr int kBlockBytes = kRowKeys * kRowBytes;
  static constexpr int kStages = DP == 128 ? 5 : 8;
  static constexpr int kRingBytes = kWarps * kStages * 2 * kBlockBytes;
  static constexpr int kJoinRows = FEW ? 8 : 16;
  static constexpr int kJoinCols = DP < 1024 / kJoinRows ? DP : 1024 / kJoinRows;
  static constexpr int kEach = kJoinRows * kJoinCols / kThreads;  // columns of a thread in a join
  static constexpr int kJoinPitch = kJoinCols + 4;
  static constexpr int kOffJoin = kRingBytes;
  static constexpr int kJoinBytes = 4 * kWarps * kJoinRows * kJoinPitch;
  static constexpr int kOffStat = kOffJoin + kJoinBytes;
  static constexpr int kOffMisc = kOffStat + 4 * 2 * kWarps * RM;
  static constexpr int kSmemBytes = kOffMisc + 256;
  static_assert(kCtas * (kSmemBytes + 1024) <= 233472, "exceeds the shared memory of an SM");
  using G = Grid<RM, kTile, 2>;
  static_assert(sizeof(JoinSmem<DP, kWarps>) <= kJoinBytes, "joins in place");
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1, float c0, float c1, float c2, float c3) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2),
        "f"(c3));
}
__device__ __forceinline__ uint32_t lds32(uint32_t ad) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(ad) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t ad) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(ad) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t ad) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(ad)
               : "memory");
  return v;
}
__device__ __forceinline__ float low_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// The larger bf16 of each half; a NaN counts as nothing.
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;

// Adds NaN to the numbers of a finished row (`out`) or its partial sums (`part`) whose group
// is NaN in a drafted token that the row's token sees: such steps and lows were left
// out of the products, where a weight of zero would not hide them.
template <int DP, int DT>
__device__ __noinline__ void add_odd4(const Args& a, int b, int h, Seq s, int tok, int d0, int d1,
                                      int col0, int col1, uint16_t* out, float* part) {
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
      else part[c] += x - x;
    }
  }
}

template <class S, int DT>
__global__ void __launch_bounds__(S::kThreads, S::kCtas)
    rows4_kernel(const __grid_constant__ Args a) {
  constexpr int RM = S::RM, DP = S::DP, NS = S::kStages, NG = DP / 32;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sbase = b200attn::ptx::smem_u32(smem);
  float* join = reinterpret_cast<float*>(smem + S::kOffJoin);
  float* stat = reinterpret_cast<float*>(smem + S::kOffStat);  // [warp][{max, sum}][RM]
  uint32_t* sums = reinterpret_cast<uint32_t*>(smem + S::kOffMisc);
  Run* found = reinterpret_cast<Run*>(smem + S::kOffMisc + 80);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r8 = lane >> 2, c4 = lane & 3;  // row and column pair of this lane in a product
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  find_run<typename S::G>(a, blockIdx.x, gridDim.x, sums, found);
  const Run& run = *found;

  const uint32_t ring = sbase + warp * (NS * 2 * S::kBlockBytes);
  const uint32_t size = static_cast<uint32_t>(a.page_size);
  const bool whole = a.page_size % kRowKeys == 0;  // a block lies in one page

  // ------------------------------------------------------------- loads
  // The place of the next tile to load; its page numbers are read one tile ahead.
  Place ld = run.p;
  bool more = !run.done(ld);
  int page = -1, page_row = 0, ld_keys = 0;
  const uint32_t inv_size = 0xffffffffu / size + 1u;  // 0 for size 1
  auto look_up = [&]() {
    const int key = ld.t * S::kTile + warp * kRowKeys + (whole ? 0 : (lane & 15));
    ld_keys = ld.s.len + ld.s.drafts - (ld.t * S::kTile + warp * kRowKeys);
    page = -1;
    page_row = 0;
    if (key < ld.s.len + ld.s.drafts) {
      // key / size or one more: key is below 2^30
      uint32_t slot = size == 1u ? key : __umulhi(key, inv_size);
      page_row = key - static_cast<int>(slot * size);
      if (page_row < 0) {
        --slot;
        page_row += static_cast<int>(size);
      }
      page = __ldg(a.table + ld.b * a.table_stride + slot);
    }
  };
  if (more) look_up();
  int stage = 0;  // stage the next loads go to
  // Rows side by side: a block's keys and values are 2 kPieces / 32 loads of 16 bytes a lane, of
  // which the middle one takes the end of the keys and the beginning of the values.
  const bool tight = whole && a.k_row == S::kRowBytes && a.v_row == S::kRowBytes;
  constexpr int kKeyLoads = S::kBlockBytes / 512, kRest = S::kBlockBytes % 512;
  static_assert(kRest == 256, "half a load of 16 bytes a lane");
  auto issue = [&]() {
    if (more) {
      if (page >= a.pages || (page < 0 && (whole ? 0 : (lane & 15)) < ld_keys)) {
        report_error(a.err, B200_ATTN_DEVERR_BOUNDS);
        page = -1;
      }
      const uint32_t dst = ring + stage * (2 * S::kBlockBytes) + 16 * lane;
      if (tight && page >= 0 && ld_keys >= kRowKeys) {
        const uint8_t* ks = a.k + ld.h * a.k_head + page * a.k_page + page_row * S::kRowBytes + 16 * lane;
        const uint8_t* vs = a.v + ld.h * a.v_head + page * a.v_page + page_row * S::kRowBytes + 16 * lane;
#pragma unroll
        for (int u = 0; u < kKeyLoads; ++u) cp_async16(dst + 512 * u, ks + 512 * u, 16u);
        cp_async16(dst + 512 * kKeyLoads, lane < 16 ? ks + 512 * kKeyLoads : vs - kRest, 16u);
#pragma unroll
        for (int u = 0; u < kKeyLoads; ++u)
          cp_async16(dst + 512 * (kKeyLoads + 1) + 512 * u, vs + kRest + 512 * u, 16u);
      } else {
#pragma unroll 1
        for (int x = lane; x < 2 * S::kBlockBytes / 16; x += 32) {
          const bool value = x >= S::kBlockBytes / 16;
          const int y = value ? x - S::kBlockBytes / 16 : x;
          const int r = y / S::kPieces, piece = y - r * S::kPieces;
          const int pg = whole ? page : __shfl_sync(0xffffffffu, page, r);
          const int64_t at = whole ? page_row + r : __shfl_sync(0xffffffffu, page_row, r);
          const uint8_t* src = value ? a.v : a.k;
          const bool ok = pg >= 0 && r < ld_keys;
          if (ok)
            src += value ? ld.h * a.v_head + pg * a.v_page + at * a.v_row + 16 * piece
                         : ld.h * a.k_head + pg * a.k_page + at * a.k_row + 16 * piece;
          cp_async16(dst - 16 * lane + 16 * x, src, ok ? 16u : 0u);
        }
      }
      if (++ld.t == ld.tiles) ld = next_unit<typename S::G>(a, ld);
      more = !run.done(ld);
      if (more) look_up();
    }
    cp_async_commit();
    stage = stage + 1 == NS ? 0 : stage + 1;
  };
#pragma unroll 1
  for (int s = 0; s < NS - 1; ++s) issue();

  Place pl = run.p;
  int use = 0;  // stage of the tile at hand

#pragma unroll 1
  while (!run.done(pl)) {
    const int t0 = pl.t;
    const int n = run.tiles(pl);
    const int keys = pl.s.len + pl.s.drafts;
    const int rows = min(RM, pl.s.drafts * a.group - pl.rt * RM);

    // ----------------------------------------------------------- queries
    // Row r8 (and r8 + 8) as fp16 operands, times the power of two that brings the row's
    // largest number to 2^13..2^14; the pairs that meet the codes' high half bytes, by 1/16 more.
    uint32_t qf[DP / 16][4];
    uint32_t qs[4];   // the sums of the four groups, in three bf16 numbers
    float to_log2[2];  // from the products' unit to that of the exponents
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      float x[DP / 16][4];
      const int r = r8 + 8 * hh;
      const bool live = hh < S::kHalves && r < rows;
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
        if (live && d < a.head_dim) {
          if constexpr (NG == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(src + 2 * d);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(src + 2 * d);
            w[0] = v.x, w[1] = v.y;
          }
        }
        sum[g] = 0.f;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          const float2 f = unpack_pair<DT>(w[i]);
          big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
          sum[g] += f.x + f.y;
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
        qf[i][hh] = pack_pair<B200_ATTN_DTYPE_FP16>(x[i][0] * up, x[i][1] * up);
        qf[i][2 + hh] =
            pack_pair<B200_ATTN_DTYPE_FP16>(x[i][2] * up * 0.0625f, x[i][3] * up * 0.0625f);
      }
      float mine = 0.f;  // the sum of group c4, in the unit of the products
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
        if (g == c4) mine = sum[g] * up * 0x1p-24f;
      }
      const uint32_t hi = pack_pair<B200_ATTN_DTYPE_BF16>(mine, 0.f);
      const float rest = mine - low_half(hi);
      const uint32_t mid = pack_pair<B200_ATTN_DTYPE_BF16>(rest, 0.f);
      const uint32_t lo = pack_pair<B200_ATTN_DTYPE_BF16>(rest - low_half(mid), 0.f);
      qs[hh] = hi | mid << 16;
      qs[2 + hh] = lo;
      to_log2[hh] = a.scale_log2 * 0x1p24f * __uint_as_float(static_cast<uint32_t>(e - 13) << 23);
    }

    // Sums of the step products, transposed: rows of the product are numbers (places i and i + 1
    // of group g, for columns r8 of the value's row), its columns the unit's rows.
    float o[S::kHalves][2 * NG][4];
    float ol[2][4];  // this lane's keys' sums of weight times low
    float m[2], l[2];
#pragma unroll
    for (int hh = 0; hh < S::kHalves; ++hh) {
#pragma unroll
      for (int x = 0; x < 2 * NG; ++x)
        o[hh][x][0] = o[hh][x][1] = o[hh][x][2] = o[hh][x][3] = 0.f;
      m[hh] = -INFINITY;
      l[hh] = 0.f;
#pragma unroll
      for (int g = 0; g < 4; ++g) ol[hh][g] = 0.f;
    }
    // Steps are multiplied by 2^(141 - top), which keeps them, and the weights times them,
    // below 2^15; top is the exponent of the largest so far (2^-100 at least).
    uint32_t top_step = 27u;
    float step_up = __uint_as_float((268u - 27u) << 23);
    bool odd = false;  // a drafted token's step or low was not finite

#pragma unroll 1
    for (int t = t0; t < t0 + n; ++t) {
      issue();
      cp_async_wait<NS - 1>();
      __syncwarp();
      const uint32_t kb = ring + use * (2 * S::kBlockBytes), vb = kb + S::kBlockBytes;
      use = use + 1 == NS ? 0 : use + 1;
      const int k0 = t * S::kTile + warp * kRowKeys;
      if (k0 < keys) {
        // ------------------------------------------------------- scores
        float s[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t row = kb + (8 * x + r8) * S::kRowBytes, at = row + c4 * (S::kCodes / 4);
          uint32_t w[NG];
          if constexpr (NG == 4) {
            const uint4 v = lds128(at);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
          } else {
            const uint2 v = lds64(at);
            w[0] = v.x, w[1] = v.y;
          }
          uint32_t low;
          asm volatile("{\n.reg .u16 h;\nld.shared.u16 h, [%1];\nmov.b32 %0, {h, h};\n}"
                       : "=r"(low)
                       : "r"(row + S::kCodes + 8 + 2 * c4)
                       : "memory");
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          mma16816<B200_ATTN_DTYPE_BF16>(acc, qs, low, low);
          const uint32_t meta = kb + (8 * x + 2 * c4) * S::kRowBytes + S::kCodes;
          const uint2 s0 = lds64(meta), s1 = lds64(meta + S::kRowBytes);  // steps of the lane's two keys
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float p[4];
            if constexpr (NG == 4) {
              mma_f16(p, qf[2 * g], w[g] & kLow, w[g] & kHigh, 0.f, 0.f, 0.f, 0.f);
              const uint32_t v = w[g] >> 8;
              mma_f16(p, qf[2 * g + 1], v & kLow, v & kHigh, p[0], p[1], p[2], p[3]);
            } else {
              const uint32_t v = g & 1 ? w[g / 2] >> 8 : w[g / 2];
              mma_f16(p, qf[g], v & kLow, v & kHigh, 0.f, 0.f, 0.f, 0.f);
            }
            const uint32_t a0 = g < 2 ? s0.x : s0.y, a1 = g < 2 ? s1.x : s1.y;
            const float f0 = g & 1 ? high_half(a0) : low_half(a0);
            const float f1 = g & 1 ? high_half(a1) : low_half(a1);
            acc[0] = fmaf(f0, p[0], acc[0]);
            acc[1] = fmaf(f1, p[1], acc[1]);
            if constexpr (!S::FEW) {
              acc[2] = fmaf(f0, p[2], acc[2]);
              acc[3] = fmaf(f1, p[3], acc[3]);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) s[x][e] = acc[e];
        }
        // steps and lows of the values of the lane's keys 2 c4, 2 c4 + 1, and 8 further
        uint4 meta[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          meta[i] = lds128(vb + (8 * (i >> 1) + 2 * c4 + (i & 1)) * S::kRowBytes + S::kCodes);
        if (k0 + kRowKeys > pl.s.len) {
          // drafted tokens, or past the last key
#pragma unroll
          for (int e = 0; e < 2 * S::kHalves; ++e) {
            const int row = pl.rt * RM + r8 + (e >> 1) * 8;
            const int tok = min(row / a.group, a.tokens - 1);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int j = k0 + 8 * x + 2 * c4 + (e & 1) - pl.s.len;
              if (j >= 0 && (j >= pl.s.drafts || !sees(a, pl.b, tok, j))) s[x][e] = -INFINITY;
            }
          }
          // A hidden value must not reach a row as 0 x NaN: it becomes 0 here and is added
          // below to the rows that see it.
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (k0 + 8 * (i >> 1) + 2 * c4 + (i & 1) < pl.s.len) continue;
            uint32_t* w = reinterpret_cast<uint32_t*>(&meta[i]);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t f = non_finite<B200_ATTN_DTYPE_BF16>(w[y]);
              odd |= f != 0u;
              w[y] &= ~f;
            }
          }
        }
        // ------------------------------------------------------ softmax
        // running maximum and largest step; the sums so far are rescaled only where one grew
        uint32_t big = max_bf16x2(max_bf16x2(max_bf16x2(meta[0].x, meta[0].y), max_bf16x2(meta[1].x, meta[1].y)),
                                  max_bf16x2(max_bf16x2(meta[2].x, meta[2].y), max_bf16x2(meta[3].x, meta[3].y)));
        big = max_bf16x2(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = max_bf16x2(big, __shfl_xor_sync(0xffffffffu, big, 2));
        uint32_t e0 = (big >> 7) & 0xffu, e1 = big >> 23;
        e0 = e0 == 255u ? 0u : e0;  // all of them NaN
        e1 = e1 == 255u ? 0u : e1;
        const uint32_t now_step = max(top_step, max(e0, e1));
        bool grew = now_step > top_step;
        float alpha[2] = {1.f, 1.f};
#pragma unroll
        for (int hh = 0; hh < S::kHalves; ++hh) {
          float top = fmaxf(fmaxf(s[0][2 * hh], s[0][2 * hh + 1]),
                            fmaxf(s[1][2 * hh], s[1][2 * hh + 1]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float now = fmaxf(m[hh], top * to_log2[hh]);
          grew |= now > m[hh];
          alpha[hh] = now == -INFINITY ? 1.f : b200attn::ptx::ex2_approx(m[hh] - now);
          m[hh] = now;
        }
        if (__any_sync(0xffffffffu, grew)) {
          // 2^(top_step - now_step), in two factors: they may lie 254 apart
          const float d0 = __uint_as_float((127u - (now_step - top_step) / 2) << 23);
          const float d1 = __uint_as_float((127u - (now_step - top_step + 1) / 2) << 23);
          top_step = now_step;
          step_up = __uint_as_float((268u - top_step) << 23);
#pragma unroll
          for (int hh = 0; hh < S::kHalves; ++hh) {
            l[hh] *= alpha[hh];
#pragma unroll
            for (int g = 0; g < 4; ++g) ol[hh][g] *= alpha[hh];
            // rows 2 c4 and 2 c4 + 1, whose factors lie in the lanes of those rows
            const float f = alpha[hh] * d0;
            const float f0 = __shfl_sync(0xffffffffu, f, 8 * c4);
            const float f1 = __shfl_sync(0xffffffffu, f, 8 * c4 + 4);
#pragma unroll
            for (int x = 0; x < 2 * NG; ++x) {
              o[hh][x][0] = o[hh][x][0] * f0 * d1;
              o[hh][x][1] = o[hh][x][1] * f1 * d1;
              o[hh][x][2] = o[hh][x][2] * f0 * d1;
              o[hh][x][3] = o[hh][x][3] * f1 * d1;
            }
          }
        }
        float p[2][4], pu[2][4];  // weights, and times the steps' factor
#pragma unroll
        for (int hh = 0; hh < S::kHalves; ++hh) {
          const float base = m[hh] == -INFINITY ? 0.f : m[hh];
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              p[x][2 * hh + e] =
                  b200attn::ptx::ex2_approx(fmaf(s[x][2 * hh + e], to_log2[hh], -base));
              l[hh] += p[x][2 * hh + e];
              pu[x][2 * hh + e] = p[x][2 * hh + e] * step_up;
            }
        }
        // ------------------------------------------------------- values
        uint32_t w[4][NG / 2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t at =
              vb + (8 * (i >> 1) + 2 * c4 + (i & 1)) * S::kRowBytes + r8 * (S::kCodes / 8);
          if constexpr (NG == 4) {
            const uint2 v = lds64(at);
            w[i][0] = v.x, w[i][1] = v.y;
          } else {
            w[i][0] = lds32(at);
          }
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float st[4], lw[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t sw = g < 2 ? meta[i].x : meta[i].y, lo = g < 2 ? meta[i].z : meta[i].w;
            st[i] = g & 1 ? high_half(sw) : low_half(sw);
            lw[i] = g & 1 ? high_half(lo) : low_half(lo);
          }
          uint32_t pf[S::kHalves][2];
#pragma unroll
          for (int hh = 0; hh < S::kHalves; ++hh)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              pf[hh][x] = pack_pair<B200_ATTN_DTYPE_FP16>(pu[x][2 * hh] * st[2 * x],
                                                          pu[x][2 * hh + 1] * st[2 * x + 1]);
              ol[hh][g] = fmaf(p[x][2 * hh], lw[2 * x], ol[hh][g]);
              ol[hh][g] = fmaf(p[x][2 * hh + 1], lw[2 * x + 1], ol[hh][g]);
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
            const uint32_t vf[4] = {(v0 >> 8 * y) & kLow, (v0 >> 8 * y) & kHigh,
                                    (v1 >> 8 * y) & kLow, (v1 >> 8 * y) & kHigh};
#pragma unroll
            for (int hh = 0; hh < S::kHalves; ++hh) {
              mma16816<B200_ATTN_DTYPE_FP16>(o[hh][NG / 2 * g + y], vf, pf[hh][0], pf[hh][1]);
            }
          }
        }
      }
      __syncwarp();  // the stage is free once every lane has read it
    }

    // ------------------------------------------- join the warps' results
    const Place done = pl;
    const bool first = t0 == 0, last = t0 + n == pl.tiles;
    pl.t += n;
    if (pl.t == pl.tiles) pl = next_unit<typename S::G>(a, pl);
    // the steps' factor and the codes' 2^-24 leave the sums (in two factors)
    const float unit0 = __uint_as_float((127u + top_step / 2) << 23);
    const float unit1 = __uint_as_float((127u + (top_step + 1) / 2 - 141u + 24u) << 23);
#pragma unroll
    for (int hh = 0; hh < S::kHalves; ++hh) {
      float v = l[hh];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      if (c4 == 0) {
        stat[(2 * warp) * RM + 8 * hh + r8] = m[hh];
        stat[(2 * warp + 1) * RM + 8 * hh + r8] = v;
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        ol[hh][g] += __shfl_xor_sync(0xffffffffu, ol[hh][g], 1);
        ol[hh][g] += __shfl_xor_sync(0xffffffffu, ol[hh][g], 2);
      }
    }
    const bool any_odd = __syncthreads_or(odd);
    // of row r8, and of rows 2 c4 and 2 c4 + 1
    float scale[2], scale_c[2][2];
#pragma unroll
    for (int hh = 0; hh < S::kHalves; ++hh) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < S::kWarps; ++w) top = fmaxf(top, stat[2 * w * RM + 8 * hh + r8]);
      scale[hh] = top == -INFINITY ? 0.f : b200attn::ptx::ex2_approx(m[hh] - top);
      scale_c[hh][0] = __shfl_sync(0xffffffffu, scale[hh], 8 * c4) * unit0;
      scale_c[hh][1] = __shfl_sync(0xffffffffu, scale[hh], 8 * c4 + 4) * unit0;
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
      // numbers DP / 4 g + NG r8 + i of rows 2 c4 and 2 c4 + 1, whose lows' sums lie in the lanes
      // of those rows
#pragma unroll
      for (int g = c0 / (DP / 4); g < (c0 + kC) / (DP / 4); ++g)
#pragma unroll
        for (int hh = 0; hh < S::kHalves; ++hh) {
          float* d = join + (warp * S::kJoinRows + 8 * hh + 2 * c4) * kPitch + DP / 4 * g - c0 + NG * r8;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float low = __shfl_sync(0xffffffffu, ol[hh][g] * scale[hh], 8 * c4 + 4 * e);
            float v[NG];
#pragma unroll
            for (int i = 0; i < NG; ++i)
              v[i] = fmaf(o[hh][NG / 2 * g + i / 2][2 * (i & 1) + e] * scale_c[hh][e],
                          i & 1 ? unit1 * 0.0625f : unit1, low);
            if constexpr (NG == 4)
              *reinterpret_cast<float4*>(d + e * kPitch) = make_float4(v[0], v[1], v[2], v[3]);
            else
              *reinterpret_cast<float2*>(d + e * kPitch) = make_float2(v[0], v[1]);
          }
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
                         finish ? reinterpret_cast<uint16_t*>(out) : nullptr, part + r * DP);
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
}

// -------------------------------------------------------------------- host
using namespace b200paged;

using AnyShape = Shape4<false, 128>;  // tiles and CTAs do not depend on the instance
static_assert(AnyShape::kTile == Shape4<true, 64>::kTile && AnyShape::kCtas == Shape4<true, 64>::kCtas,
              "one division of the work");

int64_t rows_of(const b200_tree_attn_params* p) { return p->tokens * (p->heads / p->cache.kv_heads); }

int64_t row_tiles(const b200_tree_attn_params* p) {
  return (rows_of(p) + AnyShape::RM - 1) / AnyShape::RM;
}

int64_t units_of(const b200_tree_attn_params* p) {
  return p->cache.batch * p->cache.kv_heads * row_tiles(p);
}

int64_t runs_of(const b200_tree_attn_params* p, int64_t sms) {
  const int64_t keys = p->cache.slots * p->cache.page_size;
  const double tiles = static_cast<double>(units_of(p)) *
                       static_cast<double>((keys + AnyShape::kTile - 1) / AnyShape::kTile);
  const int64_t most = (sms < kMaxSms ? sms : kMaxSms) * AnyShape::kCtas;
  return tiles < static_cast<double>(most) ? static_cast<int64_t>(tiles) : most;
}

template <int DP, int DT>
int32_t run_width(const Args& a, int runs, int64_t units, bool spread, int device, cudaStream_t s) {
  using Few = Shape4<true, DP>;
  using One = Shape4<false, DP>;
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
  if (static_cast<double>(units_of(p)) *
          static_cast<double>(c.slots * c.page_size / AnyShape::kTile + 4) > 2e9)
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
  return round16(8 * units_of(p)) + 2 * runs_of(p, kMaxSms) * 4 * AnyShape::RM * (dp + 2);
}

extern "C" int32_t b200_cache4_attn_fwd(const b200_tree_attn_params* p, int64_t head_dim,
                                        int32_t dtype, void* stream) {
  int32_t rc = b200_cache4_attn_check(p, head_dim, dtype);
  if (rc != B200_ATTN_OK) return rc;
  if (!p->workspace || p->workspace_bytes < b200_cache4_attn_workspace_bytes(p, head_dim, dtype))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(p->workspace) & 15u) return B200_ATTN_ERR_ALIGNMENT;
  b200paged::DeviceScope scope;
  if ((rc = scope.enter(p->q, "q is not a device pointer")) != B200_ATTN_OK) return rc;
  Args a{};
  if ((rc = b200attn::resolve_error_word(p->cache.error_word, &a.err)) != B200_ATTN_OK) return rc;
  fill_args(p, 2, 2, head_dim, &a);
  a.unit_rows = AnyShape::RM;
  a.row_tiles = static_cast<int32_t>(row_tiles(p));
  a.scale_log2 = p->scale * 1.4426950408889634f;
  const int64_t units = units_of(p);
  a.desc = static_cast<int2*>(p->workspace);
  a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(p->workspace) + round16(8 * units));
  const int runs = static_cast<int>(runs_of(p, b200paged::sm_count(scope.device)));
  a.runs = runs;
  // as for caches of 16 bits: long contexts of several rows are joined by a kernel of their own
  const bool spread = rows_of(p) > 4 && p->cache.slots * p->cache.page_size >= 12 * AnyShape::kTile &&
                      runs >= 8 * units;
  if (!spread && units <= B200_TREE_ATTN_COUNTERS) a.counters = p->counters;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = head_dim > 64;
  if (dtype == B200_ATTN_DTYPE_BF16)
    return wide ? run_width<128, B200_ATTN_DTYPE_BF16>(a, runs, units, spread, scope.device, s)
                : run_width<64, B200_ATTN_DTYPE_BF16>(a, runs, units, spread, scope.device, s);
  return wide ? run_width<128, B200_ATTN_DTYPE_FP16>(a, runs, units, spread, scope.device, s)
              : run_width<64, B200_ATTN_DTYPE_FP16>(a, runs, units, spread, scope.device, s);
}
