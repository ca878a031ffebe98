// tree_attn_rows.cuh — drafted-token attention for few rows (up to 32 a key
// head), 16-bit caches: single tokens and small trees.
//
// Mathematics, for a row q over the keys it sees, in one pass over blocks of keys:
//   s = scale log2(e) q.k,  m' = max(m, max s),  w = 2^(s - m'),
//   l' = l 2^(m - m') + sum w,  O' = O 2^(m - m') + sum w v,  out = O / l.
// What bounds it is HBM: R rows do 4 R D operations for the 4 D bytes of a key
// and value, far below the tensor cores' rate, so the kernel is built to keep
// loads in flight.  The warps of a CTA share a key tile, 16 keys each, and a
// warp never waits for another: it fetches its own keys and values into its own
// ring of shared memory (cp.async, 16 bytes a lane, zero-filled past the last
// key), multiplies them with mma m16n8k16 (rows of the queries are the M side),
// and keeps its own running maximum, sum and fp32 output sums.  The ring runs on
// over unit borders, so the loads of the next sequence are in flight while the
// warps of this one join their results in shared memory.  The matrix instruction of
// a warp is enough here: on 64 sequences of 0 to 8191 keys (one token, 4 rows) the tensor
// pipe is active 18 % of the time, and the fifth-generation one has no tile below 64 rows.
// Measured (bf16, D 128, 8 key heads): those 64 sequences, 1.07 GB, 174 us = 6.2 TB/s, 95 %
// of the rate of a plain copy; 16 rows over 131001 keys, 537 MB, 103 us, of
// which about 10 are the joins of the units cut over 37 CTAs each; one token over 1000 keys
// 13.2 us (12.9 us on the device alone), which is the launch, one chain of dependent loads
// (length, table, keys) and the join.  Prefetching the next blocks into L2 by bulk instructions instead of a deep ring:
// 244 us against 226 us at the time.
#pragma once

#include <type_traits>

#include "tree_attn.cuh"

namespace b200tree {

constexpr int kRowKeys = 16;  // keys of a warp's block

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <int DT>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (DT == B200_ATTN_DTYPE_BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int DT>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if constexpr (DT == B200_ATTN_DTYPE_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <int DT>
__device__ __forceinline__ float2 unpack_pair(uint32_t w) {
  if constexpr (DT == B200_ATTN_DTYPE_BF16)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// The 16-bit elements of a word that are not finite, as a mask of all-ones halves.
template <int DT>
__device__ __forceinline__ uint32_t non_finite(uint32_t w) {
  constexpr uint32_t kExp = DT == B200_ATTN_DTYPE_BF16 ? 0x7f807f80u : 0x7c007c00u;
  return __vcmpeq2(w & kExp, kExp);
}

// Shape of an instance: MT row tiles of 16 (FEW: up to 8 rows of one tile, whose other half
// is left out of the softmax), head dim padded to DP.
template <int MT_, bool FEW_, int DP_>
struct RowShape {
  static constexpr int MT = MT_, DP = DP_, RM = 16 * MT_;
  static constexpr bool FEW = FEW_;
  // One row tile: two CTAs of 4 warps on an SM, so that one reads while the other joins;
  // two row tiles need the SM for one CTA of 8.
  static constexpr int kWarps = MT == 1 ? 4 : 8, kThreads = 32 * kWarps;
  static constexpr int kCtas = 8 / kWarps;          // on an SM
  static constexpr int kTile = kWarps * kRowKeys;   // keys of a tile
  static constexpr int kHalves = FEW ? 1 : 2;  // halves of 8 rows of a tile
  static_assert(!FEW || MT == 1, "up to 8 rows");
  static constexpr int kRowBytes = 2 * DP;
  static constexpr int kPieces = kRowBytes / 16;
  static constexpr int kBlockBytes = kRowKeys * kRowBytes;     // one warp's keys or values
  static constexpr int kStages = DP == 128 ? 3 : 6;            // 192 KB of loads in flight
  static constexpr int kRingBytes = kWarps * kStages * 2 * kBlockBytes;
  static constexpr int kEach = MT == 1 ? 4 : 2;                // columns of a thread in a join
  static constexpr int kCols = kEach * kThreads / RM;          // columns joined at a time
  static constexpr int kJoinPitch = kCols + 4;
  static constexpr int kOffQ = kRingBytes;
  static constexpr int kOffJoin = kOffQ + RM * kRowBytes;
  static constexpr int kOffStat = kOffJoin + 4 * kWarps * RM * kJoinPitch;
  static constexpr int kOffMisc = kOffStat + 4 * 2 * kWarps * RM;
  static constexpr int kSmemBytes = kOffMisc + 256;
  static_assert(kSmemBytes <= 232448, "exceeds the shared memory of a block");
  using G = Grid<RM, kTile, 2>;
  static_assert(sizeof(JoinSmem<DP, kWarps>) <= 4 * kWarps * RM * kJoinPitch, "joins in place");
};

template <class S, int DT>
__global__ void __launch_bounds__(S::kThreads, S::kCtas) rows_kernel(const __grid_constant__ Args a) {
  constexpr int RM = S::RM, DP = S::DP, MT = S::MT, NS = S::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sbase = b200attn::ptx::smem_u32(smem);
  float* join = reinterpret_cast<float*>(smem + S::kOffJoin);
  float* stat = reinterpret_cast<float*>(smem + S::kOffStat);  // [warp][{max, sum}][RM]
  uint32_t* sums = reinterpret_cast<uint32_t*>(smem + S::kOffMisc);
  Run* found = reinterpret_cast<Run*>(smem + S::kOffMisc + 80);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  find_run<typename S::G>(a, blockIdx.x, gridDim.x, sums, found);
  const Run& run = *found;

  const int pieces = a.head_dim / 8;
  const uint32_t ring = sbase + warp * (NS * 2 * S::kBlockBytes);
  const uint32_t size = static_cast<uint32_t>(a.page_size);
  const bool whole = a.page_size % kRowKeys == 0;  // a block lies in one page

  // ------------------------------------------------------------- queries
  constexpr int kQPieces = RM * S::kPieces / S::kThreads > 0 ? RM * S::kPieces / S::kThreads : 1;
  uint4 qreg[kQPieces];
  auto fetch_q = [&](const Place& p) {
    const int rows = min(RM, p.s.drafts * a.group - p.rt * RM);
#pragma unroll
    for (int u = 0; u < kQPieces; ++u) {
      const int x = tid + u * S::kThreads;
      const int r = x / S::kPieces, piece = x % S::kPieces;
      qreg[u] = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows && piece < pieces) {
        const int row = p.rt * RM + r, i = row / a.group;
        qreg[u] = *reinterpret_cast<const uint4*>(
            a.q + p.b * a.q_seq + (p.h * a.group + row - i * a.group) * a.q_head + i * a.q_tok +
            16 * piece);
      }
    }
  };
  auto store_q = [&]() {
#pragma unroll
    for (int u = 0; u < kQPieces; ++u) {
      const int x = tid + u * S::kThreads;
      const int r = x / S::kPieces, piece = x % S::kPieces;
      if (r < RM)
        *reinterpret_cast<uint4*>(smem + S::kOffQ + r * S::kRowBytes + ((piece ^ (r & 7)) << 4)) =
            qreg[u];
    }
  };

  Place pl = run.p;
  const bool any = !run.done(pl);
  if (any) fetch_q(pl);

  // ------------------------------------------------------------- loads
  // The place of the next tile to load; its page numbers are read one tile ahead.
  Place ld = run.p;
  bool more = !run.done(ld);  // tiles are still to be loaded
  int page = -1, page_row = 0, ld_keys = 0;
  auto look_up = [&]() {
    const int key = ld.t * S::kTile + warp * kRowKeys + (whole ? 0 : (lane & 15));
    ld_keys = ld.s.len + ld.s.drafts - (ld.t * S::kTile + warp * kRowKeys);
    page = -1;
    page_row = 0;
    if (key < ld.s.len + ld.s.drafts) {
      const uint32_t slot = static_cast<uint32_t>(key) / size;
      page = __ldg(a.table + ld.b * a.table_stride + slot);
      page_row = static_cast<int>(static_cast<uint32_t>(key) - slot * size);
    }
  };
  if (more) look_up();
  int stage = 0;  // stage the next loads go to
  constexpr int kRowsAt = 32 / S::kPieces;  // rows a warp loads at a time
  constexpr int kPlaces = 8 / kRowsAt;
  const int piece = lane % S::kPieces, r0 = lane / S::kPieces;
  uint32_t place[kPlaces];  // of this lane's piece in its rows among 8
#pragma unroll
  for (int i = 0; i < kPlaces; ++i) {
    const int r = r0 + i * kRowsAt;
    place[i] = r * S::kRowBytes + ((piece ^ r) << 4);
  }
  auto issue = [&]() {
    if (more) {
      if (page >= a.pages || (page < 0 && (whole ? 0 : (lane & 15)) < ld_keys)) {
        report_error(a.err, B200_ATTN_DEVERR_BOUNDS);
        page = -1;
      }
      const uint32_t dst = ring + stage * (2 * S::kBlockBytes);
      const int64_t head_k = ld.h * a.k_head, head_v = ld.h * a.v_head;
      if (whole && page >= 0 && ld_keys >= kRowKeys && a.head_dim == DP) {
        // a whole block of one page
        const int64_t at = page_row + r0;
        const uint8_t* ks = a.k + page * a.k_page + head_k + at * a.k_row + 16 * piece;
        const uint8_t* vs = a.v + page * a.v_page + head_v + at * a.v_row + 16 * piece;
#pragma unroll
        for (int i = 0; i < kRowKeys / kRowsAt; ++i) {
          // rows 8 apart have the same swizzle
          const uint32_t off = dst + place[i % kPlaces] + (i / kPlaces) * (8 * S::kRowBytes);
          cp_async16(off, ks, 16u);
          cp_async16(off + S::kBlockBytes, vs, 16u);
          ks += kRowsAt * a.k_row;
          vs += kRowsAt * a.v_row;
        }
      } else
#pragma unroll 1
      for (int i = 0; i < kRowKeys / kRowsAt; ++i) {
        const int r = r0 + i * kRowsAt;
        const int pg = whole ? page : __shfl_sync(0xffffffffu, page, r);
        const int pr = whole ? page_row + r : __shfl_sync(0xffffffffu, page_row, r);
        const bool ok = pg >= 0 && r < ld_keys && piece < pieces;
        const uint8_t* ks = a.k;
        const uint8_t* vs = a.v;
        if (ok) {
          ks += pg * a.k_page + head_k + pr * a.k_row + 16 * piece;
          vs += pg * a.v_page + head_v + pr * a.v_row + 16 * piece;
        }
        const uint32_t off = r * S::kRowBytes + ((piece ^ (r & 7)) << 4);
        cp_async16(dst + off, ks, ok ? 16u : 0u);
        cp_async16(dst + S::kBlockBytes + off, vs, ok ? 16u : 0u);
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

  if (any) store_q();
  __syncthreads();
  int use = 0;  // stage of the tile at hand
  const int g = lane >> 2, t2 = (lane & 3) * 2;  // row and column pair of this lane in a product
  const int mat = lane >> 3, mrow = lane & 7;    // matrix and row this lane addresses

#pragma unroll 1
  while (!run.done(pl)) {
    const int t0 = pl.t;
    const int n = run.tiles(pl);
    const int keys = pl.s.len + pl.s.drafts;
    float o[MT][DP / 8][4];
    float m[MT][2], l[MT][2];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      m[i][0] = m[i][1] = -INFINITY;
      l[i][0] = l[i][1] = 0.f;
#pragma unroll
      for (int x = 0; x < DP / 8; ++x) o[i][x][0] = o[i][x][1] = o[i][x][2] = o[i][x][3] = 0.f;
    }
    uint32_t qf[MT == 1 ? DP / 16 : 1][4];
    auto load_q_frag = [&](uint32_t (&f)[4], int i, int kk) {
      const int r = 16 * i + (mat & 1) * 8 + mrow;
      ldmatrix_x4(f, sbase + S::kOffQ + r * S::kRowBytes + (((2 * kk + (mat >> 1)) ^ (r & 7)) << 4));
    };
    if constexpr (MT == 1) {
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) load_q_frag(qf[kk], 0, kk);
    }
    bool odd = false;  // a drafted token's value was not finite

#pragma unroll 1
    for (int t = t0; t < t0 + n; ++t) {
      issue();
      cp_async_wait<NS - 1>();
      __syncwarp();
      const uint32_t kb = ring + use * (2 * S::kBlockBytes), vb = kb + S::kBlockBytes;
      use = use + 1 == NS ? 0 : use + 1;
      const int k0 = t * S::kTile + warp * kRowKeys;
      if (k0 < keys) {
        float s[MT][2][4];
        float s2[2][4];  // one row tile: the odd steps' sums, for shorter chains of products
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          s2[x][0] = s2[x][1] = s2[x][2] = s2[x][3] = 0.f;
#pragma unroll
          for (int i = 0; i < MT; ++i) s[i][x][0] = s[i][x][1] = s[i][x][2] = s[i][x][3] = 0.f;
        }
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          uint32_t b[4];
          const int r = (mat >> 1) * 8 + mrow;
          ldmatrix_x4(b, kb + r * S::kRowBytes + (((2 * kk + (mat & 1)) ^ (r & 7)) << 4));
          if constexpr (MT == 1) {
            mma16816<DT>(kk & 1 ? s2[0] : s[0][0], qf[kk], b[0], b[1]);
            mma16816<DT>(kk & 1 ? s2[1] : s[0][1], qf[kk], b[2], b[3]);
          } else {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              uint32_t f[4];
              load_q_frag(f, i, kk);
              mma16816<DT>(s[i][0], f, b[0], b[1]);
              mma16816<DT>(s[i][1], f, b[2], b[3]);
            }
          }
        }
        if constexpr (MT == 1) {
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 2 * S::kHalves; ++e) s[0][x][e] += s2[x][e];
        }
        if (k0 + kRowKeys > pl.s.len) {
          // drafted tokens, or past the last key
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 2 * S::kHalves; ++e) {
              const int row = pl.rt * RM + 16 * i + g + (e >> 1) * 8;
              const int tok = min(row / a.group, a.tokens - 1);
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const int j = k0 + 8 * x + t2 + (e & 1) - pl.s.len;
                if (j >= 0 && (j >= pl.s.drafts || !sees(a, pl.b, tok, j))) s[i][x][e] = -INFINITY;
              }
            }
          // A hidden value must not reach a row as 0 x infinity: elements that
          // are not finite become 0 here and are added below to the rows that see them.
          const uint32_t f0 = vb + lane * 16;
#pragma unroll
          for (int u = 0; u < S::kBlockBytes / 512; ++u) {
            uint32_t w[4];
            const uint32_t ad = f0 + 512 * u;
            const int r = (16 * lane + 512 * u) / S::kRowBytes;
            if (k0 + r < pl.s.len) continue;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(ad)
                         : "memory");
            uint32_t any = 0u;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t f = non_finite<DT>(w[y]);
              any |= f;
              w[y] &= ~f;
            }
            if (any) {
              odd = true;
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(ad), "r"(w[0]),
                           "r"(w[1]), "r"(w[2]), "r"(w[3])
                           : "memory");
            }
          }
          __syncwarp();
        }
        // running maximum; the sums so far are rescaled only where it grew
        bool grew = false;
        float alpha[MT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int hh = 0; hh < S::kHalves; ++hh) {
            float top = fmaxf(fmaxf(s[i][0][2 * hh], s[i][0][2 * hh + 1]),
                              fmaxf(s[i][1][2 * hh], s[i][1][2 * hh + 1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float now = fmaxf(m[i][hh], top * a.scale_log2);
            grew |= now > m[i][hh];
            alpha[i][hh] = now == -INFINITY ? 1.f : b200attn::ptx::ex2_approx(m[i][hh] - now);
            m[i][hh] = now;
          }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int i = 0; i < MT; ++i) {
#pragma unroll
            for (int hh = 0; hh < S::kHalves; ++hh) {
              l[i][hh] *= alpha[i][hh];
#pragma unroll
              for (int x = 0; x < DP / 8; ++x) {
                o[i][x][2 * hh] *= alpha[i][hh];
                o[i][x][2 * hh + 1] *= alpha[i][hh];
              }
            }
          }
        }
        uint32_t pf[MT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            if (hh >= S::kHalves) {
              pf[i][1] = pf[i][3] = 0u;
              break;
            }
            const float base = m[i][hh] == -INFINITY ? 0.f : m[i][hh];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float p0 = b200attn::ptx::ex2_approx(fmaf(s[i][x][2 * hh], a.scale_log2, -base));
              const float p1 =
                  b200attn::ptx::ex2_approx(fmaf(s[i][x][2 * hh + 1], a.scale_log2, -base));
              // weights are rounded to the element type for the product; their sum is
              // taken of the rounded ones, so a row of few keys stays exact
              const uint32_t w = pack_pair<DT>(p0, p1);
              const float2 r = unpack_pair<DT>(w);
              pf[i][2 * x + hh] = w;
              l[i][hh] += r.x + r.y;
            }
          }
        }
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) {
          uint32_t b[4];
          const int r = (mat & 1) * 8 + mrow;
          ldmatrix_x4_trans(b, vb + r * S::kRowBytes + (((2 * x + (mat >> 1)) ^ (r & 7)) << 4));
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            mma16816<DT>(o[i][2 * x], pf[i], b[0], b[1]);
            mma16816<DT>(o[i][2 * x + 1], pf[i], b[2], b[3]);
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
    const bool again = !run.done(pl);
    if (again) fetch_q(pl);  // on its way while the results are joined
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float v = l[i][hh];
        v += __shfl_xor_sync(0xffffffffu, v, 1);
        v += __shfl_xor_sync(0xffffffffu, v, 2);
        if ((lane & 3) == 0) {
          stat[(2 * warp) * RM + 16 * i + 8 * hh + g] = m[i][hh];
          stat[(2 * warp + 1) * RM + 16 * i + 8 * hh + g] = v;
        }
      }
    const bool any_odd = __syncthreads_or(odd);
    float scale[MT][2];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < S::kWarps; ++w)
          top = fmaxf(top, stat[2 * w * RM + 16 * i + 8 * hh + g]);
        scale[i][hh] = top == -INFINITY ? 0.f : b200attn::ptx::ex2_approx(m[i][hh] - top);
      }
    const int rows = min(RM, done.s.drafts * a.group - done.rt * RM);
    float* part = a.partial + static_cast<int64_t>(2 * blockIdx.x + (first ? 1 : 0)) * (RM * (DP + 2));
    const bool finish = first && last;
    // The warps' sums go through shared memory, some columns at a time; a thread adds
    // kEach columns of a row.  Up to 8 rows (a token of 8 query heads): twice the columns of half
    // the rows.
    auto join_columns = [&](auto row_count, auto col_count) {
      constexpr int kR = decltype(row_count)::value, kC = decltype(col_count)::value;
      constexpr int kPitch = kC + 4;
      static_assert(kR * kC == S::kEach * S::kThreads, "kEach columns a thread");
      static_assert(kR * kPitch <= RM * S::kJoinPitch, "in place");
      const int r = tid / (kC / S::kEach), c = (tid % (kC / S::kEach)) * S::kEach;
      float top = -INFINITY, total = 0.f;
#pragma unroll
      for (int w = 0; w < S::kWarps; ++w) top = fmaxf(top, stat[2 * w * RM + r]);
#pragma unroll
      for (int w = 0; w < S::kWarps; ++w) {
        const float mw = stat[2 * w * RM + r];
        if (mw != -INFINITY)
          total += stat[(2 * w + 1) * RM + r] * b200attn::ptx::ex2_approx(mw - top);
      }
      const float inv = total == 0.f ? 0.f : 1.f / total;
      const int row = done.rt * RM + r, tok = row / a.group;
      uint8_t* out = a.o + done.b * a.o_seq + (done.h * a.group + row - tok * a.group) * a.o_head +
                     tok * a.o_tok;
#pragma unroll
      for (int c0 = 0; c0 < DP; c0 += kC) {
        if (c0) __syncthreads();
#pragma unroll
        for (int i = 0; i < (kR > 16 ? MT : 1); ++i)
#pragma unroll
          for (int x = 0; x < kC / 8; ++x) {
            float* d = join + (warp * kR + 16 * i + g) * kPitch + 8 * x + t2;
            const float* src = o[i][c0 / 8 + x];
            *reinterpret_cast<float2*>(d) = make_float2(src[0] * scale[i][0], src[1] * scale[i][0]);
            if (kR > 8)
              *reinterpret_cast<float2*>(d + 8 * kPitch) =
                  make_float2(src[2] * scale[i][1], src[3] * scale[i][1]);
          }
        __syncthreads();
        float2 acc[S::kEach / 2];
#pragma unroll
        for (int e = 0; e < S::kEach / 2; ++e) acc[e] = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < S::kWarps; ++w)
#pragma unroll
          for (int e = 0; e < S::kEach / 2; ++e) {
            const float2 v =
                *reinterpret_cast<const float2*>(join + (w * kR + r) * kPitch + c + 2 * e);
            acc[e].x += v.x;
            acc[e].y += v.y;
          }
#pragma unroll
        for (int e = 0; e < S::kEach / 2; ++e) {
          if (!finish)
            *reinterpret_cast<float2*>(part + r * DP + c0 + c + 2 * e) = acc[e];
          else if (r < rows && c0 + c < a.head_dim)
            *reinterpret_cast<uint32_t*>(out + 2 * (c0 + c + 2 * e)) =
                pack_pair<DT>(acc[e].x * inv, acc[e].y * inv);
        }
      }
      if (any_odd && r < rows)
        for (int c0 = c; c0 < DP; c0 += kC)
          add_odd<DT>(a, done.b, done.h, done.s, tok, t0 * S::kTile - done.s.len,
                      (t0 + n) * S::kTile - done.s.len, c0, min(a.head_dim, c0 + S::kEach),
                      finish ? reinterpret_cast<uint16_t*>(out) : nullptr, part + r * DP, 1);
      if (!finish && c == 0) {
        part[RM * DP + r] = top;
        part[RM * DP + RM + r] = total;
      }
    };
    if constexpr (S::FEW) {
      join_columns(std::integral_constant<int, 8>{}, std::integral_constant<int, 64>{});
    } else {
      join_columns(std::integral_constant<int, RM>{}, std::integral_constant<int, S::kCols>{});
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
    if (again) store_q();  // the queries' fragments are in registers, or read between the barriers
    __syncthreads();
  }
  zero_unused_rows(a, 2, S::kThreads);
}

}  // namespace b200tree
