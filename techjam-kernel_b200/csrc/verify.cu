// verify.cu — the check of drafted tokens against the target's probabilities
// (definition: b200_verify.h).
//
// A cluster of CTAs walks the tree of one sequence.  Only the rows of the nodes on the path
// are read, each by all CTAs of the cluster, a contiguous share a warp; the CTAs
// exchange their sums through distributed shared memory and all take the same decisions.  A
// step down the tree is one pass over a row: the sum of e^(l / T).  What is left after k refusals of
// drafts with probabilities q, each time normalised, is
//   max(p - t_k q, 0) / F(t_k),  F(t) = sum of max(p - t q, 0),  t_1 = 1,  t_(k+1) = t_k + F(t_k),
// (max(y / Z - q, 0) of y = max(a p - b q, 0) is max(a / Z p - (b / Z + 1) q, 0)): a refusal takes
// one more pass over the row of the target, which lies in L2 by then, and that of the drafter,
// whatever was refused before it.  The last pass's sums, a warp each, say in which share
// the next token lies; it is divided among the warps of its CTA once more, and one warp
// scans the part.
// Exponentials and sums are 64-bit: among 32000 cumulated weights a sum that is off by 1e-8
// would pick a neighbour once in some thousand draws.  The exponentials need no maximum
// beforehand: e^(l / T) does not leave the range of 64 bits unless |l / T| is over 600, and such
// a row is summed again relative to its maximum.
//
// Bound by the latency of passes that follow one another, each a wait for its row, a barrier of the
// cluster and the next decision: 64 sequences with trees of 16 nodes, vocabulary 100003, take 130 us
// where the rows on the paths are 12 us of bytes, with the issue slots half used, the 64-bit pipe a
// fifth and L1 half (of rows that do not start on four numbers each number is a load); 64 chains of 8
// nodes, vocabulary 32000, 43 us.  With a pass over the row for each refusal before (what is left
// taken again step by step) those trees took 412 us, and with a maximum first the chains 51.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <mutex>

#include "b200_verify.h"
#include "byte_range.h"
#include "error_word.cuh"
#include "paged_host.h"
#include "sm100_ptx.cuh"
#include "tree_attn.cuh"

namespace b200verify {

using b200attn::report_error;
using b200tree::Elem;

namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps, kMaxCluster = 16;
constexpr uint32_t kAll = 0xffffffffu;

struct Args {
  const uint8_t* logits;
  int64_t l_seq, l_node;  // bytes
  const uint8_t* probs;   // null: drafts count as certain
  int64_t q_seq, q_node;
  const uint8_t* tokens;
  int64_t t_seq;  // elements
  const float* uniforms;
  int64_t u_seq;
  const int32_t* parents;  // null: a chain
  int64_t p_seq;
  const int32_t* lens;
  int32_t* paths;
  int32_t* counts;
  int64_t* next;
  double inv_temp;  // 0: the largest logit
  int32_t nodes, vocab, share;  // share: numbers of a warp, a multiple of 4
  int32_t probs_type, wide_tokens;
  bool probs_vec;
  bool keep;  // a row's exponentials fit in shared memory
  int32_t* err;
};

struct Exchange {  // what a CTA tells the others
  double sum;
  float top;   // largest number
  int32_t at;  // its place
  int32_t bad;
};

// Shared memory of a CTA: what the nodes need lies behind the fixed part, and the exponentials of
// the CTA's share of the row behind that.
struct Smem {
  Exchange told[2][kMaxCluster];
  Exchange warp[kWarps];
  double part_sum[kWarps];
  double power[64];  // 2^(j / 64)
};
struct Views {
  int32_t* parent;
  int32_t* token;
  float* uniform;
  float* logit;      // the target's for the node's token, in its parent's row
  float* prob;       // the drafter's
  int32_t* refused;  // tokens refused at this node that have no weight any more
  int32_t* path;
  double* kept;
};
constexpr int kNodeArrays = 7;
__host__ __device__ inline int nodes_padded(int nodes) { return (nodes + 3) & ~3; }

__device__ __forceinline__ Views views_of(uint8_t* smem, int nodes) {
  int32_t* p = reinterpret_cast<int32_t*>(smem + sizeof(Smem));
  const int n = nodes_padded(nodes);
  return Views{p, p + n, reinterpret_cast<float*>(p + 2 * n), reinterpret_cast<float*>(p + 3 * n),
               reinterpret_cast<float*>(p + 4 * n), p + 5 * n, p + 6 * n,
               reinterpret_cast<double*>(p + kNodeArrays * n)};
}

// Four numbers of a row from number v on; `vec`: by one load where all four are there.
template <int DT, class T = typename Elem<DT>::T>
__device__ __forceinline__ void load4(const uint8_t* row, int v, int end, bool vec, float fill,
                                      float (&x)[4]) {
  const T* p = reinterpret_cast<const T*>(row) + v;
  if (vec && v + 4 <= end) {
    if constexpr (sizeof(T) == 4) {
      const float4 w = __ldg(reinterpret_cast<const float4*>(p));
      x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w;
    } else {
      union {
        uint2 w;
        T e[4];
      } u;
      u.w = __ldg(reinterpret_cast<const uint2*>(p));
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = Elem<DT>::widen(u.e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = v + i < end ? Elem<DT>::widen(p[i]) : fill;
  }
}

__device__ __forceinline__ float as_prob(float q) { return q > 0.f ? q : 0.f; }

__device__ __forceinline__ void probs4(const Args& a, const uint8_t* row, int v, int end,
                                       float (&q)[4]) {
  if (a.probs_type == B200_ATTN_DTYPE_FP32)
    load4<B200_ATTN_DTYPE_FP32>(row, v, end, a.probs_vec, 0.f, q);
  else if (a.probs_type == B200_ATTN_DTYPE_BF16)
    load4<B200_ATTN_DTYPE_BF16>(row, v, end, a.probs_vec, 0.f, q);
  else
    load4<B200_ATTN_DTYPE_FP16>(row, v, end, a.probs_vec, 0.f, q);
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = as_prob(q[i]);
}

__device__ __forceinline__ float one_prob(const Args& a, const uint8_t* row, int v) {
  if (a.probs_type == B200_ATTN_DTYPE_FP32) return as_prob(reinterpret_cast<const float*>(row)[v]);
  if (a.probs_type == B200_ATTN_DTYPE_BF16)
    return as_prob(__bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[v]));
  return as_prob(__half2float(reinterpret_cast<const __half*>(row)[v]));
}

// The node that the path has reached.  Number v has the weight max(scale e^((l - top) / T) - t q, 0),
// or 0 where it is one of `refused`.
struct Node {
  const uint8_t* row;
  const uint8_t* probs;
  double top, scale, t;
  int refused;
};

// e^z for z up to 700, and 0 below -700: 2^(k / 64) from a table times a polynomial for the rest
// (Tang, "Table-driven implementation of the exponential function in IEEE floating-point
// arithmetic", 1989).  |r| <= ln 2 / 128: the first term left out is below 4e-14 of the result, and
// r is off by 1e-13 at most.
__device__ __forceinline__ double exp_of(const double* power, double z) {
  constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: the sum's low bits are the integer
  const double t = fma(z, 92.332482616893656877, kRound);  // 64 / ln 2
  const int k = __double2loint(t);
  const double r = fma(t - kRound, -0.010830424696249145, z);  // ln 2 / 64
  double p = fma(r, 1.0 / 24.0, 1.0 / 6.0);
  p = fma(r, p, 0.5);
  p = fma(r * r, p, r);
  const double w = power[k & 63];
  const double y = fma(w, p, w);
  return z > -700.0 ? __hiloint2double(__double2hiint(y) + ((k >> 6) << 20), __double2loint(y)) : 0.0;
}

__device__ __forceinline__ double weight(const Args& a, const Smem& sm, float l, double top) {
  // (a difference of logits is exact, and 0 for the largest whatever the temperature)
  return exp_of(sm.power, (static_cast<double>(l) - top) * a.inv_temp);
}

// e^((l - top) / T) of four numbers, into or out of the CTA's kept ones (`kept`: the first's).
__device__ __forceinline__ void keep4(double* kept, const double (&e)[4]) {
  reinterpret_cast<double2*>(kept)[0] = make_double2(e[0], e[1]);
  reinterpret_cast<double2*>(kept)[1] = make_double2(e[2], e[3]);
}

// The weights of four numbers from v on; `base`: the CTA's first number.
template <int DT, bool VEC>
__device__ __forceinline__ void weights4(const Args& a, const Smem& sm, const Views& vw,
                                         const Node& n, int v, int base, int end, double (&y)[4]) {
  float q[4] = {0.f, 0.f, 0.f, 0.f};
  if (n.t != 0.0) probs4(a, n.probs, v, end, q);
  if (a.keep) {
    const double2* p = reinterpret_cast<const double2*>(vw.kept + (v - base));
    const double2 e0 = p[0], e1 = p[1];
    y[0] = e0.x, y[1] = e0.y, y[2] = e1.x, y[3] = e1.y;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (v + i >= end) y[i] = 0.0;
  } else {
    float l[4];
    load4<DT>(n.row, v, end, VEC, -INFINITY, l);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = weight(a, sm, l[i], n.top);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    y[i] = fmax(fma(y[i], n.scale, -n.t * static_cast<double>(q[i])), 0.0);
  for (int j = 0; j < n.refused; ++j) {
    const uint32_t x = static_cast<uint32_t>(vw.refused[j] - v);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (x == i) y[i] = 0.0;
  }
}

template <class T>
__device__ __forceinline__ T warp_total(T x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(kAll, x, o);
  return x;
}

// A row's first pass, of numbers [begin, end) by a warp: the sum of e^((l - top) / T), the largest
// logit and whether one is NaN or +infinity; at temperature 0 the place of the largest instead of
// the sum.
template <int DT, bool VEC>
__device__ __noinline__ Exchange first_pass(const Args& a, const Smem& sm, const Views& vw,
                                            const uint8_t* row, double top, int base, int begin,
                                            int end) {
  constexpr int kDeep = 4;  // loads in flight
  const int lane = threadIdx.x & 31;
  Exchange x{0.0, -INFINITY, 0x7fffffff, 0};
  double sum[2] = {0.0, 0.0};
  bool bad = false;
  for (int v = begin + 4 * lane; v < end; v += 128 * kDeep) {
    float l[kDeep][4];
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      if (v + 128 * u < end) {
        load4<DT>(row, v + 128 * u, end, VEC, -INFINITY, l[u]);
      } else {
        l[u][0] = l[u][1] = l[u][2] = l[u][3] = -INFINITY;
      }
    }
#pragma unroll
    for (int u = 0; u < kDeep; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) bad |= !(l[u][i] < INFINITY);
    if (a.inv_temp == 0.0) {
#pragma unroll
      for (int u = 0; u < kDeep; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (l[u][i] > x.top) {
            x.top = l[u][i];
            x.at = v + 128 * u + i;
          }
    } else {
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        double e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x.top = fmaxf(x.top, l[u][i]);
          e[i] = weight(a, sm, l[u][i], top);
          sum[i & 1] += e[i];
        }
        if (a.keep && v + 128 * u < end) keep4(vw.kept + (v + 128 * u - base), e);
      }
    }
  }
  x.sum = warp_total(sum[0] + sum[1]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float high = __shfl_xor_sync(kAll, x.top, o);
    const int at = __shfl_xor_sync(kAll, x.at, o);
    if (high > x.top || (high == x.top && at < x.at)) {
      x.top = high;
      x.at = at;
    }
  }
  x.bad = __any_sync(kAll, bad);
  return x;
}

// The sum of the weights of numbers [begin, end), by a warp.
template <int DT, bool VEC>
__device__ __noinline__ double sum_pass(const Args& a, const Smem& sm, const Views& vw,
                                        const Node& n, int base, int begin, int end) {
  double sum = 0.0;
#pragma unroll 2
  for (int v = begin + 4 * (threadIdx.x & 31); v < end; v += 128) {
    double y[4];
    weights4<DT, VEC>(a, sm, vw, n, v, base, end, y);
    sum += (y[0] + y[1]) + (y[2] + y[3]);
  }
  return warp_total(sum);
}

__device__ __forceinline__ void take(Exchange& x, const Exchange& y) {
  x.sum += y.sum;
  if (y.top > x.top || (y.top == x.top && y.at < x.at)) {
    x.top = y.top;
    x.at = y.at;
  }
  x.bad |= y.bad;
}

// Every warp's x to all: those of this CTA into sm.warp, the CTAs' into sm.told[turn], and what they
// come to.  By all threads of all CTAs.  Two slots in turn: a CTA writes a slot again when all
// have passed the barrier after reading it.
__device__ __noinline__ Exchange share_out(Smem& sm, int turn, const Exchange x, uint32_t rank,
                                           uint32_t ctas) {
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm.warp[threadIdx.x >> 5] = x;
  __syncthreads();
  if (threadIdx.x < ctas) {
    Exchange mine = sm.warp[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) take(mine, sm.warp[w]);
    const uint32_t at = b200attn::ptx::mapa_shared(
        b200attn::ptx::smem_u32(&sm.told[turn][rank]), threadIdx.x);
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(mine.sum) : "memory");
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 8), "f"(mine.top) : "memory");
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at + 12), "r"(mine.at) : "memory");
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at + 16), "r"(mine.bad) : "memory");
  }
  b200attn::ptx::cluster_sync();
  Exchange all = sm.told[turn][0];
#pragma unroll
  for (uint32_t c = 1; c < kMaxCluster; ++c)
    if (c < ctas) take(all, sm.told[turn][c]);
  return all;
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) verify_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(16) uint8_t raw[];
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  const Views vw = views_of(raw, a.nodes);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ctas = gridDim.x, rank = blockIdx.x;  // one cluster a sequence
  const int64_t b = blockIdx.y;
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();

  int n = a.lens ? a.lens[b] : a.nodes;
  if (n < 0 || n > a.nodes) {
    if (tid == 0 && rank == 0) report_error(a.err, B200_ATTN_DEVERR_BOUNDS);
    n = 0;
  }
  if (tid < 64) sm.power[tid] = exp2(tid / 64.0);
  const uint8_t* logits = a.logits + b * a.l_seq;
  const uint8_t* probs = a.probs ? a.probs + b * a.q_seq : nullptr;
  for (int i = tid; i < n; i += kThreads) {
    int parent = a.parents ? a.parents[b * a.p_seq + i] : i - 1;
    vw.uniform[i] = a.uniforms[b * a.u_seq + i];
    if (i == 0) {
      vw.parent[0] = -1;
      continue;
    }
    const int64_t t = a.wide_tokens ? reinterpret_cast<const int64_t*>(a.tokens)[b * a.t_seq + i]
                                    : reinterpret_cast<const int32_t*>(a.tokens)[b * a.t_seq + i];
    const bool known = t >= 0 && t < a.vocab;
    if (parent < -1 || parent >= i || !known) {
      if (rank == 0) report_error(a.err, B200_ATTN_DEVERR_BOUNDS);
      parent = -1;
    }
    vw.parent[i] = parent;
    vw.token[i] = static_cast<int>(t);
    if (parent >= 0) {
      const uint8_t* row = logits + parent * a.l_node;
      vw.logit[i] = Elem<DT>::widen(reinterpret_cast<const typename Elem<DT>::T*>(row)[t]);
      if (probs) vw.prob[i] = one_prob(a, probs + parent * a.q_node, static_cast<int>(t));
    }
  }
  // every CTA of the cluster runs: its shared memory may be written
  b200attn::ptx::cluster_sync();

  const int base = min(static_cast<int64_t>(a.vocab), static_cast<int64_t>(rank * kWarps) * a.share);
  const int begin = min(static_cast<int64_t>(a.vocab),
                        static_cast<int64_t>(rank * kWarps + warp) * a.share);
  const int end = min(static_cast<int64_t>(a.vocab), begin + static_cast<int64_t>(a.share));
  int turn = 0, length = 0, at = 0;
  int64_t next = -1;
  bool teller = rank == 0;  // this CTA writes the next token
  Node node{};

  auto first_of = [&]() {
    turn ^= 1;
    return share_out(sm, turn, first_pass<DT, VEC>(a, sm, vw, node.row, node.top, base, begin, end), rank, ctas);
  };
  auto sum_of = [&]() {
    turn ^= 1;
    return share_out(sm, turn, Exchange{sum_pass<DT, VEC>(a, sm, vw, node, base, begin, end), 0.f, 0, 0}, rank,
                     ctas).sum;
  };

  while (n > 0) {
    // --------------------------------------------------- a node: its sum of weights
    if (tid == 0 && rank == 0) vw.path[length] = at;
    ++length;
    node = Node{logits + at * a.l_node, probs ? probs + at * a.q_node : nullptr, 0.0, 1.0, 0.0, 0};
    Exchange all = first_of();
    if (all.bad || all.top == -INFINITY) break;  // no distribution
    if (fabs(static_cast<double>(all.top) * a.inv_temp) > 600.0) {
      node.top = static_cast<double>(all.top);
      all = first_of();
    }
    const double inv = 1.0 / all.sum;

    // --------------------------------------------------- its children in order
    int kept = -1;
    double gone = 0.0;       // weight of the refused tokens, where drafts count as certain
    bool summed = true;      // sm.warp and told hold the sums of the weights as they are now
    double left = all.sum;   // in all
    const int likeliest = all.at;
    for (int i0 = at + 1; i0 < n && kept < 0; i0 += 32) {
      uint32_t mask = __ballot_sync(kAll, i0 + lane < n && vw.parent[i0 + lane] == at);
      while (mask != 0u && kept < 0) {
        const int c = i0 + __ffs(mask) - 1;
        mask &= mask - 1;
        if (a.inv_temp == 0.0) {
          if (vw.token[c] == likeliest && vw.uniform[c] < 1.f) kept = c;
          continue;
        }
        const double e = weight(a, sm, vw.logit[c], node.top);
        const double u = static_cast<double>(vw.uniform[c]);
        if (!probs) {
          bool again = false;
          for (int j = 0; j < node.refused; ++j) again |= vw.refused[j] == vw.token[c];
          if (again) continue;
          if (u * (all.sum - gone) < e) {
            kept = c;
          } else if (all.sum - gone - e > 0.0) {  // something is left without it
            gone += e;
            __syncthreads();
            if (tid == 0) vw.refused[node.refused] = vw.token[c];
            __syncthreads();
            ++node.refused;
            summed = false;
          }
          continue;
        }
        const double q = static_cast<double>(vw.prob[c]);
        if (u * q * left < fmax(fma(e, node.scale, -node.t * q), 0.0)) {
          kept = c;
          continue;
        }
        // the weights so far were e, or max(p - t q, 0), which add up to `left`
        const Node before = node;
        node.t = node.t == 0.0 ? 1.0 : node.t + left;
        node.scale = inv;
        const double rest = sum_of();
        summed = rest > 0.0;
        if (summed) {
          left = rest;
        } else {
          node = before;
        }
      }
    }
    if (kept >= 0) {
      at = kept;
      continue;
    }
    // ------------------------------------------------------- the next token
    if (a.inv_temp == 0.0) {
      next = likeliest;
      break;
    }
    if (!summed) left = sum_of();
    // (refusals leave something: only the rounding of a sum lets one too many through)
    while (!(left > 0.0) && node.refused > 0) {
      --node.refused;
      left = sum_of();
    }
    const double goal = static_cast<double>(vw.uniform[0]) * left;
    // the CTA, then the warp, then the part of its share that the goal lies in: the first
    // whose end is past it, or else the last with any weight
    double before = 0.0;
    auto find = [&](auto sums, int count) {
      double cum = before, from = before;
      int best = -1;
      for (int i = 0; i < count; ++i) {
        const double s = sums(i);
        if (s > 0.0) {
          best = i;
          from = cum;
          if (cum + s > goal) break;
        }
        cum += s;
      }
      before = from;
      return best;
    };
    const int cta = find([&](int i) { return sm.told[turn][i].sum; }, static_cast<int>(ctas));
    teller = cta == static_cast<int>(rank);
    if (!teller) break;
    const int owner = find([&](int i) { return sm.warp[i].sum; }, kWarps);
    const int part = (a.share / 4 + kWarps - 1) / kWarps * 4;
    const int from = min(static_cast<int64_t>(a.vocab),
                         static_cast<int64_t>(rank * kWarps + owner) * a.share);
    const int to = min(static_cast<int64_t>(a.vocab), from + static_cast<int64_t>(a.share));
    const double mine = sum_pass<DT, VEC>(a, sm, vw, node, base, min(to, from + warp * part),
                                          min(to, from + (warp + 1) * part));
    if (lane == 0) sm.part_sum[warp] = mine;
    __syncthreads();
    const int which = find([&](int i) { return sm.part_sum[i]; }, kWarps);
    if (warp == 0) {
      const int stop = min(to, from + (which + 1) * part);
      int found = -1, last = -1;
      for (int v0 = from + which * part; v0 < stop && found < 0; v0 += 128) {
        const int v = v0 + 4 * lane;
        double y[4] = {0.0, 0.0, 0.0, 0.0};
        if (v < stop) weights4<DT, VEC>(a, sm, vw, node, v, base, stop, y);
        double mine4 = (y[0] + y[1]) + (y[2] + y[3]), cum = mine4;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double t = __shfl_up_sync(kAll, cum, o);
          if (lane >= o) cum += t;
        }
        const double all = __shfl_sync(kAll, cum, 31);
        double run = before + (cum - mine4);
        int first = -1, some = -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          run += y[i];
          if (y[i] > 0.0) {
            some = v + i;
            if (first < 0 && run > goal) first = v + i;
          }
        }
        const uint32_t hit = __ballot_sync(kAll, first >= 0), any = __ballot_sync(kAll, some >= 0);
        if (hit) found = __shfl_sync(kAll, first, __ffs(hit) - 1);
        if (any) last = __shfl_sync(kAll, some, 31 - __clz(any));
        before += all;
      }
      next = found >= 0 ? found : last;
    }
    break;
  }
  // ---------------------------------------------------------------- results
  if (rank == 0) {
    __syncthreads();
    for (int i = tid; i < a.nodes; i += kThreads)
      a.paths[b * a.nodes + i] = i < length ? vw.path[i] : -1;
    if (tid == 0) a.counts[b] = length;
  }
  if (teller && tid == 0) a.next[b] = next;
}

// -------------------------------------------------------------------- host
using namespace b200paged;

// Shared memory of a CTA, up to half an SM's.
constexpr int64_t kMostSmem = 100 * 1024;
int64_t fixed_bytes(int nodes) { return sizeof(Smem) + 4ll * kNodeArrays * nodes_padded(nodes); }
int64_t kept_bytes(int64_t share) { return 8 * kWarps * share; }

template <void (*kKernel)(Args)>
int32_t launch_cluster(const Args& a, unsigned ctas, int64_t batch, int device, cudaStream_t stream) {
  static std::once_flag once[kMaxDevices];
  static cudaError_t err[kMaxDevices];
  std::call_once(once[device], [&] {
    err[device] = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
    if (err[device] == cudaSuccess)
      err[device] = cudaFuncSetAttribute(kKernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  });
  if (err[device] != cudaSuccess) {
    set_error(cudaGetErrorString(err[device]));
    return B200_ATTN_ERR_LAUNCH;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas, static_cast<unsigned>(batch));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = fixed_bytes(a.nodes) + (a.keep ? kept_bytes(a.share) : 0);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kKernel, a);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error(cudaGetErrorString(e));
    return B200_ATTN_ERR_LAUNCH;
  }
  count_launch();
  return B200_ATTN_OK;
}
// Rows of four numbers can be read by one load.
bool by_fours(const void* base, const int64_t* stride, const int64_t* extent, int64_t eb) {
  if (reinterpret_cast<uintptr_t>(base) % (4 * eb)) return false;
  for (int d = 0; d < 2; ++d)
    if (extent[d] > 1 && stride[d] % 4) return false;
  return true;
}

template <int DT>
int32_t run(const Args& a, bool vec, unsigned ctas, int64_t batch, int device, cudaStream_t s) {
  return vec ? launch_cluster<verify_kernel<DT, true>>(a, ctas, batch, device, s)
             : launch_cluster<verify_kernel<DT, false>>(a, ctas, batch, device, s);
}

}  // namespace
}  // namespace b200verify

using namespace b200verify;

extern "C" int32_t b200_verify_check(const b200_verify_params* p) {
  using b200attn::may_overlap;
  using b200attn::stretches_of;
  if (!p || !p->logits || !p->tokens || !p->uniforms || !p->paths || !p->counts || !p->next ||
      p->reserved != 0 || (p->wide_tokens & ~1))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (p->batch < 1 || p->batch > 65535 || p->nodes < 1 || p->nodes > B200_VERIFY_MAX_NODES ||
      p->vocab < 1 || p->vocab > B200_VERIFY_MAX_VOCAB)
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (!(p->temperature >= 0.0) || !std::isfinite(p->temperature) ||
      (p->temperature > 0.0 && !std::isfinite(1.0 / p->temperature)))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (!known_dtype(p->dtype) || (p->draft_probs && !known_dtype(p->draft_dtype)))
    return B200_ATTN_ERR_UNSUPPORTED;
  const int64_t eb = elem_bytes(p->dtype), qb = elem_bytes(p->draft_dtype);
  const int64_t tb = p->wide_tokens ? 8 : 4;
  const int64_t extent[2] = {p->batch, p->nodes}, rows[2] = {p->batch, p->nodes - 1};
  for (int d = 0; d < 2; ++d)
    if ((extent[d] > 1 && p->logits_stride[d] < 0) ||
        (p->draft_probs && rows[d] > 1 && p->draft_stride[d] < 0))
      return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (p->batch > 1 && (p->token_stride < 0 || p->uniform_stride < 0 || p->parent_stride < 0))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(p->logits) % eb ||
      (p->draft_probs && reinterpret_cast<uintptr_t>(p->draft_probs) % qb) ||
      reinterpret_cast<uintptr_t>(p->tokens) % tb || (reinterpret_cast<uintptr_t>(p->next) & 7u) ||
      ((reinterpret_cast<uintptr_t>(p->uniforms) | reinterpret_cast<uintptr_t>(p->parents) |
        reinterpret_cast<uintptr_t>(p->draft_lens) | reinterpret_cast<uintptr_t>(p->paths) |
        reinterpret_cast<uintptr_t>(p->counts)) & 3u))
    return B200_ATTN_ERR_ALIGNMENT;
  // no output shares a byte with an input or another output
  const b200attn::Stretches outs[3] = {
      stretches_of(p->paths, nullptr, nullptr, 0, p->batch * p->nodes, 4),
      stretches_of(p->counts, nullptr, nullptr, 0, p->batch, 4),
      stretches_of(p->next, nullptr, nullptr, 0, p->batch, 8)};
  for (int i = 0; i < 3; ++i) {
    const auto& o = outs[i];
    for (int j = 0; j < i; ++j)
      if (may_overlap(o, outs[j])) return B200_ATTN_ERR_INVALID_ARGUMENT;
    if (may_overlap(o, stretches_of(p->logits, p->logits_stride, extent, 2, p->vocab, eb)) ||
        (p->draft_probs && p->nodes > 1 &&
         may_overlap(o, stretches_of(p->draft_probs, p->draft_stride, rows, 2, p->vocab, qb))) ||
        may_overlap(o, stretches_of(p->tokens, &p->token_stride, &p->batch, 1, p->nodes, tb)) ||
        may_overlap(o, stretches_of(p->uniforms, &p->uniform_stride, &p->batch, 1, p->nodes, 4)) ||
        (p->parents &&
         may_overlap(o, stretches_of(p->parents, &p->parent_stride, &p->batch, 1, p->nodes, 4))) ||
        (p->draft_lens && may_overlap(o, stretches_of(p->draft_lens, nullptr, nullptr, 0, p->batch, 4))))
      return B200_ATTN_ERR_INVALID_ARGUMENT;
  }
  return B200_ATTN_OK;
}

extern "C" int32_t b200_verify_drafts(const b200_verify_params* p, void* stream) {
  int32_t rc = b200_verify_check(p);
  if (rc != B200_ATTN_OK) return rc;
  b200paged::DeviceScope scope;
  if ((rc = scope.enter(p->logits, "logits are not device memory")) != B200_ATTN_OK) return rc;
  Args a{};
  if ((rc = b200attn::resolve_error_word(p->error_word, &a.err)) != B200_ATTN_OK) return rc;
  const int64_t eb = elem_bytes(p->dtype), qb = elem_bytes(p->draft_dtype);
  const int64_t extent[2] = {p->batch, p->nodes}, rows[2] = {p->batch, p->nodes - 1};
  a.logits = static_cast<const uint8_t*>(p->logits);
  a.l_seq = p->logits_stride[0] * eb;
  a.l_node = p->logits_stride[1] * eb;
  if (p->draft_probs && p->temperature > 0.0) {
    a.probs = static_cast<const uint8_t*>(p->draft_probs);
    a.q_seq = p->draft_stride[0] * qb;
    a.q_node = p->draft_stride[1] * qb;
    a.probs_type = p->draft_dtype;
    a.probs_vec = by_fours(p->draft_probs, p->draft_stride, rows, qb);
  }
  a.tokens = static_cast<const uint8_t*>(p->tokens);
  a.t_seq = p->token_stride;
  a.uniforms = p->uniforms;
  a.u_seq = p->uniform_stride;
  a.parents = p->parents;
  a.p_seq = p->parent_stride;
  a.lens = p->draft_lens;
  a.paths = p->paths;
  a.counts = p->counts;
  a.next = p->next;
  a.inv_temp = p->temperature > 0.0 ? 1.0 / p->temperature : 0.0;
  a.nodes = static_cast<int32_t>(p->nodes);
  a.vocab = static_cast<int32_t>(p->vocab);
  a.wide_tokens = p->wide_tokens;
  // So many CTAs that four of them, with a row's exponentials, fit on an SM up to a vocabulary of
  // about 110 thousand (three up to 149 thousand, two up to 200 thousand; past that each pass computes
  // them again).  Trees of 16 nodes with probabilities, us for 1 / 32 / 64 sequences; in brackets with
  // exponentials that are computed again:
  //   vocabulary    1 CTA             2               4               8               16
  //     4096    29 / 33 / 33   24 / 27 / 25    21 / 23 / 25    23 / 27 / 31    27 / 37 / 65
  //    16384                                   18 / 33 / 39    16 / 31 / 37    19 / 44 / 68
  //    53248                                   64 / 98 / 107   37 / 55 / 62    31 / 49 / 88
  //   100003                                   59 / 176 / 184  38 / 86 / 153   27 / 76 / 131
  //                                                           [39 / 111 / 125 27 / 93 / 148]
  //   128256                                   64 / 215 / 285  39 / 129 / 173  27 / 94 / 186
  //                                                                           [27 / 96 / 173]
  //   151936                                   76 / 268 / 321  45 / 152 / 185  33 / 133 / 255
  //                                                                           [33 / 124 / 213]
  // By the vocabulary alone: a row of 4096 numbers would be faster with 2 CTAs, and 64 sequences of
  // wide ones with 8, where one sequence would take a third more.
  const unsigned ctas = p->vocab > 53248 ? 16 : (p->vocab > 16384 ? 8 : (p->vocab > 4096 ? 4 : 1));
  const int64_t warps = static_cast<int64_t>(ctas) * kWarps;
  a.share = static_cast<int32_t>((p->vocab + 4 * warps - 1) / (4 * warps) * 4);
  a.keep = a.inv_temp != 0.0 && fixed_bytes(a.nodes) + kept_bytes(a.share) <= kMostSmem;
  const bool vec = by_fours(p->logits, p->logits_stride, extent, eb);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (p->dtype) {
    case B200_ATTN_DTYPE_BF16: return run<B200_ATTN_DTYPE_BF16>(a, vec, ctas, p->batch, scope.device, s);
    case B200_ATTN_DTYPE_FP16: return run<B200_ATTN_DTYPE_FP16>(a, vec, ctas, p->batch, scope.device, s);
    default: return run<B200_ATTN_DTYPE_FP32>(a, vec, ctas, p->batch, scope.device, s);
  }
}
