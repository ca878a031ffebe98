// cache4.cu — append to and read from the paged cache held in 4 bits
// (format: b200_cache4.h).
//
// A thread takes 8 numbers of a key row and the same 8 of the value row; the 2 or 4 threads
// of a group find its smallest and largest number by shuffles.  Bound by HBM for
// large calls: a vector of D numbers is read once and D / 2 + 16 bytes are written.
#include <cuda_runtime.h>

#include <cstdint>

#include "b200_cache4.h"
#include "byte_range.h"
#include "error_word.cuh"
#include "paged_host.h"
#include "sm100_ptx.cuh"
#include "tree_attn.cuh"

namespace b200cache4 {

using b200attn::report_error;
using b200tree::Elem;

namespace {

constexpr int kThreads = 256;

struct Call {
  uint8_t* k;  // pools
  uint8_t* v;
  int64_t k_layer, k_page, k_head, k_row;  // bytes
  int64_t v_layer, v_page, v_head, v_row;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  uint8_t* kx;  // vectors
  uint8_t* vx;
  int64_t kx_layer, kx_seq, kx_head, kx_tok;  // bytes
  int64_t vx_layer, vx_seq, vx_head, vx_tok;
  const int32_t* counts;
  int32_t batch, slots, pages, page_size, heads, tokens, head_dim;
  int32_t* err;
};

// The thread's vector: sequence, token, head and eighth-of-numbers `x` of it.
struct Place {
  int b, j, h, x;
};

template <int P>
__device__ __forceinline__ bool place_of(const Call& c, Place* p) {
  constexpr uint32_t kParts = P / 8;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const uint32_t per_tok = c.heads * kParts;
  const int64_t per_seq = static_cast<int64_t>(c.tokens) * per_tok;
  p->b = static_cast<int>(idx / per_seq);
  const uint32_t rest = static_cast<uint32_t>(idx - p->b * per_seq);
  p->j = static_cast<int>(rest / per_tok);
  const uint32_t in = rest - p->j * per_tok;
  p->h = static_cast<int>(in / kParts);
  p->x = static_cast<int>(in % kParts);
  return p->b < c.batch;
}

// The page and row of token lens[b] + j; false where there is none (reported).
__device__ __forceinline__ bool find_row(const Call& c, int b, int j, int* page, uint32_t* row) {
  const int len = c.lens[b];
  const uint32_t at = static_cast<uint32_t>(len) + j, slot = at / static_cast<uint32_t>(c.page_size);
  int p = -1;
  if (len >= 0 && slot < static_cast<uint32_t>(c.slots)) p = c.table[b * c.table_stride + slot];
  if (p < 0 || p >= c.pages) {
    report_error(c.err, B200_ATTN_DEVERR_BOUNDS);
    return false;
  }
  *page = p;
  *row = at - slot * c.page_size;
  return true;
}

template <int DT>
__device__ __forceinline__ void load8(const uint8_t* src, float (&x)[8]) {
  using E = Elem<DT>;
  union {
    uint4 w[E::kBytes / 2];
    typename E::T e[8];
  } u;
#pragma unroll
  for (int i = 0; i < E::kBytes / 2; ++i) u.w[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = E::widen(u.e[i]);
}

// The bf16 number at or below x.
__device__ __forceinline__ float bf16_down(float x) {
  const uint32_t u = __float_as_uint(x), cut = u & 0xffff0000u;
  return __uint_as_float((u & 0x80000000u) && (u & 0xffffu) ? cut + 0x10000u : cut);
}

// a - b as a rounded difference and what the rounding left off (Knuth's two-sum).
__device__ __forceinline__ float2 difference(float a, float b) {
  const float d = a - b, x = a - d;
  return make_float2(d, (x - b) + (a - (d + x)));
}

// The bf16 number at or above a fifteenth of span.x + span.y >= 0.  The quotient is rounded, so its
// neighbours are looked at too: 15 times a bf16 number is exact.
__device__ __forceinline__ float step_of(float2 span) {
  auto enough = [&](uint32_t bits) {
    const float c = 15.f * __uint_as_float(bits);
    return c > span.x || (c == span.x && span.y <= 0.f);
  };
  if (span.x == 0.f) return 0.f;
  if (!(span.x < INFINITY)) return INFINITY;
  uint32_t u = __float_as_uint(span.x / 15.f) & 0xffff0000u;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (!enough(u)) u += 0x10000u;
  return __uint_as_float(u);
}

struct Coded {
  uint32_t code[8];
  float step, low;
};

// The codes of the thread's 8 numbers and its group's step and low.  `there`: the numbers
// lie inside the vector.  By whole warps.
template <int P>
__device__ __forceinline__ Coded encode(const float (&x)[8], bool there) {
  constexpr int kLanes = P / 32;  // of a group
  Coded r;
  float lo = INFINITY, hi = -INFINITY;
  if (there) {
    float odd = 0.f;  // NaN where a number is not finite
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
      odd = fmaf(x[i], 0.f, odd);
    }
    if (odd != 0.f) lo = -INFINITY;
  }
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (lo == INFINITY) lo = hi = 0.f;  // a group past the vector
  r.low = bf16_down(lo);
  r.step = step_of(difference(hi, r.low));
  if (r.step > 0.f && r.step < 0x1p-100f) r.step = 0x1p-100f;
  const bool fine = isfinite(r.low) && isfinite(r.step);
  const float inv = fine && r.step > 0.f ? 1.f / r.step : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // x - low = d.x + d.y; what is left of d.x after t steps is exact, so the code is the
    // nearest one, with ties to even
    const float2 d = there && fine ? difference(x[i], r.low) : make_float2(0.f, 0.f);
    int t = __float2int_rn(d.x * inv);
    const float left = 2.f * fmaf(-static_cast<float>(t), r.step, d.x);
    const bool tie_up = d.y > 0.f || (d.y == 0.f && (t & 1));
    const bool tie_down = d.y < 0.f || (d.y == 0.f && (t & 1));
    if (left > r.step || (left == r.step && tie_up)) ++t;
    else if (left < -r.step || (left == -r.step && tie_down)) --t;
    r.code[i] = static_cast<uint32_t>(max(0, min(15, t)));
  }
  if (!fine) r.step = r.low = __uint_as_float(0x7fc00000u);
  return r;
}

// Part x (8 numbers) of a row of codes, as keys or values lie: see the header.
template <int P>
__device__ __forceinline__ void put_key_codes(uint8_t* row, int x, const uint32_t (&c)[8]) {
  if constexpr (P == 128) {
    uint32_t w = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= c[i] << (4 * (2 * (i / 4) + i % 4 / 2 + 4 * (i % 2)));
    *reinterpret_cast<uint32_t*>(row + 16 * (x % 4) + 4 * (x / 4)) = w;
  } else {
    const int g = x / 2;
#pragma unroll
    for (int y = 0; y < 8; y += 4) {
      uint8_t* at = row + 8 * (2 * (x % 2) + y / 4) + 4 * (g / 2) + g % 2;
      at[0] = static_cast<uint8_t>(c[y] | c[y + 2] << 4);
      at[2] = static_cast<uint8_t>(c[y + 1] | c[y + 3] << 4);
    }
  }
}
template <int P>
__device__ __forceinline__ void put_value_codes(uint8_t* row, int x, const uint32_t (&c)[8]) {
  if constexpr (P == 128) {
#pragma unroll
    for (int y = 0; y < 8; y += 4)
      *reinterpret_cast<uint16_t*>(row + 8 * (2 * (x % 4) + y / 4) + 2 * (x / 4)) =
          static_cast<uint16_t>(c[y] | c[y + 1] << 4 | c[y + 2] << 8 | c[y + 3] << 12);
  } else {
#pragma unroll
    for (int y = 0; y < 8; y += 2)
      row[4 * (4 * (x % 2) + y / 2) + x / 2] = static_cast<uint8_t>(c[y] | c[y + 1] << 4);
  }
}
template <int P>
__device__ __forceinline__ void get_key_codes(const uint8_t* row, int x, uint32_t (&c)[8]) {
  if constexpr (P == 128) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(row + 16 * (x % 4) + 4 * (x / 4));
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = w >> (4 * (2 * (i / 4) + i % 4 / 2 + 4 * (i % 2))) & 15u;
  } else {
    const int g = x / 2;
#pragma unroll
    for (int y = 0; y < 8; y += 4) {
      const uint8_t* at = row + 8 * (2 * (x % 2) + y / 4) + 4 * (g / 2) + g % 2;
      c[y] = at[0] & 15u;
      c[y + 2] = at[0] >> 4;
      c[y + 1] = at[2] & 15u;
      c[y + 3] = at[2] >> 4;
    }
  }
}
template <int P>
__device__ __forceinline__ void get_value_codes(const uint8_t* row, int x, uint32_t (&c)[8]) {
  if constexpr (P == 128) {
#pragma unroll
    for (int y = 0; y < 8; y += 4) {
      const uint32_t w =
          *reinterpret_cast<const uint16_t*>(row + 8 * (2 * (x % 4) + y / 4) + 2 * (x / 4));
#pragma unroll
      for (int i = 0; i < 4; ++i) c[y + i] = w >> (4 * i) & 15u;
    }
  } else {
#pragma unroll
    for (int y = 0; y < 8; y += 2) {
      const uint32_t w = row[4 * (4 * (x % 2) + y / 2) + x / 2];
      c[y] = w & 15u;
      c[y + 1] = w >> 4;
    }
  }
}

__device__ __forceinline__ uint16_t bf16_bits(float x) {
  return static_cast<uint16_t>(__float_as_uint(x) >> 16);
}
__device__ __forceinline__ float of_bf16(uint16_t x) {
  return __uint_as_float(static_cast<uint32_t>(x) << 16);
}

template <int P, int DT>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ Call c) {
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  Place p;
  bool mine = place_of<P>(c, &p);
  int page = 0;
  uint32_t row = 0;
  if (mine) {
    const int count = c.counts ? c.counts[p.b] : c.tokens;
    if (count < 0 || count > c.tokens) {
      report_error(c.err, B200_ATTN_DEVERR_BOUNDS);
      mine = false;
    }
    mine = mine && p.j < count && find_row(c, p.b, p.j, &page, &row);
  }
  const bool there = mine && 8 * p.x < c.head_dim;
  const int64_t l = blockIdx.y;
  float k[8], v[8];
  if (there) {
    const int at = 8 * Elem<DT>::kBytes * p.x;
    load8<DT>(c.kx + l * c.kx_layer + p.b * c.kx_seq + p.h * c.kx_head + p.j * c.kx_tok + at, k);
    load8<DT>(c.vx + l * c.vx_layer + p.b * c.vx_seq + p.h * c.vx_head + p.j * c.vx_tok + at, v);
  }
  const Coded kc = encode<P>(k, there), vc = encode<P>(v, there);
  if (!mine) return;
  uint8_t* kr = c.k + l * c.k_layer + page * c.k_page + p.h * c.k_head + row * c.k_row;
  uint8_t* vr = c.v + l * c.v_layer + page * c.v_page + p.h * c.v_head + row * c.v_row;
  put_key_codes<P>(kr, p.x, kc.code);
  put_value_codes<P>(vr, p.x, vc.code);
  if (p.x % (P / 32) == 0) {
    const int g = p.x / (P / 32);
    uint16_t* km = reinterpret_cast<uint16_t*>(kr + P / 2) + g;
    uint16_t* vm = reinterpret_cast<uint16_t*>(vr + P / 2) + g;
    km[0] = bf16_bits(kc.step);
    km[4] = bf16_bits(kc.low);
    vm[0] = bf16_bits(vc.step);
    vm[4] = bf16_bits(vc.low);
  }
}

template <int DT>
__device__ __forceinline__ void store8(uint8_t* dst, const float (&x)[8]) {
  using E = Elem<DT>;
  union {
    uint4 w[E::kBytes / 2];
    typename E::T e[8];
  } u;
#pragma unroll
  for (int i = 0; i < 8; ++i) u.e[i] = E::round(x[i]);
#pragma unroll
  for (int i = 0; i < E::kBytes / 2; ++i) reinterpret_cast<uint4*>(dst)[i] = u.w[i];
}

template <int P, int DT>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ Call c) {
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  Place p;
  if (!place_of<P>(c, &p) || 8 * p.x >= c.head_dim) return;
  const int count = c.counts ? c.counts[p.b] : c.tokens;
  if (count < 0 || count > c.tokens) report_error(c.err, B200_ATTN_DEVERR_BOUNDS);
  const int64_t l = blockIdx.y;
  float k[8], v[8];
  int page;
  uint32_t row;
  if (count <= c.tokens && p.j < count && find_row(c, p.b, p.j, &page, &row)) {
    const uint8_t* kr = c.k + l * c.k_layer + page * c.k_page + p.h * c.k_head + row * c.k_row;
    const uint8_t* vr = c.v + l * c.v_layer + page * c.v_page + p.h * c.v_head + row * c.v_row;
    const int g = p.x / (P / 32);
    const uint16_t* km = reinterpret_cast<const uint16_t*>(kr + P / 2) + g;
    const uint16_t* vm = reinterpret_cast<const uint16_t*>(vr + P / 2) + g;
    uint32_t kc[8], vc[8];
    get_key_codes<P>(kr, p.x, kc);
    get_value_codes<P>(vr, p.x, vc);
    const float ks = of_bf16(km[0]), kl = of_bf16(km[4]), vs = of_bf16(vm[0]), vl = of_bf16(vm[4]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      k[i] = fmaf(ks, static_cast<float>(kc[i]), kl);
      v[i] = fmaf(vs, static_cast<float>(vc[i]), vl);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = v[i] = 0.f;
  }
  const int at = 8 * Elem<DT>::kBytes * p.x;
  store8<DT>(c.kx + l * c.kx_layer + p.b * c.kx_seq + p.h * c.kx_head + p.j * c.kx_tok + at, k);
  store8<DT>(c.vx + l * c.vx_layer + p.b * c.vx_seq + p.h * c.vx_head + p.j * c.vx_tok + at, v);
}

// -------------------------------------------------------------------- host
using namespace b200paged;
using b200attn::may_overlap;
using b200attn::stretches_of;

// Checks both entry points' arguments and fills the call; `out`: the vectors are written.
int32_t fill(const b200_cache* c, int64_t head_dim, int32_t dtype, const b200_cache_rows* rows,
             bool out, Call* a, int64_t* threads) {
  const int32_t rc = b200_cache_check(c);
  if (rc != B200_ATTN_OK) return rc;
  const int32_t bytes = b200_cache4_row_bytes(head_dim);
  if (bytes == 0 || !known_dtype(dtype)) return B200_ATTN_ERR_UNSUPPORTED;
  if (c->dtype != B200_ATTN_DTYPE_BF16 || 2 * c->head_dim != bytes || !c->seq_lens || !rows ||
      !rows->k || !rows->v || rows->tokens < 1)
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  const int64_t eb = elem_bytes(dtype);
  const int64_t extent[4] = {c->layers, c->batch, c->kv_heads, rows->tokens};
  if (!vectors_aligned(rows->k, rows->k_stride, extent, 4, eb) ||
      !vectors_aligned(rows->v, rows->v_stride, extent, 4, eb) ||
      (reinterpret_cast<uintptr_t>(rows->counts) & 3u))
    return B200_ATTN_ERR_ALIGNMENT;
  const int64_t parts = (head_dim <= 64 ? 64 : 128) / 8;
  if (rows->tokens > 0x3fffffff || rows->tokens * c->kv_heads * parts > 0x7fffffffll ||
      c->batch * rows->tokens * c->kv_heads * parts > (1ll << 38))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  *threads = c->batch * rows->tokens * c->kv_heads * parts;
  // what is written shares no byte with what is read, nor with itself
  const int64_t pool[4] = {c->layers, c->pages, c->kv_heads, c->page_size};
  const auto kp = stretches_of(c->k, c->k_stride, pool, 4, c->head_dim, 2);
  const auto vp = stretches_of(c->v, c->v_stride, pool, 4, c->head_dim, 2);
  const auto kx = stretches_of(rows->k, rows->k_stride, extent, 4, head_dim, eb);
  const auto vx = stretches_of(rows->v, rows->v_stride, extent, 4, head_dim, eb);
  if (may_overlap(kx, kp) || may_overlap(kx, vp) || may_overlap(vx, kp) || may_overlap(vx, vp))
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  if (out) {
    if (may_overlap(kx, vx)) return B200_ATTN_ERR_INVALID_ARGUMENT;
    for (int d = 0; d < 4; ++d)
      if (extent[d] > 1 && (rows->k_stride[d] == 0 || rows->v_stride[d] == 0))
        return B200_ATTN_ERR_INVALID_ARGUMENT;
    for (const auto& o : {kx, vx})
      if (may_overlap(o, stretches_of(c->page_table, &c->table_stride, &c->batch, 1, c->slots, 4)) ||
          may_overlap(o, stretches_of(c->seq_lens, nullptr, nullptr, 0, c->batch, 4)) ||
          (rows->counts && may_overlap(o, stretches_of(rows->counts, nullptr, nullptr, 0, c->batch, 4))))
        return B200_ATTN_ERR_INVALID_ARGUMENT;
  }
  a->k = static_cast<uint8_t*>(c->k);
  a->v = static_cast<uint8_t*>(c->v);
  a->k_layer = 2 * c->k_stride[0];
  a->k_page = 2 * c->k_stride[1];
  a->k_head = 2 * c->k_stride[2];
  a->k_row = 2 * c->k_stride[3];
  a->v_layer = 2 * c->v_stride[0];
  a->v_page = 2 * c->v_stride[1];
  a->v_head = 2 * c->v_stride[2];
  a->v_row = 2 * c->v_stride[3];
  a->table = c->page_table;
  a->table_stride = c->table_stride;
  a->lens = c->seq_lens;
  a->kx = static_cast<uint8_t*>(const_cast<void*>(rows->k));
  a->vx = static_cast<uint8_t*>(const_cast<void*>(rows->v));
  a->kx_layer = eb * rows->k_stride[0];
  a->kx_seq = eb * rows->k_stride[1];
  a->kx_head = eb * rows->k_stride[2];
  a->kx_tok = eb * rows->k_stride[3];
  a->vx_layer = eb * rows->v_stride[0];
  a->vx_seq = eb * rows->v_stride[1];
  a->vx_head = eb * rows->v_stride[2];
  a->vx_tok = eb * rows->v_stride[3];
  a->counts = rows->counts;
  a->batch = static_cast<int32_t>(c->batch);
  a->slots = static_cast<int32_t>(c->slots);
  a->pages = static_cast<int32_t>(c->pages);
  a->page_size = static_cast<int32_t>(c->page_size);
  a->heads = static_cast<int32_t>(c->kv_heads);
  a->tokens = static_cast<int32_t>(rows->tokens);
  a->head_dim = static_cast<int32_t>(head_dim);
  return B200_ATTN_OK;
}

template <int P, int DT>
int32_t run(bool out, const Call& a, dim3 grid, cudaStream_t s) {
  return launch(out ? read_kernel<P, DT> : append_kernel<P, DT>, grid, dim3(kThreads), 0, s, a);
}

int32_t run_call(const b200_cache* c, int64_t head_dim, int32_t dtype, const b200_cache_rows* rows,
                 bool out, void* stream) {
  Call a{};
  int64_t threads = 0;
  int32_t rc = fill(c, head_dim, dtype, rows, out, &a, &threads);
  if (rc != B200_ATTN_OK) return rc;
  DeviceScope scope;
  if ((rc = scope.enter(c->k, "the pools are not device memory")) != B200_ATTN_OK) return rc;
  if ((rc = resolve_error_word(c->error_word, &a.err)) != B200_ATTN_OK) return rc;
  const dim3 grid(static_cast<unsigned>((threads + kThreads - 1) / kThreads),
                  static_cast<unsigned>(c->layers));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = head_dim > 64;
  switch (dtype) {
    case B200_ATTN_DTYPE_BF16:
      return wide ? run<128, B200_ATTN_DTYPE_BF16>(out, a, grid, s)
                  : run<64, B200_ATTN_DTYPE_BF16>(out, a, grid, s);
    case B200_ATTN_DTYPE_FP16:
      return wide ? run<128, B200_ATTN_DTYPE_FP16>(out, a, grid, s)
                  : run<64, B200_ATTN_DTYPE_FP16>(out, a, grid, s);
    default:
      return wide ? run<128, B200_ATTN_DTYPE_FP32>(out, a, grid, s)
                  : run<64, B200_ATTN_DTYPE_FP32>(out, a, grid, s);
  }
}

}  // namespace
}  // namespace b200cache4

extern "C" int32_t b200_cache4_row_bytes(int64_t head_dim) {
  if (head_dim < 8 || head_dim > 128 || head_dim % 8) return 0;
  return head_dim <= 64 ? 48 : 80;
}

extern "C" int32_t b200_cache4_append(const b200_cache* c, int64_t head_dim, int32_t dtype,
                                      const b200_cache_rows* rows, void* stream) {
  return b200cache4::run_call(c, head_dim, dtype, rows, false, stream);
}

extern "C" int32_t b200_cache4_read(const b200_cache* c, int64_t head_dim, int32_t dtype,
                                    const b200_cache_rows* rows, void* stream) {
  return b200cache4::run_call(c, head_dim, dtype, rows, true, stream);
}
