// cache4.cu — append to and read from the paged cache held in 4 bits
// (format: b200_cache4.h).
//
// append: a thread takes a group of a key or value vector, 16 or 32 numbers, so what is done once a
// group (its ends, step and low) is shared by many numbers; the four threads of a vector exchange
// words to write rows 8 or 16 bytes at a time.  read: a thread takes 8 numbers of a key and the same
// 8 of the value.
//
// Bound by the issue of instructions.  16 prompts of up to 2048 tokens, 16 thousand in all, of 8 heads of
// 128 bf16 numbers, keys and values: append 42 us, where its bytes take 13 at the copy rate, with 34
// instructions a number and 76 % of the issue slots used; read, which writes the rows behind the
// counts too, 34 us, bytes 24, 12 instructions a number and 74 %.  A lane of append
// reads 64 bytes that lie together, so each 32-byte sector is asked for twice, the second time from
// L1.  A thread for 8 numbers, whose group's ends went through shuffles, and every code settled
// exactly: 177 us for both.  A thread a vector (append 80 us) kept 128 numbers in registers, a
// warp a vector spent most of its time in shuffles.
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
constexpr int kParts = 8;  // threads of a token's key and value of a head

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
  uint32_t inv_tok, inv_size;  // for divisions by the threads of a token and by the page size
  int32_t* err;
};

// x / d with inv = 2^32 / d rounded up (0 for d = 1): the product is the quotient or one more.
__host__ __device__ inline uint32_t inverse_of(uint32_t d) { return 0xffffffffu / d + 1u; }
__device__ __forceinline__ uint32_t divided(uint32_t x, uint32_t d, uint32_t inv) {
  if (d == 1u) return x;
  const uint32_t q = __umulhi(x, inv);
  return q * d > x ? q - 1u : q;
}

// The thread's group: token, head, keys or values, group.  blockIdx: threads of a sequence, layers,
// sequences.  The threads of a vector are lanes 4 n to 4 n + 3 of a warp.
struct Place {
  int j, h, g;
  bool value;
};

__device__ __forceinline__ bool place_of(const Call& c, Place* p) {
  const uint32_t idx = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t per_tok = c.heads * kParts;
  const uint32_t j = divided(idx, per_tok, c.inv_tok), in = idx - j * per_tok;
  p->j = static_cast<int>(j);
  p->h = static_cast<int>(in / kParts);
  p->value = in % kParts >= 4;
  p->g = static_cast<int>(in % 4);
  return j < static_cast<uint32_t>(c.tokens);
}

// The page and row of token lens[b] + j; false where there is none (reported).
__device__ __forceinline__ bool find_row(const Call& c, int b, int j, int* page, uint32_t* row) {
  const int len = c.lens[b];
  const uint32_t at = static_cast<uint32_t>(len) + j, slot = divided(at, c.page_size, c.inv_size);
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
__device__ __forceinline__ void load8(const uint8_t* src, float* x) {
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

// The bf16 number at or above a fifteenth of span.x + span.y >= 0; infinity where the span passes fp32.
// The quotient is rounded, so its neighbours are looked at too: 15 times a bf16 number is exact.
__device__ __forceinline__ float step_of(float2 span) {
  auto enough = [&](uint32_t bits) {
    const float c = 15.f * __uint_as_float(bits);
    return c > span.x || (c == span.x && span.y <= 0.f);
  };
  if (span.x == 0.f) return 0.f;
  if (!(span.x < INFINITY)) return INFINITY;
  uint32_t u = __float_as_uint(span.x * (1.f / 15.f)) & 0xffff0000u;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (!enough(u)) u += 0x10000u;
  return __uint_as_float(u);
}

// The nearest whole number to (x - low) / step, ties to even, where `code` is it but for a rounding
// of the quotient: x - low = d.x + d.y, and what is left of d.x after `code` steps is exact.
__device__ __forceinline__ float settled(float x, float step, float low, float code) {
  const float2 d = difference(x, low);
  const float left = 2.f * fmaf(-code, step, d.x);
  const bool odd = static_cast<int>(code) & 1;
  const bool tie_up = d.y > 0.f || (d.y == 0.f && odd), tie_down = d.y < 0.f || (d.y == 0.f && odd);
  if (left > step || (left == step && tie_up)) code += 1.f;
  else if (left < -step || (left == -step && tie_down)) code -= 1.f;
  return fmaxf(0.f, fminf(15.f, code));
}

// Codes in place of the group's first n numbers (a multiple of 8; 0 for the others), its step and its
// low.
template <int G>
__device__ __forceinline__ float2 encode(float (&x)[G], int n) {
  float lo = INFINITY, hi = -INFINITY, odd = 0.f;  // NaN where a number is not finite
#pragma unroll
  for (int i = 0; i < G; ++i) {
    if (i < n) {
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
      odd = fmaf(x[i], 0.f, odd);
    }
  }
  if (odd != 0.f) lo = -INFINITY;
  if (n <= 0) lo = hi = 0.f;
  float low = bf16_down(lo), step = step_of(difference(hi, low));
  if (step > 0.f && step < 0x1p-100f) step = 0x1p-100f;
  if (!(isfinite(low) && isfinite(step))) {
    step = low = __uint_as_float(0x7fc00000u);
    n = 0;
  }
  if (!(step > 0.f)) n = 0;
  constexpr float kRound = 12582912.f;  // 1.5 2^23
  const float inv = __frcp_rn(step);
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const float f = (x[i] - low) * inv;
    float code = (f + kRound) - kRound;
    // next to a border the quotient's rounding could decide
    if (i < n && fabsf(f - code) > 0.5f - 0x1p-14f) code = settled(x[i], step, low, code);
    x[i] = i < n ? code : 0.f;
  }
  return make_float2(step, low);
}

// a + 16 b + 256 c + 4096 d of codes, as a whole number.
__device__ __forceinline__ uint32_t four(float a, float b, float c, float d) {
  const float v = fmaf(fmaf(fmaf(d, 16.f, c), 16.f, b), 16.f, a);
  return __float_as_uint(v + 8388608.f) & 0xffffu;
}
__device__ __forceinline__ uint32_t two(float a, float b) {
  return __float_as_uint(fmaf(b, 16.f, a) + 8388608.f) & 0xffu;
}

// The 4 x 4 words of four lanes, transposed: word i of lane k becomes word k of lane i.  By whole
// warps.
__device__ __forceinline__ void transpose(uint32_t (&w)[4]) {
  const bool one = threadIdx.x & 1, two = threadIdx.x & 2;
  uint32_t a = __shfl_xor_sync(0xffffffffu, one ? w[0] : w[1], 1);
  uint32_t b = __shfl_xor_sync(0xffffffffu, one ? w[2] : w[3], 1);
  if (one) w[0] = a, w[2] = b;
  else w[1] = a, w[3] = b;
  a = __shfl_xor_sync(0xffffffffu, two ? w[0] : w[2], 2);
  b = __shfl_xor_sync(0xffffffffu, two ? w[1] : w[3], 2);
  if (two) w[0] = a, w[1] = b;
  else w[2] = a, w[3] = b;
}

// The codes of group g of a row, as keys or values lie (see the header): lane g of the row's four
// writes quarter g of the row's codes.  By whole warps; `mine`: there is a row.
template <int P>
__device__ __forceinline__ void put_codes(uint8_t* row, int g, bool value, const float (&c)[P / 4],
                                          bool mine) {
  uint32_t w[4];
  if constexpr (P == 128) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* x = c + 8 * i;
      w[i] = value ? four(x[0], x[1], x[2], x[3]) | four(x[4], x[5], x[6], x[7]) << 16
                   : four(x[0], x[2], x[4], x[6]) | four(x[1], x[3], x[5], x[7]) << 16;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* x = c + 4 * i;
      w[i] = value ? two(x[0], x[1]) | two(x[2], x[3]) << 8
                   : (two(x[0], x[2]) | two(x[1], x[3]) << 16) << (8 * (g % 2));
    }
  }
  transpose(w);
  if (!mine) return;
  if constexpr (P == 128) {
    uint4 o = make_uint4(w[0], w[1], w[2], w[3]);
    if (value)
      o = make_uint4(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410),
                     __byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632));
    reinterpret_cast<uint4*>(row)[g] = o;
  } else {
    uint2 o = make_uint2(w[0] | w[1], w[2] | w[3]);
    if (value) {
      const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);
      o = make_uint2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
    }
    reinterpret_cast<uint2*>(row)[g] = o;
  }
}

__device__ __forceinline__ uint16_t bf16_bits(float x) {
  return static_cast<uint16_t>(__float_as_uint(x) >> 16);
}
__device__ __forceinline__ float of_bf16(uint16_t x) {
  return __uint_as_float(static_cast<uint32_t>(x) << 16);
}

// Rows in and out of a thread's pool and vectors.
struct Sides {
  uint8_t* row;  // of the pool
  uint8_t* x;    // the group's first number in the vector
};
template <int P, int DT>
__device__ __forceinline__ Sides sides_of(const Call& c, const Place& p, int page, uint32_t row) {
  const int64_t b = blockIdx.z, l = blockIdx.y;
  const int at = P / 4 * Elem<DT>::kBytes * p.g;
  return p.value ? Sides{c.v + l * c.v_layer + page * c.v_page + p.h * c.v_head + row * c.v_row,
                         c.vx + l * c.vx_layer + b * c.vx_seq + p.h * c.vx_head + p.j * c.vx_tok + at}
                 : Sides{c.k + l * c.k_layer + page * c.k_page + p.h * c.k_head + row * c.k_row,
                         c.kx + l * c.kx_layer + b * c.kx_seq + p.h * c.kx_head + p.j * c.kx_tok + at};
}

template <int P, int DT>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ Call c) {
  constexpr int G = P / 4;
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  Place p;
  bool mine = place_of(c, &p);
  int page = 0;
  uint32_t row = 0;
  if (mine) {
    const int count = c.counts ? c.counts[blockIdx.z] : c.tokens;
    if (count < 0 || count > c.tokens) {
      report_error(c.err, B200_ATTN_DEVERR_BOUNDS);
      mine = false;
    }
    mine = mine && p.j < count && find_row(c, blockIdx.z, p.j, &page, &row);
  }
  if (!__any_sync(0xffffffffu, mine)) return;
  const Sides to = sides_of<P, DT>(c, p, page, row);
  const int n = mine ? min(G, c.head_dim - G * p.g) : 0;
  float x[G];
#pragma unroll
  for (int i = 0; i < G; i += 8) {
    if (i < n) {
      load8<DT>(to.x + i * Elem<DT>::kBytes, x + i);
    } else {
#pragma unroll
      for (int y = 0; y < 8; ++y) x[i + y] = 0.f;
    }
  }
  const float2 meta = encode(x, n);
  put_codes<P>(to.row, p.g, p.value, x, mine);
  if (!mine) return;
  uint16_t* m = reinterpret_cast<uint16_t*>(to.row + P / 2) + p.g;
  m[0] = bf16_bits(meta.x);
  m[4] = bf16_bits(meta.y);
}

template <int DT>
__device__ __forceinline__ void store8(uint8_t* dst, const float* x) {
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

// Part x (8 numbers) of a row's codes.
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

// Whether low + step code, rounded to fp32, can lie halfway between two numbers of a 16-bit type
// without being there.  With the exponents l and s of two numbers of 8 bits and code < 16 the sum is a
// multiple of 2^(min(s, l) - 7) below 2^(max(s + 6, l + 2)): exact in fp32 for -11 <= l - s <= 15.  Past
// that step code is less than half a step of the type from low, which of bf16 and of normal fp16
// numbers is one itself.
template <int DT>
__device__ __forceinline__ bool may_round(float step, float low) {
  if constexpr (DT == B200_ATTN_DTYPE_FP32) return false;
  const float near = step * 0x1p-11f;
  return fabsf(low) < (DT == B200_ATTN_DTYPE_FP16 ? fmaxf(near, 0x1p-14f) : near);
}

// Writes a thread's numbers where that is so, each rounded once: the sum becomes, where it is not an
// fp32 number, the neighbour whose last bit is 1, which is never halfway between two of the 16-bit
// type, so the second rounding is that of the sum.
template <int P, int DT>
__device__ __noinline__ void store_sums(const uint8_t* kr, const uint8_t* vr, int x, uint8_t* kd,
                                        uint8_t* vd) {
  const int g = x / (P / 32);
  uint32_t codes[2][8];
  get_key_codes<P>(kr, x, codes[0]);
  get_value_codes<P>(vr, x, codes[1]);
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint16_t* m = reinterpret_cast<const uint16_t*>((s ? vr : kr) + P / 2) + g;
    const float step = of_bf16(m[0]), low = of_bf16(m[4]);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float code = static_cast<float>(codes[s][i]);
      const float below = __fmaf_rd(step, code, low), above = __fmaf_ru(step, code, low);
      y[i] = __float_as_uint(below) & 1u ? below : above;
    }
    store8<DT>(s ? vd : kd, y);
  }
}

// A thread gives 8 numbers of a key and the same 8 of the value, so that neighbours write side by
// side (a group a thread as above: 46 us against 34 us for 33 thousand rows of 8 heads).
template <int P, int DT>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ Call c) {
  b200attn::ptx::launch_dependents();
  b200attn::ptx::grid_dependency_wait();
  const uint32_t idx = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t per_tok = c.heads * (P / 8);
  const uint32_t tok = divided(idx, per_tok, c.inv_tok), in = idx - tok * per_tok;
  const int j = static_cast<int>(tok), h = static_cast<int>(in / (P / 8)), x = static_cast<int>(in % (P / 8));
  if (j >= c.tokens || 8 * x >= c.head_dim) return;
  const int64_t b = blockIdx.z, l = blockIdx.y;
  const int count = c.counts ? c.counts[b] : c.tokens;
  if (count < 0 || count > c.tokens) report_error(c.err, B200_ATTN_DEVERR_BOUNDS);
  const int at = 8 * Elem<DT>::kBytes * x;
  uint8_t* kd = c.kx + l * c.kx_layer + b * c.kx_seq + h * c.kx_head + j * c.kx_tok + at;
  uint8_t* vd = c.vx + l * c.vx_layer + b * c.vx_seq + h * c.vx_head + j * c.vx_tok + at;
  const uint8_t *kr = nullptr, *vr = nullptr;
  float k[8], v[8];
  bool again = false;
  int page;
  uint32_t row;
  if (count <= c.tokens && j < count && find_row(c, b, j, &page, &row)) {
    kr = c.k + l * c.k_layer + page * c.k_page + h * c.k_head + row * c.k_row;
    vr = c.v + l * c.v_layer + page * c.v_page + h * c.v_head + row * c.v_row;
    const int g = x / (P / 32);
    const uint16_t* km = reinterpret_cast<const uint16_t*>(kr + P / 2) + g;
    const uint16_t* vm = reinterpret_cast<const uint16_t*>(vr + P / 2) + g;
    uint32_t kc[8], vc[8];
    get_key_codes<P>(kr, x, kc);
    get_value_codes<P>(vr, x, vc);
    const float ks = of_bf16(km[0]), kl = of_bf16(km[4]), vs = of_bf16(vm[0]), vl = of_bf16(vm[4]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // (a code under the exponent of 2^23 is that number and the code)
      k[i] = fmaf(ks, __uint_as_float(kc[i] | 0x4b000000u) - 8388608.f, kl);
      v[i] = fmaf(vs, __uint_as_float(vc[i] | 0x4b000000u) - 8388608.f, vl);
    }
    again = may_round<DT>(ks, kl) || may_round<DT>(vs, vl);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = v[i] = 0.f;
  }
  store8<DT>(kd, k);
  store8<DT>(vd, v);
  if (again) store_sums<P, DT>(kr, vr, x, kd, vd);  // (in place of the stores: 47.1 us against 44.6)
}

// -------------------------------------------------------------------- host
using namespace b200paged;
using b200attn::may_overlap;
using b200attn::stretches_of;

// Checks both entry points' arguments and fills the call; `out`: the vectors are written.
// threads: of a sequence.
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
  const int64_t parts = out && head_dim > 64 ? 16 : kParts;  // threads of a token's heads, each
  if (rows->tokens > 0x3fffffff || rows->tokens * c->kv_heads * parts > 0x7fffffffll - kThreads)
    return B200_ATTN_ERR_INVALID_ARGUMENT;
  *threads = rows->tokens * c->kv_heads * parts;
  a->inv_tok = inverse_of(static_cast<uint32_t>(c->kv_heads * parts));
  a->inv_size = inverse_of(static_cast<uint32_t>(c->page_size));
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
  const bool wide = head_dim > 64;
  const dim3 grid(static_cast<unsigned>((threads + kThreads - 1) / kThreads),
                  static_cast<unsigned>(c->layers), static_cast<unsigned>(c->batch));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
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
