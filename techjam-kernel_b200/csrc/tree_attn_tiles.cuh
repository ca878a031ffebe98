// tree_attn_tiles.cuh — what the drafted-token attention kernels on the fifth-generation
// tensor cores share: bounded waits, tensor-memory accesses and packed arithmetic.
#pragma once

#include <cstdint>

#include "tree_attn.cuh"

namespace b200tree {
namespace {

namespace ptx = b200attn::ptx;

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

}  // namespace
}  // namespace b200tree
