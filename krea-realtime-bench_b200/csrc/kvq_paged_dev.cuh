// Device code shared by the two attention kernels over the paged cache: bulk copies,
// code bits to values.
#pragma once

#include <cuda_bf16.h>

#include "kvq_paged.cuh"
#include "kvq_sm100.cuh"

namespace kvq {
namespace paged {

// Waits for the phase of `parity`, as sm100::mbar_wait, but polls first: a thread that
// try_wait suspends comes back 1000 to 2500 cycles after the phase completed, which in a
// pipeline of 2000-cycle steps is a step; test_wait answers in about 100. A wait that
// is still unfinished after kPolls polls goes on as the bounded, suspending one.
constexpr int kPolls = 512;
__device__ __forceinline__ bool mbar_test(const uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(sm100::smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool poll_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* status, long long limit) {
#pragma unroll 1
  for (int i = 0; i < kPolls; ++i)
    if (mbar_test(bar, parity)) return true;
  return sm100::mbar_wait(bar, parity, abort, status, limit);
}
// The same by a converged warp.
__device__ __forceinline__ bool poll_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort, int* status,
                                               long long limit) {
#pragma unroll 1
  for (int i = 0; i < kPolls; ++i)
    if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
  return sm100::mbar_wait_warp(bar, parity, abort, status, limit);
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 ld_shared_v2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t ld_shared_u16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  const __nv_bfloat162 r = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b),
                                   *reinterpret_cast<__nv_bfloat162*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// int4 codes (code = q + 8) at bits 0-3 and 16-19, or 4-7 and 20-23, of a word -> bf16x2
// (q / 4, q / 4), exact, one logic operation and one FMA each and no shift:
//   low   ored into the mantissa of 128: 128 + code, times 1/4, minus 34;
//   high  bits 4-7 of a bf16 are its lowest exponent bit and the top of its mantissa, and
//         a bf16 with that exponent or none is linear in its bits: code * 2^-129, times
//         2^127, minus 2.
// With four times the scale the product is q * s, rounded once.
// (x & m) | o as one instruction: from the C expression the compiler made two.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t m, uint32_t o) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(m), "r"(o));
  return y;
}
__device__ __forceinline__ uint32_t int4_low(uint32_t x) {
  return hfma2(and_or(x, 0x000F000Fu, 0x43004300u), 0x3E803E80u, 0xC208C208u);
}
__device__ __forceinline__ uint32_t int4_high(uint32_t x) { return hfma2(x & 0x00F000F0u, 0x7F007F00u, 0xC000C000u); }
constexpr uint32_t kFour = 0x40804080u;  // bf16x2 (4, 4)
// Bytes at bits 0-7 and 16-23 (code = q + 128) -> bf16x2 (q, q). The low seven bits give
// 128 + code % 128, from which 256 is taken, or 128 where the top bit is set.
__device__ __forceinline__ uint32_t int8_pair(uint32_t x) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(d) : "r"(x), "r"(0x00800080u), "r"(0x43804380u));  // (x & m) ^ o
  return hsub2(and_or(x, 0x007F007Fu, 0x43004300u), d);
}

// Most channel groups that an aligned run of N channels meets.
template <class L, int N>
__host__ __device__ constexpr int most_groups() {
  int most = 0;
  for (int c = 0; c < D; c += N) {
    int n = 0;
    for (int g = 0; g < L::G; ++g) n += L::E[g] < c + N && L::E[g + 1] > c;
    most = n > most ? n : most;
  }
  return most;
}

}  // namespace paged
}  // namespace kvq
