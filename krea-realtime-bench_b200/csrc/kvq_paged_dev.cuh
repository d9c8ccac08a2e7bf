// Device code shared by the two attention kernels over the paged cache: bulk copies,
// code bits to values.
#pragma once

#include <cuda_bf16.h>

#include "kvq_paged.cuh"
#include "kvq_sm100.cuh"

namespace kvq {
namespace paged {

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar))
               : "memory");
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
// Nibbles at bits 0-3 and 16-19 (code = q + 8) -> bf16x2 (q, q): 128 + code - 136.
__device__ __forceinline__ uint32_t int4_pair(uint32_t x) { return hsub2((x & 0x000F000Fu) | 0x43004300u, 0x43084308u); }
// Bytes at bits 0-7 and 16-23 (code = q + 128) -> bf16x2 (q, q). The low seven bits give
// 128 + code % 128, from which 256 is taken, or 128 where the top bit is set.
__device__ __forceinline__ uint32_t int8_pair(uint32_t x) {
  return hsub2((x & 0x007F007Fu) | 0x43004300u, (x & 0x00800080u) ^ 0x43804380u);
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
