// Device code shared by the two attention kernels over the paged cache: bulk copies,
// code bits to values.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

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
// (x & m) | o as one instruction: from the C expression the compiler made two.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t m, uint32_t o) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(m), "r"(o));
  return y;
}
// int4 codes (code = q + 8) at bits 0-3 and 16-19 of a word -> bf16x2 (q / 4, q / 4), exact:
// 128 + code, times 1/4, minus 34. With four times the scale the product is q * s, rounded once.
__device__ __forceinline__ uint32_t int4_low(uint32_t x) {
  return hfma2(and_or(x, 0x000F000Fu, 0x43004300u), 0x3E803E80u, 0xC208C208u);
}
constexpr uint32_t kFour = 0x40804080u;  // bf16x2 (4, 4)
// Bytes at bits 0-7 and 16-23 (code = q + 128) -> bf16x2 (q, q). The low seven bits give
// 128 + code % 128, from which 256 is taken, or 128 where the top bit is set.
__device__ __forceinline__ uint32_t int8_pair(uint32_t x) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(d) : "r"(x), "r"(0x00800080u), "r"(0x43804380u));  // (x & m) ^ o
  return hsub2(and_or(x, 0x007F007Fu, 0x43004300u), d);
}

// The attention multiplies in fp16 rather than bf16: an int4 code times a bf16 scale has
// eleven significant bits, which fp16 holds and bf16 rounds to eight; with bf16 products
// the output's error against 64 bits was 3.7e-3, of which the rounding of the output is
// 1.7e-3. fp16 ends at 65504 and thins out below 2^-14, so a token with a key or value
// scale beyond [kScaleLeast, kScaleMost] is multiplied as if its scales were 2^-e times
// as large, and a query row likewise: logits get the power of two back in fp32, softmax
// weights get a value's, relative to a power of two F that each output row keeps for
// itself. Tokens and rows that have none keep their bits. Groups down to 2^-22 of a
// token's largest so keep all that fp16 has of them (int4: down to 2^-25 all their bits),
// those below 2^-33 become 0. A group whose codes are all zero is stored with the scale 1,
// which does not count.
__device__ __forceinline__ uint32_t h16mul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h16fma2(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b), *reinterpret_cast<__half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h16add2(uint32_t a, uint32_t b) {
  const __half2 r = __hadd2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Codes at the same places as above -> f16x2 (q, q), exact: 1024 + code - 1032, and
// (1024 + 16 code) / 16 - 72; for int8 1024 + code - 1152.
__device__ __forceinline__ uint32_t int4_low_f16(uint32_t x) {
  return h16add2(and_or(x, 0x000F000Fu, 0x64006400u), 0xE408E408u);
}
__device__ __forceinline__ uint32_t int4_high_f16(uint32_t x) {
  return h16fma2(and_or(x, 0x00F000F0u, 0x64006400u), 0x2C002C00u, 0xD480D480u);
}
__device__ __forceinline__ uint32_t int8_pair_f16(uint32_t x) {
  return h16add2(and_or(x, 0x00FF00FFu, 0x64006400u), 0xE480E480u);
}
constexpr uint32_t kScaleLeast = 0x3880, kScaleMost = 0x4400;  // bf16 2^-14, 512 (127 * 512 < 65504)
constexpr uint32_t kQueryLeast = 0x3880, kQueryMost = 0x4700;  // bf16 2^-14, 2^15
// bits of a bf16 >= 0 outside [least, most]
__device__ __forceinline__ bool beyond(uint32_t bits, uint32_t least, uint32_t most) { return bits - least > most - least; }
// 2^e, |e| <= 126
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
// Exponent to take out of a token whose largest and least scales (of groups that are not
// zero) have these bits: the largest ends below 512, the least at 2^-14 or above if the
// largest leaves room for that; 0 where both do.
__device__ __forceinline__ int scale_exponent(uint32_t most, uint32_t least) {
  if (most <= kScaleMost && least >= kScaleLeast) return 0;
  const int down = static_cast<int>(most >> 7) - 127 - 8, up = static_cast<int>(least >> 7) - 127 + 14;
  return most > kScaleMost ? min(down, 119) : max(max(down, up), -110);
}
// The largest and least of the scales that lanes differing in the bits FIRST, 2 FIRST, ... ,
// LAST of their number have, in one exchange.
template <int FIRST, int LAST>
__device__ __forceinline__ void extremes_of_lanes(uint32_t& most, uint32_t& least) {
  uint32_t x = most << 16 | (0xFFFFu - least);
#pragma unroll
  for (int d = FIRST; d <= LAST; d <<= 1) x = __vmaxu2(x, __shfl_xor_sync(0xffffffffu, x, d));
  most = x >> 16;
  least = 0xFFFFu - (x & 0xFFFFu);
}
// Bits of the scale that a group of zeros is stored with: no other group needs a look at its
// codes to tell.
constexpr uint32_t kScaleOne = 0x3F80;
// What a token without any such group has: its weight counts nowhere but in the sum.
constexpr int kNoScale = -110;
// Exponent to take out of a query row whose largest and least magnitudes (of elements that
// are not 0) have these bits: the largest ends below 2^15, the least at 2^-14 or above if the
// largest leaves room for that. No further, so that products with huge keys stay in range.
__device__ __forceinline__ int query_exponent(uint32_t most, uint32_t least) {
  if (most <= kQueryMost && least >= kQueryLeast) return 0;
  const int down = static_cast<int>(most >> 7) - 127 - 14, up = static_cast<int>(least >> 7) - 127 + 14;
  return most > kQueryMost ? down : max(max(down, up), -110);
}
// What a row's logits are multiplied with: the softmax scale with the power of two taken out
// of the row's query. Never 0, which would make a masked logit NaN; logits of so small a
// scale are 0 either way.
__device__ __forceinline__ float row_scale_of(float scale_log2, int e) { return fmaxf(scale_log2 * pow2i(e), 0x1p-126f); }
// Largest finite magnitude among eight bf16, as bits.
__device__ __forceinline__ uint32_t most_of(const uint4& v) {
  uint32_t m = 0;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = w[i] & 0x7FFFu, hi = (w[i] >> 16) & 0x7FFFu;
    m = max(m, lo < 0x7F80u ? lo : 0u);
    m = max(m, hi < 0x7F80u ? hi : 0u);
  }
  return m;
}
// Least magnitude other than 0 among eight bf16, as bits, or one less (0x8000 or more: none).
// A 0 in a low half takes one from the high half, where a 1 then counts as none.
__device__ __forceinline__ uint32_t least_of(const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t m = 0xFFFFFFFFu;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __vminu2(m, (w[i] & 0x7FFF7FFFu) - 0x00010001u);
  return min(min(m & 0xFFFFu, m >> 16), 0xFFFEu) + 1;
}
// A row's running maximum m stands kBias below the logit it was taken from and moves only
// when some logit lies more than kLag + kBias above it, so the softmax weights 2^(x - m)
// end at 2^15, and the largest of a row is 2^7 at least. fp16 holds weights of 2^-21 of that
// with all their bits, and those of 2^-32 at all: without the bias 200 tokens under a first
// token that leads by 17 nats and has the value 0 came out 7 % off.
constexpr float kBias = 7.0f, kLag = 8.0f;
// The F of an output row once a weight times its value's power of two has been 2^top, given
// what F has to be for the row so far: F less what the maximum has risen since, which for a
// row that had seen nothing is all it can be. Leaves room below fp16's end; 0 where that
// leaves what an ordinary row has (top = kBias at least), so that those end up there.
__device__ __forceinline__ float next_f(float f, float top) {
  const float n = fmaxf(f, ceilf(top) - (kBias + kLag));
  return top == -INFINITY ? f : (n >= -kLag && n < 0.0f ? 0.0f : n);
}
// Eight bf16 times 2^-e -> fp16 (exact for normal results).
__device__ __forceinline__ uint4 to_f16(const uint4& v, int e) {
  const float f = pow2i(-e);
  uint4 o;
  o.x = pack_f16x2(bf16lo_to_f32(v.x) * f, bf16hi_to_f32(v.x) * f);
  o.y = pack_f16x2(bf16lo_to_f32(v.y) * f, bf16hi_to_f32(v.y) * f);
  o.z = pack_f16x2(bf16lo_to_f32(v.z) * f, bf16hi_to_f32(v.z) * f);
  o.w = pack_f16x2(bf16lo_to_f32(v.w) * f, bf16hi_to_f32(v.w) * f);
  return o;
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

// Bit q: group base + q has a code other than zero's among the N channels from ch on, whose
// codes are at `src` in shared memory; bits of groups whose scale is not 1 are of no use.
// Groups are made of channel pairs. Rarely called, and a function of its own: inlined it cost
// the loops around it 2 to 3 % in registers and instruction cache.
template <class L, int BITS, int N>
__device__ __noinline__ uint32_t used_groups(uint32_t src, int ch, int base) {
  constexpr int kPerWord = 32 / BITS;
  uint32_t used = 0;
#pragma unroll 1
  for (int i = 0; i < N * BITS / 32; ++i, src += 4, ch += kPerWord) {
    uint32_t x;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(src));
    x ^= BITS == 4 ? 0x88888888u : 0x80808080u;
#pragma unroll
    for (int c = 0; c < kPerWord; c += 2)
      if ((x >> (BITS * c)) & ((1u << (2 * BITS)) - 1)) used |= 1u << (group_at<L>(ch + c) - base);
  }
  return used;
}

}  // namespace paged
}  // namespace kvq
