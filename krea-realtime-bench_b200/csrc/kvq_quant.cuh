// Quantization arithmetic of one (token, head) row, shared by the append / rebuild
// kernels and the paged append: per-group absmax, scale and codes, bit-exact to
// the reference torch path (see kvq_quant.cu for the derivation).
#pragma once

#include <utility>

#include "kvq_common.cuh"

namespace kvq {

constexpr int kQD = 128;  // head_dim of the specialised kernels

// Absolute values of a bf16x2 word, max'ed into m with NaN propagation.
__device__ __forceinline__ uint32_t absmax_bf16x2(uint32_t m, uint32_t w) {
  uint32_t a = w & 0x7FFF7FFFu;
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(a));
  return r;
}

// Division-free code of x: returns the bit pattern of rne(x/s) + magic, whose low
// byte is the offset code (see file comment). `fast` groups only.
__device__ __forceinline__ uint32_t code_fast(float x, float s, float r, float magic) {
  float y0 = __fmul_rn(x, r);
  float rem = __fmaf_rn(-y0, s, x);
  float y = __fmaf_rn(rem, r, y0);
  return __float_as_uint(__fadd_rn(y, magic));
}

// Reference formula with the IEEE divide; clamps so non-finite inputs give codes
// in range (they are outside the parity contract).
__device__ __forceinline__ uint32_t code_exact(float x, float s, float qmax, float magic) {
  float y = __fdiv_rn(x, s);
  y = fminf(fmaxf(y, -qmax), qmax);
  return __float_as_uint(__fadd_rn(y, magic));
}

template <int BITS>
struct QuantConsts {
  static constexpr int kQmax = (1 << (BITS - 1)) - 1;
  // 1.5 * 2^23 + offset: adding it rounds to the nearest even integer and puts
  // code + offset in the low bits of the result.
  static constexpr float kMagic = 12582912.0f + (BITS == 4 ? 8.0f : 128.0f);
  static constexpr int kCodeBytes = BITS == 4 ? kQD / 2 : kQD;  // per row
};

// Group scale s = amax / qmax without a divide: q0 = amax * r, rem = amax - q0 * qmax
// (FMA), s = q0 + rem * r (FMA), r = RN(1/qmax). Equal to the IEEE quotient for
// every positive finite bf16 amax (exhaustively checked by the oracle's
// kvqo_check_scale_div); non-finite amax take the IEEE divide.
template <int QMAX>
__device__ __forceinline__ float group_scale(float amax) {
  if (!(amax <= 3.0e38f)) return __fdiv_rn(amax, static_cast<float>(QMAX));
  const float r = QMAX == 7 ? 0.142857149243354797f : 0.00787401571869850159f;
  const float q0 = __fmul_rn(amax, r);
  const float rem = __fmaf_rn(-q0, static_cast<float>(QMAX), amax);
  return __fmaf_rn(rem, r, q0);
}

// __byte_perm selectors that replace byte p of the first operand with byte 0 of
// the second and keep the other three
__device__ constexpr uint32_t kInsertByte[4] = {0x3214u, 0x3240u, 0x3410u, 0x4210u};

template <int LO, int HI, int BITS, int G_INDEX>
__device__ __forceinline__ void quant_group(const uint32_t (&w)[64], uint32_t (&ow)[BITS == 4 ? 16 : 32],
                                            uint16_t& scale_out, uint32_t& slow_mask) {
  using C = QuantConsts<BITS>;
  static_assert(LO % 2 == 0 && HI % 2 == 0 && LO < HI, "groups must start and end on even channels");
  uint32_t m = 0;
#pragma unroll
  for (int k = LO / 2; k < HI / 2; ++k) m = absmax_bf16x2(m, w[k]);
  float amax;
  {
    uint32_t lo = m << 16, hi = m & 0xFFFF0000u;
    float a = __uint_as_float(lo), b = __uint_as_float(hi);
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(amax) : "f"(a), "f"(b));  // NaN if either is NaN
  }
  float s = group_scale<C::kQmax>(amax);
  s = (s > 0.0f) ? s : 1.0f;  // quant_kv.py:152 (also maps NaN to 1, like torch.where)
  scale_out = f32_to_bf16_bits(s);
  // groups with a tiny or non-finite amax are recomputed with the IEEE divide by
  // quant_fix_slow after staging; the fast chain below still runs for them (any
  // value it produces is overwritten)
  if (!((amax >= 0x1p-100f) && (amax <= 3.0e38f))) slow_mask |= 1u << G_INDEX;
  // reciprocal within one ulp of 1/s: hardware approximation + one Newton step
  // (the code formula holds for any such r, kvqo_check_fast_codes_rcp)
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  r = __fmaf_rn(r, __fmaf_rn(-s, r, 1.0f), r);
  // the per-element chain on packed f32x2: two channels per instruction
  const float2 r2 = make_float2(r, r), ns2 = make_float2(-s, -s);
  const float2 mg2 = make_float2(C::kMagic, C::kMagic);
#pragma unroll
  for (int k = LO / 2; k < HI / 2; ++k) {
    const float2 x = make_float2(bf16lo_to_f32(w[k]), bf16hi_to_f32(w[k]));
    const float2 y0 = __fmul2_rn(x, r2);
    const float2 rem = __ffma2_rn(y0, ns2, x);
    const float2 t = __fadd2_rn(__ffma2_rn(rem, r2, y0), mg2);
    const uint32_t c0 = __float_as_uint(t.x), c1 = __float_as_uint(t.y);
    if constexpr (BITS == 4) {
      // low byte of c0 + 16 * c1 is the packed pair (code bytes are < 16)
      const uint32_t pair = c0 + (c1 << 4);
      ow[k >> 2] = __byte_perm(ow[k >> 2], pair, kInsertByte[k & 3]);
    } else {
      const uint32_t half = __byte_perm(c0, c1, 0x0040);
      ow[k >> 1] = __byte_perm(ow[k >> 1], half, (k & 1) ? 0x5410u : 0x3254u);
    }
  }
}

template <class L, int BITS, int... Gs>
__device__ __forceinline__ void quant_row(const uint32_t (&w)[64], uint32_t (&ow)[BITS == 4 ? 16 : 32],
                                          uint16_t (&sc)[L::G], uint32_t& slow_mask,
                                          std::integer_sequence<int, Gs...>) {
  (quant_group<L::E[Gs], L::E[Gs + 1], BITS, Gs>(w, ow, sc[Gs], slow_mask), ...);
}

template <class L, int... Is>
__device__ __forceinline__ void fill_edges(int (&e)[L::G + 1], std::integer_sequence<int, Is...>) {
  ((e[Is] = std::integral_constant<int, L::E[Is]>::value), ...);
}

}  // namespace kvq
