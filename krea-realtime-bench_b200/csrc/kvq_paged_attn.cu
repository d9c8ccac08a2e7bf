// Attention of a chunk of new tokens over the paged quantized cache (sm_100a).
//
// One CTA of four warps per (query token, query head). Each warp walks every
// fourth visible token: lane l holds channels 4l..4l+3 of q, K and V; the dot
// product is reduced over the warp; m, l and the unnormalised output are kept in
// fp32 with the online softmax, and the four warps' states are joined at the end:
//   m = max m_w, O = sum_w 2^(m_w - m) O_w / sum_w 2^(m_w - m) l_w.
#include <cmath>

#include "kvq_paged.cuh"

namespace kvq {
namespace paged {

struct AttnArgs {
  Pages p;
  const uint16_t* q;
  int64_t q_stride;
  const uint8_t* k_pages;
  const uint8_t* v_pages;
  uint16_t* out;
  int64_t out_stride;
  float* lse;
  int group;  // query heads per KV head
  int causal;
  int64_t window, sink;
  float scale_log2;
};

// Channels 4l..4l+3 of a stored row.
template <class L, int BITS>
__device__ __forceinline__ float4 load4(const uint8_t* rec, int row, int lane, int g0, int g1) {
  using R = Rec<L, BITS>;
  const uint16_t* sc = reinterpret_cast<const uint16_t*>(rec + R::kCodes) + row * L::G;
  const float s0 = bf16_bits_to_f32(__ldg(sc + g0)), s1 = bf16_bits_to_f32(__ldg(sc + g1));
  int c[4];
  if constexpr (BITS == 4) {
    const uint32_t w = __ldg(reinterpret_cast<const uint16_t*>(rec + row * R::CW) + lane);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = static_cast<int>((w >> (4 * i)) & 15u) - 8;
  } else {
    const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(rec + row * R::CW) + lane);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = static_cast<int>((w >> (8 * i)) & 255u) - 128;
  }
  return make_float4(c[0] * s0, c[1] * s0, c[2] * s1, c[3] * s1);
}

template <class L, int KB, int VB>
__global__ void __launch_bounds__(128) rows_kernel(const __grid_constant__ AttnArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ float sm_o[4][D];
  __shared__ float sm_m[4], sm_l[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tok = blockIdx.x, hq = blockIdx.y, h = hq / a.group;
  int s = 0;
  for (int hi = a.p.n_seqs - 1; s < hi;) {  // the last sequence that starts at or before tok
    const int mid = (s + hi + 1) >> 1;
    if (__ldg(&a.p.seqs[mid].q_first) <= tok) s = mid; else hi = mid - 1;
  }
  const kvq_paged_seq sq = a.p.seqs[s];
  const int pos = sq.kv_len - sq.q_len + (tok - sq.q_first);
  const int end = a.causal ? min(pos + 1, sq.kv_len) : sq.kv_len;
  const int64_t first = a.window > 0 ? max(static_cast<int64_t>(0), pos - a.window + 1) : 0;
  const int64_t kept = a.window > 0 ? min(a.sink, first) : 0;

  const uint2 qw = *reinterpret_cast<const uint2*>(a.q + tok * a.q_stride + hq * D + 4 * lane);
  const float4 q = make_float4(bf16lo_to_f32(qw.x), bf16hi_to_f32(qw.x), bf16lo_to_f32(qw.y), bf16hi_to_f32(qw.y));
  const int g0 = group_at<L>(4 * lane), g1 = group_at<L>(4 * lane + 2);
  float m = -1.0e30f, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto visit = [&](int j) {
    bool ok;
    const int64_t b = a.p.block(s, h, j / kBlock, ok);
    const float4 k = load4<L, KB>(a.k_pages + b * Rec<L, KB>::kBytes, j % kBlock, lane, g0, g1);
    float d = q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) d += __shfl_xor_sync(0xffffffffu, d, i);
    d *= a.scale_log2;
    const float mn = fmaxf(m, d), alpha = exp2f(m - mn), w = exp2f(d - mn);
    const float4 v = load4<L, VB>(a.v_pages + b * Rec<L, VB>::kBytes, j % kBlock, lane, g0, g1);
    o = make_float4(o.x * alpha + w * v.x, o.y * alpha + w * v.y, o.z * alpha + w * v.z, o.w * alpha + w * v.w);
    l = l * alpha + w;
    m = mn;
  };
  for (int64_t j = warp; j < kept; j += 4) visit(static_cast<int>(j));
  for (int64_t j = first + warp; j < end; j += 4) visit(static_cast<int>(j));

  *reinterpret_cast<float4*>(&sm_o[warp][4 * lane]) = o;
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
  __syncthreads();
  const float mm = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
  float total = 0.0f, acc = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = exp2f(sm_m[w] - mm);
    total += f * sm_l[w];
    acc += f * sm_o[w][threadIdx.x];
  }
  a.out[tok * a.out_stride + hq * D + threadIdx.x] = f32_to_bf16_bits(total == 0.0f ? 0.0f : acc / total);
  if (a.lse && threadIdx.x == 0)
    a.lse[static_cast<int64_t>(tok) * gridDim.y + hq] =
        total == 0.0f ? -INFINITY : 0.69314718055994531f * (mm + log2f(total));
}

}  // namespace paged
}  // namespace kvq

using namespace kvq;

extern "C" int kvq_paged_attention(const void* q, int64_t q_token_stride, const kvq_paged_cache* cache,
                                   const kvq_paged_batch* batch, void* out, int64_t out_token_stride, float* lse,
                                   int n_q_heads, int causal, int64_t window, int64_t sink, float softmax_scale,
                                   void* stream) {
  clear_error();
  int layout = 0;
  int rc = paged::check_cache(cache, batch, &layout);
  if (rc) return rc;
  KVQ_REQUIRE(n_q_heads >= 1 && n_q_heads <= 65535 && n_q_heads % cache->n_heads == 0, KVQ_ERR_ARG,
              "%d query heads are not a multiple of %d KV heads", n_q_heads, cache->n_heads);
  KVQ_REQUIRE(window >= 0 && sink >= 0, KVQ_ERR_ARG, "window and sink must be >= 0");
  KVQ_REQUIRE(std::isfinite(softmax_scale), KVQ_ERR_ARG, "softmax_scale must be finite");
  if (batch->n_seqs == 0 || batch->n_new == 0) return KVQ_OK;
  KVQ_REQUIRE(q && out, KVQ_ERR_ARG, "NULL q or out pointer");
  KVQ_REQUIRE(q_token_stride >= (int64_t)n_q_heads * paged::D && out_token_stride >= (int64_t)n_q_heads * paged::D,
              KVQ_ERR_ARG, "token strides must be >= heads*head_dim");
  KVQ_REQUIRE((reinterpret_cast<uintptr_t>(q) & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0 &&
                  q_token_stride % 8 == 0 && out_token_stride % 8 == 0,
              KVQ_ERR_ALIGN, "q and out must be 16-byte aligned with token strides that are multiples of 8");
  KVQ_REQUIRE((reinterpret_cast<uintptr_t>(lse) & 3) == 0, KVQ_ERR_ALIGN, "lse must be 4-byte aligned");
  rc = require_sm100();
  if (rc) return rc;
  paged::AttnArgs a;
  a.p = paged::make_pages(cache, batch);
  a.q = static_cast<const uint16_t*>(q);
  a.q_stride = q_token_stride;
  a.k_pages = static_cast<const uint8_t*>(cache->k_pages);
  a.v_pages = static_cast<const uint8_t*>(cache->v_pages);
  a.out = static_cast<uint16_t*>(out);
  a.out_stride = out_token_stride;
  a.lse = lse;
  a.group = n_q_heads / cache->n_heads;
  a.causal = causal ? 1 : 0;
  a.window = window;
  a.sink = sink;
  a.scale_log2 = (softmax_scale > 0.0f ? softmax_scale : 1.0f / sqrtf(128.0f)) * 1.4426950408889634f;
  const dim3 grid(static_cast<unsigned>(batch->n_new), n_q_heads);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return paged::with_layout(layout, [&](auto l) {
    using L = decltype(l);
    return paged::with_bits(cache->k_bits, cache->v_bits, [&](auto b) {
      using B = decltype(b);
      paged::rows_kernel<L, B::k, B::v><<<grid, 128, 0, st>>>(a);
      return check_launch("kvq_paged_attention");
    });
  });
}
