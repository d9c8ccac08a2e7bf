// Attention of a batch's new tokens over the paged quantized cache: argument checks
// and launches (kvq_paged_attention).
#include <cmath>

#include "kvq_paged.cuh"
#include "kvq_sm100.cuh"

using namespace kvq;

extern "C" int kvq_paged_attention(const void* q, int64_t q_token_stride, const kvq_paged_cache* cache,
                                   const kvq_paged_batch* batch, void* out, int64_t out_token_stride, float* lse,
                                   int n_q_heads, int causal, int64_t window, int64_t sink, float softmax_scale,
                                   const kvq_paged_plan_info* info, const int32_t* plan, void* workspace,
                                   uint32_t* counters, void* stream) {
  clear_error();
  int layout = 0;
  int rc = paged::check_cache(cache, batch, &layout);
  if (rc) return rc;
  KVQ_REQUIRE(n_q_heads >= 1 && n_q_heads <= 65535 && n_q_heads % cache->n_heads == 0, KVQ_ERR_ARG,
              "%d query heads are not a multiple of %d KV heads", n_q_heads, cache->n_heads);
  KVQ_REQUIRE(window >= 0 && sink >= 0, KVQ_ERR_ARG, "window and sink must be >= 0");
  KVQ_REQUIRE(std::fabs(softmax_scale) <= 1e38f, KVQ_ERR_ARG, "softmax_scale must be at most 1e38");
  if (batch->n_seqs == 0 || batch->n_new == 0) return KVQ_OK;
  KVQ_REQUIRE(q && out, KVQ_ERR_ARG, "NULL q or out pointer");
  KVQ_REQUIRE(q_token_stride >= (int64_t)n_q_heads * paged::D && out_token_stride >= (int64_t)n_q_heads * paged::D,
              KVQ_ERR_ARG, "token strides must be >= heads*head_dim");
  KVQ_REQUIRE((reinterpret_cast<uintptr_t>(q) & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0 &&
                  q_token_stride % 8 == 0 && out_token_stride % 8 == 0,
              KVQ_ERR_ALIGN, "q and out must be 16-byte aligned with token strides that are multiples of 8");
  KVQ_REQUIRE((reinterpret_cast<uintptr_t>(lse) & 3) == 0, KVQ_ERR_ALIGN, "lse must be 4-byte aligned");
  KVQ_REQUIRE(info && plan, KVQ_ERR_ARG, "NULL plan");
  KVQ_REQUIRE((reinterpret_cast<uintptr_t>(plan) & 15) == 0, KVQ_ERR_ALIGN, "the plan must be 16-byte aligned");
  KVQ_REQUIRE(info->n_units == 0 || (workspace && counters), KVQ_ERR_ARG, "the plan needs a workspace and counters");
  KVQ_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, KVQ_ERR_ALIGN,
              "the workspace must be 256-byte aligned");
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
  a.n_q_heads = n_q_heads;
  a.causal = causal ? 1 : 0;
  a.window = window;
  a.sink = sink;
  a.scale_log2 = (softmax_scale > 0.0f ? softmax_scale : 1.0f / sqrtf(128.0f)) * 1.4426950408889634f;
  a.items = reinterpret_cast<const paged::Item*>(plan);
  a.cta_first = info->n_row_items == info->n_row_ctas
                    ? nullptr
                    : plan + static_cast<int64_t>(info->n_row_items + info->n_tile_items) * paged::kItemWords;
  a.ws = static_cast<float*>(workspace);
  a.ctr = counters;
  a.wait_cycles = sm100::kWaitCycles;
  rc = status_word(&a.status);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (info->n_tile_items > 0) {
    paged::AttnArgs t = a;
    t.items += info->n_row_items;
    t.ws = reinterpret_cast<float*>(static_cast<char*>(workspace) + info->tile_workspace_offset);
    rc = paged::launch_tiles(t, layout, cache->k_bits, cache->v_bits, info->n_tile_items, st);
    if (rc) return rc;
  }
  if (info->n_row_ctas > 0) {
    rc = paged::launch_rows(a, layout, cache->k_bits, cache->v_bits, info->row_tile, info->n_row_ctas, st);
    if (rc) return rc;
  }
  return check_launch("kvq_paged_attention");
}
