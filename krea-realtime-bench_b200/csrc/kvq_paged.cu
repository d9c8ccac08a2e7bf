// Paged quantized cache: writing new tokens into their pages and reading tokens
// back (sm_100a), and the checks shared with the attention over it.
//
// Append. Per (token, head) row x and channel group g: s_g = max_g |x| / qmax (1
// where that is 0), code = rne(x / s_g) + offset, stored scale bf16(s_g): the
// arithmetic of kvq_quantize, bit for bit, with rows going to pages.
#include "kvq_paged.cuh"
#include "kvq_quant.cuh"

namespace kvq {
namespace paged {

int check_format(const kvq_paged_cache* c, int* layout) {
  KVQ_REQUIRE(c != nullptr, KVQ_ERR_ARG, "NULL cache");
  KVQ_REQUIRE(c->head_dim == D, KVQ_ERR_UNSUPPORTED, "the paged cache supports head_dim 128, got %d", c->head_dim);
  KVQ_REQUIRE((c->k_bits == 4 && c->v_bits == 4) || (c->k_bits == 8 && (c->v_bits == 4 || c->v_bits == 8)),
              KVQ_ERR_UNSUPPORTED, "the paged cache holds K/V in 4/4, 8/4 or 8/8 bits, got %d/%d", c->k_bits,
              c->v_bits);
  KVQ_REQUIRE(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 || c->page_size == 128,
              KVQ_ERR_UNSUPPORTED, "page_size must be 16, 32, 64 or 128, got %d", c->page_size);
  KVQ_REQUIRE(c->n_heads >= 1 && c->n_heads <= 65535, KVQ_ERR_ARG, "n_heads %d out of range", c->n_heads);
  KVQ_REQUIRE(c->n_pages >= 1 && c->n_pages * c->page_size < ((int64_t)1 << 31), KVQ_ERR_ARG,
              "n_pages %lld out of range", (long long)c->n_pages);
  const int id = resolve_layout(c->chan_band, c->head_dim, c->n_groups, nullptr);
  if (id < 0) return id;
  KVQ_REQUIRE(id != kLayoutGeneric, KVQ_ERR_UNSUPPORTED,
              "the paged cache supports the bands, bands2, bands4, blind32 and blind64 group maps");
  *layout = id;
  return KVQ_OK;
}

int check_cache(const kvq_paged_cache* c, const kvq_paged_batch* b, int* layout) {
  const int rc = check_format(c, layout);
  if (rc) return rc;
  KVQ_REQUIRE(b != nullptr, KVQ_ERR_ARG, "NULL batch");
  KVQ_REQUIRE(c->k_pages && c->v_pages, KVQ_ERR_ARG, "NULL page pointer");
  KVQ_REQUIRE((reinterpret_cast<uintptr_t>(c->k_pages) & 15) == 0 && (reinterpret_cast<uintptr_t>(c->v_pages) & 15) == 0,
              KVQ_ERR_ALIGN, "pages must be 16-byte aligned");
  const int64_t lim = ((int64_t)1 << 31) - 1;
  KVQ_REQUIRE(b->n_seqs >= 0 && b->n_new >= 0 && b->n_tokens >= 0 && b->n_new_blocks >= 0 && b->n_blocks >= 0 &&
                  b->n_new <= lim && b->n_tokens <= lim && b->table_stride >= 0,
              KVQ_ERR_ARG, "bad batch");
  KVQ_REQUIRE(b->n_seqs == 0 || (b->table && b->seqs), KVQ_ERR_ARG, "NULL table or sequence pointer");
  KVQ_REQUIRE((reinterpret_cast<uintptr_t>(b->table) & 3) == 0 && (reinterpret_cast<uintptr_t>(b->seqs) & 15) == 0,
              KVQ_ERR_ALIGN, "the table must be 4-byte and the sequences 16-byte aligned");
  return KVQ_OK;
}

Pages make_pages(const kvq_paged_cache* c, const kvq_paged_batch* b) {
  Pages p;
  p.table = b->table;
  p.table_stride = b->table_stride;
  p.seqs = b->seqs;
  p.n_seqs = b->n_seqs;
  p.n_heads = c->n_heads;
  p.n_pages = static_cast<int>(c->n_pages);
  p.page_shift = 0;
  while ((kBlock << p.page_shift) < c->page_size) ++p.page_shift;
  return p;
}

// ---------------------------------------------------------------- append
struct AppendArgs {
  Pages p;
  const uint16_t* x[2];  // K, V
  int64_t stride[2];
  uint8_t* pages[2];
};

// Rare path: the groups flagged in slow_mask (amax below 2^-100, above 3e38 or not
// finite) with the IEEE divide; NaN counts as 0, magnitudes above 3e38 as 3e38.
template <class L, int BITS>
__device__ __noinline__ void fix_slow(const uint16_t* x, uint32_t slow_mask, uint8_t* codes, uint16_t* scales) {
  using C = QuantConsts<BITS>;
  constexpr float q = static_cast<float>(C::kQmax), top = 3.0e38f;
  int edges[L::G + 1];
  fill_edges<L>(edges, std::make_integer_sequence<int, L::G + 1>{});
  for (int g = 0; slow_mask; ++g, slow_mask >>= 1) {
    if (!(slow_mask & 1u)) continue;
    float amax = 0.0f;
    for (int c = edges[g]; c < edges[g + 1]; ++c) {
      const float v = fabsf(bf16_bits_to_f32(x[c]));
      amax = fmaxf(amax, v == v ? fminf(v, top) : 0.0f);
    }
    float s = __fdiv_rn(amax, q);
    s = s > 0.0f ? s : 1.0f;
    scales[g] = f32_to_bf16_bits(s);
    for (int c = edges[g]; c < edges[g + 1]; ++c) {
      float v = bf16_bits_to_f32(x[c]);
      v = v == v ? v : 0.0f;
      const uint32_t code = code_exact(v, s, q, C::kMagic) & 0xFFu;
      if constexpr (BITS == 4) {
        uint8_t& o = codes[c >> 1];
        o = (c & 1) ? static_cast<uint8_t>((o & 0x0F) | (code << 4)) : static_cast<uint8_t>((o & 0xF0) | code);
      } else {
        codes[c] = static_cast<uint8_t>(code);
      }
    }
  }
}

// One thread per row: 16 tokens of a storage block x 8 heads per CTA.
template <class L, int BITS>
__device__ __forceinline__ void append_row(const AppendArgs& a, int which, int s, int blk, int row, int h, int tok) {
  using R = Rec<L, BITS>;
  const uint16_t* x = a.x[which] + tok * a.stride[which] + h * D;
  uint32_t w[64];
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    const uint4 v = ld_global_nc_v4(x + 8 * c);
    w[4 * c] = v.x;
    w[4 * c + 1] = v.y;
    w[4 * c + 2] = v.z;
    w[4 * c + 3] = v.w;
  }
  uint32_t ow[BITS == 4 ? 16 : 32];
#pragma unroll
  for (int i = 0; i < (BITS == 4 ? 16 : 32); ++i) ow[i] = 0;
  uint16_t sc[L::G];
  uint32_t slow = 0;
  quant_row<L, BITS>(w, ow, sc, slow, std::make_integer_sequence<int, L::G>{});
  bool ok;
  uint8_t* rec = a.pages[which] + a.p.block(s, h, blk, ok) * R::kBytes;
  if (!ok) return;
  uint8_t* codes = rec + row * R::CW;
  uint16_t* scales = reinterpret_cast<uint16_t*>(rec + R::kCodes) + row * L::G;
#pragma unroll
  for (int i = 0; i < R::CW / 16; ++i)
    st_global_v4(codes + 16 * i, make_uint4(ow[4 * i], ow[4 * i + 1], ow[4 * i + 2], ow[4 * i + 3]));
#pragma unroll
  for (int g = 0; g < L::G; ++g) scales[g] = sc[g];
  if (slow) fix_slow<L, BITS>(x, slow, codes, scales);
}

template <class L, int KB, int VB>
__global__ void __launch_bounds__(128) append_kernel(const __grid_constant__ AppendArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.y * 8 + (threadIdx.x >> 4);
  const int s = find_seq<true>(a.p, blockIdx.x);
  const kvq_paged_seq q = a.p.seqs[s];
  const int start = q.kv_len - q.q_len;
  const int blk = start / kBlock + (static_cast<int>(blockIdx.x) - q.q_block);
  const int row = threadIdx.x & (kBlock - 1);
  const int pos = blk * kBlock + row;
  if (h >= a.p.n_heads || pos < start || pos >= q.kv_len) return;
  const int tok = q.q_first + pos - start;
  if (blockIdx.z == 0)
    append_row<L, KB>(a, 0, s, blk, row, h, tok);
  else
    append_row<L, VB>(a, 1, s, blk, row, h, tok);
}

// ---------------------------------------------------------------- read
struct ReadArgs {
  Pages p;
  const uint8_t* pages[2];
  uint16_t* out[2];
  int64_t stride[2];
};

// 16 lanes per row, 8 channels each.
template <class L, int BITS>
__device__ __forceinline__ void read_row(const ReadArgs& a, int which, const uint8_t* rec, int row, int h, int tok) {
  using R = Rec<L, BITS>;
  const int lane = threadIdx.x & 15;
  const uint16_t* scales = reinterpret_cast<const uint16_t*>(rec + R::kCodes) + row * L::G;
  uint32_t o[4];
  uint2 w;
  if constexpr (BITS == 4) {
    w.x = __ldg(reinterpret_cast<const uint32_t*>(rec + row * R::CW) + lane);
  } else {
    w = __ldg(reinterpret_cast<const uint2*>(rec + row * R::CW) + lane);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float s = bf16_bits_to_f32(__ldg(scales + group_at<L>(8 * lane + 2 * i)));
    float lo, hi;
    if constexpr (BITS == 4) {
      lo = static_cast<float>(static_cast<int>((w.x >> (8 * i)) & 15u) - 8);
      hi = static_cast<float>(static_cast<int>((w.x >> (8 * i + 4)) & 15u) - 8);
    } else {
      const uint32_t v = (i < 2 ? w.x : w.y) >> (16 * (i & 1));
      lo = static_cast<float>(static_cast<int>(v & 255u) - 128);
      hi = static_cast<float>(static_cast<int>((v >> 8) & 255u) - 128);
    }
    o[i] = pack_bf16x2(lo * s, hi * s);
  }
  st_global_v4(a.out[which] + tok * a.stride[which] + h * D + 8 * lane, make_uint4(o[0], o[1], o[2], o[3]));
}

template <class L, int KB, int VB, bool NEW>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ ReadArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int s = find_seq<NEW>(a.p, blockIdx.x);
  const kvq_paged_seq q = a.p.seqs[s];
  const int start = NEW ? q.kv_len - q.q_len : 0;
  const int blk = start / kBlock + (static_cast<int>(blockIdx.x) - (NEW ? q.q_block : q.kv_block));
  const int row = threadIdx.x >> 4;
  const int pos = blk * kBlock + row;
  if (pos < start || pos >= q.kv_len) return;
  const int tok = (NEW ? q.q_first : q.kv_first) + pos - start;
  const int h = blockIdx.y;
  bool ok;
  const int64_t b = a.p.block(s, h, blk, ok);
  if (blockIdx.z == 0)
    read_row<L, KB>(a, 0, a.pages[0] + b * Rec<L, KB>::kBytes, row, h, tok);
  else
    read_row<L, VB>(a, 1, a.pages[1] + b * Rec<L, VB>::kBytes, row, h, tok);
}

static int check_rows(const void* k, int64_t ks, const void* v, int64_t vs, int n_heads, const char* what) {
  KVQ_REQUIRE(k && v, KVQ_ERR_ARG, "NULL %s pointer", what);
  KVQ_REQUIRE(ks >= (int64_t)n_heads * D && vs >= (int64_t)n_heads * D, KVQ_ERR_ARG,
              "%s token strides must be >= heads*head_dim", what);
  KVQ_REQUIRE((reinterpret_cast<uintptr_t>(k) & 15) == 0 && (reinterpret_cast<uintptr_t>(v) & 15) == 0 &&
                  ks % 8 == 0 && vs % 8 == 0,
              KVQ_ERR_ALIGN, "%s must be 16-byte aligned with token strides that are multiples of 8", what);
  return KVQ_OK;
}

}  // namespace paged
}  // namespace kvq

using namespace kvq;

extern "C" int kvq_paged_append(const void* k, int64_t k_token_stride, const void* v, int64_t v_token_stride,
                                const kvq_paged_cache* cache, const kvq_paged_batch* batch, void* stream) {
  clear_error();
  int layout = 0;
  int rc = paged::check_cache(cache, batch, &layout);
  if (rc) return rc;
  if (batch->n_seqs == 0 || batch->n_new == 0) return KVQ_OK;
  rc = paged::check_rows(k, k_token_stride, v, v_token_stride, cache->n_heads, "k and v");
  if (rc) return rc;
  rc = require_sm100();
  if (rc) return rc;
  paged::AppendArgs a;
  a.p = paged::make_pages(cache, batch);
  a.x[0] = static_cast<const uint16_t*>(k);
  a.x[1] = static_cast<const uint16_t*>(v);
  a.stride[0] = k_token_stride;
  a.stride[1] = v_token_stride;
  a.pages[0] = static_cast<uint8_t*>(cache->k_pages);
  a.pages[1] = static_cast<uint8_t*>(cache->v_pages);
  const dim3 grid(static_cast<unsigned>(batch->n_new_blocks), (cache->n_heads + 7) / 8, 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return paged::with_layout(layout, [&](auto l) {
    using L = decltype(l);
    return paged::with_bits(cache->k_bits, cache->v_bits, [&](auto b) {
      using B = decltype(b);
      paged::append_kernel<L, B::k, B::v><<<grid, 128, 0, st>>>(a);
      return check_launch("kvq_paged_append");
    });
  });
}

extern "C" int kvq_paged_read(const kvq_paged_cache* cache, const kvq_paged_batch* batch, int new_only, void* k_out,
                              int64_t k_out_token_stride, void* v_out, int64_t v_out_token_stride, void* stream) {
  clear_error();
  int layout = 0;
  int rc = paged::check_cache(cache, batch, &layout);
  if (rc) return rc;
  if (batch->n_seqs == 0 || (new_only ? batch->n_new : batch->n_tokens) == 0) return KVQ_OK;
  rc = paged::check_rows(k_out, k_out_token_stride, v_out, v_out_token_stride, cache->n_heads, "k_out and v_out");
  if (rc) return rc;
  rc = require_sm100();
  if (rc) return rc;
  paged::ReadArgs a;
  a.p = paged::make_pages(cache, batch);
  a.pages[0] = static_cast<const uint8_t*>(cache->k_pages);
  a.pages[1] = static_cast<const uint8_t*>(cache->v_pages);
  a.out[0] = static_cast<uint16_t*>(k_out);
  a.out[1] = static_cast<uint16_t*>(v_out);
  a.stride[0] = k_out_token_stride;
  a.stride[1] = v_out_token_stride;
  const dim3 grid(static_cast<unsigned>(new_only ? batch->n_new_blocks : batch->n_blocks), cache->n_heads, 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return paged::with_layout(layout, [&](auto l) {
    using L = decltype(l);
    return paged::with_bits(cache->k_bits, cache->v_bits, [&](auto b) {
      using B = decltype(b);
      if (new_only)
        paged::read_kernel<L, B::k, B::v, true><<<grid, 256, 0, st>>>(a);
      else
        paged::read_kernel<L, B::k, B::v, false><<<grid, 256, 0, st>>>(a);
      return check_launch("kvq_paged_read");
    });
  });
}
