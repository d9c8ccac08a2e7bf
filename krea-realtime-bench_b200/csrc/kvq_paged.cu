// Paged quantized cache: writing new tokens into their pages and reading tokens
// back (sm_100a), and the checks shared with the attention over it.
//
// Append. Per (token, head) row x and channel group g: s_g = max_g |x| / qmax (1
// where that is 0), code = rne(x / s_g) + offset, stored scale bf16(s_g): the
// arithmetic of kvq_quantize, bit for bit, with rows going to pages.
#include <algorithm>

#include "kvq_paged_dev.cuh"
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
                  b->n_new <= lim && b->n_tokens <= lim && b->n_new_blocks <= lim && b->n_blocks <= lim &&
                  b->table_stride >= 0,
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

constexpr int kHeadsPerCta = 8;                      // heads of one tile
constexpr int kTileRowsA = kBlock * kHeadsPerCta;    // rows of one tile, a thread each

// 16-byte chunk c of row r in the staged input and in the staged codes: the XOR spreads
// the threads' equal chunks of consecutive rows over the banks.
__device__ __forceinline__ int in_slot(int r, int c) { return r * 16 + (c ^ (r & 7)); }
template <int BITS>
__device__ __forceinline__ int code_slot(int r, int c) {
  return BITS == 4 ? r * 4 + (c ^ ((r >> 1) & 3)) : r * 8 + (c ^ (r & 7));
}

// Rare path: the groups flagged in slow_mask (amax below 2^-100, above 3e38 or not
// finite) with the IEEE divide; NaN counts as 0, magnitudes above 3e38 as 3e38.
template <class L, int BITS>
__device__ __noinline__ void fix_slow(const uint4* tin, int r, uint32_t slow_mask, uint4* sm_codes, uint16_t* scales) {
  using C = QuantConsts<BITS>;
  constexpr float q = static_cast<float>(C::kQmax), top = 3.0e38f;
  int edges[L::G + 1];
  fill_edges<L>(edges, std::make_integer_sequence<int, L::G + 1>{});
  auto value = [&](int c) {
    const float v = bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(tin + in_slot(r, c >> 3))[c & 7]);
    return v == v ? v : 0.0f;
  };
  for (int g = 0; slow_mask; ++g, slow_mask >>= 1) {
    if (!(slow_mask & 1u)) continue;
    float amax = 0.0f;
    for (int c = edges[g]; c < edges[g + 1]; ++c) amax = fmaxf(amax, fminf(fabsf(value(c)), top));
    float s = __fdiv_rn(amax, q);
    s = s > 0.0f ? s : 1.0f;
    scales[g] = f32_to_bf16_bits(s);
    for (int c = edges[g]; c < edges[g + 1]; ++c) {
      const uint32_t code = code_exact(value(c), s, q, C::kMagic) & 0xFFu;
      const int b = BITS == 4 ? c >> 1 : c;
      uint8_t& o = reinterpret_cast<uint8_t*>(sm_codes + code_slot<BITS>(r, b >> 4))[b & 15];
      if constexpr (BITS == 4)
        o = (c & 1) ? static_cast<uint8_t>((o & 0x0F) | (code << 4)) : static_cast<uint8_t>((o & 0xF0) | code);
      else
        o = static_cast<uint8_t>(code);
    }
  }
}

// Bound by latency at few tokens; at many by memory and the quantization's instructions
// alike (4680 tokens of 40 heads, bands4: 129 MB in 29.4 us, 4.4 TB/s, 69 % of the issue
// slots; 9 prompts of 129 to 1531 tokens, 10 heads, int8: 14.0 us; 24 single tokens of 8
// heads 3.5 us on the device). One CTA per tile of 16 tokens
// (one storage block) x 8 heads of K or V: the rows arrive by cp.async (a token's heads
// are contiguous: 2 KB runs), thread r quantizes row r = 16 head + token, and each head's
// record, contiguous in its page, is written with 16-byte stores; a block that the step
// fills partly is written row by row. Several CTAs per SM overlap the three phases.
template <class L, int BITS>
__device__ __forceinline__ void append_tile(const AppendArgs& a, int which, int s, int blk, int row0, int n_tok, int tok0,
                                            uint8_t* smem) {
  using R = Rec<L, BITS>;
  constexpr int CCH = R::CW / 16;  // code chunks per row
  uint4* tin = reinterpret_cast<uint4*>(smem);
  uint4* sm_codes = tin + kTileRowsA * 16;
  uint16_t* sm_sc = reinterpret_cast<uint16_t*>(sm_codes + kTileRowsA * CCH);
  const int tid = threadIdx.x;
  const int h0 = blockIdx.y * kHeadsPerCta, nh = min(kHeadsPerCta, a.p.n_heads - h0);
  // tokens row0 .. row0 + n_tok of the block; copies in the order of memory
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(tin));
  for (int i = tid; i < n_tok * nh * 16; i += kTileRowsA) {
    const int c = i & 15, j = i >> 4, t = j / nh, h = j - t * nh, r = h * kBlock + row0 + t;
    const uint16_t* src = a.x[which] + static_cast<int64_t>(tok0 + t) * a.stride[which] + (h0 + h) * D + 8 * c;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + in_slot(r, c) * 16), "l"(src) : "memory");
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  const int t = tid & (kBlock - 1), h = tid >> 4;
  if (h < nh && t >= row0 && t < row0 + n_tok) {
    uint32_t w[64];
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const uint4 v = tin[in_slot(tid, c)];
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
#pragma unroll
    for (int c = 0; c < CCH; ++c)
      sm_codes[code_slot<BITS>(tid, c)] = make_uint4(ow[4 * c], ow[4 * c + 1], ow[4 * c + 2], ow[4 * c + 3]);
#pragma unroll
    for (int g = 0; g < L::G; ++g) sm_sc[tid * L::G + g] = sc[g];
    if (slow) fix_slow<L, BITS>(tin, tid, slow, sm_codes, sm_sc + tid * L::G);
  }
  __syncthreads();
  bool ok;
  const int64_t rec = a.p.block(s, h0, blk, ok);  // the next head's record is (1 << page_shift) records on
  if (!ok) return;
  uint8_t* out = a.pages[which] + rec * R::kBytes;
  const int64_t head_bytes = static_cast<int64_t>(R::kBytes) << a.p.page_shift;
  for (int i = tid; i < n_tok * nh * CCH; i += kTileRowsA) {
    const int hh = i / (n_tok * CCH), k = i - hh * (n_tok * CCH), r = row0 + k / CCH, c = k % CCH;
    st_global_v4(out + hh * head_bytes + r * R::CW + 16 * c, sm_codes[code_slot<BITS>(hh * kBlock + r, c)]);
  }
  if (n_tok == kBlock) {
    constexpr int SCH = 2 * L::G;  // 16-byte chunks of a block's scales
    for (int i = tid; i < nh * SCH; i += kTileRowsA) {
      const int hh = i / SCH, c = i - hh * SCH;
      st_global_v4(out + hh * head_bytes + R::kCodes + 16 * c, reinterpret_cast<const uint4*>(sm_sc + hh * kBlock * L::G)[c]);
    }
  } else {
    for (int i = tid; i < n_tok * nh * L::G; i += kTileRowsA) {
      const int hh = i / (n_tok * L::G), k = i - hh * (n_tok * L::G);
      reinterpret_cast<uint16_t*>(out + hh * head_bytes + R::kCodes)[row0 * L::G + k] =
          sm_sc[(hh * kBlock + row0) * L::G + k];
    }
  }
}

template <class L, int BITS>
constexpr int append_smem() {
  return kTileRowsA * (256 + Rec<L, BITS>::CW + 2 * L::G);
}

template <class L, int KB, int VB>
__global__ void __launch_bounds__(kTileRowsA, 3) append_kernel(const __grid_constant__ AppendArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  pdl_wait();
  pdl_launch_dependents();
  const int s = find_seq<true>(a.p, blockIdx.x);
  const kvq_paged_seq q = a.p.seqs[s];
  const int start = q.kv_len - q.q_len;
  const int blk = max(start, 0) / kBlock + (static_cast<int>(blockIdx.x) - q.q_block);
  const int row0 = max(start - blk * kBlock, 0), n_tok = min(kBlock, q.kv_len - blk * kBlock) - row0;
  if (n_tok <= 0) return;
  const int tok0 = q.q_first + blk * kBlock + row0 - start;
  if (blockIdx.z == 0)
    append_tile<L, KB>(a, 0, s, blk, row0, n_tok, tok0, smem);
  else
    append_tile<L, VB>(a, 1, s, blk, row0, n_tok, tok0, smem);
}

// ---------------------------------------------------------------- read
struct ReadArgs {
  Pages p;
  const uint8_t* pages[2];
  uint16_t* out[2];
  int64_t stride[2];
};

// Bound by memory (32760 tokens of 40 heads, bands4: 902 MB in 165 us, 5.46 TB/s, 83 % of
// what a copy reaches). One CTA per storage block and tensor, all heads, 16 lanes per row and
// eight channels per lane, so a warp reads contiguous codes and writes 256-byte rows.
// kHeadsAtOnce heads are loaded before the first is converted. An aligned run of eight
// channels meets at most two groups.
constexpr int kHeadsAtOnce = 4;

template <class L, int BITS>
__device__ __forceinline__ void read_block(const ReadArgs& a, int which, int64_t rec, int row, bool live, int64_t tok) {
  using R = Rec<L, BITS>;
  const int lane = threadIdx.x & 15;
  const int ga = group_at<L>(8 * lane), gb = group_at<L>(8 * lane + 7);
  int split = 4;  // first channel pair of the second group
#pragma unroll
  for (int i = 3; i > 0; --i)
    if (group_at<L>(8 * lane + 2 * i) != ga) split = i;
  const uint8_t* src = a.pages[which] + rec * R::kBytes + row * R::CW + lane * (BITS);
  const uint8_t* sc = a.pages[which] + rec * R::kBytes + R::kCodes + row * L::G * 2;
  const int64_t head_bytes = static_cast<int64_t>(R::kBytes) << a.p.page_shift;
  uint16_t* dst = a.out[which] + tok * a.stride[which] + 8 * lane;
  for (int h0 = 0; h0 < a.p.n_heads; h0 += kHeadsAtOnce) {
    uint2 w[kHeadsAtOnce];
    uint32_t sa[kHeadsAtOnce], sb[kHeadsAtOnce];
#pragma unroll
    for (int i = 0; i < kHeadsAtOnce; ++i) {
      if (h0 + i < a.p.n_heads && live) {
        const uint8_t* q = src + (h0 + i) * head_bytes;
        if constexpr (BITS == 4)
          w[i].x = __ldg(reinterpret_cast<const uint32_t*>(q));
        else
          w[i] = __ldg(reinterpret_cast<const uint2*>(q));
        const uint16_t* s = reinterpret_cast<const uint16_t*>(sc + (h0 + i) * head_bytes);
        sa[i] = __ldg(s + ga);
        sb[i] = __ldg(s + gb);
      }
    }
#pragma unroll
    for (int i = 0; i < kHeadsAtOnce; ++i) {
      if (h0 + i < a.p.n_heads && live) {
        uint32_t o[4];
        uint32_t pa = sa[i] * 0x10001u, pb = sb[i] * 0x10001u;
        if constexpr (BITS == 4) {
          pa = hmul2(pa, kFour);
          pb = hmul2(pb, kFour);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t v;
          if constexpr (BITS == 4)
            v = int4_low(__byte_perm(w[i].x, w[i].x >> 4, (4 + j) << 8 | j));
          else
            v = int8_pair(__byte_perm(j < 2 ? w[i].x : w[i].y, 0, (j & 1) ? 0x4342 : 0x4140));
          o[j] = hmul2(v, j >= split ? pb : pa);
        }
        st_global_v4(dst + (h0 + i) * D, make_uint4(o[0], o[1], o[2], o[3]));
      }
    }
  }
}

template <class L, int KB, int VB, bool NEW>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ ReadArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int s = find_seq<NEW>(a.p, blockIdx.x);
  const kvq_paged_seq q = a.p.seqs[s];
  const int start = NEW ? q.kv_len - q.q_len : 0;
  const int blk = max(start, 0) / kBlock + (static_cast<int>(blockIdx.x) - (NEW ? q.q_block : q.kv_block));
  const int row = threadIdx.x >> 4;
  const int pos = blk * kBlock + row;
  const bool live = pos >= start && pos < q.kv_len;
  if (blk * kBlock >= q.kv_len) return;
  const int64_t tok = static_cast<int64_t>(NEW ? q.q_first : q.kv_first) + pos - start;
  bool ok;
  const int64_t rec = a.p.block(s, 0, blk, ok);
  if (blockIdx.y == 0)
    read_block<L, KB>(a, 0, rec, row, live, tok);
  else
    read_block<L, VB>(a, 1, rec, row, live, tok);
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
  const dim3 grid(static_cast<unsigned>(batch->n_new_blocks), (cache->n_heads + paged::kHeadsPerCta - 1) / paged::kHeadsPerCta, 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return paged::with_layout(layout, [&](auto l) {
    using L = decltype(l);
    return paged::with_bits(cache->k_bits, cache->v_bits, [&](auto b) {
      using B = decltype(b);
      constexpr int smem = std::max(paged::append_smem<L, B::k>(), paged::append_smem<L, B::v>());
      static_assert(smem <= 227 * 1024, "shared memory");
      static bool configured[64];
      int dev = 0;
      cudaGetDevice(&dev);
      if (dev < 0 || dev >= 64 || !configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(paged::append_kernel<L, B::k, B::v>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        KVQ_REQUIRE(e == cudaSuccess, KVQ_ERR_CUDA, "cudaFuncSetAttribute(paged append): %s", cudaGetErrorString(e));
        if (dev >= 0 && dev < 64) configured[dev] = true;
      }
      cudaError_t e = launch_pdl(paged::append_kernel<L, B::k, B::v>, grid, paged::kTileRowsA, smem, st, a);
      KVQ_REQUIRE(e == cudaSuccess, KVQ_ERR_CUDA, "kvq_paged_append: launch failed: %s", cudaGetErrorString(e));
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
  const dim3 grid(static_cast<unsigned>(new_only ? batch->n_new_blocks : batch->n_blocks), 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return paged::with_layout(layout, [&](auto l) {
    using L = decltype(l);
    return paged::with_bits(cache->k_bits, cache->v_bits, [&](auto b) {
      using B = decltype(b);
      cudaError_t e = new_only ? launch_pdl(paged::read_kernel<L, B::k, B::v, true>, grid, 256, 0, st, a)
                               : launch_pdl(paged::read_kernel<L, B::k, B::v, false>, grid, 256, 0, st, a);
      KVQ_REQUIRE(e == cudaSuccess, KVQ_ERR_CUDA, "kvq_paged_read: launch failed: %s", cudaGetErrorString(e));
      return check_launch("kvq_paged_read");
    });
  });
}
