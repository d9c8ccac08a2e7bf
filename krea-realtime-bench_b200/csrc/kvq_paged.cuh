// Paged cache: addressing shared by the append, read and attention kernels.
#pragma once

#include <type_traits>
#include <utility>

#include "kvq_common.cuh"

namespace kvq {
namespace paged {

constexpr int D = 128;
constexpr int kBlock = 16;  // tokens of one storage block

// Bytes of one storage block: 16 code rows, then 16 rows of G bf16 scales.
template <class L, int BITS>
struct Rec {
  static constexpr int CW = BITS == 4 ? D / 2 : D;
  static constexpr int kCodes = kBlock * CW;
  static constexpr int kBytes = kCodes + kBlock * L::G * 2;
  static_assert(kBytes % 16 == 0, "blocks are copied 16 bytes at a time");
};

// Group of a channel that is known only at run time.
template <class L, int... Is>
__device__ __forceinline__ int group_at(int ch, std::integer_sequence<int, Is...>) {
  return (0 + ... + (ch >= std::integral_constant<int, L::E[Is + 1]>::value ? 1 : 0));
}
template <class L>
__device__ __forceinline__ int group_at(int ch) {
  return group_at<L>(ch, std::make_integer_sequence<int, L::G - 1>{});
}

// The batch and one of the cache's two pools, as the kernels take them.
struct Pages {
  const int32_t* table;
  int64_t table_stride;
  const kvq_paged_seq* seqs;
  int n_seqs, n_heads, n_pages;
  int page_shift;  // log2(blocks per page)

  // Storage block `blk` (token / 16) of sequence s, head h, as a block index of
  // the pool; `ok` is false where the table entry lies outside the pool.
  __device__ __forceinline__ int64_t block(int s, int h, int blk, bool& ok) const {
    int id = __ldg(table + s * table_stride + (blk >> page_shift));
    ok = static_cast<unsigned>(id) < static_cast<unsigned>(n_pages);
    id = ok ? id : 0;
    return (((static_cast<int64_t>(id) * n_heads + h) << page_shift) | (blk & ((1 << page_shift) - 1)));
  }
};

// First block and sequence of storage block `i` of the batch (all tokens, or the
// new ones): the sequence whose block sums enclose i.
template <bool NEW>
__device__ __forceinline__ int find_seq(const Pages& p, int i) {
  int lo = 0, hi = p.n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    const int first = NEW ? __ldg(&p.seqs[mid].q_block) : __ldg(&p.seqs[mid].kv_block);
    if (first <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Checks that hold for every entry point; fills the group layout.
int check_cache(const kvq_paged_cache* c, const kvq_paged_batch* b, int* layout);
Pages make_pages(const kvq_paged_cache* c, const kvq_paged_batch* b);

// Calls f(Layout{}) for the layout id.
template <class F>
int with_layout(int layout, F&& f) {
  switch (layout) {
    case kLayoutBands: return f(LayoutBands{});
    case kLayoutBands2: return f(LayoutBands2{});
    case kLayoutBands4: return f(LayoutBands4{});
    case kLayoutBlind32: return f(LayoutBlind32{});
    case kLayoutBlind64: return f(LayoutBlind64{});
    default: break;
  }
  set_error("internal: unhandled layout %d", layout);
  return KVQ_ERR_UNSUPPORTED;
}
template <int K, int V>
struct Bits {
  static constexpr int k = K, v = V;
};
template <class F>
int with_bits(int k_bits, int v_bits, F&& f) {
  if (k_bits == 4) return f(Bits<4, 4>{});
  return v_bits == 4 ? f(Bits<8, 4>{}) : f(Bits<8, 8>{});
}

}  // namespace paged
}  // namespace kvq
