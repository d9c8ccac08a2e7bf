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

// One piece of attention work: rows [row0, row0 + n_rows) of a sequence and KV head
// over entries [jb, je) of the list of storage blocks the rows see: blocks [0, n_sink),
// then first, first + 1, ... ; part `part` of `parts`, its partial result in workspace
// slot `slot` + part, its unit counted in counter `unit`; start = position of the
// sequence's first query, q_first = its index. (kvq_paged_plan)
struct alignas(16) Item {
  int32_t seq, head, row0, n_rows, n_sink, first, jb, je, part, parts, unit, slot;
  int32_t kv_len, start, q_first, reserved;
  __host__ __device__ __forceinline__ int block_at(int j) const { return j < n_sink ? j : first + (j - n_sink); }
};
static_assert(sizeof(Item) == 64, "the plan's layout");
constexpr int kItemWords = 16;

// Workspace of one part: O [rows][128] unnormalised, then m, l, F and an unused one per row
// (fp32): the running maximum, the sum, and the power of two that O is kept divided by.
__host__ __device__ constexpr int slot_floats(int rows) { return rows * (D + 4); }
// Most parts of a unit: joining them is serial work of one block.
constexpr int kMaxParts = 128;

// What both attention kernels take.
struct AttnArgs {
  Pages p;
  const uint16_t* q;
  int64_t q_stride;
  const uint8_t* k_pages;
  const uint8_t* v_pages;
  uint16_t* out;
  int64_t out_stride;
  float* lse;
  int group, n_q_heads;
  int causal;
  int64_t window, sink;
  float scale_log2;
  const Item* items;
  const int32_t* cta_first;
  float* ws;
  unsigned* ctr;
  int* status;  // the device status word (kvq_device_status)
  long long wait_cycles;
};

// Tokens [lo, hi) and [0, kept) that the query at position pos sees.
struct Seen {
  int lo, hi, kept;
};
__device__ __forceinline__ Seen seen_by(const AttnArgs& a, int pos, int kv_len) {
  Seen s;
  s.hi = a.causal ? min(pos + 1, kv_len) : kv_len;
  const int64_t lo = a.window > 0 ? static_cast<int64_t>(pos) + 1 - a.window : 0;
  s.lo = static_cast<int>(lo > 0 ? lo : 0);
  s.kept = a.window > 0 ? static_cast<int>(min(a.sink, static_cast<int64_t>(s.hi > 0 ? s.hi : 0))) : 0;
  return s;
}

// Workspace of one part in the kernel for many rows: two Q tiles of float4 [33][128 rows],
// 32 columns of O and one of (m, l, F).
constexpr int kTileRows = 256;
constexpr int64_t kTileSlotBytes = 2 * 33 * 128 * 16;

int launch_tiles(const AttnArgs& a, int layout, int k_bits, int v_bits, int n_items, cudaStream_t st);
// Resident blocks per SM of the kernel for few rows.
int rows_ctas_per_sm(int layout, int k_bits, int v_bits, int row_tile);
int launch_rows(const AttnArgs& a, int layout, int k_bits, int v_bits, int row_tile, int n_ctas, cudaStream_t st);

// Checks that hold for every entry point; fills the group layout.
int check_format(const kvq_paged_cache* c, int* layout);
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
