// Host-side plan of one attention step over a paged batch (kvq_paged_plan).
#include <algorithm>
#include <cstring>
#include <new>
#include <vector>

#include "kvq_paged.cuh"

namespace kvq {
namespace paged {

struct Unit {
  int32_t seq, row0, n_rows, n_sink, first, n;  // n: entries of the block list
};

// The storage blocks that rows [row0, row0 + n_rows) of a sequence see between them.
static Unit make_unit(int seq, int kv_len, int q_len, int group, int row0, int n_rows, int causal, int64_t window,
                      int64_t sink) {
  const int64_t start = static_cast<int64_t>(kv_len) - q_len;
  const int64_t p0 = start + row0 / group, p1 = start + (row0 + n_rows - 1) / group;
  const int64_t hi = std::max<int64_t>(0, causal ? std::min<int64_t>(p1 + 1, kv_len) : kv_len);
  const int64_t lo = window > 0 ? std::min(hi, std::max<int64_t>(0, p0 + 1 - window)) : 0;
  const int64_t kept = window > 0 ? std::min(sink, hi) : 0;
  const int64_t b1 = (hi + kBlock - 1) / kBlock;
  const int64_t b0 = std::min(lo / kBlock, b1);
  const int64_t ns = std::min((kept + kBlock - 1) / kBlock, b0);
  return Unit{seq, row0, n_rows, static_cast<int32_t>(ns), static_cast<int32_t>(b0),
              static_cast<int32_t>(ns + b1 - b0)};
}

struct Plan {
  std::vector<Item> rows, tiles;
  std::vector<int32_t> cta_first;
  int units = 0, slots = 0, tile_slots = 0, row_tile = 8;
};

// Few rows: the work of all units is one line of blocks (an empty unit counts as
// one), cut into equal pieces, one per resident block of the device, so every block
// streams the same number of bytes whatever the lengths are; a piece is made of the
// whole or partial units it meets. No piece is shorter than kMinBlocks blocks, and
// no unit gets more than kMaxParts parts.
constexpr int kMinBlocks = 8;

static void cut_rows(const std::vector<Unit>& units, int n_heads, int n_sms, Plan* p) {
  int64_t total = 0, longest = 0;
  for (const Unit& u : units) {
    total += static_cast<int64_t>(std::max(u.n, 1)) * n_heads;
    longest = std::max<int64_t>(longest, u.n);
  }
  if (total == 0) return;
  const int64_t most = static_cast<int64_t>(n_sms) * kRowCtasPerSm;
  int64_t piece = std::max<int64_t>({(total + most - 1) / most, kMinBlocks, (longest + kMaxParts - 2) / (kMaxParts - 1)});
  const int64_t n_ctas = (total + piece - 1) / piece;
  p->cta_first.push_back(0);
  int64_t at = 0;  // position on the line
  for (const Unit& u : units) {
    const int len = std::max(u.n, 1);
    for (int h = 0; h < n_heads; ++h, at += len) {
      const int64_t c0 = at / piece, c1 = (at + len - 1) / piece;
      const int parts = static_cast<int>(c1 - c0 + 1);
      for (int64_t c = c0; c <= c1; ++c) {
        while (static_cast<int64_t>(p->cta_first.size()) <= c)
          p->cta_first.push_back(static_cast<int32_t>(p->rows.size()));
        const int64_t b = std::max(c * piece, at) - at, e = std::min((c + 1) * piece, at + len) - at;
        p->rows.push_back(Item{u.seq, h, u.row0, u.n_rows, u.n_sink, u.first, static_cast<int32_t>(std::min<int64_t>(b, u.n)),
                               static_cast<int32_t>(std::min<int64_t>(e, u.n)), static_cast<int32_t>(c - c0), parts,
                               parts > 1 ? p->units : -1, parts > 1 ? p->slots : -1});
      }
      if (parts > 1) {
        ++p->units;
        p->slots += parts;
      }
    }
  }
  while (static_cast<int64_t>(p->cta_first.size()) <= n_ctas)
    p->cta_first.push_back(static_cast<int32_t>(p->rows.size()));
}

// Many rows: one block of the device per item and SM, started in the order of the list.
// Long units first, whole while much work is left; later ones are cut so that no piece is
// longer than an equal share of the work that is left, and the last ones to run
// end together. No piece is shorter than kMinTiles tiles of four storage blocks, no
// unit has more than kMaxTileParts parts (their join is serial work of one block).
constexpr int kMinTiles = 8, kMaxTileParts = 32;

static void cut_tiles(std::vector<Unit>& units, int n_heads, int n_sms, Plan* p) {
  std::stable_sort(units.begin(), units.end(), [](const Unit& a, const Unit& b) { return a.n > b.n; });
  int64_t left = 0;
  for (const Unit& u : units) left += static_cast<int64_t>((u.n + 3) / 4) * n_heads;
  for (const Unit& u : units) {
    const int64_t t = (u.n + 3) / 4;
    for (int h = 0; h < n_heads; ++h, left -= t) {
      const int64_t piece = std::max<int64_t>(kMinTiles, left / n_sms);
      const int parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((t + piece - 1) / piece, kMaxTileParts)));
      for (int i = 0; i < parts; ++i)
        p->tiles.push_back(Item{u.seq, h, u.row0, u.n_rows, u.n_sink, u.first, static_cast<int32_t>(4 * (t * i / parts)),
                                static_cast<int32_t>(std::min<int64_t>(u.n, 4 * (t * (i + 1) / parts))), i, parts,
                                parts > 1 ? p->units : -1, parts > 1 ? p->tile_slots : -1});
      if (parts > 1) {
        ++p->units;
        p->tile_slots += parts;
      }
    }
  }
}

// Up to kFewRows rows of a sequence and KV head go to the kernel for few rows.
constexpr int kFewRows = 16;

static int make_plan(const int32_t* kv_lens, const int32_t* q_lens, int n_seqs, int n_heads, int group, int causal,
                     int64_t window, int64_t sink, int n_sms, Plan* p) {
  std::vector<Unit> few, many;
  for (int s = 0; s < n_seqs; ++s) {
    const int64_t rows = static_cast<int64_t>(q_lens[s]) * group;
    const int tile = rows <= kFewRows ? kFewRows : kTileRows;
    for (int64_t r = 0; r < rows; r += tile) {
      const int n = static_cast<int>(std::min<int64_t>(tile, rows - r));
      (rows <= kFewRows ? few : many)
          .push_back(make_unit(s, kv_lens[s], q_lens[s], group, static_cast<int>(r), n, causal, window, sink));
      if (rows <= kFewRows && rows > 8) p->row_tile = 16;
    }
  }
  KVQ_REQUIRE(static_cast<int64_t>(few.size() + many.size()) * n_heads < (1 << 24), KVQ_ERR_ARG,
              "too many rows for one launch");
  cut_rows(few, n_heads, n_sms, p);
  cut_tiles(many, n_heads, n_sms, p);
  return KVQ_OK;
}

}  // namespace paged
}  // namespace kvq

using namespace kvq;

extern "C" int kvq_paged_plan(const int32_t* kv_lens, const int32_t* q_lens, int n_seqs, int n_heads, int n_q_heads,
                              int causal, int64_t window, int64_t sink, int n_sms, int32_t* out, int64_t capacity,
                              kvq_paged_plan_info* info) {
  clear_error();
  KVQ_REQUIRE(info != nullptr, KVQ_ERR_ARG, "NULL info");
  KVQ_REQUIRE(n_seqs >= 0 && n_sms >= 1 && (n_seqs == 0 || (kv_lens && q_lens)), KVQ_ERR_ARG, "bad lengths");
  KVQ_REQUIRE(n_heads >= 1 && n_heads <= 65535 && n_q_heads >= n_heads && n_q_heads <= 65535 && n_q_heads % n_heads == 0,
              KVQ_ERR_ARG, "%d query heads are not a multiple of %d KV heads", n_q_heads, n_heads);
  KVQ_REQUIRE(window >= 0 && sink >= 0, KVQ_ERR_ARG, "window and sink must be >= 0");
  const int group = n_q_heads / n_heads;
  for (int s = 0; s < n_seqs; ++s) {
    KVQ_REQUIRE(kv_lens[s] >= 0 && q_lens[s] >= 0, KVQ_ERR_ARG, "negative length of sequence %d", s);
    KVQ_REQUIRE(static_cast<int64_t>(q_lens[s]) * group < ((int64_t)1 << 31), KVQ_ERR_ARG, "too many queries");
  }
  try {
    paged::Plan p;
    const int rc = paged::make_plan(kv_lens, q_lens, n_seqs, n_heads, group, causal ? 1 : 0, window, sink, n_sms, &p);
    if (rc) return rc;
    *info = kvq_paged_plan_info{};
    info->n_row_items = static_cast<int32_t>(p.rows.size());
    info->n_row_ctas = p.cta_first.empty() ? 0 : static_cast<int32_t>(p.cta_first.size()) - 1;
    info->n_tile_items = static_cast<int32_t>(p.tiles.size());
    info->row_tile = p.row_tile;
    info->n_units = p.units;
    info->words = static_cast<int64_t>(p.rows.size() + p.tiles.size()) * 12 + static_cast<int64_t>(p.cta_first.size());
    info->tile_workspace_offset = (static_cast<int64_t>(p.slots) * paged::slot_floats(p.row_tile) * 4 + 255) / 256 * 256;
    info->workspace_bytes = info->tile_workspace_offset + p.tile_slots * paged::kTileSlotBytes;
    if (!out) return KVQ_OK;
    KVQ_REQUIRE(capacity >= info->words, KVQ_ERR_ARG, "the plan needs %lld words", (long long)info->words);
    auto put = [&out](const void* src, size_t words) {
      if (words) std::memcpy(out, src, words * 4);
      out += words;
    };
    put(p.rows.data(), p.rows.size() * 12);
    put(p.tiles.data(), p.tiles.size() * 12);
    put(p.cta_first.data(), p.cta_first.size());
  } catch (const std::bad_alloc&) {
    set_error("kvq_paged_plan: out of host memory");
    return KVQ_ERR_ARG;
  }
  return KVQ_OK;
}
