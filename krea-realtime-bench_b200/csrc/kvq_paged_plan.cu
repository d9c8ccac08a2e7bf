// Host-side plan of one attention step over a paged batch (kvq_paged_plan).
#include <algorithm>
#include <cstring>
#include <functional>
#include <new>
#include <vector>

#include "kvq_paged.cuh"

namespace kvq {
namespace paged {

struct Unit {
  int32_t seq, row0, n_rows, n_sink, first, n;  // n: entries of the block list
  int32_t kv_len, start, q_first;
};

// The storage blocks that rows [row0, row0 + n_rows) of a sequence see between them.
static Unit make_unit(int seq, int kv_len, int q_len, int64_t q_first, int group, int row0, int n_rows, int causal,
                      int64_t window, int64_t sink) {
  const int64_t start = static_cast<int64_t>(kv_len) - q_len;
  const int64_t p0 = start + row0 / group, p1 = start + (row0 + n_rows - 1) / group;
  const int64_t hi = std::max<int64_t>(0, causal ? std::min<int64_t>(p1 + 1, kv_len) : kv_len);
  const int64_t lo = window > 0 ? std::min(hi, std::max<int64_t>(0, p0 + 1 - window)) : 0;
  const int64_t kept = window > 0 ? std::min(sink, hi) : 0;
  const int64_t b1 = (hi + kBlock - 1) / kBlock;
  const int64_t b0 = std::min(lo / kBlock, b1);
  const int64_t ns = std::min((kept + kBlock - 1) / kBlock, b0);
  return Unit{seq, row0, n_rows, static_cast<int32_t>(ns), static_cast<int32_t>(b0), static_cast<int32_t>(ns + b1 - b0),
              kv_len, static_cast<int32_t>(start), static_cast<int32_t>(q_first)};
}

static Item make_item(const Unit& u, int head, int64_t jb, int64_t je, int part, int parts, int unit, int slot) {
  return Item{u.seq, head, u.row0, u.n_rows, u.n_sink, u.first, static_cast<int32_t>(jb), static_cast<int32_t>(je), part,
              parts, parts > 1 ? unit : -1, parts > 1 ? slot : -1, u.kv_len, u.start, u.q_first, 0};
}

struct Plan {
  std::vector<Item> rows, tiles;
  std::vector<int32_t> cta_first;
  int units = 0, slots = 0, tile_slots = 0, row_tile = 8, row_ctas = 0;
};

// Few rows. Two ways to cut the units, by an estimate in microseconds of the blocks'
// work: rounds of kRound storage blocks (two for each warp of a block of threads), the
// join of a unit's parts, and what any join costs; for 8 and 16 rows, fitted to graph
// replays of 1 to 8 sequences of 400 to 8000 tokens, 8 KV heads. It says nothing of what an
// item costs, and the first way is not tried below 9 storage blocks: batches of short
// contexts, whose whole units become items one after the other on a line, are far from
// one wave's latency (64 sequences of 16 tokens 49 us, of 20 to 300 tokens 31, one of 100 14).
// - Each unit by itself into equal parts, of which all are resident at once: a block of
//   threads has one item and waits for its data once.
// - The units as one line of storage blocks (an empty unit counts as one), cut into equal
//   pieces, one per resident block of threads: each streams the same number of bytes
//   whatever the lengths are; a piece is made of the whole or partial units it meets, two
//   joins in the common case.
// Measured: 8 sequences of 3000 tokens by units 15.7 us, as a line 18.9; one of 8000 in 16
// parts a head 11.8, in 32 12.9; one of 400 whole 7.3, in two parts 8.6; one of 1561 in 7
// parts 8.5, in 4 11.0. No unit gets more than kMaxParts parts.
constexpr int kRound = 8;
constexpr double kRoundCost[2] = {1.4, 1.9}, kRowPart[2] = {0.17, 0.44}, kRowJoin = 3.0;

static double row_cost(int row_tile, int64_t piece, int64_t parts) {
  const int w = row_tile > 8;
  return kRoundCost[w] * static_cast<double>((piece + kRound - 1) / kRound) +
         (parts > 1 ? kRowJoin + kRowPart[w] * static_cast<double>(parts) : 0.0);
}

static void cut_rows(const std::vector<Unit>& units, int n_heads, int64_t n_resident, Plan* p) {
  int64_t total = 0, longest = 0;
  for (const Unit& u : units) {
    total += static_cast<int64_t>(std::max(u.n, 1)) * n_heads;
    longest = std::max<int64_t>(longest, u.n);
  }
  if (total == 0) return;
  int64_t piece = std::max<int64_t>(
      {(total + n_resident - 1) / n_resident, 2 * kRound, (longest + kMaxParts - 2) / (kMaxParts - 1)});
  const int64_t n_ctas = (total + piece - 1) / piece;
  // the line, as two items a block of threads
  double least = row_cost(p->row_tile, piece + kRound, (longest + piece - 1) / piece + 1) + kRowJoin;
  int64_t by_unit = 0;  // piece of the first way
  if (static_cast<int64_t>(units.size()) * n_heads <= n_resident) {
    for (int64_t c = 2 * kRound; c < longest + kRound; c += kRound) {
      const int64_t parts = (longest + c - 1) / c;
      const double cost = row_cost(p->row_tile, (longest + parts - 1) / parts, parts);
      if (parts > kMaxParts || cost >= least) continue;
      int64_t all = 0;
      for (const Unit& u : units) all += std::max<int64_t>(1, (u.n + c - 1) / c) * n_heads;
      if (all > n_resident) continue;
      least = cost;
      by_unit = c;
    }
    if (longest == 0) by_unit = kRound;  // nothing to see: the rows still have to be written
  }
  p->rows.reserve(units.size() * n_heads + n_ctas);
  if (by_unit) {
    for (const Unit& u : units)
      for (int h = 0; h < n_heads; ++h) {
        const int64_t parts = std::max<int64_t>(1, (u.n + by_unit - 1) / by_unit);
        for (int64_t k = 0; k < parts; ++k)
          p->rows.push_back(make_item(u, h, u.n * k / parts, u.n * (k + 1) / parts, static_cast<int>(k),
                                      static_cast<int>(parts), p->units, p->slots));
        if (parts > 1) {
          ++p->units;
          p->slots += static_cast<int>(parts);
        }
      }
    p->row_ctas = static_cast<int>(p->rows.size());
    return;
  }
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
        p->rows.push_back(make_item(u, h, std::min<int64_t>(b, u.n), std::min<int64_t>(e, u.n), static_cast<int>(c - c0),
                                    parts, p->units, p->slots));
      }
      if (parts > 1) {
        ++p->units;
        p->slots += parts;
      }
    }
  }
  while (static_cast<int64_t>(p->cta_first.size()) <= n_ctas)
    p->cta_first.push_back(static_cast<int32_t>(p->rows.size()));
  p->row_ctas = static_cast<int>(n_ctas);
}

// Many rows: one CTA per item and SM, started in the order of the list, long units first.
// Which units are cut into parts, and into how many, is chosen by simulating that list
// on the SMs for a few ways to cut it: none; all units, the units behind the last full
// wave, or those and one wave more, into the smallest equal pieces of which there are
// at most one to three waves. Costs in tiles of 64 tokens, measured (a tile of two Q
// tiles takes about 2100 cycles): kItemCost for an item (fill, epilogue), kPartCost
// more for a part's partial sums, kJoinCost and kJoinPart per part for the join.
// Lists of more than kSimWaves waves are left whole: the last wave is a small share.
constexpr double kItemCost = 4.0, kPartCost = 0.5, kJoinCost = 1.5, kJoinPart = 0.5;
constexpr int kMinTiles = 4, kMaxTileParts = 32, kSimWaves = 8;

struct Cut {
  size_t from;    // units (heads multiplied) from this one on are cut
  int64_t piece;  // into the fewest parts of at most this many tiles (0: none are)
  int parts(size_t i, int64_t t) const {
    if (i < from || piece <= 0) return 1;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((t + piece - 1) / piece, kMaxTileParts)));
  }
};

static double simulate(const std::vector<Unit>& units, int n_heads, int n_sms, const Cut& cut) {
  std::vector<double> busy(static_cast<size_t>(n_sms), 0.0);  // heap of the SMs' finishing times
  const std::greater<double> later;
  double end = 0.0;
  size_t i = 0;
  for (const Unit& u : units) {
    const int64_t t = (u.n + 3) / 4;
    const double pace = u.n_rows > 128 ? 1.0 : 0.65;  // measured: 0.62 int4, 0.69 int8
    for (int h = 0; h < n_heads; ++h, ++i) {
      const int parts = cut.parts(i, t);
      const double cost = pace * static_cast<double>(t) / parts + kItemCost + (parts > 1 ? kPartCost : 0.0);
      for (int k = 0; k < parts; ++k) {
        std::pop_heap(busy.begin(), busy.end(), later);
        busy.back() += cost + (parts > 1 && k + 1 == parts ? kJoinCost + kJoinPart * parts : 0.0);
        end = std::max(end, busy.back());
        std::push_heap(busy.begin(), busy.end(), later);
      }
    }
  }
  return end;
}

static void cut_tiles(std::vector<Unit>& units, int n_heads, int n_sms, Plan* p) {
  if (units.empty()) return;
  std::stable_sort(units.begin(), units.end(), [](const Unit& a, const Unit& b) { return a.n > b.n; });
  const size_t n = units.size() * n_heads, wave = static_cast<size_t>(n_sms);
  Cut best{n, 0};
  if (n <= kSimWaves * wave) {
    double least = simulate(units, n_heads, n_sms, best);
    const size_t rest = n % wave;
    const size_t tail[3] = {n, rest, rest + wave};
    for (int m = 0; m < 3; ++m) {
      if (tail[m] == 0 || tail[m] > n || (m > 0 && tail[m] == n)) continue;
      for (int k = 1; k <= 3; ++k) {
        // the smallest piece that gives at most k waves
        Cut c{n - tail[m], 0};
        int64_t lo = kMinTiles, hi = (units.front().n + 3) / 4 + 1;
        while (lo < hi) {
          c.piece = (lo + hi) / 2;
          size_t pieces = 0, i = 0;
          for (const Unit& u : units)
            for (int h = 0; h < n_heads; ++h, ++i)
              if (i >= c.from) pieces += c.parts(i, (u.n + 3) / 4);
          if (pieces <= wave * k) hi = c.piece; else lo = c.piece + 1;
        }
        c.piece = lo;
        const double end = simulate(units, n_heads, n_sms, c);
        if (end < least * 0.98) {  // a cut has to be worth something
          least = end;
          best = c;
        }
      }
    }
  }
  size_t i = 0;
  for (const Unit& u : units) {
    const int64_t t = (u.n + 3) / 4;
    for (int h = 0; h < n_heads; ++h, ++i) {
      const int parts = best.parts(i, t);
      for (int k = 0; k < parts; ++k)
        p->tiles.push_back(make_item(u, h, 4 * (t * k / parts), std::min<int64_t>(u.n, 4 * (t * (k + 1) / parts)), k, parts,
                                     p->units, p->tile_slots));
      if (parts > 1) {
        ++p->units;
        p->tile_slots += parts;
      }
    }
  }
}

// Up to kFewRows rows of a sequence and KV head go to the kernel for few rows: 16 rows,
// 64 sequences of 946 to 16384 tokens, 8 KV heads 253 us, on the other kernel 401. Up to
// kMidRows do, in tiles of 16 rows that each read the cache, where all sequences are such
// and the work is at most kMidBlocks storage blocks per resident block of threads: 24 rows,
// one sequence of 1561 tokens 13.1 us, on the other kernel 21.9; 64 rows, one of 8000 tokens
// (54 blocks) 24.4, 33.4; 8 sequences of 3000 tokens, 24 rows (81 blocks) 31.7, 34.6; 8 of
// 1500, 64 rows (81) 27.5, 25.7; 12 with 32 to 48 rows, int8 (126) 44.8, 39.3: at the limit
// each is a tenth faster for one of two batches. Rows on both sides of 16 cost two launches
// else: 12 sequences with 16 to 24 rows 31.1, 51.7. (17 to 64 rows beside a sequence with
// more go to the other kernel without a measurement.)
constexpr int kFewRows = 16, kMidRows = 64, kMidBlocks = 80;

static int make_plan(const kvq_paged_cache* c, int layout, const int32_t* kv_lens, const int32_t* q_lens, int n_seqs,
                     int group, int causal, int64_t window, int64_t sink, int n_sms, Plan* p) {
  auto resident = [&](int row_tile) {
    return static_cast<int64_t>(n_sms) * rows_ctas_per_sm(layout, c->k_bits, c->v_bits, row_tile);
  };
  int64_t most = 0, q_sum = 0, n_least = 0;  // rows of a sequence and KV head, queries, fewest units
  for (int s = 0; s < n_seqs; ++s) {
    const int64_t rows = static_cast<int64_t>(q_lens[s]) * group;
    most = std::max(most, rows);
    q_sum += q_lens[s];
    n_least += (rows + kTileRows - 1) / kTileRows;
  }
  KVQ_REQUIRE(q_sum < ((int64_t)1 << 31) && n_least * c->n_heads < (1 << 24), KVQ_ERR_ARG, "too many rows for one launch");
  std::vector<Unit> few, many;
  auto split = [&](int64_t limit) {
    few.clear();
    many.clear();
    int64_t q_first = 0, blocks = 0;
    for (int s = 0; s < n_seqs; ++s) {
      const int64_t rows = static_cast<int64_t>(q_lens[s]) * group;
      const int tile = rows <= limit ? kFewRows : kTileRows;
      for (int64_t r = 0; r < rows; r += tile) {
        const int n = static_cast<int>(std::min<int64_t>(tile, rows - r));
        const Unit u = make_unit(s, kv_lens[s], q_lens[s], q_first, group, static_cast<int>(r), n, causal, window, sink);
        (rows <= limit ? few : many).push_back(u);
        if (rows <= limit) blocks += u.n;
        if (rows <= limit && rows > 8) p->row_tile = 16;
      }
      q_first += q_lens[s];
    }
    return blocks * c->n_heads;
  };
  if (most <= kFewRows || most > kMidRows) {
    split(kFewRows);
  } else if (split(kMidRows) > kMidBlocks * resident(16)) {
    p->row_tile = 8;
    split(kFewRows);
  }
  KVQ_REQUIRE(static_cast<int64_t>(few.size() + many.size()) * c->n_heads < (1 << 24), KVQ_ERR_ARG,
              "too many rows for one launch");
  cut_rows(few, c->n_heads, resident(p->row_tile), p);
  cut_tiles(many, c->n_heads, n_sms, p);
  return KVQ_OK;
}

}  // namespace paged
}  // namespace kvq

using namespace kvq;

extern "C" int kvq_paged_plan(const kvq_paged_cache* cache, const int32_t* kv_lens, const int32_t* q_lens, int n_seqs,
                              int n_q_heads, int causal, int64_t window, int64_t sink, int n_sms, int32_t* out,
                              int64_t capacity, kvq_paged_plan_info* info) {
  clear_error();
  int layout = 0;
  int rc = paged::check_format(cache, &layout);
  if (rc) return rc;
  const int n_heads = cache->n_heads;
  KVQ_REQUIRE(info != nullptr, KVQ_ERR_ARG, "NULL info");
  KVQ_REQUIRE(n_seqs >= 0 && n_sms >= 1 && (n_seqs == 0 || (kv_lens && q_lens)), KVQ_ERR_ARG, "bad lengths");
  KVQ_REQUIRE(n_q_heads >= n_heads && n_q_heads <= 65535 && n_q_heads % n_heads == 0,
              KVQ_ERR_ARG, "%d query heads are not a multiple of %d KV heads", n_q_heads, n_heads);
  KVQ_REQUIRE(window >= 0 && sink >= 0, KVQ_ERR_ARG, "window and sink must be >= 0");
  const int group = n_q_heads / n_heads;
  for (int s = 0; s < n_seqs; ++s) {
    KVQ_REQUIRE(kv_lens[s] >= 0 && q_lens[s] >= 0, KVQ_ERR_ARG, "negative length of sequence %d", s);
    KVQ_REQUIRE(static_cast<int64_t>(q_lens[s]) * group < ((int64_t)1 << 31), KVQ_ERR_ARG, "too many queries");
  }
  try {
    paged::Plan p;
    rc = paged::make_plan(cache, layout, kv_lens, q_lens, n_seqs, group, causal ? 1 : 0, window, sink, n_sms, &p);
    if (rc) return rc;
    *info = kvq_paged_plan_info{};
    info->n_row_items = static_cast<int32_t>(p.rows.size());
    info->n_row_ctas = p.row_ctas;
    info->n_tile_items = static_cast<int32_t>(p.tiles.size());
    info->row_tile = p.row_tile;
    info->n_units = p.units;
    info->words = static_cast<int64_t>(p.rows.size() + p.tiles.size()) * paged::kItemWords + static_cast<int64_t>(p.cta_first.size());
    info->tile_workspace_offset = (static_cast<int64_t>(p.slots) * paged::slot_floats(p.row_tile) * 4 + 255) / 256 * 256;
    info->workspace_bytes = info->tile_workspace_offset + p.tile_slots * paged::kTileSlotBytes;
    if (!out) return KVQ_OK;
    KVQ_REQUIRE(capacity >= info->words, KVQ_ERR_ARG, "the plan needs %lld words", (long long)info->words);
    auto put = [&out](const void* src, size_t words) {
      if (words) std::memcpy(out, src, words * 4);
      out += words;
    };
    put(p.rows.data(), p.rows.size() * paged::kItemWords);
    put(p.tiles.data(), p.tiles.size() * paged::kItemWords);
    put(p.cta_first.data(), p.cta_first.size());
  } catch (const std::bad_alloc&) {
    set_error("kvq_paged_plan: out of host memory");
    return KVQ_ERR_ARG;
  }
  return KVQ_OK;
}
