// Attention of many query rows per KV head over the paged quantized cache (sm_100a):
// prompt chunks, denoising blocks, drafts of grouped heads: tcgen05.mma with TMEM
// accumulators. Bound by the softmax step of a warp (~1700 of a 64-token tile's ~2000
// cycles: S out of TMEM, maximum, exponentials, P into TMEM), which the MMAs of the other Q
// tile overlap, and under a long load by the power limit. Measured: 4680 queries of 40
// heads over 32760 tokens 3.4 to 3.85 ms by the clock that the power left (815 to 925
// TFLOP/s), 2000 queries of 40 heads over 18720 tokens, causal, 0.79 to 0.87 ms; 12
// sequences with 4 to 6 new tokens, 8 query heads per KV head, 2705 to 6240 tokens, int8:
// 40.5 us, of which ~15 are launch, set-up, first tiles and the join.
//
// One CTA of 16 warps per item of the plan: up to 256 rows (two Q tiles of 128) of a
// sequence and KV head, row = query * group + grouped head, over its list of 16-token
// storage blocks; a KV tile is four consecutive entries of that list (64 tokens), so the
// kept first tokens and a sliding window need no tokens between them.
//   warps 0-3 / 4-7  softmax of Q tile 0 / 1: thread r owns row r (TMEM lane r); all
//                    eight first gather the Q rows into the MMA's layout
//   warps 8-9/10-11  converters of K / V: four lanes per row, 32 channels each, codes and
//                    scales from the staged records to 128B-swizzled fp16 tiles
//   warps 12 / 15    producers of K / V: a storage block is contiguous, one bulk copy
//   warps 13 / 14    one thread each issuing the tcgen05.mma of Q tile 0 / 1:
//                    S_x = Q_x K^T (M128 N64 K128), O_x += P_x V (M128 N128 K64, P in TMEM)
// The pipeline is that of the contiguous-window attention kernel (S double-buffered,
// S_x(j+2) issued behind PV_x(j), one commit per tile and Q tile, K and V as separate
// streams): see there for what was measured. What differs: rows of different lengths
// of sight, and items of one Q tile, whose two softmax sets take turns with the KV tiles and
// join their results at the end (24 to 72 rows over 12480 tokens, int4: 188 us for 148 such
// items; one set, the other's warps converting too: 218). A tile that some row of the Q tile does not see whole takes a masked step
// (a 64-bit mask per row; a masked logit is -inf); the running maximum starts at -1e30,
// so a row without any visible token ends with l = 0 and is stored as 0.
// Roundings: Q, K, V and P are fp16 for the MMAs (K and V exact for int4 codes; see
// kScaleLeast); S, m, l, O are fp32.
#include <cmath>

#include "kvq_paged_dev.cuh"

namespace kvq {
namespace paged {
using namespace sm100;
namespace tiles {

constexpr int BM = 128, BN = 64;
constexpr int kThreads = 512;
constexpr int kProdWarp = 12, kMmaWarp = 13, kProdWarpV = 15;
constexpr uint32_t kTmemCols = 512, kColO = 0, kColS = 256;
constexpr int kKVTile = BN * D * 2;  // 16 KB: two SWIZZLE_128B atoms (channels 0-63, 64-127)
constexpr int kAtom = BN * 128;
constexpr int kQTile = BM * D * 2;
constexpr int kQAtom = BM * 128;

// Shared memory: fp16 stages of K and V, staged records, the Q tiles. Three fp16 stages of
// K and five of V (a K stage is free two tiles before a V stage, and both tiles must be
// ready before S(j)) and three staged tiles where the codes are small: 794 us for 2000 new
// tokens of 40 heads over 18720, against 808 with four stages each. int8 codes leave two staged
// tiles, and with both tensors int8 four stages of V.
template <class L, int KB, int VB>
struct Geo {
  static constexpr int kRecK = Rec<L, KB>::kBytes, kRecV = Rec<L, VB>::kBytes;
  static constexpr int kStageK = 4 * kRecK, kStageV = 4 * kRecV;
  static constexpr int NK = 3, NV = VB == 8 ? 4 : 5;
  static constexpr int LK = KB == 8 ? 2 : 3, LV = KB == 8 ? 2 : 3;
  static constexpr int kReady = 8;  // see at the converters
  static constexpr int kOffK = 0;
  static constexpr int kOffV = kOffK + NK * kKVTile;
  // Q tile 1, then Q tile 0: an item of one Q tile has two more stages of V in the other's place
  static constexpr int NV1 = NV + kQTile / kKVTile;
  static_assert(NK < kReady && NV1 < kReady, "no tile may be converted before the barrier of the one kReady before it completes");
  static constexpr int kOffQ = kOffV + NV * kKVTile;
  static constexpr int kOffCK = kOffQ + 2 * kQTile;
  static constexpr int kOffCV = kOffCK + LK * kStageK;
  static constexpr int kOffBar = (kOffCV + LV * kStageV + 15) / 16 * 16;
  // barriers; index + stages of K for V
  static constexpr int bLdFull = 0, bLdEmpty = bLdFull + LK + LV, bReady = bLdEmpty + LK + LV,
                       bKvEmpty = bReady + kReady, bQReady = bKvEmpty + NK + NV1, bSFull = bQReady + 2,
                       bPFull = bSFull + 4, bOReady = bPFull + 4, bOFinal = bOReady + 2, bMmaDone = bOFinal + 2,
                       kNumBars = bMmaDone + 2;
  static constexpr int kOffMisc = (kOffBar + kNumBars * 8 + 15) / 16 * 16;
  // Of the last kExpK key tiles and kExpV value tiles: the exponent taken out of each token,
  // and a byte per converter warp that says whether there is any. A slot is written again
  // only after softmax step j has ended: tile j + 8 is converted after S(j + 8 - NK) or, with
  // up to NV1 stages, after S(j + 5) has been found complete by its softmax warps, and with it
  // every step up to the fifth before it has ended, in each order of the two Q tiles' or
  // the two shares' steps.
  static constexpr int kExpK = 8, kExpV = 8;
  static_assert(kExpK >= NK + 5 && kExpV >= NV1 + 1, "rings of exponents");
  static constexpr int kOffExpK = kOffMisc + 32, kOffExpV = kOffExpK + kExpK * BN;
  static constexpr int kOffWideK = kOffExpV + kExpV * BN, kOffWideV = kOffWideK + 4 * kExpK;
  static constexpr int kOffExpQ = kOffWideV + 4 * kExpV;  // the exponent taken out of each query row
  static constexpr int kSmemBytes = kOffExpQ + 2 * BM;
  static_assert(kSmemBytes <= 227 * 1024, "one CTA per SM must fit");
  static_assert(kOffCK % 16 == 0 && kOffCV % 16 == 0, "bulk copies");
};

__device__ __forceinline__ uint32_t tile_off(int r, int c) {
  return static_cast<uint32_t>((c >> 3) * kAtom + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Converters: four lanes per row, lane t channels 32t..32t+31.
template <class L, int BITS>
struct Converter {
  static constexpr int KG = most_groups<L, 32>();
  int base;
  uint32_t sel[KG == 1 ? 1 : 16];
  // Lanes 2 and 3 of a row write atom 1: taking their 16-byte chunks in the order 2, 3, 0,
  // 1 keeps the eight lanes of a store phase on different banks.
  __device__ __forceinline__ void init(int t) {
    base = group_at<L>(32 * t);
    if constexpr (KG > 1) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int w = (i >> 2) ^ (t & 2);
        const uint32_t l = 2 * (group_at<L>(32 * t + 8 * w + 2 * (i & 3)) - base);
        sel[i] = l | (l + 1) << 4 | l << 8 | (l + 1) << 12;
      }
    }
  }
  // This lane's codes and scales of one row: row rr of record block `rec`.
  struct Raw {
    uint32_t w[BITS], x[KG];  // 4 or 8 words of codes
    uint32_t src;             // and where they are
  };
  __device__ __forceinline__ Raw load(uint32_t rec, int rr, int t) const {
    using R = Rec<L, BITS>;
    Raw u;
    const uint32_t src = u.src = rec + rr * R::CW + t * (R::CW / 4);
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) {
      const uint4 v = ld_shared_v4(src + 16 * i);
      u.w[4 * i] = v.x;
      u.w[4 * i + 1] = v.y;
      u.w[4 * i + 2] = v.z;
      u.w[4 * i + 3] = v.w;
    }
    const uint32_t sc = rec + R::kCodes + rr * L::G * 2;
#pragma unroll
    for (int q = 0; q < KG; ++q) u.x[q] = ld_shared_u16(sc + 2 * (KG == 1 ? base : min(base + q, L::G - 1)));
    return u;
  }
  // One loaded row, to row r of the tile at dst. EXACT: takes a power of two out of a row
  // beyond (kScaleLeast, kScaleMost) and returns its exponent; else converts as if there
  // were none and keeps this lane's extremes of live rows' scales.
  template <bool EXACT>
  __device__ __forceinline__ int row(const Raw& u, uint32_t dst, int r, int t, bool live, uint32_t& least,
                                     uint32_t& most) const {
    const uint32_t (&w)[BITS] = u.w;
    const uint32_t (&x)[KG] = u.x;
    uint32_t top = 0, low = 0xFFFFu, used = live ? ~0u : 0u;  // rows past the end hold anything
    if constexpr (EXACT) {
      bool one = false;
#pragma unroll
      for (int q = 0; q < KG; ++q) one |= x[q] == kScaleOne;
      if (__any_sync(0xffffffffu, one)) used &= used_groups<L, BITS, 32>(u.src, 32 * t, base);
    }
#pragma unroll
    for (int q = 0; q < KG; ++q) {
      if (EXACT && !((used >> q) & 1u)) continue;
      top = max(top, x[q]);
      low = min(low, x[q]);
    }
    float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int q = 0; q < KG; ++q) f[q] = (used >> q) & 1u ? __uint_as_float(x[q] << 16) : 0.0f;
    uint32_t s01, s23 = 0;
    int e = 0;
    if constexpr (EXACT) {
      extremes_of_lanes<1, 2>(top, low);
      e = !live ? 0 : top == 0 ? kNoScale : scale_exponent(top, low);
#pragma unroll
      for (int q = 0; q < KG; ++q) f[q] *= pow2i(-e);
    } else if (live) {
      most = max(most, top);
      least = min(least, low);
    }
    s01 = pack_f16x2(f[0], f[KG == 1 ? 0 : 1]);
    if constexpr (KG > 2) s23 = pack_f16x2(f[2], f[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int hi = t & 2;  // word i ^ hi
      uint32_t o[4];
      if constexpr (BITS == 4) {
        const uint32_t v = hi ? w[i ^ 2] : w[i], y = v >> 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t b = __byte_perm(v, y, (4 + j) << 8 | j);
          o[j] = int4_low_f16(b);
        }
      } else {
        const uint32_t v = hi ? w[2 * (i ^ 2)] : w[2 * i], y = hi ? w[2 * (i ^ 2) + 1] : w[2 * i + 1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t b = __byte_perm(j < 2 ? v : y, 0, (j & 1) ? 0x4342 : 0x4140);
          o[j] = int8_pair_f16(b);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t sp = KG == 1 ? s01 : __byte_perm(s01, s23, sel[KG == 1 ? 0 : 4 * i + j]);
        o[j] = h16mul2(o[j], sp);
      }
      st_shared_v4(dst + tile_off(r, 4 * t + (i ^ hi)), o[0], o[1], o[2], o[3]);
    }
    return e;
  }
};

// idesc_bf16 with fp16 for both operands.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, int b_mn_major) {
  return idesc_bf16(m, n, b_mn_major) & ~((7u << 7) | (7u << 10));
}

template <class L, int KB, int VB>
__global__ void __launch_bounds__(kThreads, 1) tiles_kernel(const __grid_constant__ AttnArgs a) {
  using GEO = Geo<L, KB, VB>;
  constexpr int NK = GEO::NK, NV = GEO::NV, LK = GEO::LK, LV = GEO::LV;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  if (sbase & 1023) {  // the swizzled tiles need it
    if (threadIdx.x == 0) atomicExch(a.status, kDevTimeout);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + GEO::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + GEO::kOffMisc);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + GEO::kOffMisc + 8);
  volatile int* last = abort + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long lim = a.wait_cycles;
  pdl_wait();
  pdl_launch_dependents();
  const Item it = a.items[blockIdx.x];
  const int nq = it.n_rows > BM ? 2 : 1;
  const int n_blk = it.je - it.jb;  // entries of the block list
  const int nkv = (n_blk + 3) / 4;
  // With one Q tile its two sets of softmax warps share the KV tiles: set (and MMA thread) x
  // takes tiles x, x + 2, ..., and the two partial results are joined at the end.
  const bool shared = nq == 1;
  const int stride = shared ? 2 : 1, n_vs = shared ? GEO::NV1 : NV;

  // where row n of the item reads its query and writes its output
  auto place = [&](int n, int64_t& tok, int& h) {
    const int row = it.row0 + n, i = row / a.group;
    tok = it.q_first + i;
    h = it.head * a.group + row - i * a.group;
  };
  // Offset of row n's head in q (0: out); a division, so each lane makes one and rows are
  // passed around by shuffles.
  auto q_offset = [&](int n, int64_t stride) {
    int64_t tok;
    int h;
    place(min(n, it.n_rows - 1), tok, h);
    return tok * stride + h * D;
  };
  auto q_at = [](int x) { return static_cast<uint32_t>(GEO::kOffQ + (1 - x) * kQTile); };
  // A warp's n_out (at most 32) output rows, n0.. of the item, staged in the Q buffer, to
  // global memory: half a warp per row, 256 contiguous bytes.
  auto store_rows = [&](int n0, int n_out) {
    const int64_t mine = q_offset(n0 + lane, a.out_stride);
#pragma unroll 4
    for (int k = 0; k < n_out / 2; ++k) {
      const int i = 2 * k + (lane >> 4), n = n0 + i, rr = n & (BM - 1), c = lane & 15;
      const int64_t to = __shfl_sync(0xffffffffu, mine, i);
      const uint32_t stage = sbase + q_at(n >> 7);
      if (n < it.n_rows)
        st_global_v4(a.out + to + 8 * c, ld_shared_v4(stage + (c >> 3) * kQAtom + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)));
    }
  };
  auto stage_chunk = [&](uint32_t stage, int r, int ch, const float* v, float f) {
    st_shared_v4(stage + (ch >> 3) * kQAtom + r * 128 + (((ch & 7) ^ (r & 7)) << 4),
                 pack_bf16x2(v[0] * f, v[1] * f), pack_bf16x2(v[2] * f, v[3] * f), pack_bf16x2(v[4] * f, v[5] * f),
                 pack_bf16x2(v[6] * f, v[7] * f));
  };
  auto store_lse = [&](int n, float m, float l) {
    if (a.lse && n < it.n_rows) {
      int64_t tok;
      int h;
      place(n, tok, h);
      a.lse[tok * a.n_q_heads + h] = l == 0.0f ? -INFINITY : 0.69314718055994531f * (m + log2f(l));
    }
  };

  // The exponent to take out of a query row of which each lane of half a warp has a part.
  auto row_exponent = [&](uint32_t most, uint32_t least) {
    if (!__any_sync(0xffffffffu, most > kQueryMost || least < kQueryLeast)) return 0;
    extremes_of_lanes<1, 8>(most, least);
    return query_exponent(most, least);
  };
  // Ahead of the set-up of the barriers: the Q rows, gathered by the eight softmax warps
  // (two rows at a time) and converted to fp16, and the producers' first look-ups.
  int q_wide = 0;     // whether a power of two was taken out of any query row
  int64_t where = 0;  // producer lane i: the pool block of list entry 32 k + i
  auto look_up = [&](int j) {
    const int e = it.jb + 4 * j + lane;
    bool ok;
    if (e < it.je) where = a.p.block(it.seq, it.head, it.block_at(e), ok);
  };
  if (warp < 8) {
    const int64_t mine = q_offset(16 * (lane >> 1) + 2 * warp + (lane & 1), a.q_stride);
#pragma unroll 4
    for (int k = 0; k < 8 * nq; ++k) {
      const int n = 16 * k + (tid >> 4), c = tid & 15, r = n & (BM - 1);
      const int64_t from = __shfl_sync(0xffffffffu, mine, 2 * k + (lane >> 4));
      const uint32_t dst = sbase + q_at(n >> 7) + (c >> 3) * kQAtom + r * 128 + (((c & 7) ^ (r & 7)) << 4);
      uint4 v = make_uint4(0, 0, 0, 0);
      if (n < it.n_rows) v = ld_global_nc_v4(a.q + from + 8 * c);
      const int e = row_exponent(most_of(v), least_of(v));
      q_wide |= e;
      if (c == 0) smem[GEO::kOffExpQ + n] = static_cast<uint8_t>(e);
      if (n < it.n_rows) v = to_f16(v, e);
      st_shared_v4(dst, v.x, v.y, v.z, v.w);
    }
  } else if (warp == kProdWarp || warp == kProdWarpV) {
    look_up(0);
  }

  if (tid == 0) {
    for (int i = 0; i < LK + LV; ++i) {
      mbar_init(&bars[GEO::bLdFull + i], 1);
      mbar_init(&bars[GEO::bLdEmpty + i], 2);  // a tensor's converter warps
    }
    for (int i = 0; i < NK + GEO::NV1; ++i) mbar_init(&bars[GEO::bKvEmpty + i], nq);
    for (int i = 0; i < GEO::kReady; ++i) mbar_init(&bars[GEO::bReady + i], 4);
    for (int x = 0; x < 2; ++x) {
      mbar_init(&bars[GEO::bQReady + x], 8);  // the eight gathering warps
      mbar_init(&bars[GEO::bSFull + 2 * x], 1);
      mbar_init(&bars[GEO::bSFull + 2 * x + 1], 1);
      mbar_init(&bars[GEO::bPFull + 2 * x], 4);
      mbar_init(&bars[GEO::bPFull + 2 * x + 1], 4);
      mbar_init(&bars[GEO::bOReady + x], 1);
      mbar_init(&bars[GEO::bOFinal + x], 1);
      mbar_init(&bars[GEO::bMmaDone + x], 1);
    }
    *abort = 0;
    for (int i = 0; i < GEO::kExpK + GEO::kExpV; ++i) *reinterpret_cast<uint32_t*>(smem + GEO::kOffWideK + 4 * i) = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  q_wide = __syncthreads_or(q_wide);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 8) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(&bars[GEO::bQReady]);
      mbar_arrive(&bars[GEO::bQReady + 1]);
    }
  }
  if (warp < 8) {
    // ------------------------------------------------ softmax (Q tile or share of the tiles x)
    const int x = warp >> 2;
    const int r = tid - x * BM;
    const int xq = shared ? 0 : x;  // Q tile
    const int n = xq * BM + r;
    const int n_mine = shared ? (nkv - x + 1) / 2 : nkv;  // KV tiles of set x
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lane_off + kColO + 128 * x;
    const uint32_t tS0 = tmem + lane_off + kColS + 128 * x;
    const int n_last = min(xq * BM + BM, it.n_rows) - 1;
    const Seen see = seen_by(a, it.start + (it.row0 + min(n, it.n_rows - 1)) / a.group, it.kv_len);
    const Seen first = seen_by(a, it.start + (it.row0 + xq * BM) / a.group, it.kv_len);
    const Seen fin = seen_by(a, it.start + (it.row0 + n_last) / a.group, it.kv_len);
    float m = -1.0e30f, l = 0.0f, F = 0.0f;  // O is kept divided by 2^F
    bool ok = true, s_ready = false;  // s_ready: S of the coming tile was already found complete
    // this row's softmax scale, with the power of two taken out of its query
    float row_scale = a.scale_log2;
    if (q_wide) row_scale = row_scale_of(a.scale_log2, static_cast<int8_t>(smem[GEO::kOffExpQ + n]));
    // wide_k, wide_v: a byte per converter warp of the tile, and whose rows' exponents count
    auto exps16 = [&](uint32_t wide, uint32_t at, int block) {
      return (wide >> (8 * (block >> 1))) & 255u ? ld_shared_v4(at + 16 * block) : make_uint4(0, 0, 0, 0);
    };
    // step i of this set, tile j
    auto step = [&](const int i_, const int j, const uint32_t wide_k, const uint32_t wide_v, auto masked) -> bool {
      constexpr bool MASK = decltype(masked)::value;
      const uint32_t tS = tS0 + 64 * (i_ & 1);
      uint32_t s0[32], s1[32];
      tmem_ld32x2_wait(tS, tS + 32, s0, s1);
      if constexpr (MASK) {
        if (wide_k) {  // powers of two taken out of the tile's keys
          const uint32_t at = sbase + GEO::kOffExpK + (j % GEO::kExpK) * BN;
#pragma unroll
          for (int c = 0; c < 32; c += 16) {
            const uint4 u = exps16(wide_k, at, c / 16), v = exps16(wide_k, at, 2 + c / 16);
            const uint32_t eu[4] = {u.x, u.y, u.z, u.w}, ev[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              s0[c + i] = __float_as_uint(__uint_as_float(s0[c + i]) * pow2i(static_cast<int8_t>(eu[i >> 2] >> (8 * (i & 3)))));
              s1[c + i] = __float_as_uint(__uint_as_float(s1[c + i]) * pow2i(static_cast<int8_t>(ev[i >> 2] >> (8 * (i & 3)))));
            }
          }
        }
        uint32_t mk[2] = {0, 0};  // bit c: column c is seen
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int e = it.jb + 4 * j + b;
          if (e < it.je) {
            const int tb = it.block_at(e) * kBlock;
            auto below = [&](int lim_) { return (1u << max(0, min(kBlock, lim_ - tb))) - 1u; };
            const uint32_t bits = below(see.hi) & (~below(see.lo) | below(see.kept)) & 0xFFFFu;
            mk[b >> 1] |= bits << (16 * (b & 1));
          }
        }
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          if (!((mk[0] >> c) & 1u)) s0[c] = 0xFF800000u;  // -inf
          if (!((mk[1] >> c) & 1u)) s1[c] = 0xFF800000u;
        }
      }
      float pm[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) pm[i] = -INFINITY;
#pragma unroll
      for (int c = 0; c < 32; ++c) pm[c & 7] = fmax3(pm[c & 7], __uint_as_float(s0[c]), __uint_as_float(s1[c]));
      const float mt =
          fmax3(fmax3(pm[0], pm[1], pm[2]), fmax3(pm[3], pm[4], pm[5]), fmaxf(pm[6], pm[7])) * row_scale;
      bool rescale = false;
      const float m_old = m;
      float alpha = 1.0f;
      if (i_ == 0) {
        m = fmaxf(m, mt - kBias);
      } else if (mt - m > kBias + kLag) {
        rescale = true;
        alpha = ex2f(m - (mt - kBias));
        m = mt - kBias;
        l *= alpha;
      }
      const float nm = -m;
      float alpha_o = alpha;
      uint32_t pw[32];
      const float2 sc2 = make_float2(row_scale, row_scale), nm2 = make_float2(nm, nm);
      float2 sum2 = make_float2(0.0f, 0.0f);
      auto half = [&](const uint32_t (&sv)[32], int base) {
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const float2 xx =
              __ffma2_rn(make_float2(__uint_as_float(sv[2 * c]), __uint_as_float(sv[2 * c + 1])), sc2, nm2);
          const float p0 = ex2f(xx.x), p1 = ex2f(xx.y);
          sum2 = __fadd2_rn(sum2, make_float2(p0, p1));
          pw[base / 2 + c] = pack_f16x2(p0, p1);
        }
      };
      half(s0, 0);
      if constexpr (MASK) {
        half(s1, 32);
        if (__any_sync(0xffffffffu, wide_v != 0 || F != 0.0f)) {
          // weights times the powers of two taken out of the values, relative to 2^F, in
          // log2: y = s * scale - m + e. F grows where 2^(y - F) would leave fp16.
          const uint32_t at = sbase + GEO::kOffExpV + (j % GEO::kExpV) * BN;
          auto exps_of = [&](int c, float (&e)[16]) {
            const uint4 u = exps16(wide_v, at, c / 16);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 16; ++i) e[i] = static_cast<float>(static_cast<int8_t>(w[i >> 2] >> (8 * (i & 3))));
          };
          float top = -INFINITY;
#pragma unroll
          for (int c = 0; c < 32; c += 16) {
            float e0[16], e1[16];
            exps_of(c, e0);
            exps_of(32 + c, e1);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              s0[c + i] = __float_as_uint(fmaf(__uint_as_float(s0[c + i]), row_scale, nm) + e0[i]);
              s1[c + i] = __float_as_uint(fmaf(__uint_as_float(s1[c + i]), row_scale, nm) + e1[i]);
              top = fmax3(top, __uint_as_float(s0[c + i]), __uint_as_float(s1[c + i]));
            }
          }
          F += m_old - m;
          const float Fn = next_f(F, top);
          alpha_o = ex2f(F - Fn);  // alpha's part in F has been taken
          rescale = rescale || (i_ > 0 && Fn != F);
          F = Fn;
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            pw[c] = pack_f16x2(ex2f(__uint_as_float(s0[2 * c]) - F), ex2f(__uint_as_float(s0[2 * c + 1]) - F));
            pw[16 + c] = pack_f16x2(ex2f(__uint_as_float(s1[2 * c]) - F), ex2f(__uint_as_float(s1[2 * c + 1]) - F));
          }
        }
        tmem_st16(tS, pw);
      } else {
        tmem_st16(tS, pw);
        half(s1, 32);
      }
      tmem_st16(tS + 16, pw + 16);
      l += sum2.x + sum2.y;
      if (__any_sync(0xffffffffu, rescale)) {
        // O_x must hold every product up to PV_x(i-1) before it is rescaled: wait for
        // S_x(i+1), issued behind PV_x(i-1), or at the last tile for the commit behind it
        const bool tail = i_ + 1 == n_mine;
        if (!poll_wait_warp(&bars[tail ? GEO::bOReady + x : GEO::bSFull + 2 * x + ((i_ + 1) & 1)],
                            tail ? 0u : static_cast<uint32_t>(((i_ + 1) >> 1) & 1), abort, a.status, lim))
          return false;
        tc_fence_after();
#pragma unroll 1
        for (int k = 0; k < 8; ++k) {
          uint32_t o[16];
          tmem_ld16_wait(tO + 16 * k, o);
#pragma unroll
          for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha_o);
          tmem_st16(tO + 16 * k, o);
        }
        tmem_wait_st();
      }
      s_ready = i_ + 1 < n_mine && mbar_test(&bars[GEO::bSFull + 2 * x + ((i_ + 1) & 1)], ((i_ + 1) >> 1) & 1);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[GEO::bPFull + 2 * x + (i_ & 1)]);
      return true;
    };
    int vs = shared ? x : 0;  // V stage of this set's tile i - 2
    for (int i = 0; i < n_mine; ++i) {
      const int j = shared ? 2 * i + x : i;
      if (!__all_sync(0xffffffffu, s_ready) &&
          !poll_wait_warp(&bars[GEO::bSFull + 2 * x + (i & 1)], (i >> 1) & 1, abort, a.status, lim)) {
        ok = false;
        break;
      }
      // S_x(i) complete: set x no longer reads its K stage, and PV_x(i-2) (issued before
      // it) is complete: nor that V stage
      if ((warp & 3) == 0 && lane == 0) {
        mbar_arrive(&bars[GEO::bKvEmpty + j % NK]);
        if (i >= 2) {
          mbar_arrive(&bars[GEO::bKvEmpty + NK + vs]);
          vs += stride;
          if (vs >= n_vs) vs -= n_vs;
        }
      }
      tc_fence_after();
      const uint32_t wide_k = *reinterpret_cast<volatile uint32_t*>(smem + GEO::kOffWideK + 4 * (j % GEO::kExpK));
      const uint32_t wide_v = *reinterpret_cast<volatile uint32_t*>(smem + GEO::kOffWideV + 4 * (j % GEO::kExpV));
      const int e0 = it.jb + 4 * j;
      const int ta = it.block_at(e0) * kBlock, tz = it.block_at(e0 + 3) * kBlock + kBlock;
      const bool whole = e0 + 4 <= it.je && tz <= first.hi && (ta >= fin.lo || tz <= first.kept);
      ok = __all_sync(0xffffffffu, whole && wide_k == 0 && wide_v == 0 && F == 0.0f) 
               ? step(i, j, 0, 0, std::false_type{})
               : step(i, j, wide_k, wide_v, std::true_type{});
      if (!ok) break;
    }
    // what the rows of O, of this set and of the other, are multiplied with when they are joined
    float of = 1.0f, of1 = 0.0f;
    bool done = ok && n_mine > 0 && poll_wait_warp(&bars[GEO::bOFinal + x], 0, abort, a.status, lim);
    // Shared tiles: set 1 leaves its row in the stages of K and V, float4 column c of row r
    // at [c][r] and (m, l, F) behind them, and set 0 adds it to its own. No MMA reads the
    // stages any more. Sums and O each have their own greatest term, m and m + F: O times
    // 2^F may be beyond fp32 until it is divided by the sum.
    const uint32_t other = sbase + GEO::kOffK + r * 16;
    if (shared && nkv > 0) {
      if (x == 1) {
        if (poll_wait_warp(&bars[GEO::bOFinal], 0, abort, a.status, lim)) {
          tc_fence_after();
#pragma unroll 1
          for (int k = 0; k < 4 && done; ++k) {
            uint32_t o[32];
            tmem_ld32_wait(tO + 32 * k, o);
#pragma unroll
            for (int c = 0; c < 8; ++c)
              st_shared_v4(other + (8 * k + c) * BM * 16, o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
          }
          st_shared_v4(other + 32 * BM * 16, __float_as_uint(m), __float_as_uint(l), __float_as_uint(F), 0);
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (x == 0) {
        const uint4 u = ld_shared_v4(other + 32 * BM * 16);
        const float m1 = __uint_as_float(u.x), l1 = __uint_as_float(u.y), mf1 = m1 + __uint_as_float(u.z);
        const float mx = fmaxf(m, m1), mf = fmaxf(m + F, mf1);
        l = l * ex2f(m - mx) + l1 * ex2f(m1 - mx);
        of = ex2f(m + F - mf);
        of1 = ex2f(mf1 - mf);
        m = mx;
        F = mf - mx;
      }
    }
    const bool both = shared && nkv > 1;  // set 1 had tiles
    // 32 columns of the joined row of O, divided by 2^F
    auto fetch = [&](int k, float (&v)[32]) {
      if (done) {
        uint32_t o[32];
        tmem_ld32_wait(tO + 32 * k, o);
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = __uint_as_float(o[c]) * of;
        if (both) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint4 u = ld_shared_v4(other + (8 * k + c) * BM * 16);
            v[4 * c] = fmaf(__uint_as_float(u.x), of1, v[4 * c]);
            v[4 * c + 1] = fmaf(__uint_as_float(u.y), of1, v[4 * c + 1]);
            v[4 * c + 2] = fmaf(__uint_as_float(u.z), of1, v[4 * c + 2]);
            v[4 * c + 3] = fmaf(__uint_as_float(u.w), of1, v[4 * c + 3]);
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = 0.0f;
      }
    };
    if (x < nq) {
      if (it.parts > 1) {
        // one part of a unit: unnormalised O row, m and l for the join. float4 column c of
        // row r at [c][r]: a warp's 32 rows are contiguous
        tc_fence_after();
        float4* dst = reinterpret_cast<float4*>(a.ws) + (static_cast<int64_t>(it.slot + it.part) * 2 + x) * 33 * BM + r;
#pragma unroll 1
        for (int k = 0; k < 4; ++k) {
          float v[32];
          fetch(k, v);
#pragma unroll
          for (int c = 0; c < 8; ++c) dst[(8 * k + c) * BM] = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
        }
        dst[32 * BM] = make_float4(m, l, F, 0.0f);
        __threadfence();
      } else if (done || (nkv == 0 && poll_wait_warp(&bars[GEO::bQReady + x], 0, abort, a.status, lim))) {
        // (no tiles: Q_x has landed before its buffer is reused below)
        tc_fence_after();
        const float inv = l == 0.0f ? 0.0f : 1.0f / l, pow_f = ex2f(F);
        of *= inv;
        of1 *= inv;
        store_lse(n, m, l);
        const uint32_t stage = sbase + q_at(x);  // Q_x is no longer read
#pragma unroll 1
        for (int k = 0; k < 4; ++k) {
          float v[32];
          fetch(k, v);
#pragma unroll
          for (int c = 0; c < 4; ++c) stage_chunk(stage, r, 4 * k + c, v + 8 * c, pow_f);
        }
        __syncwarp();
        store_rows(warp * 32, 32);
      }
    }
  } else if (warp < kProdWarp) {
    // ------------------------------------------------------------ converters
    // K(j) and V(j) count on one barrier, which the MMA threads wait for before S(j): V a
    // little early, so that softmax step j finds V's exponents as well as K's. An arrival
    // does not say whose it is, so no warp may arrive for tile j + kReady before all four
    // have for tile j: with fewer stages than kReady, a tile j + kReady takes a stage that a
    // tile behind j had, which is free only after that tile's S, and all four warps, each
    // in the order of the tiles, have arrived for it.
    const int is_v = (warp >> 1) & 1;
    constexpr int rows = 32;  // of this warp
    const int t = lane & 3, r0 = (warp & 1) * rows + (lane >> 2);
    auto convert = [&](auto conv, uint32_t codes, uint32_t tiles, int n_ld, int n_kv, uint64_t* ld_full, uint64_t* ld_empty,
                       uint64_t* kv_empty, uint8_t* exps, uint8_t* wide, int n_exp, int rec, int stage_bytes) {
      conv.init(t);
      bool ready = false;
      // stages and phases are counted, not divided out: the ring sizes are not known here
      int ls = 0, ks = 0, slot = 0;
      uint32_t ld_phase = 0, kv_phase = 1;  // of the next waits; kv_phase counts from the second round
      for (int j = 0; j < nkv; ++j) {
        // usually already found ready at the end of the last tile
        if (!__all_sync(0xffffffffu, ready)) {
          if (!poll_wait_warp(&ld_full[ls], ld_phase, abort, a.status, lim)) break;
          if (j >= n_kv && !poll_wait_warp(&kv_empty[ks], kv_phase, abort, a.status, lim)) break;
        }
        const uint32_t dst = tiles + ks * kKVTile;
        uint32_t least = kScaleLeast, most = 0;
        auto convert_rows = [&](auto exact, auto unroll) {
          constexpr bool EXACT = decltype(exact)::value;
          int any = 0;
          auto load = [&](int r) { return conv.load(codes + ls * stage_bytes + (r >> 4) * rec, r & 15, t); };
          auto next = load(r0);
#pragma unroll(decltype(unroll)::value)
          for (int p = 0; p < rows; p += 8) {
            // the next row's loads are in flight while this one is converted
            const int r = r0 + p, e = it.jb + 4 * j + (r >> 4);
            const auto raw = next;
            if (p + 8 < rows) next = load(r + 8);
            const bool live = e < it.je && it.block_at(e) * kBlock + (r & 15) < it.kv_len;
            const int x = conv.template row<EXACT>(raw, dst, r, t, live, least, most);
            if constexpr (EXACT) {
              any |= x;
              if (t == 0) exps[slot * BN + r] = static_cast<uint8_t>(x);
            }
          }
          return any;
        };
        // The conversion is what items of one Q tile wait for, and four rows at a time have the
        // most in flight (165 us, one at a time 205, for 195 tiles in each of 148 items); two Q
        // tiles wait for their softmax, and the shorter loop is easier on the instruction
        // caches (2000 new tokens over 18720: 797 us, four at a time 814).
        int any = shared ? convert_rows(std::false_type{}, std::integral_constant<int, 4>{})
                         : convert_rows(std::false_type{}, std::integral_constant<int, 1>{});
        if (__any_sync(0xffffffffu, most > kScaleMost || least < kScaleLeast))
          any = __any_sync(0xffffffffu, convert_rows(std::true_type{}, std::integral_constant<int, 1>{}) != 0);
        if (lane == 0) wide[4 * slot + r0 / rows] = static_cast<uint8_t>(any);
        uint64_t* const read = &ld_empty[ls];
        if (++ls == n_ld) ls = 0, ld_phase ^= 1;
        if (++ks == n_kv) ks = 0, kv_phase ^= 1;
        if (++slot == n_exp) slot = 0;
        ready = mbar_test(&ld_full[ls], ld_phase);
        ready = (j + 1 < n_kv || mbar_test(&kv_empty[ks], kv_phase)) && ready && j + 1 < nkv;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(read);
          mbar_arrive(&bars[GEO::bReady + j % GEO::kReady]);
        }
      }
    };
    const uint32_t codes = sbase + (is_v ? GEO::kOffCV : GEO::kOffCK), dst = sbase + (is_v ? GEO::kOffV : GEO::kOffK);
    uint64_t* const ld_full = bars + GEO::bLdFull + (is_v ? LK : 0);
    uint64_t* const ld_empty = bars + GEO::bLdEmpty + (is_v ? LK : 0);
    uint64_t* const kv_empty = bars + GEO::bKvEmpty + (is_v ? NK : 0);
    uint8_t* const exps = smem + (is_v ? GEO::kOffExpV : GEO::kOffExpK);
    uint8_t* const wide = smem + (is_v ? GEO::kOffWideV : GEO::kOffWideK);
    const int n_exp = is_v ? GEO::kExpV : GEO::kExpK;
    // one copy of the loop where K and V have the same format: the instruction caches
    // hold four different loops per sub-partition as it is
    if (KB == VB || !is_v)
      convert(Converter<L, KB>{}, codes, dst, is_v ? LV : LK, is_v ? n_vs : NK, ld_full, ld_empty, kv_empty, exps, wide, n_exp,
              GEO::kRecK, GEO::kStageK);
    else
      convert(Converter<L, VB>{}, codes, dst, LV, n_vs, ld_full, ld_empty, kv_empty, exps, wide, n_exp, GEO::kRecV,
              GEO::kStageV);
  } else if (warp == kProdWarp || warp == kProdWarpV) {
    // ------------------------------------------------------------ producers
    const bool pv = warp != kProdWarp;
    const int n_ld = pv ? LV : LK;
    const uint32_t rec = pv ? GEO::kRecV : GEO::kRecK;
    const uint8_t* pages = pv ? a.v_pages : a.k_pages;
    uint64_t* full = bars + GEO::bLdFull + (pv ? LK : 0);
    uint64_t* empty = bars + GEO::bLdEmpty + (pv ? LK : 0);
    const uint32_t base = sbase + (pv ? GEO::kOffCV : GEO::kOffCK);
    int issued = 0, ls = 0;
    uint32_t phase = 1;
    for (int j = 0; j < nkv; ++j) {
      if (j > 0 && (j & 7) == 0) look_up(j);
      if (j >= n_ld && !poll_wait_warp(&empty[ls], phase, abort, a.status, lim)) break;
      const int nb = min(4, n_blk - 4 * j);
      if (lane == 0) mbar_arrive_expect_tx(&full[ls], nb * rec);
      __syncwarp();
      const int64_t blk = __shfl_sync(0xffffffffu, where, 4 * (j & 7) + (lane & 3));
      if (lane < nb) bulk_load(base + (4 * ls + lane) * rec, pages + blk * rec, rec, &full[ls]);
      issued = j + 1;
      if (++ls == n_ld) ls = 0, phase ^= 1;
    }
    // leave no copy into this CTA's shared memory in flight
    if (lane == 0)
      for (int j = max(0, issued - n_ld); j < issued; ++j) mbar_drain(&full[j % n_ld], (j / n_ld) & 1, a.status, lim);
    __syncwarp();
  } else {
    // ------------------------------------------------------------ MMA issuers
    const int x = warp - kMmaWarp;
    if (lane == 0) {
      constexpr uint32_t idS = idesc_f16(BM, BN, 0);
      constexpr uint32_t idPV = idesc_f16(BM, D, 1);
      const uint32_t tS0 = tmem + kColS + 128 * x, tO = tmem + kColO + 128 * x;
      // descriptors address shared memory in units of 16 bytes
      const uint64_t dq = smem_desc_sw128(sbase + q_at(shared ? 0 : x), 16, 1024);
      const uint64_t dk = smem_desc_sw128(sbase + GEO::kOffK, 16, 1024);
      const uint64_t dv = smem_desc_sw128(sbase + GEO::kOffV, kAtom, 1024);
      const int n_mine = shared ? (nkv - x + 1) / 2 : nkv;
      auto tile = [&](int i) { return shared ? 2 * i + x : i; };
      auto issue_s = [&](int i) {
        const uint64_t k = dk + static_cast<uint64_t>((tile(i) % NK) * (kKVTile >> 4));
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          mma_bf16_ss(tS0 + 64 * (i & 1), dq + (((kk >> 2) * kQAtom + (kk & 3) * 32) >> 4),
                      k + (((kk >> 2) * kAtom + (kk & 3) * 32) >> 4), idS, kk > 0);
        mma_commit(&bars[GEO::bSFull + 2 * x + (i & 1)]);
      };
      int vs = shared ? x : 0;
      auto issue_pv = [&](int i) {
        const uint64_t v = dv + static_cast<uint64_t>(vs * (kKVTile >> 4));
        const uint32_t p = tS0 + 64 * (i & 1);
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)
          mma_bf16_ts(tO, p + 8 * kk, v + ((kk * 2048) >> 4), idPV, (i > 0 || kk > 0) ? 1u : 0u);
        vs += stride;
        if (vs >= n_vs) vs -= n_vs;
      };
      auto ready_at = [&](int i) { return &bars[GEO::bReady + tile(i) % GEO::kReady]; };
      auto ready_phase = [&](int i) { return static_cast<uint32_t>((tile(i) / GEO::kReady) & 1); };
      auto wait_ready = [&](int i) { return poll_wait(ready_at(i), ready_phase(i), abort, a.status, lim); };
      bool ok = n_mine > 0 && poll_wait(&bars[GEO::bQReady + x], 0, abort, a.status, lim);
      for (int i = 0; i < 2 && i < n_mine && ok; ++i) {
        if (!(ok = wait_ready(i))) break;
        tc_fence_after();
        issue_s(i);
      }
      // A test of a barrier takes this thread over 100 cycles even where its phase has
      // completed, and a tile's issue is what it has time for: the next tile's is tested
      // before S(i+2) is issued, and waited for only if that failed.
      bool ready = n_mine > 2 && ok && mbar_test(ready_at(2), ready_phase(2));
      for (int i = 0; i < n_mine && ok; ++i) {
        if (!(ok = poll_wait(&bars[GEO::bPFull + 2 * x + (i & 1)], (i >> 1) & 1, abort, a.status, lim))) break;
        tc_fence_after();
        issue_pv(i);
        if (i + 2 < n_mine) {
          if (!ready && !(ok = wait_ready(i + 2))) break;
          ready = i + 3 < n_mine && mbar_test(ready_at(i + 3), ready_phase(i + 3));
          tc_fence_after();
          issue_s(i + 2);
        } else if (i + 2 == n_mine) {
          mma_commit(&bars[GEO::bOReady + x]);
        }
      }
      if (ok) mma_commit(&bars[GEO::bOFinal + x]);
      // all MMAs issued by this thread have completed before TMEM is released
      mma_commit(&bars[GEO::bMmaDone + x]);
      mbar_drain(&bars[GEO::bMmaDone + x], 0, a.status, lim);
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
  if (it.parts > 1) {
    // the part that ends last joins them, in part order
    if (tid == 0) {
      const unsigned old = atomicAdd(a.ctr + it.unit, 1u);
      *last = old == static_cast<unsigned>(it.parts - 1);
      if (*last) a.ctr[it.unit] = 0u;  // ready for the next launch
    }
    __syncthreads();
    if (*last) {
      // All 16 warps: a thread has one row and a half (two Q tiles) or a quarter of its
      // columns, so that the loads of eight float4 and two parts are in flight.
      __threadfence();
      const int n = tid & (nq * BM - 1), x = n >> 7, r = n & (BM - 1);
      const int n_col = 16 * nq / 2, c0 = (tid / (nq * BM)) * n_col;  // float4 columns of this thread
      const int64_t pstride = static_cast<int64_t>(2) * 33 * BM;
      const float4* src = reinterpret_cast<const float4*>(a.ws) + (static_cast<int64_t>(it.slot) * 2 + x) * 33 * BM + r;
      float mx = -1.0e30f, mf = -1.0e30f, lsum = 0.0f;
#pragma unroll 4
      for (int p = 0; p < it.parts; ++p) {
        const float4 ml = __ldcg(src + p * pstride + 32 * BM);
        mx = fmaxf(mx, ml.x);
        mf = fmaxf(mf, ml.x + ml.z);
      }
#pragma unroll 4
      for (int p = 0; p < it.parts; ++p) {
        const float4 ml = __ldcg(src + p * pstride + 32 * BM);
        lsum = fmaf(ml.y, ex2f(ml.x - mx), lsum);
      }
      const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum, pow_f = ex2f(mf - mx);
      if (c0 == 0) store_lse(n, mx, lsum);
      const uint32_t stage = sbase + q_at(x);
#pragma unroll 1
      for (int g = c0; g < c0 + n_col; g += 8) {
        float acc[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) acc[i] = 0.0f;
#pragma unroll 2
        for (int p = 0; p < it.parts; ++p) {
          const float4 ml = __ldcg(src + p * pstride + 32 * BM);
          const float f = ex2f(ml.x + ml.z - mf);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const float4 v = __ldcg(src + p * pstride + (g + c) * BM);
            acc[4 * c] = fmaf(v.x, f, acc[4 * c]);
            acc[4 * c + 1] = fmaf(v.y, f, acc[4 * c + 1]);
            acc[4 * c + 2] = fmaf(v.z, f, acc[4 * c + 2]);
            acc[4 * c + 3] = fmaf(v.w, f, acc[4 * c + 3]);
          }
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) acc[i] *= inv;
#pragma unroll
        for (int c = 0; c < 4; ++c) stage_chunk(stage, r, g / 2 + c, acc + 8 * c, pow_f);
      }
      __syncthreads();
      store_rows(warp * 8 * nq, 8 * nq);
    }
  }
}

}  // namespace tiles

int launch_tiles(const AttnArgs& a, int layout, int k_bits, int v_bits, int n_items, cudaStream_t st) {
  return with_layout(layout, [&](auto lt) {
    using L = decltype(lt);
    return with_bits(k_bits, v_bits, [&](auto bt) -> int {
      using B = decltype(bt);
      auto kernel = tiles::tiles_kernel<L, B::k, B::v>;
      constexpr int smem = tiles::Geo<L, B::k, B::v>::kSmemBytes;
      static bool configured[64];
      int dev = 0;
      cudaGetDevice(&dev);
      if (dev < 0 || dev >= 64 || !configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        KVQ_REQUIRE(e == cudaSuccess, KVQ_ERR_CUDA, "cudaFuncSetAttribute(paged tiles): %s", cudaGetErrorString(e));
        if (dev >= 0 && dev < 64) configured[dev] = true;
      }
      cudaError_t e = launch_pdl(kernel, static_cast<unsigned>(n_items), tiles::kThreads, smem, st, a);
      KVQ_REQUIRE(e == cudaSuccess, KVQ_ERR_CUDA, "kvq_paged_attention: launch failed: %s", cudaGetErrorString(e));
      return KVQ_OK;
    });
  });
}

}  // namespace paged
}  // namespace kvq
