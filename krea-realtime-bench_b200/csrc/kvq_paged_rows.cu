// Attention of few query rows per KV head over the paged quantized cache (sm_100a):
// single tokens, short drafts. Every K and V record of a KV head is read once for all its
// rows. Memory-bound with int8 records; with int4 ones, of half the bytes and as many
// instructions, bound by the issue slots (64 % used, and the ALU 53 %). Measured, 64
// sequences of 946 to 16384 tokens, 8 KV heads, 40 query heads: int4 636 MB in 174 to 177 us
// (3.6 TB/s), int8 1203 MB in 212 us (5.7 of the 6.55 that a copy reaches); two sequences of
// 107 and 131 thousand tokens, int8 K and int4 V: 571 MB in 123 us (4.6 TB/s). A step with
// scales beyond fp16's range is repeated: the int4 batch takes 2.3 times as long if all are.
//
// A CTA of four warps streams its pieces of the plan (kvq_paged_plan) one after the
// other; warp w takes every fourth pair of 16-token storage blocks of a piece. A block's K
// and V records are contiguous, so a stage of the warp's ring is filled by four bulk
// copies (no tensor map) while the other stage is worked on; the warps never wait for
// each other inside a piece. Per block (tokens j, rows n, channels c; mma.sync m16n8k16, fp32 out):
//   S^T[j, n] = sum_c K[j, c] q[n, c]      A = K from registers, B = q held in registers
//   p = 2^(S^T scale - m_n)                m_n moves (and O, l are rescaled) only when some
//                                          logit exceeds it by more than kLag + kBias, one
//                                          vote per block otherwise
//   O^T[c, n] += sum_j V[j, c] p[j, n]     A = V from registers, B = p (transposed, movmatrix)
// Tokens are the M side, so 8 rows cost one N = 8 instruction. tcgen05 would need
// the dequantized tile in shared memory (2 x 256 bytes per row through the shared-
// memory port, more than it moves at memory speed); mma.sync takes it from registers.
// Codes become values in registers, two per instruction: code bits are ored into the
// mantissa of fp16 1024 and the offset subtracted (exact), then times the scale, exact for
// int4; see kScaleLeast for what fp16 does not hold. p is rounded to fp16, S, m, l and O
// are fp32. The order of channels and
// of tokens inside a fragment is free as long as A and B agree: lane (g, t) = (lane /
// 4, lane % 4) holds channels 32t..32t+31 of K rows and channels 16g..16g+15 of V
// rows, 8 or 16 contiguous bytes of shared memory.
// The warps' (m, l, F, O) are joined in shared memory, parts of a unit in the workspace.
#include <cmath>

#include "kvq_paged_dev.cuh"

namespace kvq {
namespace paged {
using namespace sm100;

constexpr int kWarps = 4;
constexpr int kRowThreads = 32 * kWarps;

template <class L, int KB, int VB, int NT>
struct RowGeo {
  static constexpr int kRecK = Rec<L, KB>::kBytes, kRecV = Rec<L, VB>::kBytes;
  // most channel groups of a lane's 32 key channels, of its 16 value channels
  static constexpr int kKG = most_groups<L, 32>(), kVG = most_groups<L, 16>();
  static_assert(kKG <= 4 && kVG <= 3, "group selection");
  static constexpr int kStage = 2 * (kRecK + kRecV);  // two storage blocks
  static constexpr int kStages = 2;
  static constexpr int kRing = kStages * kStage;  // one warp's
  static constexpr int kOffML = kWarps * kRing;
  static constexpr int kOffBar = kOffML + kWarps * 8 * NT * 16;
  static constexpr int kOffMisc = kOffBar + kWarps * kStages * 8;
  static constexpr int kSmemBytes = kOffMisc + 16;
  // resident blocks: shared memory, and registers (168 a thread for three, 255 for two; with
  // four, and spills, 5 to 20 % slower)
  static constexpr int kFit = (228 * 1024) / (kSmemBytes + 1024);
  static constexpr int kCtas = kFit < (NT == 1 ? 3 : 2) ? kFit : (NT == 1 ? 3 : 2);
  static_assert(kRing >= 8 * NT * D * 4, "the join fits a warp's ring");
  static_assert(kRecK % 16 == 0 && kStage % 16 == 0, "bulk copies");
};

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <class L, int KB, int VB, int NT>
__global__ void __launch_bounds__(kRowThreads, (RowGeo<L, KB, VB, NT>::kCtas)) rows_kernel(const __grid_constant__ AttnArgs a) {
  using GEO = RowGeo<L, KB, VB, NT>;
  static_assert(GEO::kStages == 2, "stage and phase below");
  constexpr int kRows = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + GEO::kOffBar) + warp * GEO::kStages;
  volatile int* abort = reinterpret_cast<volatile int*>(smem + GEO::kOffMisc);
  volatile int* last = abort + 1;
  uint8_t* ring = smem + warp * GEO::kRing;
  float4* sm_ml = reinterpret_cast<float4*>(smem + GEO::kOffML);  // [warp][row] (m, l, F)
  if (lane == 0) {
    for (int i = 0; i < GEO::kStages; ++i) mbar_init(&bars[i], 1);
    fence_mbar_init();
  }
  if (tid == 0) *abort = 0;
  __syncthreads();

  // this lane's channel groups: K channels 32t.., V channels 16g..
  const int kbase = group_at<L>(32 * t), vbase = group_at<L>(16 * g);
  uint32_t ksel[GEO::kKG == 1 ? 1 : 16];
  if constexpr (GEO::kKG > 1) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int c = 32 * t + 8 * (i >> 2) + (i & 3);
      const uint32_t la = 2 * (group_at<L>(c) - kbase), lb = 2 * (group_at<L>(c + 4) - kbase);
      ksel[i] = la | (la + 1) << 4 | lb << 8 | (lb + 1) << 12;
    }
  }
  // first channel pair of this lane's second and third V group (8: none)
  int ve1 = 8, ve2 = 8;
  if constexpr (GEO::kVG > 1) {
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      const int l = group_at<L>(16 * g + 2 * i) - vbase;
      if (l >= 1) ve1 = i;
      if (l >= 2) ve2 = i;
    }
  }
  // physical token of S row r: a permutation that spreads both K and V reads over the banks
  auto token_of = [](int r) { return r ^ ((r >> 1) & 1); };

  // what lanes 0-3 copy at each step
  const uint32_t copy_bytes = (lane & 1) ? GEO::kRecV : GEO::kRecK;
  const uint8_t* copy_src = (lane & 1) ? a.v_pages : a.k_pages;
  const uint32_t copy_dst = smem_u32(ring) + ((lane >> 1) & 1) * (GEO::kStage / 2) + ((lane & 1) ? GEO::kRecK : 0);
  // this lane's K row and V rows inside a stage, codes and scales
  const uint32_t k_codes = smem_u32(ring) + token_of(g) * Rec<L, KB>::CW + t * (KB * 4);
  const uint32_t k_scales = smem_u32(ring) + Rec<L, KB>::kCodes + token_of(g) * L::G * 2;
  const int vt0 = token_of(2 * t), vt1 = token_of(2 * t + 1);  // and 8 more
  const uint32_t v_ring = smem_u32(ring) + GEO::kRecK;
  const uint32_t v_codes0 = v_ring + vt0 * Rec<L, VB>::CW + g * (2 * VB), v_codes1 = v_codes0 + (vt1 - vt0) * Rec<L, VB>::CW;
  const uint32_t v_scales0 = v_ring + Rec<L, VB>::kCodes + vt0 * L::G * 2, v_scales1 = v_scales0 + (vt1 - vt0) * L::G * 2;

  pdl_wait();
  pdl_launch_dependents();
  uint32_t step = 0;  // blocks this warp has consumed, over all pieces: stage and phase
  // one item per block: no list of first items
  const int i0 = a.cta_first ? __ldg(a.cta_first + blockIdx.x) : static_cast<int>(blockIdx.x);
  const int i1 = a.cta_first ? __ldg(a.cta_first + blockIdx.x + 1) : i0 + 1;
  for (int ii = i0; ii < i1; ++ii) {
    const Item it = a.items[ii];
    // this warp's pairs of list entries: 2 (warp + kWarps k) and the next
    const int n_blk = it.je - it.jb, n_pair = (n_blk + 1) / 2;
    int n_mine = n_pair > warp ? (n_pair - warp + kWarps - 1) / kWarps : 0;
    if (__any_sync(0xffffffffu, *abort)) n_mine = 0;  // a wait gave up: only the counting goes on
    const uint32_t step0 = step;
    auto entry = [&](int k) { return 2 * (warp + kWarps * k); };  // relative to jb

    // copies: lanes 2i, 2i + 1 look up the two blocks of step base + i, 16 steps at a time;
    // lanes 0-3 copy the step's records: K, V of the first block, K, V of the second
    uint32_t where = 0;
    auto issue = [&](int k) {
      if ((k & 15) == 0) {
        const int e = entry(k + (lane >> 1)) + (lane & 1);
        bool ok;
        if (e < n_blk) where = static_cast<uint32_t>(a.p.block(it.seq, it.head, it.block_at(it.jb + e), ok));
      }
      const uint32_t b = __shfl_sync(0xffffffffu, where, 2 * (k & 15) + ((lane >> 1) & 1));
      const uint32_t st = (step0 + k) & 1;
      const bool two = entry(k) + 1 < n_blk;
      if (lane == 0) mbar_arrive_expect_tx(&bars[st], two ? GEO::kStage : GEO::kStage / 2);
      __syncwarp();
      if (lane < (two ? 4 : 2))
        bulk_load(copy_dst + st * GEO::kStage, copy_src + static_cast<uint64_t>(b) * copy_bytes, copy_bytes, &bars[st]);
    };
    // q fragments: rows 8 nt + g, channels (32t + 8i + 2h + {0, 4}) and the next two; the
    // loads are under way while the first copies are looked up
    uint4 qv[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int n = 8 * nt + g;
      const int row = it.row0 + min(n, it.n_rows - 1);
      const int i = row / a.group;
      const uint4* src = reinterpret_cast<const uint4*>(a.q + static_cast<int64_t>(it.q_first + i) * a.q_stride +
                                                        (it.head * a.group + row - i * a.group) * D + 32 * t);
#pragma unroll
      for (int w = 0; w < 4; ++w) qv[nt][w] = ld_global_nc_v4(src + w);
    }
    if (n_mine > 0) issue(0);
    uint32_t qf[NT][8][2];
    float sc[NT][2];  // softmax scale of rows 8 nt + 2t, + 2t + 1, with the power of two taken from the row
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint32_t most = max(max(most_of(qv[nt][0]), most_of(qv[nt][1])), max(most_of(qv[nt][2]), most_of(qv[nt][3])));
      uint32_t least = min(min(least_of(qv[nt][0]), least_of(qv[nt][1])), min(least_of(qv[nt][2]), least_of(qv[nt][3])));
      extremes_of_lanes<1, 2>(most, least);
      const int e = query_exponent(most, least);
#pragma unroll
      for (int i = 0; i < 2; ++i) sc[nt][i] = row_scale_of(a.scale_log2, __shfl_sync(0xffffffffu, e, 4 * (2 * t + i)));
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint4 v = 8 * nt + g < it.n_rows ? to_f16(qv[nt][w], e) : make_uint4(0, 0, 0, 0);
        qf[nt][2 * w][0] = __byte_perm(v.x, v.z, 0x5410);
        qf[nt][2 * w][1] = __byte_perm(v.x, v.z, 0x7632);
        qf[nt][2 * w + 1][0] = __byte_perm(v.y, v.w, 0x5410);
        qf[nt][2 * w + 1][1] = __byte_perm(v.y, v.w, 0x7632);
      }
    }

    // what the rows 8 nt + 2t, + 2t + 1 see, and what all rows of the item see
    Seen see[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = it.row0 + min(8 * nt + 2 * t + e, it.n_rows - 1);
        see[nt][e] = seen_by(a, it.start + row / a.group, it.kv_len);
      }
    const Seen first = seen_by(a, it.start + it.row0 / a.group, it.kv_len);
    const Seen final_ = seen_by(a, it.start + (it.row0 + it.n_rows - 1) / a.group, it.kv_len);

    float o[NT][8][4], m[NT][2], l[NT][2], F[NT][2];  // O is kept divided by 2^F
    bool f_any = false;                               // whether any row's F is not 0
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.0f;
      m[nt][0] = m[nt][1] = -1.0e30f;
      l[nt][0] = l[nt][1] = F[nt][0] = F[nt][1] = 0.0f;
    }

    for (int k = 0; k < n_mine; ++k) {
      const uint32_t st = (step0 + k) & 1;
      // the other stage: every lane has read it (the __syncwarp that ended the last step)
      if (k + 1 < n_mine) issue(k + 1);
      const uint32_t phase = ((step0 + k) >> 1) & 1;
      if (!__all_sync(0xffffffffu, mbar_try_wait(smem_u32(&bars[st]), phase))) {
        const bool ok = mbar_wait(&bars[st], phase, abort, a.status, a.wait_cycles);
        if (!__all_sync(0xffffffffu, ok)) {
          // copies in flight land before the shared memory is given up
          mbar_drain(&bars[st], phase, a.status, a.wait_cycles);
          if (k + 1 < n_mine) mbar_drain(&bars[st ^ 1], ((step0 + k + 1) >> 1) & 1, a.status, a.wait_cycles);
          break;
        }
      }
      const uint32_t at = st * GEO::kStage;
      const int e0 = it.jb + entry(k);
      const bool two = e0 + 1 < it.je;
      const int ta = it.block_at(e0) * kBlock, tz = it.block_at(e0 + 1) * kBlock;  // first tokens of the blocks
      const bool whole = two && tz + kBlock <= first.hi && (ta >= final_.lo || tz + kBlock <= first.kept);

      // ---- S^T of storage block bb. EXACT: with a power of two taken out of the tokens beyond
      // (kScaleLeast, kScaleMost); else as if there were none, keeping the scales' extremes.
      uint32_t least = kScaleLeast, most = 0;
      auto scores = [&](const uint32_t off, float (&acc)[NT][4], auto exact) {
        constexpr bool EXACT = decltype(exact)::value;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[nt][e] = 0.0f;
        uint32_t kw[2][KB == 4 ? 4 : 8], ks01[2], ks23[2];
        float back[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t src = k_codes + off + 8 * r * Rec<L, KB>::CW;
#pragma unroll
          for (int w = 0; w < KB / 4; ++w) {
            const uint4 v = ld_shared_v4(src + 16 * w);
            kw[r][4 * w] = v.x;
            kw[r][4 * w + 1] = v.y;
            kw[r][4 * w + 2] = v.z;
            kw[r][4 * w + 3] = v.w;
          }
          const uint32_t from = k_scales + off + 8 * r * L::G * 2;
          uint32_t x[GEO::kKG], top = 0, low = 0xFFFFu;
          float f[GEO::kKG];
          uint32_t used = ~0u;
          bool one = false;
#pragma unroll
          for (int q = 0; q < GEO::kKG; ++q) {
            x[q] = ld_shared_u16(from + 2 * (GEO::kKG == 1 ? kbase : min(kbase + q, L::G - 1)));
            one |= x[q] == kScaleOne;
          }
          if (EXACT && __any_sync(0xffffffffu, one)) used = used_groups<L, KB, 32>(src, 32 * t, kbase);
#pragma unroll
          for (int q = 0; q < GEO::kKG; ++q) {
            if (EXACT && !((used >> q) & 1u)) continue;
            top = max(top, x[q]);
            low = min(low, x[q]);
          }
#pragma unroll
          for (int q = 0; q < GEO::kKG; ++q) f[q] = (used >> q) & 1u ? __uint_as_float(x[q] << 16) : 0.0f;
          if constexpr (EXACT) {
            extremes_of_lanes<1, 2>(top, low);
            const int e = top == 0 ? 0 : scale_exponent(top, low);
            back[r] = pow2i(e);
#pragma unroll
            for (int q = 0; q < GEO::kKG; ++q) f[q] *= pow2i(-e);
          } else {
            most = max(most, top);
            least = min(least, low);
          }
          ks01[r] = pack_f16x2(f[0], f[GEO::kKG > 1 ? 1 : 0]);
          ks23[r] = 0;
          if constexpr (GEO::kKG > 2) ks23[r] = pack_f16x2(f[2], f[GEO::kKG > 3 ? 3 : 2]);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t f[2][4];
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t v;
              if constexpr (KB == 4) {
                const uint32_t x = j < 2 ? kw[r][w] : kw[r][w] >> 8;
                v = (j & 1) ? int4_high_f16(x) : int4_low_f16(x);
              } else {
                v = int8_pair_f16(__byte_perm(kw[r][2 * w], kw[r][2 * w + 1], j | j << 4 | (4 + j) << 8 | (4 + j) << 12));
              }
              uint32_t sp = ks01[r];
              if constexpr (GEO::kKG > 1) sp = __byte_perm(ks01[r], ks23[r], ksel[4 * w + j]);
              f[r][j] = h16mul2(v, sp);
            }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816(acc[nt], f[0][2 * h], f[1][2 * h], f[0][2 * h + 1], f[1][2 * h + 1], qf[nt][2 * w + h][0],
                       qf[nt][2 * w + h][1]);
        }
        if constexpr (EXACT) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][e] *= back[e >> 1];
        }
      };
      float s[2][NT][4];
      scores(at, s[0], std::false_type{});
      scores(at + GEO::kStage / 2, s[1], std::false_type{});

      // ---- V's scales, of this lane's tokens: S rows 2t, 2t + 1, 8 + 2t, 9 + 2t, of block bb
      auto value_scales = [&](const uint32_t off, const int first_token, const bool any_live, uint32_t (&vs)[2][GEO::kVG],
                              float (&ve)[2], auto exact) {
        constexpr bool EXACT = decltype(exact)::value;
        float f[4][GEO::kVG];
        int ex[4] = {0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t from = ((u & 1) ? v_scales1 : v_scales0) + off + (u >> 1) * 8 * L::G * 2;
          // rows past the end hold anything: as zeros they add nothing
          const bool live = whole || (any_live && first_token + ((u & 1) ? vt1 : vt0) + (u >> 1) * 8 < it.kv_len);
          uint32_t used = live ? ~0u : 0u, top = 0, low = 0xFFFFu, xs[GEO::kVG];
          bool one = false;
#pragma unroll
          for (int q = 0; q < GEO::kVG; ++q) {
            xs[q] = ld_shared_u16(from + 2 * (GEO::kVG == 1 ? vbase : min(vbase + q, L::G - 1)));
            one |= xs[q] == kScaleOne;
          }
          if (EXACT && __any_sync(0xffffffffu, one))
            used &= used_groups<L, VB, 16>(((u & 1) ? v_codes1 : v_codes0) + off + (u >> 1) * 8 * Rec<L, VB>::CW, 16 * g, vbase);
#pragma unroll
          for (int q = 0; q < GEO::kVG; ++q) {
            const uint32_t x = (used >> q) & 1u ? xs[q] : 0;
            top = max(top, x);
            if (!EXACT || ((used >> q) & 1u)) low = min(low, x);
            f[u][q] = __uint_as_float(x << 16);
          }
          if constexpr (EXACT) {
            extremes_of_lanes<4, 16>(top, low);
            ex[u] = !live ? 0 : top == 0 ? kNoScale : scale_exponent(top, low);
#pragma unroll
            for (int q = 0; q < GEO::kVG; ++q) f[u][q] *= pow2i(-ex[u]);
          } else {
            most = max(most, top);
            least = min(least, live ? low : kScaleLeast);
          }
        }
        if constexpr (EXACT) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int ea = __shfl_sync(0xffffffffu, ex[2 * r], g >> 1), eb = __shfl_sync(0xffffffffu, ex[2 * r + 1], g >> 1);
            ve[r] = static_cast<float>((g & 1) ? eb : ea);
          }
        }
#pragma unroll
        for (int q = 0; q < GEO::kVG; ++q) {
          vs[0][q] = pack_f16x2(f[0][q], f[1][q]);
          vs[1][q] = pack_f16x2(f[2][q], f[3][q]);
        }
      };
      uint32_t vs[2][2][GEO::kVG];
      float ve[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};  // exponents taken out of the tokens of S rows g, 8 + g
      value_scales(at, ta, true, vs[0], ve[0], std::false_type{});
      value_scales(at + GEO::kStage / 2, tz, two, vs[1], ve[1], std::false_type{});
      bool wide_v = false;
      // Rows past the end hold anything, zeros where nothing was written yet, and those of K
      // have counted above (a test per row there cost 3 % of a decode batch): where there are
      // some, the live rows' scales are looked at again.
      auto live_beyond = [&]() {
        bool far = false;
#pragma unroll 1
        for (int bb = 0; bb < (two ? 2 : 1); ++bb) {
          const uint32_t off = at + bb * (GEO::kStage / 2);
          const int n_live = it.kv_len - (bb ? tz : ta);
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int q = 0; q < GEO::kKG; ++q) {
              const uint32_t x = ld_shared_u16(k_scales + off + 8 * r * L::G * 2 + 2 * min(kbase + q, L::G - 1));
              far |= token_of(g) + 8 * r < n_live && beyond(x, kScaleLeast, kScaleMost);
            }
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int q = 0; q < GEO::kVG; ++q) {
              const uint32_t x = ld_shared_u16(((u & 1) ? v_scales1 : v_scales0) + off + (u >> 1) * 8 * L::G * 2 +
                                               2 * min(vbase + q, L::G - 1));
              far |= ((u & 1) ? vt1 : vt0) + (u >> 1) * 8 < n_live && beyond(x, kScaleLeast, kScaleMost);
            }
        }
        return far;
      };
      if (__any_sync(0xffffffffu, most > kScaleMost || least < kScaleLeast) &&
          (whole || __any_sync(0xffffffffu, live_beyond()))) {
        // rare: once more, with the powers of two
#pragma unroll 1
        for (int bb = 0; bb < 2; ++bb) {
          float sx[NT][4], vx[2];
          uint32_t vsx[2][GEO::kVG];
          scores(at + bb * (GEO::kStage / 2), sx, std::true_type{});
          value_scales(at + bb * (GEO::kStage / 2), bb ? tz : ta, !bb || two, vsx, vx, std::true_type{});
          wide_v = __any_sync(0xffffffffu, vx[0] != 0.0f || vx[1] != 0.0f) || wide_v;
#pragma unroll
          for (int b = 0; b < 2; ++b)
            if (b == bb) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[b][nt][e] = sx[nt][e];
#pragma unroll
              for (int q = 0; q < GEO::kVG; ++q) {
                vs[b][0][q] = vsx[0][q];
                vs[b][1][q] = vsx[1][q];
              }
              ve[b][0] = vx[0];
              ve[b][1] = vx[1];
            }
        }
      }

      // ---- softmax weights
      uint32_t pf[NT][2][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (!whole) {
#pragma unroll
          for (int bb = 0; bb < 2; ++bb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = (bb ? tz : ta) + 8 * (e >> 1) + token_of(g);
              const Seen& v = see[nt][e & 1];
              if (!(j < v.hi && (j >= v.lo || j < v.kept)) || (bb && !two)) s[bb][nt][e] = -INFINITY;
            }
        }
        const float mx0 = fmaxf(fmaxf(s[0][nt][0], s[0][nt][2]), fmaxf(s[1][nt][0], s[1][nt][2])) * sc[nt][0];
        const float mx1 = fmaxf(fmaxf(s[0][nt][1], s[0][nt][3]), fmaxf(s[1][nt][1], s[1][nt][3])) * sc[nt][1];
        if (__any_sync(0xffffffffu, mx0 - m[nt][0] > kBias + kLag || mx1 - m[nt][1] > kBias + kLag)) {
          float n0 = mx0, n1 = mx1;
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, x));
            n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, x));
          }
          n0 = fmaxf(n0 - kBias, m[nt][0]);
          n1 = fmaxf(n1 - kBias, m[nt][1]);
          const float a0 = ex2f(m[nt][0] - n0), a1 = ex2f(m[nt][1] - n1);
          l[nt][0] *= a0;
          l[nt][1] *= a1;
          if (wide_v || f_any) {  // F follows, and O below
            F[nt][0] += m[nt][0] - n0;
            F[nt][1] += m[nt][1] - n1;
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              o[nt][i][0] *= a0;
              o[nt][i][1] *= a1;
              o[nt][i][2] *= a0;
              o[nt][i][3] *= a1;
            }
          }
          m[nt][0] = n0;
          m[nt][1] = n1;
        }
#pragma unroll
        for (int bb = 0; bb < 2; ++bb) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) p[e] = ex2f(fmaf(s[bb][nt][e], sc[nt][e & 1], -m[nt][e & 1]));
          l[nt][0] += p[0] + p[2];
          l[nt][1] += p[1] + p[3];
          pf[nt][bb][0] = transpose8x8(pack_f16x2(p[0], p[1]));
          pf[nt][bb][1] = transpose8x8(pack_f16x2(p[2], p[3]));
        }
      }
      if (wide_v || f_any) {
        f_any = false;
        // weights times the powers of two taken out of the values, relative to 2^F, in log2:
        // y = s * scale - m + e. F grows where 2^(y - F) would leave fp16.
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int bb = 0; bb < 2; ++bb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[bb][nt][e] = fmaf(s[bb][nt][e], sc[nt][e & 1], -m[nt][e & 1]) + ve[bb][e >> 1];
              top[e & 1] = fmaxf(top[e & 1], s[bb][nt][e]);
            }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], d));
            const float Fn = next_f(F[nt][i], top[i]);
            const float back = ex2f(F[nt][i] - Fn);
            F[nt][i] = Fn;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              o[nt][c][i] *= back;
              o[nt][c][2 + i] *= back;
            }
          }
#pragma unroll
          for (int bb = 0; bb < 2; ++bb)
#pragma unroll
            for (int r = 0; r < 2; ++r)
              pf[nt][bb][r] = transpose8x8(pack_f16x2(ex2f(s[bb][nt][2 * r] - F[nt][0]), ex2f(s[bb][nt][2 * r + 1] - F[nt][1])));
          f_any = __any_sync(0xffffffffu, F[nt][0] != 0.0f || F[nt][1] != 0.0f) || f_any;
        }
      }

      // ---- O^T
#pragma unroll
      for (int bb = 0; bb < 2; ++bb) {
        const uint32_t off = at + bb * (GEO::kStage / 2);
        uint32_t vw[4][VB == 4 ? 2 : 4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t src = ((u & 1) ? v_codes1 : v_codes0) + off + (u >> 1) * 8 * Rec<L, VB>::CW;
          if constexpr (VB == 4) {
            const uint2 v = ld_shared_v2(src);
            vw[u][0] = v.x;
            vw[u][1] = v.y;
          } else {
            const uint4 v = ld_shared_v4(src);
            vw[u][0] = v.x;
            vw[u][1] = v.y;
            vw[u][2] = v.z;
            vw[u][3] = v.w;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // channels 16g + 2i (rows g) and 16g + 2i + 1 (rows 8 + g)
          uint32_t f[2][2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t sp = vs[bb][u][0];
            if (GEO::kVG > 1) sp = i >= ve1 ? vs[bb][u][GEO::kVG > 1 ? 1 : 0] : sp;
            if (GEO::kVG > 2) sp = i >= ve2 ? vs[bb][u][GEO::kVG > 2 ? 2 : 0] : sp;
            if constexpr (VB == 4) {
              const int b = i & 3;  // the byte with both channels, of either token
              const uint32_t x = __byte_perm(vw[2 * u][i >> 2], vw[2 * u + 1][i >> 2], b | b << 4 | (4 + b) << 8 | (4 + b) << 12);
              f[u][0] = h16mul2(int4_low_f16(x), sp);
              f[u][1] = h16mul2(int4_high_f16(x), sp);
            } else {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int c = 2 * i + e, b = c & 3;
                f[u][e] = h16mul2(int8_pair_f16(__byte_perm(vw[2 * u][c >> 2], vw[2 * u + 1][c >> 2],
                                                      b | b << 4 | (4 + b) << 8 | (4 + b) << 12)), sp);
              }
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816(o[nt][i], f[0][0], f[0][1], f[1][0], f[1][1], pf[nt][bb][0], pf[nt][bb][1]);
        }
      }
      __syncwarp();
    }
    step = step0 + n_mine;

    // ---- join the warps: each leaves (m, l, F, O) in its own ring, whose copies are all
    // consumed. Sums and O each have their own greatest term, m and m + F: O times 2^F may
    // be beyond fp32 until it is divided by the sum.
    float* mine = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[nt][e];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
        const int n = 8 * nt + 2 * t + e;
        if (g == 0) sm_ml[warp * kRows + n] = make_float4(m[nt][e], x, F[nt][e], 0.0f);
        float4* dst = reinterpret_cast<float4*>(mine + n * D + 16 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          dst[i] = make_float4(o[nt][2 * i][e], o[nt][2 * i][2 + e], o[nt][2 * i + 1][e], o[nt][2 * i + 1][2 + e]);
      }
    }
    __syncthreads();
    float* slot = it.parts > 1 ? a.ws + static_cast<int64_t>(it.slot + it.part) * slot_floats(kRows) : nullptr;
    // Rows are dealt to the warps, lane i has channels 4i..4i+3.
    auto finish = [&](int n, float4 acc, float mm, float total, float f) {
      const int row = it.row0 + n, i = row / a.group;
      const int64_t tok = it.q_first + i;
      const int h = it.head * a.group + row - i * a.group;
      const float inv = total == 0.0f ? 0.0f : 1.0f / total, of = ex2f(f);
      *reinterpret_cast<uint2*>(a.out + tok * a.out_stride + h * D + 4 * lane) =
          make_uint2(pack_bf16x2(acc.x * inv * of, acc.y * inv * of), pack_bf16x2(acc.z * inv * of, acc.w * inv * of));
      if (a.lse && lane == 0)
        a.lse[tok * a.n_q_heads + h] = total == 0.0f ? -INFINITY : 0.69314718055994531f * (mm + log2f(total));
    };
    auto add = [](float4& acc, float f, const float4& v) {
      acc = make_float4(fmaf(f, v.x, acc.x), fmaf(f, v.y, acc.y), fmaf(f, v.z, acc.z), fmaf(f, v.w, acc.w));
    };
    for (int n = warp; n < it.n_rows; n += kWarps) {
      float mm = -1.0e30f, total = 0.0f;
      float4 ml[kWarps];
      bool wide = false;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        ml[w] = sm_ml[w * kRows + n];
        mm = fmaxf(mm, ml[w].x);
        wide = wide || ml[w].z != 0.0f;
      }
      float mf = -1.0e30f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mf = fmaxf(mf, ml[w].x + ml[w].z);
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2f(ml[w].x - mm);
        total += f * ml[w].y;
        add(acc, ex2f(ml[w].x + ml[w].z - mf), reinterpret_cast<const float4*>(smem + w * GEO::kRing + n * D * 4)[lane]);
      }
      if (slot) {
        reinterpret_cast<float4*>(slot + n * D)[lane] = acc;
        if (lane == 0) reinterpret_cast<float4*>(slot + kRows * D)[n] = make_float4(mm, total, mf - mm, 0.0f);
      } else {
        finish(n, acc, mm, total, mf - mm);
      }
    }
    if (slot) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const unsigned old = atomicAdd(a.ctr + it.unit, 1u);
        *last = old == static_cast<unsigned>(it.parts - 1);
        if (*last) a.ctr[it.unit] = 0u;  // ready for the next launch
      }
      __syncthreads();
      if (*last) {
        // All parts are in the workspace: join them in part order, kAtOnce parts of a row in
        // flight per warp, with the online rescaling between those groups.
        __threadfence();
        constexpr int kAtOnce = 16;
        const float* base = a.ws + static_cast<int64_t>(it.slot) * slot_floats(kRows);
        for (int n = warp; n < it.n_rows; n += kWarps) {
          float mm = -1.0e30f, mf = -1.0e30f, total = 0.0f;
          float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int p0 = 0; p0 < it.parts; p0 += kAtOnce) {
            const float* sp = base + static_cast<int64_t>(p0) * slot_floats(kRows);
            const int np = it.parts - p0;
            float4 ml = make_float4(-1.0e30f, 0.0f, 0.0f, 0.0f);
            if (lane < min(np, kAtOnce))
              ml = __ldcg(reinterpret_cast<const float4*>(sp + lane * slot_floats(kRows) + kRows * D) + n);
            float4 v[kAtOnce];
#pragma unroll
            for (int q = 0; q < kAtOnce; ++q)
              v[q] = q < np ? __ldcg(reinterpret_cast<const float4*>(sp + q * slot_floats(kRows) + n * D) + lane)
                            : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float top = fmaxf(ml.x, mm), top_f = fmaxf(ml.x + ml.z, mf);
#pragma unroll
            for (int x = 8; x > 0; x >>= 1) {
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
              top_f = fmaxf(top_f, __shfl_xor_sync(0xffffffffu, top_f, x));
            }
            top = __shfl_sync(0xffffffffu, top, 0);  // lanes 0-15 hold the parts
            top_f = __shfl_sync(0xffffffffu, top_f, 0);
            const float f0 = ex2f(mf - top_f), f = ex2f(ml.x + ml.z - top_f);
            float sum = ex2f(ml.x - top) * ml.y;
#pragma unroll
            for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            total = total * ex2f(mm - top) + __shfl_sync(0xffffffffu, sum, 0);
            acc = make_float4(acc.x * f0, acc.y * f0, acc.z * f0, acc.w * f0);
#pragma unroll
            for (int q = 0; q < kAtOnce; ++q) add(acc, __shfl_sync(0xffffffffu, f, q), v[q]);
            mm = top;
            mf = top_f;
          }
          finish(n, acc, mm, total, mf - mm);
        }
      }
    }
    // the ring was written by threads: order that before the next piece's copies into it
    fence_proxy_async_smem();
    __syncthreads();
  }
}

int rows_ctas_per_sm(int layout, int k_bits, int v_bits, int row_tile) {
  return with_layout(layout, [&](auto lt) {
    using L = decltype(lt);
    return with_bits(k_bits, v_bits, [&](auto bt) -> int {
      using B = decltype(bt);
      return row_tile == 8 ? RowGeo<L, B::k, B::v, 1>::kCtas : RowGeo<L, B::k, B::v, 2>::kCtas;
    });
  });
}

int launch_rows(const AttnArgs& a, int layout, int k_bits, int v_bits, int row_tile, int n_ctas, cudaStream_t st) {
  return with_layout(layout, [&](auto lt) {
    using L = decltype(lt);
    return with_bits(k_bits, v_bits, [&](auto bt) {
      using B = decltype(bt);
      auto go = [&](auto kernel, int smem, bool* configured) -> int {
        int dev = 0;
        cudaGetDevice(&dev);
        if (dev < 0 || dev >= 64 || !configured[dev]) {
          cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
          KVQ_REQUIRE(e == cudaSuccess, KVQ_ERR_CUDA, "cudaFuncSetAttribute(paged rows): %s", cudaGetErrorString(e));
          if (dev >= 0 && dev < 64) configured[dev] = true;
        }
        cudaError_t e = launch_pdl(kernel, static_cast<unsigned>(n_ctas), kRowThreads, smem, st, a);
        KVQ_REQUIRE(e == cudaSuccess, KVQ_ERR_CUDA, "kvq_paged_attention: launch failed: %s", cudaGetErrorString(e));
        return KVQ_OK;
      };
      static bool done1[64], done2[64];
      if (row_tile == 8) return go(rows_kernel<L, B::k, B::v, 1>, RowGeo<L, B::k, B::v, 1>::kSmemBytes, done1);
      return go(rows_kernel<L, B::k, B::v, 2>, RowGeo<L, B::k, B::v, 2>::kSmemBytes, done2);
    });
  });
}

}  // namespace paged
}  // namespace kvq
