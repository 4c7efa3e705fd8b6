// Decode attention of requests that share long prefixes held once in the
// paged cache (reference KV format: uint8 codes, float32 scale per 64 values).
//
// One decode row per request reads its whole context alone: behind a shared
// prefix of p tokens that is B * p rows of K and V.  Here the query rows of a
// group -- requests x the G query heads of a KV head -- are the M side of one
// product with the prefix, which is then read and decoded once for all:
//   1. own tokens: the paged decode kernels of qkv_attn.cu, writing partials.
//   2. prefix: CTA = (2 tiles of 128 rows, KV head, split of the prefix).
//      S = Q K^T and O = P V on tcgen05 as in prompt_attn.cu; bulk copies bring
//      the codes of a block of 128 keys, eight warps turn them into fp16 tiles
//      in shared memory.
//   3. combine: out = sum 2^(m_s - m) O_s / sum 2^(m_s - m) l_s over splits.
//
// What bounds it: the prefix kernel's start (plan, page table, first copies and
// their decoding: 10000 cycles before the first scores), then the chain of a
// block (copy, decoding, scores, softmax, product): 5200 cycles a block of two
// tiles in splits of 27, with half of the issue slots used.  It is let onto the
// SMs as the own tokens' CTAs leave them.  A split costs a start, and
// its partials are written and read: 8192 keys and 64 rows over 4 KV heads by
// one CTA an SM against half as many 24 / 32 us, 20001 keys and 128 rows over
// 8 KV heads 58 / 99 us.
// Measured (own tokens, prefix, combine; 32 heads of 128): 64 rows behind 8192
// tokens, up to 512 of their own, 4 KV heads 12.8 / 28.2 / 5.8 us, 43 us in
// all (29 MB, 8.9 GFLOP); 128 rows in two groups behind 20001 and 16906, up to
// 2000 of their own, 8 KV heads 75 / 78 / 6 us, 141 us in all (354 MB, 40.5
// GFLOP); 4 rows behind 500 tokens 5.0 / 10.2 / 3.8 us.
//
// fp16 operands: a code is exact in 11 bits, and scale * code costs one
// rounding of 2^-11, where bf16 would cost 2^-8 on K, V and P each -- more than
// the output's own rounding.  fp16's range is made up for by powers of two,
// which are exact: each query row is scaled by its own absmax, K and V by the
// largest scale of each block (groups of zeros, whose scale is 1 whatever lies
// beside them, do not count), which lands at 2^(15-BITS): nothing is cut, and
// below it a scale of 8 significant bits (rows quantized as bf16) is exact for
// 2^(32-BITS), one of 11 for 2^(29-BITS).  K's power comes back into the scores.
// V's goes into them as an exponent: with v = 2^a v' the row's weights are
// 2^(s + a - m), whose products with v' add up to 2^-m sum 2^s v, and which
// times 2^-a add up to l = 2^-m sum 2^s.
#include "attn_tc.cuh"

namespace b2f {

// qkv_attn.cu: decode attention of B rows over their own pages, as partials
// (o [B * Hq][n_splits][D], then m, l pairs).
int launch_own_partials(const __nv_bfloat16* q, const uint8_t* kc, const float* ks, const uint8_t* vc, const float* vs,
                        const int32_t* table, int64_t width, const int32_t* lens, int B, int Hq, int Hkv, int D, int P,
                        int bits, float scale, int n_splits, int max_len, float* o_part, float* ml_part,
                        cudaStream_t st);

// warps 0-15 softmax, 16-19 decode K, 20-23 V, 24 issues the MMAs, 25 copies K and finds its power, 26 V
constexpr int PX_THREADS = 864;
constexpr int PX_MMA = 24, PX_COPY = 25;
constexpr int PX_BN = 128;  // keys per block
constexpr int PX_SMS = 148;
// Stages alternate K and V (it = 2 j, 2 j + 1): an even number, so that a
// stage holds one of the two only and its readers see its phases in turn.
constexpr int PX_RAW = 2;   // blocks of codes in flight
constexpr int PX_RING = 4;  // decoded tiles
struct PrefixParams {
  const __nv_bfloat16* q;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int32_t *table, *lens, *off;
  int64_t width;
  float *o_part, *ml_part;  // [CTA][256 rows][DP], [CTA][256 rows] of (m, l)
  int* quota;               // how the prefixes are split, for the combine
  float scale2;   // |softmax_scale| * log2(e)
  int negate;     // softmax_scale < 0: the MMA negates Q
  int B, Ng, Hq, Hkv, G, P, tpt, max_prefix;
  int beside;     // launched to run beside the previous kernel (see launch_prefix)
};

template <int DP, int BITS>
struct PrefixSmem {
  static constexpr int TILE = 128 * DP * 2, RB = DP * BITS / 8, DG = DP / 64;
  static constexpr int CODES = PX_BN * RB, RAW = CODES + PX_BN * DG * 4;  // codes, then scales
  static constexpr int PITCH = DP * 4 + 16;                               // bytes between output rows on their way out
  uint8_t q[2][TILE];           // at the end, with the ring, the output rows
  uint8_t ring[PX_RING][TILE];  // K_0 V_0 K_1 V_1 ..., fp16
  uint8_t raw[PX_RAW][RAW];     // the same blocks as codes
  uint16_t exchange[2][128];    // between the two threads of a row
  // Of block j (mod 8: the copies are at most 4 blocks ahead of the softmax).
  float norm[2][8];             // the power of K, of V; negative: some keys do not count
  float k_back[8];              // 1 / the power of K
  float2 v_power[8];            // a, 2^-a
  uint64_t raw_full[PX_RAW], raw_empty[PX_RAW], full[PX_RING], empty[PX_RING], q_full, s_full[2], p_full[2], pv_done[2],
      drain;
  // Block j (mod 4) has its power.  The MMA warp waits for V's before the scores
  // of j; four blocks on there is another only after P V of j.
  uint64_t norm_full[2][4];
  int item[6];  // group, first request, requests from there, prefix length, KV head, split
  int per;  // blocks a CTA of the group
  uint32_t tmem;
  int abort_flag;
};

// 4 codes (the bytes of w) as fp16 (code - top) * scale
__device__ __forceinline__ uint2 codes_to_f16(uint32_t w, uint32_t off2, uint32_t scale2) {
  const uint32_t a = prmt(w, 0x64646464u, 0x4140u), b = prmt(w, 0x64646464u, 0x4342u);  // 1024 + code
  const __half2 o = *reinterpret_cast<const __half2*>(&off2), s = *reinterpret_cast<const __half2*>(&scale2);
  const __half2 x = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&a), o), s);
  const __half2 y = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&b), o), s);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

// 16 bytes of packed codes as 128 / BITS bytes, one code each, in order
template <int BITS>
__device__ __forceinline__ void spread_codes(const uint4& q, uint32_t (&w)[32 / BITS]) {
  const uint32_t in[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BITS == 8) {
      w[i] = in[i];
    } else if constexpr (BITS == 4) {
      const uint32_t hi = (in[i] >> 4) & 0x0F0F0F0Fu, lo = in[i] & 0x0F0F0F0Fu;
      w[2 * i] = prmt(hi, lo, 0x5140u);
      w[2 * i + 1] = prmt(hi, lo, 0x7362u);
    } else {
      const uint32_t a = (in[i] >> 6) & 0x03030303u, b = (in[i] >> 4) & 0x03030303u, c = (in[i] >> 2) & 0x03030303u,
                     d = in[i] & 0x03030303u;
      const uint32_t ab01 = prmt(a, b, 0x5140u), ab23 = prmt(a, b, 0x7362u), cd01 = prmt(c, d, 0x5140u),
                     cd23 = prmt(c, d, 0x7362u);
      w[4 * i] = prmt(ab01, cd01, 0x5410u);
      w[4 * i + 1] = prmt(ab01, cd01, 0x7632u);
      w[4 * i + 2] = prmt(ab23, cd23, 0x5410u);
      w[4 * i + 3] = prmt(ab23, cd23, 0x7632u);
    }
  }
}

// The groups as the device finds them: which rows, how many pairs of tiles,
// how many blocks of keys.
struct PrefixGroup {
  int lo, hi, len, pairs, blocks;
  __device__ __forceinline__ void look(const int32_t* off, const int32_t* lens, int g, int Ng, int B, int span,
                                       int max_prefix) {
    lo = hi = len = 0;
    if (g < Ng) {
      lo = min(max(off[g], 0), B);
      hi = min(max(off[g + 1], lo), B);
      len = min(max(lens[g], 0), max_prefix);
    }
    pairs = (hi - lo + span - 1) / span;
    blocks = pairs ? (len + PX_BN - 1) / PX_BN : 0;
  }
  // how a prefix is split: by `quota` blocks a CTA, or (negative) into -quota
  __device__ __forceinline__ int splits(int quota) const {
    return quota > 0 ? (blocks + quota - 1) / quota : min(blocks, -quota);
  }
};

// How the prefixes are split, by the whole warp: the fewest blocks a CTA (to a
// 32nd) with which all fit one CTA per SM (a CTA takes the whole SM's shared
// memory), so that long and short prefixes end together; or all alike, where
// that gives the longest no more.  Measured, alike against by quota: groups of
// 8 rows behind 16000, 1000, 500 and 2000 tokens 37 / 19 us, of 64 behind
// 20001 and 2000 55 / 41, of 60 and 68 behind 20001 and 16906 72 / 76.
__device__ __forceinline__ int prefix_quota(const int32_t* off, const int32_t* lens, int Ng, int B, int span, int Hkv,
                                            int max_prefix) {
  const int lane = threadIdx.x & 31;
  PrefixGroup own;
  own.look(off, lens, lane, Ng, B, span, max_prefix);
  auto over_groups = [&](auto f) {
    f(own);
    for (int g = 32 + lane; g < Ng; g += 32) {
      PrefixGroup x;
      x.look(off, lens, g, Ng, B, span, max_prefix);
      f(x);
    }
  };
  float work = 0.f;
  int most = 1, pairs = 0;
  over_groups([&](const PrefixGroup& x) {
    work += float(x.pairs) * float(x.blocks);
    most = max(most, x.blocks);
    if (x.blocks) pairs += x.pairs;
  });
  most = __reduce_max_sync(0xffffffffu, most);
  const float even = warp_sum<32>(work) * float(Hkv) / float(PX_SMS);  // blocks a CTA if it came out even
  int quota = even < float(most) ? max(1, int(ceilf(even))) : most;
  const int alike = max(1, min(most, PX_SMS / max(1, __reduce_add_sync(0xffffffffu, pairs) * Hkv)));
  while (quota < (most + alike - 1) / alike) {
    int ctas = 0;
    over_groups([&](const PrefixGroup& x) { ctas += x.pairs * x.splits(quota); });
    if (__reduce_add_sync(0xffffffffu, ctas) * Hkv <= PX_SMS) return quota;
    quota += max(1, quota / 32);
  }
  return -alike;
}

__device__ __forceinline__ bool px_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  if (*abort_flag) return false;
  if (mbar_wait_bounded(bar, parity)) return true;
  *abort_flag = 1;
  return false;
}
template <int DP, int BITS>
__global__ void __launch_bounds__(PX_THREADS, 1) prefix_attn_kernel(const PrefixParams p) {
  if (p.beside) pdl_trigger();
  else pdl_enter();
  using SM = PrefixSmem<DP, BITS>;
  constexpr int TILE = SM::TILE, HALF = 128 * 128, NST = PX_RING;
  constexpr int RB = SM::RB, DG = SM::DG, CPR = RB / 16;  // bytes, scales, 16-byte chunks of a code row
  constexpr int LPR = CPR < 4 ? CPR : 4;                  // lanes on a row (and rows a lane has)
  constexpr int CPT = CPR / LPR;                          // chunks of a row that a lane has
  constexpr float TOP = float((1 << (BITS - 1)) - 1);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  SM& sm = *reinterpret_cast<SM*>(smem_raw);
  volatile int* abort_flag = &sm.abort_flag;
  // (the shuffles tell the compiler that roles are uniform in a warp)
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (smem_u32(smem_raw) & 1023) {  // the swizzled tiles need it; the runtime gives it
    if (tid == 0) report_timeout(nullptr);
    return;
  }

  // test control: stalled producers issue nothing (read early: it is a chain of latencies from here to the first copy)
  const bool stall = warp >= PX_COPY && producers_stalled();
  if (warp == 0) {
    const int span = 2 * p.tpt;
    const int quota = prefix_quota(p.off, p.lens, p.Ng, p.B, span, p.Hkv, p.max_prefix);
    if (blockIdx.x == 0 && lane == 0) *p.quota = quota;
    int left = blockIdx.x, g = -1, row0 = 0, rows = 0, len = 0, hk = 0, split = 0, per = 1;
    for (int g0 = 0; g0 < p.Ng && g < 0; g0 += 32) {
      PrefixGroup x;
      x.look(p.off, p.lens, g0 + lane, p.Ng, p.B, span, p.max_prefix);
      const int mine = x.splits(quota), ctas = x.pairs * mine * p.Hkv;
      int s = ctas;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += a;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, s > left);
      if (hit) {
        const int w = __ffs(hit) - 1;
        const int at = left - __shfl_sync(0xffffffffu, s - ctas, w), splits = __shfl_sync(0xffffffffu, mine, w);
        len = __shfl_sync(0xffffffffu, x.len, w);
        g = g0 + w;
        split = at % splits;
        per = quota > 0 ? quota : ((len + PX_BN - 1) / PX_BN + splits - 1) / splits;
        hk = at / splits % p.Hkv;
        row0 = __shfl_sync(0xffffffffu, x.lo, w) + at / splits / p.Hkv * span;
        rows = __shfl_sync(0xffffffffu, x.hi, w) - row0;
      } else {
        left -= __shfl_sync(0xffffffffu, s, 31);
      }
    }
    if (lane == 0) {
      sm.item[0] = g;
      sm.item[1] = row0;
      sm.item[2] = rows;
      sm.item[3] = len;
      sm.item[4] = hk;
      sm.item[5] = split;
      sm.per = per;
    }
  } else if (tid == 32) {
    for (int s = 0; s < PX_RAW; ++s) {
      mbar_init(&sm.raw_full[s], 1);
      mbar_init(&sm.raw_empty[s], 4);
    }
    for (int s = 0; s < NST; ++s) {
      mbar_init(&sm.full[s], 4);
      mbar_init(&sm.empty[s], 1);
    }
    mbar_init(&sm.q_full, 16);
    for (int i = 0; i < 8; ++i) mbar_init(&sm.norm_full[i >> 2][i & 3], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], 8);
      mbar_init(&sm.pv_done[i], 1);
    }
    mbar_init(&sm.drain, 1);
    sm.abort_flag = 0;
    fence_mbarrier_init();
  } else if (warp == PX_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
  const int g = __shfl_sync(0xffffffffu, sm.item[0], 0), row0 = __shfl_sync(0xffffffffu, sm.item[1], 0);
  const int rows = __shfl_sync(0xffffffffu, sm.item[2], 0), len = __shfl_sync(0xffffffffu, sm.item[3], 0);
  const int hk = __shfl_sync(0xffffffffu, sm.item[4], 0), split = __shfl_sync(0xffffffffu, sm.item[5], 0);
  const int per = __shfl_sync(0xffffffffu, sm.per, 0);
  const int blocks = (len + PX_BN - 1) / PX_BN;
  const int j0 = split * per;
  const int n = g < 0 ? 0 : max(0, min(blocks, j0 + per) - j0);  // this split's blocks (g < 0: a spare CTA of the grid)
  const int n_tiles = rows > p.tpt ? 2 : 1;

  if (warp >= PX_MMA) {
    if (warp == PX_MMA && n > 0) {
      // ============================ MMA issuer ==================================
      const uint32_t one = elect_lane();
      const uint32_t id_s = mma_idesc(PX_BN, false, false, p.negate), id_o = mma_idesc(DP, false, true, false);
      auto wait_all = [&](uint64_t* bar, uint32_t parity) {
        return bool(__all_sync(0xffffffffu, px_wait(bar, parity, abort_flag)));
      };
      // position in the ring
      struct Ring {
        int s = 0;
        uint32_t phase = 0;
        __device__ __forceinline__ void next() {
          if (++s == NST) s = 0, phase ^= 1;
        }
      };
      auto full_of = [&](const Ring& r) { return wait_all(&sm.full[r.s], r.phase); };
      const uint64_t q_desc = sw128_desc(sm.q[0]), k_desc = sw128_desc(sm.ring[0]),
                     v_desc = sw128_mn_desc(sm.ring[0], HALF);
      auto score = [&](int t, int stage) {  // S_t = Q_t K^T
        const uint64_t a = q_desc + uint64_t(t * (TILE >> 4)), b = k_desc + uint64_t(stage * (TILE >> 4));
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          const uint64_t at = (ks >> 2) * (HALF >> 4) + 2 * (ks & 3);
          tc_mma_ss(one, tmem + 128 * t, a + at, b + at, id_s, ks > 0);
        }
        tc_commit_by(one, &sm.s_full[t]);
      };
      // Scores are issued once V's power of their block is known: it goes into
      // them, and the softmax warps wait for the scores only.
      auto power_of = [&](int j) { return wait_all(&sm.norm_full[1][j & 3], uint32_t((j >> 2) & 1)); };
      Ring ring;
      bool ok = wait_all(&sm.q_full, 0u) && power_of(0) && full_of(ring);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < n_tiles; ++t) score(t, ring.s);
        tc_commit_by(one, &sm.empty[ring.s]);
      }
      for (int j = 0; ok && j < n; ++j) {
        ring.next();
        const Ring rv = ring;  // V_j
        ok = full_of(rv);
        if (ok && j + 1 < n) {  // K_{j+1}
          ring.next();
          ok = power_of(j + 1) && full_of(ring);
        }
        for (int t = 0; ok && t < n_tiles; ++t) {
          const uint64_t v = v_desc + uint64_t(rv.s * (TILE >> 4));
          ok = wait_all(&sm.p_full[t], uint32_t(j & 1));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < 8; ++ks)  // O_t += P_t V_j
            tc_mma_ts(one, tmem + 256 + DP * t, tmem + 128 * t + 64 * (ks >> 2) + 8 * (ks & 3), v + ks * (2048 >> 4),
                      id_o, j > 0 || ks > 0);
          tc_commit_by(one, &sm.pv_done[t]);
          if (j + 1 < n) score(t, ring.s);
        }
        if (!ok) break;
        tc_commit_by(one, &sm.empty[rv.s]);
        if (j + 1 < n) tc_commit_by(one, &sm.empty[ring.s]);
      }
      // all MMAs issued complete before TMEM is released
      tc_commit_by(one, &sm.drain);
      mbar_wait_bounded(&sm.drain, 0u, 100000000ull);
      __syncwarp();
    } else if (warp >= PX_COPY && n > 0 && !stall) {
      // ============================ copies of codes and scales ==================
      // 16 keys a lane (pages hold a multiple of 16)
      const int v = warp - PX_COPY, part = lane;  // K or V
      const int32_t* pages = p.table + int64_t(g) * p.width;
      const uint8_t* codes = v ? p.vc : p.kc;
      const float* scales = v ? p.vs : p.ks;
      // A page is loaded a block ahead, and looked at only where it is used; all
      // that a copy needs is worked out before its stage is free.
      auto entry_of = [&](int j) {
        const int key = (j0 + j) * PX_BN + 16 * part;
        return part < 8 && j < n && key < len ? key / p.P : -1;
      };
      auto page_of = [&](int entry) { return entry >= 0 ? pages[entry] : 0; };
      int entry = entry_of(0), page = page_of(entry), j = 0;
      int64_t row = 0;
      bool have = false;
      auto look = [&](int j) {  // where the lane's keys of block j are; the next block's page
        row = (int64_t(max(page, 0)) * p.Hkv + hk) * p.P + ((j0 + j) * PX_BN + 16 * part) % p.P;
        have = entry >= 0;
        entry = entry_of(j + 1);
        page = page_of(entry);
      };
      look(0);
      for (; j < n; ++j) {
        const int it = 2 * j + v, s = it % PX_RAW;
        const int valid = len - (j0 + j) * PX_BN;         // keys of the block (128 or more: all)
        const int keys = min(PX_BN, (valid + 15) & ~15);  // in whole sixteens
        if (it >= PX_RAW &&
            !__all_sync(0xffffffffu, px_wait(&sm.raw_empty[s], uint32_t((it / PX_RAW - 1) & 1), abort_flag)))
          break;
        if (lane == 0) mbar_arrive_expect_tx(&sm.raw_full[s], uint32_t(keys) * (RB + DG * 4));
        __syncwarp();
        if (have) {
          bulk_g2s(sm.raw[s] + 16 * part * RB, codes + row * RB, 16 * RB, &sm.raw_full[s]);
          bulk_g2s(sm.raw[s] + SM::CODES + 16 * part * DG * 4, scales + row * DG, 16 * DG * 4, &sm.raw_full[s]);
        }
        look(j + 1);
        // the block's power, from the largest scale (4 keys a lane), while the
        // decoding warps take the codes into registers
        if (!__all_sync(0xffffffffu, px_wait(&sm.raw_full[s], uint32_t((it / PX_RAW) & 1), abort_flag))) {
          ++j;
          break;
        }
        const float* sc = reinterpret_cast<const float*>(sm.raw[s] + SM::CODES);
        float top = 0.f;
        bool careful = valid < PX_BN;
        if (!careful) {
#pragma unroll
          for (int e = 0; e < DG; ++e) {
            const float4 x = reinterpret_cast<const float4*>(sc)[lane * DG + e];
            top = fmaxf(top, fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)));
          }
          top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
          careful = top == 1.f || top == INFINITY;
        }
        if (careful) {  // keys past the prefix, groups of zeros and infinite scales do not count
          top = 0.f;
          for (int e = 4 * DG * lane; e < min(valid * DG, 4 * DG * (lane + 1)); ++e) {
            const float x = sc[e];
            uint32_t some = x < INFINITY;
            if (x == 1.f) {
              constexpr uint32_t ZEROS = BITS == 8 ? 0x7F7F7F7Fu : BITS == 4 ? 0x77777777u : 0x55555555u;
              const uint4* at = reinterpret_cast<const uint4*>(sm.raw[s] + e * (8 * BITS));
              some = 0;
              for (int i = 0; i < BITS / 2; ++i)
                some |= (at[i].x ^ ZEROS) | (at[i].y ^ ZEROS) | (at[i].z ^ ZEROS) | (at[i].w ^ ZEROS);
            }
            if (some) top = fmaxf(top, x);
          }
          top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
        }
        if (lane == 0) {
          const float norm = top > 0.f ? fminf(pow2_inverse(top, 15 - BITS), 0x1p60f) : 0x1p60f;
          sm.norm[v][j & 7] = careful ? -norm : norm;
          if (v) sm.v_power[j & 7] = make_float2(float(127 - int(__float_as_uint(norm) >> 23)), norm);
          else sm.k_back[j & 7] = __uint_as_float((254u << 23) - __float_as_uint(norm));  // 1 / norm
          mbar_arrive(&sm.norm_full[v][j & 3]);
        }
        __syncwarp();
      }
      // the last copy issued lands before the CTA goes away (those before it were waited for)
      if (j > 0) {
        const int it = 2 * (j - 1) + v;
        mbar_wait_bounded(&sm.raw_full[it % PX_RAW], uint32_t((it / PX_RAW) & 1), 100000000ull);
      }
      __syncwarp();
    }
  } else if (warp >= 16) {
    // ============================ codes -> fp16 tiles ===========================
    // Lane t has rows t / LPR + (128 / LPR) * k and chunks t % LPR + LPR * c of
    // each: the stores of a phase's 8 lanes hit 8 different 16-byte columns of
    // the swizzled tile.
    const int v = (warp - 16) >> 2;  // K or V
    const int t = tid - 512 - 128 * v, sub = t % LPR;
    constexpr uint32_t OFF = 0x64006400u + uint32_t(TOP) * 0x00010001u;  // 1024 + TOP, twice
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int it = 2 * j + v, s = it % PX_RAW, st = it % NST;
      ok = __all_sync(0xffffffffu, ok && px_wait(&sm.raw_full[s], uint32_t((it / PX_RAW) & 1), abort_flag));
      if (!ok) break;
      // the lane's codes and scales into registers: the stage is free for the next copy
      const int valid = len - (j0 + j) * PX_BN;  // keys of the block (128 or more: all)
      const float* scales = reinterpret_cast<const float*>(sm.raw[s] + SM::CODES);
      uint4 w[LPR][CPT];
      float sc[LPR][CPT];
#pragma unroll
      for (int k = 0; k < LPR; ++k) {
        const int row = t / LPR + (128 / LPR) * k;
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
          const int chunk = sub + LPR * c;
          w[k][c] = *reinterpret_cast<const uint4*>(sm.raw[s] + row * RB + chunk * 16);
          sc[k][c] = scales[row * DG + chunk * (128 / BITS) / 64];
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.raw_empty[s]);
      ok = __all_sync(0xffffffffu, px_wait(&sm.norm_full[v][j & 3], uint32_t((j >> 2) & 1), abort_flag)) &&
           (it < NST || __all_sync(0xffffffffu, px_wait(&sm.empty[st], uint32_t((it / NST - 1) & 1), abort_flag)));
      if (!ok) break;
      const float norm = sm.norm[v][j & 7];
#pragma unroll
      for (int k = 0; k < LPR; ++k)
#pragma unroll
        for (int c = 0; c < CPT; ++c) sc[k][c] *= fabsf(norm);
      if (norm < 0.f) {
#pragma unroll
        for (int k = 0; k < LPR; ++k)
#pragma unroll
          for (int c = 0; c < CPT; ++c) {
            // past the prefix; a group of zeros beside smaller scales
            const bool passes = sc[k][c] > float(1 << (16 - BITS)) && sc[k][c] < INFINITY;
            if (t / LPR + (128 / LPR) * k >= valid || passes) sc[k][c] = 0.f;
          }
      }
#pragma unroll
      for (int k = 0; k < LPR; ++k) {
        const int row = t / LPR + (128 / LPR) * k;
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
          const __half2 h2 = __float2half2_rn(sc[k][c]);
          const uint32_t s2 = *reinterpret_cast<const uint32_t*>(&h2);
          uint32_t b[32 / BITS];
          spread_codes<BITS>(w[k][c], b);
          const int col = (sub + LPR * c) * (16 / BITS);  // first 8-value column of the chunk
#pragma unroll
          for (int x = 0; x < 16 / BITS; ++x) {
            const uint2 lo = codes_to_f16(b[2 * x], OFF, s2), hi = codes_to_f16(b[2 * x + 1], OFF, s2);
            const int cc = col + x;
            *reinterpret_cast<uint4*>(sm.ring[st] + (cc >> 3) * HALF + row * 128 + (((cc & 7) ^ (row & 7)) << 4)) =
                make_uint4(lo.x, lo.y, hi.x, hi.y);
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.full[st]);
    }
    __syncwarp();
  } else {
    // ============================ queries, softmax, partials ====================
    // Two threads a row, 64 keys (and half the columns of O) each.  The two
    // warps of 32 rows share a barrier and leave the loops together: what a
    // wait that gave up says goes through the barrier first.
    const int i = warp >> 3, h = (warp >> 2) & 1, r = tid & 127;  // tile, half of the keys, MMA row
    const int bar = 1 + 4 * i + (warp & 3);
    // MMA row r of tile i: request row0 + i * tpt + r / G, query head hk * G + r % G
    const int req = i * p.tpt + r / p.G;
    const bool live = g >= 0 && r < p.tpt * p.G && req < rows;
    const int64_t bh = int64_t(row0 + req) * p.Hq + hk * p.G + r % p.G;
    const int64_t part = int64_t(blockIdx.x) * 256 + i * 128 + r;
    auto wait_all = [&](uint64_t* b, uint32_t parity) {
      return bool(__all_sync(0xffffffffu, px_wait(b, parity, abort_flag)));
    };
    if (n <= 0) {  // rounding left this split nothing
      if (live && h == 0) *reinterpret_cast<float2*>(p.ml_part + part * 2) = make_float2(-INFINITY, 0.f);
    } else if (i < n_tiles) {
      // ---- this row's query, scaled by a power of two into fp16; a half of its columns each ----
      constexpr int QC = DP / 16;  // 16-byte pieces of a half
      uint4 w[QC];
#pragma unroll
      for (int c = 0; c < QC; ++c)
        w[c] = live ? reinterpret_cast<const uint4*>(p.q + bh * DP)[h * QC + c] : make_uint4(0u, 0u, 0u, 0u);
      float top = 0.f;
#pragma unroll
      for (int c = 0; c < QC; ++c) {
        const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&w[c]);
#pragma unroll
        for (int k = 0; k < 4; ++k) top = fmaxf(top, fmaxf(fabsf(__low2float(e[k])), fabsf(__high2float(e[k]))));
      }
      // max with the row's other thread.  The reference is the exact maximum: P
      // goes to fp16, which an error of a few in the exponent overflows or
      // empties, and rounded to 8 bits it is off by 32 at 10000.  Shared
      // memory has room for half a float per row, so each hands over two halves.
      auto join = [&](float v) {
        uint32_t other = 0;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          const uint16_t mine = uint16_t(__float_as_uint(v) >> (part ? 0 : 16));
          uint16_t theirs = 0;
          if (h) sm.exchange[i][r] = mine;
          bar_all(bar, 64);
          if (!h) {
            theirs = sm.exchange[i][r];
            sm.exchange[i][r] = mine;
          }
          bar_all(bar, 64);
          if (h) theirs = sm.exchange[i][r];
          other = other << 16 | theirs;
        }
        return max2(v, __uint_as_float(other));
      };
      const float qn = pow2_inverse(join(top), 0);
#pragma unroll
      for (int c = 0; c < QC; ++c) {
        const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&w[c]);
        uint32_t x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = pack_f16x2(__low2float(e[k]) * qn, __high2float(e[k]) * qn);
        const int cc = h * QC + c;
        *reinterpret_cast<uint4*>(sm.q[i] + (cc >> 3) * HALF + r * 128 + (((cc & 7) ^ (r & 7)) << 4)) =
            make_uint4(x[0], x[1], x[2], x[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full);
      const uint32_t lane_at = uint32_t(32 * (warp & 3)) << 16;
      const uint32_t s_at = tmem + lane_at + 128 * i + 64 * h, o_at = tmem + lane_at + 256 + DP * i + DP / 2 * h;
      const float zq = p.scale2 / qn;  // scores in base 2 = S * zq * K's power back
      float m = -INFINITY, l = 0.f;  // m: reference of the exponents
      bool ok = true, quit = false;
      for (int j = 0; j < n; ++j) {
        ok = ok && wait_all(&sm.s_full[i], uint32_t(j & 1));
        tc_fence_after();
        const float2 power = sm.v_power[j & 7];
        const float zs = fmaxf(zq * sm.k_back[j & 7], 1e-37f);  // above 0: a masked score stays -inf
        const int valid = len - (j0 + j) * PX_BN - 64 * h;  // keys of this half (64 or more: all)
        const bool masked = valid < 64;
        // the scores are read twice, 32 at a time: 64 at once and P do not fit 72 registers
        auto scores = [&](int c, uint32_t (&s)[32]) {
          tmem_ld32(s_at + c, s);
          if (masked) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (c + k >= valid) s[k] = 0xFF800000u;
          }
        };
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          uint32_t s[32];
          scores(c, s);
          mx = max2(mx, row_max(s));
        }
        mx = fmaf(mx, zs, power.x);
        // P up to 2^7 when m moves and 2^15 before it does: 11 bits for weights 2^-21 of the largest
        if (bar_or(bar, 64, !ok || j == 0 || !(mx <= m + 15.f))) {
          if (bar_or(bar, 64, !ok)) {
            quit = true;
            break;
          }
          float both = join(mx);
          if (both == INFINITY) both = __int_as_float(0x7fffffff);  // inf - inf
          const bool move = j == 0 || !(both <= m + 15.f);
          both -= 7.f;
          if (j > 0) {
            // O holds blocks up to j - 1 once their product is done
            ok = wait_all(&sm.pv_done[i], uint32_t((j - 1) & 1));
            tc_fence_after();
            const float f = move ? ex2(m - both) : 1.f;
            l *= f;
            if (__any_sync(0xffffffffu, move)) {
#pragma unroll
              for (int c = 0; c < DP / 2; c += 16) {
                uint32_t o[16];
                tmem_ld16(o_at + c, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st16(o_at + c, o);
              }
            }
          }
          if (move) m = both;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        const float from = ref - power.x;
        uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t s[32], pk[16];
          scores(32 * c, s);
          if (masked) exp_row<false, false>(s, zs, from, sum, pk);  // exact zeros
          else exp_row<false, true>(s, zs, from, sum, pk);
          tmem_st16(s_at + 16 * c, pk);  // P goes over this thread's own scores, behind their reading
        }
        const float2 l2 = f32x2_parts(add_x2(sum[0], sum[1]));
        l = fmaf(l2.x + l2.y, power.y, l);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[i]);
      }
      // ---- the partial: rows of O through shared memory, then one copy each ----
      // (the operands have been used up once both tiles' products are done)
      ok = ok && !quit && wait_all(&sm.drain, 0u);
      tc_fence_after();
      uint8_t* out = sm.q[0] + (i * 128 + r) * SM::PITCH;
      if (ok) {
        if (h) *reinterpret_cast<float*>(out + DP * 4) = l;  // behind the row: this thread's sum
#pragma unroll
        for (int c = 0; c < DP / 2; c += 16) {
          uint32_t o[16];
          tmem_ld16(o_at + c, o);
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<float4*>(out + (DP / 2 * h + c + e) * 4) =
                make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]),
                            __uint_as_float(o[e + 3]));
        }
        fence_proxy_async_smem();
      }
      bar_all(bar, 64);
      if (ok && live && h == 0) {
        bulk_s2g(p.o_part + part * DP, out, DP * 4);
        *reinterpret_cast<float2*>(p.ml_part + part * 2) = make_float2(m, l + *reinterpret_cast<const float*>(out + DP * 4));
        bulk_s2g_wait();
      }
      tc_fence_before();
    } else {
      if (lane == 0) mbar_arrive(&sm.q_full);  // the tile is not used
    }
  }
  __syncthreads();
  if (warp == PX_MMA) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
  if (tid == 0 && *abort_flag) report_timeout(nullptr);
  if (p.beside) pdl_wait();  // this kernel completes after the one it ran beside
}

// One warp per (request, head), D / 32 values a lane, over the partials of its
// prefix (if it is in a group) and of its own tokens: summed in order, 8 loads
// ahead.
struct CombineParams {
  const float *o_prefix, *ml_prefix;  // [CTA][256][D] and (m, l), as prefix_attn_kernel leaves them
  const float *o_own, *ml_own;        // [B * Hq][n_own][D] and (m, l)
  const int* quota;
  const int32_t *off, *lens, *own_lens;
  __nv_bfloat16* out;
  int Ng, B, Hq, Hkv, tpt, max_prefix, n_own, ctas;
};

template <int D>
__global__ void __launch_bounds__(256) prefix_combine_kernel(const CombineParams p) {
  pdl_enter();
  constexpr int V = D / 32;
  const int64_t bh = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (bh >= int64_t(p.B) * p.Hq) return;
  const int b = int(bh / p.Hq), h = int(bh - int64_t(b) * p.Hq), G = p.Hq / p.Hkv, span = 2 * p.tpt;
  // the group's splits, its first CTA, the request's place in it
  int ctas = 0, sp = 0, rel = 0;
  const int quota = p.Ng ? *p.quota : 1;
  for (int g0 = 0; g0 < p.Ng; g0 += 32) {
    PrefixGroup x;
    x.look(p.off, p.lens, g0 + lane, p.Ng, p.B, span, p.max_prefix);
    const int mine = x.splits(quota);
    int s = x.pairs * mine * p.Hkv;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += a;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, b >= x.lo && b < x.hi);
    if (hit) {
      const int w = __ffs(hit) - 1;
      rel = b - __shfl_sync(0xffffffffu, x.lo, w);
      sp = __shfl_sync(0xffffffffu, mine, w);
      ctas += __shfl_sync(0xffffffffu, s - x.pairs * mine * p.Hkv, w);
      break;
    }
    ctas += __shfl_sync(0xffffffffu, s, 31);
  }
  const int first = ctas + (rel / span * p.Hkv + h / G) * sp;
  if (first < 0 || first + sp > p.ctas) sp = 0;  // (group offsets that fall)
  const int count = sp + p.n_own;
  // partial s of the row: the prefix's splits, then the own tokens'
  const int64_t at = int64_t(first) * 256 + rel % span / p.tpt * 128 + rel % p.tpt * G + h % G;
  auto ml_of = [&](int s) {
    return s < sp ? reinterpret_cast<const float2*>(p.ml_prefix)[at + s * 256]
                  : reinterpret_cast<const float2*>(p.ml_own)[bh * p.n_own + s - sp];
  };
  auto row_of = [&](int s) {
    return (s < sp ? p.o_prefix + (at + s * 256) * D : p.o_own + (bh * p.n_own + s - sp) * D) + lane * V;
  };
  float top = -INFINITY;
  for (int s = lane; s < count; s += 32) top = fmaxf(top, ml_of(s).x);
  top = warp_max<32>(top);
  float acc[V], l = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.f;
  for (int c0 = 0; c0 < count; c0 += 32) {
    const int s = c0 + lane;
    const float2 x = s < count ? ml_of(s) : make_float2(0.f, 0.f);
    // an empty split wrote no partial; NaN sums stay
    const float f = x.y == 0.f ? 0.f : top == -INFINITY ? 1.f : ex2(x.x - top);
    const unsigned some = __ballot_sync(0xffffffffu, x.y != 0.f);
    l += warp_sum<32>(x.y == 0.f ? 0.f : f * x.y);
    for (int k0 = 0; k0 < min(32, count - c0); k0 += 8) {
      float v[8][V];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool on = (some >> (k0 + k)) & 1;
        const float* src = row_of(c0 + k0 + k);
        if constexpr (V == 4) {
          const float4 y = on ? *reinterpret_cast<const float4*>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[k][0] = y.x, v[k][1] = y.y, v[k][2] = y.z, v[k][3] = y.w;
        } else {
          const float2 y = on ? *reinterpret_cast<const float2*>(src) : make_float2(0.f, 0.f);
          v[k][0] = y.x, v[k][1] = y.y;
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = __shfl_sync(0xffffffffu, f, k0 + k);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = fmaf(w, v[k][e], acc[e]);
      }
    }
  }
  float inv = l != 0.f ? 1.f / l : 0.f;
  // all scores are -inf: 0 / 0 (NaN maxima, which the comparisons pass over, come with sums that are NaN)
  if (top == -INFINITY && (sp > 0 || (p.n_own > 0 && p.own_lens[b] > 0))) inv = __int_as_float(0x7fffffff);
  uint32_t y[V / 2];
#pragma unroll
  for (int e = 0; e < V / 2; ++e) y[e] = pack_bf16x2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  if constexpr (V == 4) *reinterpret_cast<uint2*>(p.out + bh * D + lane * V) = make_uint2(y[0], y[1]);
  else *reinterpret_cast<uint32_t*>(p.out + bh * D + lane * V) = y[0];
}

// With `beside` the kernel follows the requests' own-token kernel, whose
// results it does not need: it is let onto the SMs as that one's CTAs leave
// them (programmatic launch without the wait at the start).  That kernel's
// CTAs have all passed their own wait by then, so what came before it is
// complete; the wait at this kernel's end makes its completion cover both.
template <int DP, int BITS>
static int launch_prefix(const PrefixParams& p, unsigned grid, cudaStream_t st) {
  using SM = PrefixSmem<DP, BITS>;
  static_assert(sizeof(SM) <= 227 * 1024, "one CTA's shared memory");
  static_assert(2 * 128 * SM::PITCH <= (2 + PX_RING) * SM::TILE, "room for the output rows");
  constexpr auto kern = prefix_attn_kernel<DP, BITS>;
  const int set = allow_smem<kern>(int(sizeof(SM)));
  if (set != B2F_OK) return set;
  int& policy = launch_pdl_policy();
  const int before = policy;
  if (p.beside) policy = 1;
  const int rc = launch_kernel(kern, dim3{grid}, dim3{PX_THREADS}, sizeof(SM), st, p);
  policy = before;
  return rc;
}

template <int DP>
static int launch_prefix_bits(const PrefixParams& p, int bits, unsigned grid, cudaStream_t st) {
  if (bits == 8) return launch_prefix<DP, 8>(p, grid, st);
  if (bits == 4) return launch_prefix<DP, 4>(p, grid, st);
  return launch_prefix<DP, 2>(p, grid, st);
}

// Splits of the requests' own tokens: about two CTAs per SM, 256 tokens or
// more each.  Measured with up to 2000 tokens and 4 KV heads, split against
// whole: 7.3 / 23.8 us for one row, 11.5 / 23.6 for 16; 128 rows with 8 KV
// heads, which have CTAs enough, 74 us whole, 81 in splits of 1024, 159 of 256.
static int own_splits(int64_t B, int64_t Hkv, int64_t max_own) {
  if (max_own <= 0) return 0;
  const int64_t want = 296 / (B * Hkv) > 1 ? 296 / (B * Hkv) : 1, cap = max_own / 256 > 1 ? max_own / 256 : 1;
  const int64_t n = want < cap ? want : cap;
  return int(n < 64 ? n : 64);
}

// CTAs of the prefix kernel, each with room for the partials of its two tiles:
// a partial pair of tiles at most per group with rows, of which there are no
// more than rows, and more splits than one only while they fit the SMs.
static int64_t prefix_ctas(int64_t B, int64_t G, int64_t Hkv, int64_t Ng, int64_t max_prefix) {
  if (Ng <= 0 || max_prefix <= 0 || B <= 0) return 0;
  const int64_t n = (B / (2 * (128 / G)) + (Ng < B ? Ng : B)) * Hkv;
  return n > PX_SMS ? n : PX_SMS;
}

// Floats of the workspace: the partials of prefix and own tokens, the quota.
static int64_t workspace_floats(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t Ng, int64_t max_prefix,
                                int64_t max_own) {
  const int64_t rows = prefix_ctas(B, Hq / Hkv, Hkv, Ng, max_prefix) * 256 + B * Hq * own_splits(B, Hkv, max_own);
  return rows ? rows * (D + 2) + 4 : 0;
}

B2F_DEFINE_WAIT_CONTROLS(prefix_attn)

}  // namespace b2f

using namespace b2f;

extern "C" {

int64_t b2f_shared_prefix_attn_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t n_groups,
                                               int64_t max_prefix, int64_t max_own) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || Hq / Hkv > 16) return 0;
  return workspace_floats(B, Hq, Hkv, D, n_groups, max_prefix, max_own) * int64_t(sizeof(float));
}

int b2f_shared_prefix_attn(const void* q, const uint8_t* k_pages, const float* k_scales, const uint8_t* v_pages,
                           const float* v_scales, const int32_t* prefix_table, int64_t prefix_pages,
                           const int32_t* prefix_lens, const int32_t* group_offsets, int64_t n_groups,
                           const int32_t* block_table, int64_t max_pages, const int32_t* seq_lens, int64_t B,
                           int64_t Hq, int64_t Hkv, int64_t D, int64_t page_size, int bits, int group_size,
                           float softmax_scale, int64_t max_prefix, int64_t max_own, void* workspace,
                           int64_t workspace_bytes, void* out, void* stream) {
  if (!(bits == 2 || bits == 4 || bits == 8)) return B2F_ERR_UNSUPPORTED;
  if (!(D == 64 || D == 128) || group_size != 64) return B2F_ERR_UNSUPPORTED;
  if (B < 0 || n_groups < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0) return B2F_ERR_INVALID;
  if (Hq / Hkv > 16 || B > 65535 || Hkv > 4096 || B * Hq > (1 << 30) || n_groups > 65535) return B2F_ERR_UNSUPPORTED;
  if (page_size <= 0 || page_size % 16 != 0 || prefix_pages <= 0 || max_pages <= 0 || max_prefix < 0 || max_own < 0)
    return B2F_ERR_INVALID;
  if (page_size > (1 << 20) || prefix_pages * page_size > (int64_t(1) << 30) || max_pages * page_size > (int64_t(1) << 30))
    return B2F_ERR_UNSUPPORTED;
  if (B == 0) return B2F_OK;
  if (!q || !k_pages || !k_scales || !v_pages || !v_scales || !seq_lens || !out || (max_own > 0 && !block_table) ||
      (n_groups > 0 && (!prefix_lens || !group_offsets || (max_prefix > 0 && !prefix_table))))
    return B2F_ERR_INVALID;
  if (!aligned(q, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(k_scales, 16) ||
      !aligned(v_scales, 16) || !aligned(out, 16))
    return B2F_ERR_ALIGN;
  const int64_t G = Hq / Hkv, tpt = 128 / G;
  if (max_prefix > prefix_pages * page_size) max_prefix = prefix_pages * page_size;
  if (max_own > max_pages * page_size) max_own = max_pages * page_size;
  const int no = own_splits(B, Hkv, max_own);
  const int64_t ctas = prefix_ctas(B, G, Hkv, n_groups, max_prefix);
  if (ctas > 0x7fffffff) return B2F_ERR_UNSUPPORTED;
  if (ctas + no > 0) {
    if (!workspace || workspace_bytes < workspace_floats(B, Hq, Hkv, D, n_groups, max_prefix, max_own) * 4)
      return B2F_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return B2F_ERR_ALIGN;
  }
  float* o_prefix = static_cast<float*>(workspace);
  float* o_own = o_prefix + ctas * 256 * D;
  float* ml_prefix = o_own + B * Hq * no * D;
  float* ml_own = ml_prefix + ctas * 256 * 2;
  int* quota = reinterpret_cast<int*>(ml_own + B * Hq * no * 2);
  const __nv_bfloat16* qb = static_cast<const __nv_bfloat16*>(q);
  cudaStream_t st = as_stream(stream);
  int rc;
  if (no > 0) {
    rc = launch_own_partials(qb, k_pages, k_scales, v_pages, v_scales, block_table, max_pages, seq_lens, int(B), int(Hq),
                             int(Hkv), int(D), int(page_size), bits, softmax_scale, no, int(max_own), o_own, ml_own, st);
    if (rc != B2F_OK) return rc;
  }
  if (ctas > 0) {
    const float s2 = fabsf(softmax_scale) * kLog2e;
    PrefixParams p{qb, k_pages, v_pages, k_scales, v_scales, prefix_table, prefix_lens, group_offsets, prefix_pages,
                   o_prefix, ml_prefix, quota, s2 <= 1e-30f ? 1e-30f : s2, softmax_scale < 0.f, int(B), int(n_groups), int(Hq),
                   int(Hkv), int(G), int(page_size), int(tpt), int(max_prefix), no > 0};
    rc = D == 64 ? launch_prefix_bits<64>(p, bits, unsigned(ctas), st)
                 : launch_prefix_bits<128>(p, bits, unsigned(ctas), st);
    if (rc != B2F_OK) return rc;
  }
  const CombineParams c{o_prefix, ml_prefix, o_own, ml_own, quota, group_offsets, prefix_lens, seq_lens,
                        static_cast<__nv_bfloat16*>(out), ctas > 0 ? int(n_groups) : 0, int(B), int(Hq), int(Hkv),
                        int(tpt), int(max_prefix), no, int(ctas)};
  return launch_kernel(D == 64 ? prefix_combine_kernel<64> : prefix_combine_kernel<128>,
                       dim3{unsigned((B * Hq + 7) / 8)}, dim3{256}, 0, st, c);
}

}  // extern "C"
