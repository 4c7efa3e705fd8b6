// Decode attention of requests that share long prefixes held once in the
// paged cache (reference KV format: uint8 codes, float32 scale per 64 values).
//
// One decode row per request reads its whole context alone: behind a shared
// prefix of p tokens that is B * p rows of K and V.  Here the query rows of a
// group -- requests x the G query heads of a KV head -- are the M side of one
// product with the prefix, which is then read and decoded once for all:
//   1. prefix: CTA = (2 tiles of 128 rows, KV head, split of the prefix).
//      S = Q K^T and O = P V on tcgen05 as in prompt_attn.cu; four warps turn
//      the codes of a block of 128 keys into fp16 tiles in shared memory.
//   2. own tokens: the paged decode kernels of qkv_attn.cu, writing partials.
//   3. combine: out = sum 2^(m_s - m) O_s / sum 2^(m_s - m) l_s over splits.
//
// fp16 operands: a code is exact in 11 bits, and scale * code costs one
// rounding of 2^-12, where bf16 would cost 2^-9 on K, V and P each -- more than
// the output's own rounding.  fp16's range is made up for by powers of two,
// which are exact: each query row is scaled by its own absmax, K and V by the
// largest scale of the CTA's first block (2^14 up to saturation, 2^14 down to
// the first lost bit); the scores and the output are scaled back in float32.
#include "attn_tc.cuh"

namespace b2f {

// qkv_attn.cu: decode attention of B rows over their own pages, as partials
// (o [B * Hq][part_stride][D], then m, l pairs) at splits part_base...
int launch_own_partials(const __nv_bfloat16* q, const uint8_t* kc, const float* ks, const uint8_t* vc, const float* vs,
                        const int32_t* table, int64_t width, const int32_t* lens, int B, int Hq, int Hkv, int D, int P,
                        int bits, float scale, int n_splits, int max_len, float* o_part, float* ml_part,
                        int part_stride, int part_base, cudaStream_t st);

constexpr int PX_THREADS = 416;  // warps 0-7 softmax, 8-11 decode the codes, 12 issues the MMAs
constexpr int PX_BN = 128;       // keys per block
constexpr int PX_STAGES = 5;     // K and V tiles in flight

struct PrefixParams {
  const __nv_bfloat16* q;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int32_t *table, *lens, *off;
  int64_t width;
  float *o_part, *ml_part;
  float scale2;  // softmax_scale * log2(e)
  int B, Ng, Hq, Hkv, G, P, tpt, n_splits, part_stride, max_prefix;
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

__device__ __forceinline__ bool px_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (*abort_flag) return false;
  if (mbar_wait_bounded(bar, parity)) return true;
  *abort_flag = 1;
  return false;
}

template <int DP, int BITS>
__global__ void __launch_bounds__(PX_THREADS, 1) prefix_attn_kernel(const PrefixParams p) {
  pdl_enter();
  constexpr int TILE = 128 * DP * 2, HALF = 128 * 128, NST = PX_STAGES;
  constexpr int RB = DP * BITS / 8, DG = DP / 64, CPR = RB / 16;  // bytes, scales, 16-byte chunks of a code row
  constexpr int LPR = CPR < 4 ? CPR : 4;                          // lanes on a row (and rows a lane has)
  constexpr int CPT = CPR / LPR;                                  // chunks of a row that a lane has
  constexpr float TOP = float((1 << (BITS - 1)) - 1);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;               // [2][TILE]
  uint8_t* ring = smem + 2 * TILE;  // [NST][TILE], K_0 V_0 K_1 V_1 ...
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + NST * TILE);
  uint64_t *full = bars, *empty = full + NST, *q_full = empty + NST, *s_full = q_full + 1, *p_full = s_full + 2,
           *pv_done = p_full + 2, *drain = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* item = reinterpret_cast<int*>(tmem_slot + 2);        // group, first row, rows of the group
  float* red = reinterpret_cast<float*>(tmem_slot + 6);     // [2][4] largest scales of the first block
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  const int split = blockIdx.x % p.n_splits, hk = blockIdx.x / p.n_splits % p.Hkv;
  if (warp == 0) {
    int left = blockIdx.x / p.n_splits / p.Hkv, g = -1, row0 = 0, rows = 0;
    const int span = 2 * p.tpt;
    for (int g0 = 0; g0 < p.Ng && g < 0; g0 += 32) {
      int lo = 0, hi = 0;
      if (g0 + lane < p.Ng) {
        lo = min(max(p.off[g0 + lane], 0), p.B);
        hi = min(max(p.off[g0 + lane + 1], lo), p.B);
      }
      int s = (hi - lo + span - 1) / span;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += a;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, s > left);
      if (hit) {
        const int w = __ffs(hit) - 1;
        const int before = w ? __shfl_sync(0xffffffffu, s, max(w - 1, 0)) : 0;
        const int a = __shfl_sync(0xffffffffu, lo, w), b = __shfl_sync(0xffffffffu, hi, w);
        g = g0 + w;
        row0 = a + (left - before) * span;
        rows = b - row0;
      } else {
        left -= __shfl_sync(0xffffffffu, s, 31);
      }
    }
    if (lane == 0) {
      item[0] = g;
      item[1] = row0;
      item[2] = rows;
    }
  }
  if (tid == 32) {
    for (int s = 0; s < NST; ++s) {
      mbar_init(&full[s], 4);
      mbar_init(&empty[s], 1);
    }
    mbar_init(q_full, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  __syncthreads();
  const int g = item[0], row0 = item[1], rows = item[2];
  if (g < 0) return;  // a spare item of the grid
  const int len = min(max(p.lens[g], 0), p.max_prefix);
  const int blocks = (len + PX_BN - 1) / PX_BN, per = (blocks + p.n_splits - 1) / p.n_splits;
  const int j0 = split * per, n = min(blocks, j0 + per) - j0;  // this split's blocks
  const int n_tiles = rows > p.tpt ? 2 : 1;

  // MMA row r of tile i: request row0 + i * tpt + r / G, query head hk * G + r % G
  const int i = (warp >> 2) & 1, r = tid & 127;
  const int req = i * p.tpt + r / p.G;
  const bool live = warp < 8 && r < p.tpt * p.G && req < rows;
  const int64_t bh = int64_t(row0 + req) * p.Hq + hk * p.G + r % p.G;
  const int64_t part = bh * p.part_stride + split;
  if (n <= 0) {  // fewer blocks than splits
    if (live) *reinterpret_cast<float2*>(p.ml_part + part * 2) = make_float2(-INFINITY, 0.f);
    return;
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 12) {
    // ============================ MMA issuer ====================================
    {
      const uint32_t one = elect_lane();
      auto wait_all = [&](uint64_t* bar, uint32_t parity) {
        return bool(__all_sync(0xffffffffu, px_wait(bar, parity, abort_flag)));
      };
      constexpr uint32_t id_s = mma_idesc(PX_BN, false, false, false), id_o = mma_idesc(DP, false, true, false);
      auto score = [&](int t, int j) {  // S_t = Q_t K_j^T
        const uint8_t *a = sq + t * TILE, *b = ring + ((2 * j) % NST) * TILE;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
          tc_mma_ss(one, tmem + 128 * t, sw128_desc(a + (ks >> 2) * HALF) + 2 * (ks & 3),
                 sw128_desc(b + (ks >> 2) * HALF) + 2 * (ks & 3), id_s, ks > 0);
        tc_commit_by(one, &s_full[t]);
      };
      auto full_of = [&](int it) { return wait_all(&full[it % NST], uint32_t((it / NST) & 1)); };
      bool ok = wait_all(q_full, 0u) && full_of(0);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < n_tiles; ++t) score(t, 0);
        tc_commit_by(one, &empty[0]);
      }
      for (int j = 0; ok && j < n; ++j) {
        ok = full_of(2 * j + 1);
        for (int t = 0; ok && t < n_tiles; ++t) {
          ok = wait_all(&p_full[t], uint32_t(j & 1));
          if (!ok) break;
          tc_fence_after();
          const uint8_t* v = ring + ((2 * j + 1) % NST) * TILE;
#pragma unroll
          for (int ks = 0; ks < PX_BN / 16; ++ks)  // O_t += P_t V_j
            tc_mma_ts(one, tmem + 256 + DP * t, tmem + 128 * t + 8 * ks, sw128_mn_desc(v + ks * 2048, HALF), id_o,
                      j > 0 || ks > 0);
          tc_commit_by(one, &pv_done[t]);
          if (j + 1 < n) {
            if (t == 0) ok = full_of(2 * j + 2);
            if (ok) score(t, j + 1);
          }
        }
        if (!ok) break;
        tc_commit_by(one, &empty[(2 * j + 1) % NST]);
        if (j + 1 < n) tc_commit_by(one, &empty[(2 * j + 2) % NST]);
      }
      // all MMAs issued by this thread complete before TMEM is released
      tc_commit_by(one, drain);
      mbar_wait_bounded(drain, 0u, 100000000ull);
    }
    __syncwarp();
  } else if (warp >= 8) {
    // ============================ codes -> fp16 tiles ===========================
    // Lane t has rows t / LPR + (128 / LPR) * k and chunks t % LPR + LPR * c of
    // each: 64-byte runs of a row in global memory, and stores whose 8 lanes of
    // a phase hit 8 different 16-byte columns of the swizzled tile.
    const int t = tid - 256, sub = t % LPR;
    const int32_t* pages = p.table + int64_t(g) * p.width;
    const bool stall = producers_stalled();  // test control: nothing is produced
    uint4 kq[LPR][CPT], vq[LPR][CPT];
    float kscale[LPR][CPT], vscale[LPR][CPT];
    int64_t rid[LPR];
    int page[LPR];
    auto key_of = [&](int j, int k) { return (j0 + j) * PX_BN + t / LPR + (128 / LPR) * k; };
    auto load_pages = [&](int j) {
#pragma unroll
      for (int k = 0; k < LPR; ++k) {
        const int key = key_of(j, k);
        page[k] = j < n && key < len ? pages[key / p.P] : -1;
      }
    };
    auto load = [&](const uint8_t* codes, const float* scales, uint4 (&w)[LPR][CPT], float (&s)[LPR][CPT]) {
#pragma unroll
      for (int k = 0; k < LPR; ++k)
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
          const int chunk = sub + LPR * c;
          const bool in = rid[k] >= 0;
          w[k][c] = in ? *reinterpret_cast<const uint4*>(codes + rid[k] * RB + chunk * 16) : make_uint4(0u, 0u, 0u, 0u);
          s[k][c] = in ? scales[rid[k] * DG + chunk * (128 / BITS) / 64] : 0.f;
        }
    };
    auto rows_of = [&](int j) {
#pragma unroll
      for (int k = 0; k < LPR; ++k)
        rid[k] = page[k] < 0 ? -1 : (int64_t(page[k]) * p.Hkv + hk) * p.P + key_of(j, k) % p.P;
    };
    constexpr uint32_t OFF = 0x64006400u + uint32_t(TOP) * 0x00010001u;  // 1024 + TOP, twice
    auto store = [&](int it, const uint4 (&w)[LPR][CPT], const float (&s)[LPR][CPT], float norm) {
      const int st = it % NST;
      bool ok = it < NST || px_wait(&empty[st], uint32_t((it / NST - 1) & 1), abort_flag);
      ok = __all_sync(0xffffffffu, ok) && !stall;
      if (!ok) return false;
#pragma unroll
      for (int k = 0; k < LPR; ++k) {
        const int row = t / LPR + (128 / LPR) * k;
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
          const float sc = s[k][c] * norm;
          const float sat = sc > 256.f ? 256.f : sc;  // 255 * 256 is the last fp16 value; NaN stays
          const __half2 h2 = __float2half2_rn(sat);
          const uint32_t s2 = *reinterpret_cast<const uint32_t*>(&h2);
          uint32_t b[32 / BITS];
          spread_codes<BITS>(w[k][c], b);
          const int col = (sub + LPR * c) * (16 / BITS);  // first 8-value column of the chunk
#pragma unroll
          for (int x = 0; x < 16 / BITS; ++x) {
            const uint2 lo = codes_to_f16(b[2 * x], OFF, s2), hi = codes_to_f16(b[2 * x + 1], OFF, s2);
            const int cc = col + x;
            *reinterpret_cast<uint4*>(ring + st * TILE + (cc >> 3) * HALF + row * 128 + (((cc & 7) ^ (row & 7)) << 4)) =
                make_uint4(lo.x, lo.y, hi.x, hi.y);
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[st]);
      return true;
    };
    load_pages(0);
    rows_of(0);
    load(p.kc, p.ks, kq, kscale);
    load(p.vc, p.vs, vq, vscale);
    load_pages(1);
    float km = 0.f, vm = 0.f;
#pragma unroll
    for (int k = 0; k < LPR; ++k)
#pragma unroll
      for (int c = 0; c < CPT; ++c) {
        if (kscale[k][c] < INFINITY) km = fmaxf(km, kscale[k][c]);
        if (vscale[k][c] < INFINITY) vm = fmaxf(vm, vscale[k][c]);
      }
    km = warp_max<32>(km);
    vm = warp_max<32>(vm);
    if (lane == 0) {
      red[warp - 8] = km;
      red[4 + warp - 8] = vm;
    }
    named_sync(128);
    // the largest value of the first block lands in [2^(BITS-8), 2^(BITS-6))
    const float kn = pow2_inverse(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), -7);
    const float vn = pow2_inverse(fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7])), -7);
    for (int j = 0; j < n; ++j) {
      if (!store(2 * j, kq, kscale, kn)) break;
      rows_of(j + 1);
      load(p.kc, p.ks, kq, kscale);
      load_pages(j + 2);
      if (!store(2 * j + 1, vq, vscale, vn)) break;
      load(p.vc, p.vs, vq, vscale);
    }
    __syncwarp();
  } else {
    // ============================ queries, softmax, partials ====================
    float zs = 0.f;  // scores in base 2 = S * zs
    if (i < n_tiles) {
      // this thread's query row, scaled by a power of two into fp16
      uint4 w[DP / 8];
#pragma unroll
      for (int c = 0; c < DP / 8; ++c)
        w[c] = live ? reinterpret_cast<const uint4*>(p.q + bh * DP)[c] : make_uint4(0u, 0u, 0u, 0u);
      float top = 0.f;
#pragma unroll
      for (int c = 0; c < DP / 8; ++c) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w[c]);
#pragma unroll
        for (int k = 0; k < 4; ++k) top = fmaxf(top, fmaxf(fabsf(__low2float(h[k])), fabsf(__high2float(h[k]))));
      }
      const float qn = pow2_inverse(top, 0);
      zs = p.scale2 / qn;
#pragma unroll
      for (int c = 0; c < DP / 8; ++c) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w[c]);
        uint32_t x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = pack_f16x2(__low2float(h[k]) * qn, __high2float(h[k]) * qn);
        *reinterpret_cast<uint4*>(sq + i * TILE + (c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4)) =
            make_uint4(x[0], x[1], x[2], x[3]);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
    const uint32_t lane_at = uint32_t(32 * (warp & 3)) << 16;
    const uint32_t s_at = tmem + lane_at + 128 * i, o_at = tmem + lane_at + 256 + DP * i;
    float m = -INFINITY, l = 0.f;  // m: reference of the exponents
    bool ok = true;
    if (i < n_tiles) {
      for (int j = 0; j < n; ++j) {
        ok = __all_sync(0xffffffffu, px_wait(&s_full[i], uint32_t(j & 1), abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (j == 0) zs /= pow2_inverse(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), -7);
        const int valid = len - (j0 + j) * PX_BN;  // keys of the block (128 or more: all)
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t s[64];
          tmem_ld64(s_at + 64 * h, s);
#pragma unroll
          for (int c = 0; c < 64; ++c) {
            const float z = __uint_as_float(s[c]) * zs;
            if (64 * h + c < valid) mx[c & 3] = fmaxf(mx[c & 3], z);
          }
        }
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (j == 0) {
          m = top;
        } else {
          const bool move = top > m + 8.f;
          if (__any_sync(0xffffffffu, move)) {
            ok = __all_sync(0xffffffffu, px_wait(&pv_done[i], uint32_t((j - 1) & 1), abort_flag));
            if (!ok) break;
            tc_fence_after();
            const float f = move ? ex2(m - top) : 1.f;
            if (move) m = top;
            l *= f;
#pragma unroll
            for (int c = 0; c < DP; c += 32) {
              uint32_t o[32];
              tmem_ld32(o_at + c, o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tmem_st32(o_at + c, o);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t pk[2][32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t s[64];
          tmem_ld64(s_at + 64 * h, s);
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            float e[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int c = 2 * k + x;
              e[x] = 64 * h + c < valid ? ex2(fmaf(__uint_as_float(s[c]), zs, -ref)) : 0.f;
              sum[c & 3] += e[x];
            }
            pk[h][k] = pack_f16x2(e[0], e[1]);
          }
        }
        // P goes over S once every column of S has been read
        tmem_st32(s_at, pk[0]);
        tmem_st32(s_at + 32, pk[1]);
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[i]);
      }
      if (ok) {
        ok = __all_sync(0xffffffffu, px_wait(&pv_done[i], uint32_t((n - 1) & 1), abort_flag));
        tc_fence_after();
      }
      if (ok) {
        const float back = 1.f / pow2_inverse(fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7])), -7);
#pragma unroll
        for (int c = 0; c < DP; c += 32) {
          uint32_t o[32];
          tmem_ld32(o_at + c, o);
          if (live) {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *reinterpret_cast<float4*>(p.o_part + part * DP + c + k) =
                  make_float4(__uint_as_float(o[k]) * back, __uint_as_float(o[k + 1]) * back,
                              __uint_as_float(o[k + 2]) * back, __uint_as_float(o[k + 3]) * back);
          }
          __syncwarp();
        }
        if (live) *reinterpret_cast<float2*>(p.ml_part + part * 2) = make_float2(m, l);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
  if (tid == 0 && *abort_flag) report_timeout(nullptr);
}

// Splits n_prefix.. are the request's own tokens; the first n_prefix hold
// something only where the request is in a group.  One CTA per (request,
// head), one thread per value; the splits are summed in order.
__global__ void prefix_combine_kernel(const float* __restrict__ o_part, const float* __restrict__ ml_part,
                                      const int32_t* __restrict__ off, int Ng, int Hq, int n_prefix, int n, int D,
                                      __nv_bfloat16* __restrict__ out) {
  pdl_enter();
  const int64_t bh = blockIdx.x;
  const int b = int(bh / Hq);
  bool in = false;
  for (int g = threadIdx.x & 31; g < Ng; g += 32) in |= b >= off[g] && b < off[g + 1];
  const int s0 = __any_sync(0xffffffffu, in) ? 0 : n_prefix;
  const float2* ml = reinterpret_cast<const float2*>(ml_part) + bh * n;
  float top = -INFINITY;
  for (int s = s0; s < n; ++s) top = fmaxf(top, ml[s].x);
  float o = 0.f, l = 0.f;
  const int d = threadIdx.x;
  for (int s = s0; s < n; ++s) {
    const float2 x = ml[s];
    if (x.y == 0.f) continue;  // an empty split wrote no partial
    const float f = top == -INFINITY ? 1.f : ex2(x.x - top);
    o += f * o_part[(bh * n + s) * D + d];
    l += f * x.y;
  }
  out[bh * D + d] = __float2bfloat16_rn(l != 0.f ? o / l : 0.f);
}

template <int DP, int BITS>
static int launch_prefix(const PrefixParams& p, unsigned grid, cudaStream_t st) {
  auto kern = prefix_attn_kernel<DP, BITS>;
  const int smem = 1024 + (2 + PX_STAGES) * 128 * DP * 2 + 256;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return B2F_ERR_CUDA;
  }
  return launch_kernel(kern, dim3{grid}, dim3{PX_THREADS}, size_t(smem), st, p);
}

template <int DP>
static int launch_prefix_bits(const PrefixParams& p, int bits, unsigned grid, cudaStream_t st) {
  if (bits == 8) return launch_prefix<DP, 8>(p, grid, st);
  if (bits == 4) return launch_prefix<DP, 4>(p, grid, st);
  return launch_prefix<DP, 2>(p, grid, st);
}

// Splits of the prefix: enough for one CTA per SM (a CTA takes the whole
// SM's shared memory), at most one per block of keys.
static int prefix_splits(int64_t B, int64_t G, int64_t Hkv, int64_t Ng, int64_t max_prefix) {
  if (Ng <= 0 || max_prefix <= 0 || B <= 0) return 0;
  const int64_t span = 2 * (128 / G), per_group = (B + Ng - 1) / Ng;
  const int64_t ctas = Ng * ((per_group + span - 1) / span) * Hkv, blocks = (max_prefix + PX_BN - 1) / PX_BN;
  const int64_t want = 148 / ctas > 1 ? 148 / ctas : 1;
  return int(want < blocks ? want : blocks);
}

// Splits of the requests' own tokens: about two CTAs per SM, 256 tokens or
// more each (measured for the paged decode kernels at batch 1 to 64).
static int own_splits(int64_t B, int64_t Hkv, int64_t max_own) {
  if (max_own <= 0) return 0;
  const int64_t want = 296 / (B * Hkv) > 1 ? 296 / (B * Hkv) : 1, cap = max_own / 256 > 1 ? max_own / 256 : 1;
  const int64_t n = want < cap ? want : cap;
  return int(n < 64 ? n : 64);
}

B2F_DEFINE_WAIT_CONTROLS(prefix_attn)

}  // namespace b2f

using namespace b2f;

extern "C" {

int64_t b2f_shared_prefix_attn_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t n_groups,
                                               int64_t max_prefix, int64_t max_own) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || Hq / Hkv > 16) return 0;
  const int64_t n = prefix_splits(B, Hq / Hkv, Hkv, n_groups, max_prefix) + own_splits(B, Hkv, max_own);
  return B * Hq * n * (D + 2) * int64_t(sizeof(float));
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
  if (Hq / Hkv > 16 || B > 65535 || Hkv > 4096 || n_groups > 65535) return B2F_ERR_UNSUPPORTED;
  if (page_size <= 0 || page_size % 16 != 0 || prefix_pages <= 0 || max_pages <= 0 || max_prefix < 0 || max_own < 0)
    return B2F_ERR_INVALID;
  if (page_size > (1 << 20) || prefix_pages * page_size > (int64_t(1) << 30) || max_pages * page_size > (int64_t(1) << 30))
    return B2F_ERR_UNSUPPORTED;
  if (B == 0) return B2F_OK;
  if (!q || !k_pages || !k_scales || !v_pages || !v_scales || !block_table || !seq_lens || !out ||
      (n_groups > 0 && (!prefix_table || !prefix_lens || !group_offsets)))
    return B2F_ERR_INVALID;
  if (!aligned(q, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(k_scales, 8) ||
      !aligned(v_scales, 8) || !aligned(out, 16))
    return B2F_ERR_ALIGN;
  const int64_t G = Hq / Hkv, tpt = 128 / G;
  if (max_prefix > prefix_pages * page_size) max_prefix = prefix_pages * page_size;
  if (max_own > max_pages * page_size) max_own = max_pages * page_size;
  const int np = prefix_splits(B, G, Hkv, n_groups, max_prefix), no = own_splits(B, Hkv, max_own), n = np + no;
  if (n > 0) {
    if (!workspace || workspace_bytes < B * Hq * n * (D + 2) * int64_t(sizeof(float))) return B2F_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return B2F_ERR_ALIGN;
  }
  float* o_part = static_cast<float*>(workspace);
  float* ml_part = o_part + B * Hq * n * D;
  const __nv_bfloat16* qb = static_cast<const __nv_bfloat16*>(q);
  cudaStream_t st = as_stream(stream);
  int rc;
  if (np > 0) {
    // items: at most one partial pair of tiles per group
    const int64_t grid = (B / (2 * tpt) + n_groups) * Hkv * np;
    if (grid > 0x7fffffff) return B2F_ERR_UNSUPPORTED;
    PrefixParams p{qb, k_pages, v_pages, k_scales, v_scales, prefix_table, prefix_lens, group_offsets, prefix_pages,
                   o_part, ml_part, softmax_scale * kLog2e, int(B), int(n_groups), int(Hq), int(Hkv), int(G),
                   int(page_size), int(tpt), np, n, int(max_prefix)};
    rc = D == 64 ? launch_prefix_bits<64>(p, bits, unsigned(grid), st)
                 : launch_prefix_bits<128>(p, bits, unsigned(grid), st);
    if (rc != B2F_OK) return rc;
  }
  if (no > 0) {
    rc = launch_own_partials(qb, k_pages, k_scales, v_pages, v_scales, block_table, max_pages, seq_lens, int(B), int(Hq),
                             int(Hkv), int(D), int(page_size), bits, softmax_scale, no, int(max_own), o_part, ml_part, n,
                             np, st);
    if (rc != B2F_OK) return rc;
  }
  return launch_kernel(prefix_combine_kernel, dim3{unsigned(B * Hq)}, dim3{unsigned(D)}, 0, st,
                       static_cast<const float*>(o_part), static_cast<const float*>(ml_part), group_offsets,
                       np > 0 ? int(n_groups) : 0, int(Hq), np, n, int(D), static_cast<__nv_bfloat16*>(out));
}

}  // extern "C"
