// Attention of packed prompts over themselves on the 5th-generation tensor
// cores: for each sequence and query head, softmax(scale * Q K^T) V, causal or
// full, grouped heads, sequences of any length back to back.
//
// Work item = (sequence, 2 tiles of consecutive tokens, KV head).  A tile is
// 128 MMA rows = 128 / G tokens x the G query heads of the KV head, so K and V
// are staged once for all heads that share them, and only the tile's own
// tokens, not 128 of them, see a diagonal block.  Per block of 128 keys:
//   S = Q K^T        tcgen05.mma, Q and K in shared memory (TMA, 128B swizzle)
//   P = 2^(S c - m)  one thread per row: the row comes out of TMEM into
//                    registers, the running maximum m and sum l are the
//                    thread's own (no shuffles), P goes back over S as 16 bits
//   O += P V         tcgen05.mma with P read from TMEM, V as it lies (MN-major)
// Softmax in base 2, m and l and O in float32; P is rounded to the inputs'
// type because the tensor core takes both operands alike (its relative error
// is that of the output's own rounding).  m is a reference, not the exact
// maximum: it moves, and O is rescaled, only where a row's new maximum passes
// it by more than 8 (P stays below 2^8), which after the first blocks is rare,
// so the rescale lives in the softmax warps and needs no warps of its own.
//
// Warps: 0-3 softmax of tile 0, 4-7 of tile 1 (also the epilogue), 8 issues
// the MMAs, 9 the TMA loads, 10-11 mend value tiles (below).  The two tiles
// alternate on the tensor core: while it works on one, the other's softmax
// runs.
//
// Rows of V that a tile's rows must not see meet P = 0, and 0 * NaN is NaN.
// So in the blocks in which anything is masked, warps 10-11 zero the rows past
// the item's last key (they belong to other tokens or sequences) and replace
// what is not finite by 0, keeping for each column the first key with a NaN,
// +inf or -inf; the epilogue adds those back to the rows that see them.
#include "attn_tc.cuh"

namespace b2f {

constexpr int PA_THREADS = 384;
constexpr int PA_BN = 128;  // keys per block

struct PromptParams {
  const int32_t* cu;
  void* out;
  float* lse;
  float scale2;   // |softmax_scale| * log2(e)
  int negate;     // softmax_scale < 0: the MMA negates Q
  int B, T, Hq, Hkv, G, D, causal;
  int tpt;        // tokens per tile
};

template <int DP>
struct PromptSmem {
  static constexpr int TILE = 128 * DP * 2;  // bytes of a Q tile, of a K or V block
  static constexpr int STAGES = DP == 128 ? 5 : 8;
  static constexpr int BARS = 320;  // barriers, TMEM address, work item
  static constexpr int BYTES = 1024 + 2 * TILE + STAGES * TILE + BARS + 3 * DP * 4;
};

// Waits with the CTA's abort flag; false once any wait gave up.
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (*abort_flag) return false;
  if (mbar_wait_bounded(bar, parity)) return true;
  *abort_flag = 1;
  return false;
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(PA_THREADS, 1) prompt_attn_kernel(const PromptParams p,
                                                                    const __grid_constant__ CUtensorMap tmq,
                                                                    const __grid_constant__ CUtensorMap tmk,
                                                                    const __grid_constant__ CUtensorMap tmv) {
  pdl_enter();
  using SM = PromptSmem<DP>;
  constexpr int NST = SM::STAGES, TILE = SM::TILE, HALF = 128 * 128;  // HALF: 64 columns of a tile
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;               // [2][TILE]
  uint8_t* ring = smem + 2 * TILE;  // [NST][TILE], K_0 V_0 K_1 V_1 ...
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + NST * TILE);
  uint64_t *full = bars, *empty = full + NST, *q_full = empty + NST, *s_full = q_full + 1, *p_full = s_full + 2,
           *pv_done = p_full + 4, *v_raw = pv_done + 2, *v_fix = v_raw + 3, *drain = v_fix + 3;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* item = reinterpret_cast<int*>(tmem_slot + 2);                                // first row, rows, first token of the item; anything in `bad`
  int* bad = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bars) + SM::BARS);  // [3][DP] first key: NaN, +inf, -inf
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // ---- the work item -------------------------------------------------------
  const int hk = blockIdx.x % p.Hkv;
  if (warp == 0) {
    int left = blockIdx.x / p.Hkv, row0 = 0, rows = 0, pair = 0, found = 0;
    const int span = 2 * p.tpt;
    // sequence B: the rows past the last sequence
    for (int b0 = 0; b0 <= p.B && !found; b0 += 32) {
      const int b = b0 + lane;
      int lo = 0, hi = 0;
      if (b <= p.B) {
        lo = min(max(p.cu[b], 0), p.T);
        hi = b < p.B ? min(max(p.cu[b + 1], lo), p.T) : p.T;
      }
      const int n = (hi - lo + span - 1) / span;
      int s = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += a;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, s > left);
      if (hit) {
        const int w = __ffs(hit) - 1;
        row0 = __shfl_sync(0xffffffffu, lo, w);
        rows = __shfl_sync(0xffffffffu, b0 + w < p.B ? hi - lo : lo - hi, w);  // negative: rows of no sequence
        // the longest rows of a sequence first: they set the tail of the grid
        pair = __shfl_sync(0xffffffffu, s, w) - 1 - left;
        found = 1;
      } else {
        left -= __shfl_sync(0xffffffffu, s, 31);
      }
    }
    if (lane == 0) {
      item[0] = row0;
      item[1] = rows;
      item[2] = pair * span;
    }
  }
  if (tid == 32) {
    for (int s = 0; s < NST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; i < 3; ++i) {
      mbar_init(&v_raw[i], 1);
      mbar_init(&v_fix[i], 2);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    item[3] = 0;
    fence_mbarrier_init();
  }
  for (int i = tid; i < 3 * DP; i += PA_THREADS) bad[i] = 0x7fffffff;
  __syncthreads();
  const int row0 = item[0], len = item[1], tok0 = item[2];
  if (len <= 0) {
    // rows of no sequence: zeros (the grid's spare items have none)
    const int n = min(2 * p.tpt, -len - tok0);
    for (int i = tid; i < n * p.G; i += PA_THREADS) {
      const int64_t r = int64_t(row0 + tok0 + i / p.G) * p.Hq + hk * p.G + i % p.G;
      for (int d = 0; d < p.D; d += 8)
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + r * p.D + d) = make_uint4(0u, 0u, 0u, 0u);
      if (p.lse) p.lse[r] = -INFINITY;
    }
    return;
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // keys and blocks of each tile; the first block in which anything is masked
  int n_blk[2], kend = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = tok0 + i * p.tpt;
    const int e = t >= len ? 0 : p.causal ? min(len, t + p.tpt) : len;
    n_blk[i] = (e + PA_BN - 1) / PA_BN;
    kend = max(kend, e);
  }
  const int n_all = max(n_blk[0], n_blk[1]);
  // (at most 3 of them: a pair of tiles spans 256 tokens or fewer)
  const int j_mask = p.causal ? tok0 / PA_BN : len / PA_BN;

  if (warp == 9) {
    // ============================ TMA producer ==================================
    if (lane == 0 && !producers_stalled()) {  // test control: stalled producers issue nothing
      const int qrows = p.tpt * p.G;
      mbar_arrive_expect_tx(q_full, uint32_t((n_blk[1] ? 2 : 1) * (DP / 64) * qrows * 128));
      for (int i = 0; i < (n_blk[1] ? 2 : 1); ++i)
        for (int h = 0; h < DP / 64; ++h)
          tma_load_4d(sq + i * TILE + h * HALF, &tmq, 64 * h, 0, hk, row0 + tok0 + i * p.tpt, q_full);
      int it = 0;
      for (; it < 2 * n_all; ++it) {
        const int s = it % NST;
        if (it >= NST && !wait_or_abort(&empty[s], uint32_t((it / NST - 1) & 1), abort_flag)) break;
        // a value block with masked rows lands on a barrier of its own, for warps 10-11
        const bool mend = (it & 1) && (it >> 1) >= j_mask;
        uint64_t* bar = mend ? &v_raw[(it >> 1) - j_mask] : &full[s];
        if (mend) mbar_arrive(&full[s]);
        mbar_arrive_expect_tx(bar, uint32_t(TILE));
        for (int h = 0; h < DP / 64; ++h)
          tma_load_3d(ring + s * TILE + h * HALF, it & 1 ? &tmv : &tmk, 64 * h, hk, row0 + (it >> 1) * PA_BN, bar);
      }
      // copies already issued land before the CTA goes away
      mbar_wait_bounded(q_full, 0u, 100000000ull);
      for (int k = 1; k <= NST && it - k >= 0; ++k)
        mbar_wait_bounded(&full[(it - k) % NST], uint32_t(((it - k) / NST) & 1), 100000000ull);
      for (int j = j_mask; 2 * j + 1 < it; ++j) mbar_wait_bounded(&v_raw[j - j_mask], 0u, 100000000ull);
    }
    __syncwarp();
  } else if (warp >= 10) {
    // ============================ value tiles with masked rows ==================
    for (int j = j_mask; j < n_all; ++j) {
      if (!__all_sync(0xffffffffu, wait_or_abort(&v_raw[j - j_mask], 0u, abort_flag))) break;
      uint8_t* v = ring + ((2 * j + 1) % NST) * TILE;
      const int valid = min(PA_BN, kend - j * PA_BN);
      // a line = 64 columns of one key; warp 10 takes the even lines, 11 the odd
      for (int line = (warp - 10) * 4 + (lane >> 3); line < 128 * (DP / 64); line += 8) {
        const int key = line & 127, h = line >> 7, c = lane & 7;
        uint4* at = reinterpret_cast<uint4*>(v + h * HALF + key * 128 + ((c ^ (key & 7)) << 4));
        if (key >= valid) {
          *at = make_uint4(0u, 0u, 0u, 0u);
        } else if (p.causal) {
          uint4 w = *at;
          constexpr uint32_t expo = BF16 ? 0x7F80u : 0x7C00u;
          uint32_t* u = reinterpret_cast<uint32_t*>(&w);
          bool any = false;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            any |= (u[k] & expo) == expo || ((u[k] >> 16) & expo) == expo;
          if (any) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t x = (u[k >> 1] >> (16 * (k & 1))) & 0xFFFFu;
              if ((x & expo) != expo) continue;
              const int cls = (x & ~expo & 0x7FFFu) ? 0 : (x & 0x8000u) ? 2 : 1;
              atomicMin(&bad[cls * DP + 64 * h + 8 * c + k], j * PA_BN + key);
              item[3] = 1;
              u[k >> 1] &= ~(0xFFFFu << (16 * (k & 1)));
            }
            *at = w;
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_fix[j - j_mask]);
    }
    __syncwarp();
  } else if (warp == 8) {
    // ============================ MMA issuer ====================================
    {
      const uint32_t one = elect_lane();
      auto wait_all = [&](uint64_t* bar, uint32_t parity) {
        return bool(__all_sync(0xffffffffu, wait_or_abort(bar, parity, abort_flag)));
      };
      const uint32_t id_s = mma_idesc(PA_BN, BF16, false, p.negate), id_o = mma_idesc(DP, BF16, true, false);
      auto score = [&](int i, int j) {  // S_i = Q_i K_j^T
        const uint8_t *a = sq + i * TILE, *b = ring + ((2 * j) % NST) * TILE;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
          tc_mma_ss(one, tmem + 128 * i, sw128_desc(a + (ks >> 2) * HALF) + 2 * (ks & 3),
                    sw128_desc(b + (ks >> 2) * HALF) + 2 * (ks & 3), id_s, ks > 0);
        tc_commit_by(one, &s_full[i]);
      };
      auto full_of = [&](int it) { return wait_all(&full[it % NST], uint32_t((it / NST) & 1)); };
      bool ok = wait_all(q_full, 0u) && full_of(0);
      if (ok) {
        tc_fence_after();
        for (int i = 0; i < 2; ++i)
          if (n_blk[i]) score(i, 0);
        tc_commit_by(one, &empty[0]);
      }
      for (int j = 0; ok && j < n_all; ++j) {
        ok = j < j_mask ? full_of(2 * j + 1) : wait_all(&v_fix[j - j_mask], 0u);
        bool next = false;  // K_{j+1} has landed
        for (int i = 0; ok && i < 2; ++i) {
          if (j >= n_blk[i]) continue;
          const uint8_t* v = ring + ((2 * j + 1) % NST) * TILE;
          // O_i += P_i V_j, the first 64 keys while the others' P is formed
          for (int h = 0; ok && h < 2; ++h) {
            ok = wait_all(&p_full[2 * i + h], uint32_t(j & 1));
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int ks = 4 * h; ks < 4 * h + 4; ++ks)
              tc_mma_ts(one, tmem + 256 + DP * i, tmem + 128 * i + 8 * ks, sw128_mn_desc(v + ks * 2048, HALF), id_o,
                        j > 0 || ks > 0);
          }
          if (!ok) break;
          tc_commit_by(one, &pv_done[i]);
          if (j + 1 < n_blk[i]) {
            if (!next) ok = next = full_of(2 * j + 2);
            if (ok) score(i, j + 1);
          }
        }
        if (!ok) break;
        tc_commit_by(one, &empty[(2 * j + 1) % NST]);
        if (j + 1 < n_all) tc_commit_by(one, &empty[(2 * j + 2) % NST]);
      }
      // all MMAs issued by this thread complete before TMEM is released
      tc_commit_by(one, drain);
      mbar_wait_bounded(drain, 0u, 100000000ull);
    }
    __syncwarp();
  } else {
    // ============================ softmax and epilogue ==========================
    const int i = warp >> 2, r = tid & 127;  // tile, MMA row
    const int t = tok0 + i * p.tpt + r / p.G;
    const bool live = r < p.tpt * p.G && t < len;
    const int last = !live ? -1 : p.causal ? t : len - 1;  // last key the row sees
    const uint32_t lane_at = uint32_t(32 * (warp & 3)) << 16;
    const uint32_t s_at = tmem + lane_at + 128 * i, o_at = tmem + lane_at + 256 + DP * i;
    float m = -INFINITY, l = 0.f;  // m: reference of the exponents (scaled scores)
    bool ok = true;
    for (int j = 0; j < n_blk[i]; ++j) {
      ok = __all_sync(0xffffffffu, wait_or_abort(&s_full[i], uint32_t(j & 1), abort_flag));
      if (!ok) break;
      tc_fence_after();
      uint32_t s[128];
      tmem_ld128(s_at, s);
      const bool masked = j >= j_mask;
      if (masked) {
        const int rel = last - j * PA_BN;
#pragma unroll
        for (int c = 0; c < 128; ++c)
          if (c > rel) s[c] = 0xFF800000u;
      }
      const float top = row_max(s) * p.scale2;
      if (j == 0) {
        m = top;
      } else {
        const bool move = top > m + 8.f;
        if (__any_sync(0xffffffffu, move)) {
          // O holds blocks up to j - 1 once their product is done
          ok = __all_sync(0xffffffffu, wait_or_abort(&pv_done[i], uint32_t((j - 1) & 1), abort_flag));
          if (!ok) break;
          tc_fence_after();
          const float f = move ? ex2(m - top) : 1.f;
          if (move) m = top;
          l *= f;
#pragma unroll
          for (int c = 0; c < DP; c += 16) {
            uint32_t o[16];
            tmem_ld16(o_at + c, o);
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            tmem_st16(o_at + c, o);
          }
        }
      }
      const float ref = m == -INFINITY ? 0.f : m;
      uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t(&sh)[64] = *reinterpret_cast<const uint32_t(*)[64]>(&s[64 * h]);
        uint32_t pk[32];
        if (masked) exp_row<BF16, false>(sh, p.scale2, ref, sum, pk);  // exact zeros
        else exp_row<BF16, true>(sh, p.scale2, ref, sum, pk);
        tmem_st32(s_at + 32 * h, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * i + h]);
      }
      const float2 l2 = f32x2_parts(add_x2(sum[0], sum[1]));
      l += l2.x + l2.y;
    }
    if (ok && n_blk[i]) {
      ok = __all_sync(0xffffffffu, wait_or_abort(&pv_done[i], uint32_t((n_blk[i] - 1) & 1), abort_flag));
      tc_fence_after();
      const int64_t row = int64_t(row0 + t) * p.Hq + hk * p.G + r % p.G;
      const float inv = l > 0.f ? 1.f / l : l;  // l is NaN where a score is
      const bool any_bad = *const_cast<volatile int*>(&item[3]) != 0;
      if (ok) {
#pragma unroll
        for (int c = 0; c < DP; c += 32) {
          uint32_t o[32];
          tmem_ld32(o_at + c, o);
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            if (!live || c + k >= p.D) continue;
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              x[e] = __uint_as_float(o[k + e]) * inv;
              if (any_bad) {
                const int d = c + k + e;
                if (bad[d] <= t) x[e] = __int_as_float(0x7fffffff);
                if (bad[DP + d] <= t) x[e] += INFINITY;
                if (bad[2 * DP + d] <= t) x[e] -= INFINITY;
              }
            }
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = BF16 ? pack_bf16x2(x[2 * e], x[2 * e + 1]) : pack_f16x2(x[2 * e], x[2 * e + 1]);
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + row * p.D + c + k) =
                make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
        }
        if (live && p.lse) p.lse[row] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : l == 0.f ? -INFINITY : l;
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
  if (tid == 0 && *abort_flag) report_timeout(nullptr);
}

// [T, heads, D] rows as a tensor of 64-column, 128B-swizzled boxes: q with
// the heads split into KV head and head of the group (box: `rows` tokens of
// one group), k and v with box_rows tokens of one head.  Columns past D and
// rows past T read 0.
static int make_rows_map(CUtensorMap* map, const void* base, bool bf16, int64_t D, int64_t group, int64_t heads,
                         int64_t T, int64_t head_stride, int64_t row_stride, int box_group, int box_rows) {
  const bool q = group > 0;
  cuuint64_t dims[4], strides[3];
  cuuint32_t box[4], estr[4] = {1, 1, 1, 1};
  int n = 0;
  dims[n] = cuuint64_t(D), box[n] = 64, ++n;
  if (q) {
    dims[n] = cuuint64_t(group), box[n] = cuuint32_t(box_group), strides[n - 1] = cuuint64_t(head_stride) * 2, ++n;
  }
  dims[n] = cuuint64_t(heads), box[n] = 1, strides[n - 1] = cuuint64_t(head_stride) * (q ? group : 1) * 2, ++n;
  dims[n] = cuuint64_t(T), box[n] = cuuint32_t(box_rows), strides[n - 1] = cuuint64_t(row_stride) * 2, ++n;
  const CUresult r = g_encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                              cuuint32_t(n), const_cast<void*>(base), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B2F_OK : B2F_ERR_INVALID;
}

template <int DP, bool BF16>
static int launch_prompt(const PromptParams& p, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                         unsigned grid, cudaStream_t st) {
  auto kern = prompt_attn_kernel<DP, BF16>;
  const int smem = PromptSmem<DP>::BYTES;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return B2F_ERR_CUDA;
  }
  return launch_kernel(kern, dim3{grid}, dim3{PA_THREADS}, size_t(smem), st, p, mq, mk, mv);
}

B2F_DEFINE_WAIT_CONTROLS(prompt_attn)

}  // namespace b2f

using namespace b2f;

extern "C" int b2f_prompt_attn(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row,
                               int64_t k_head, const void* v, int64_t v_row, int64_t v_head, int dtype,
                               const int32_t* cu_seqlens, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                               int causal, float softmax_scale, void* out, float* lse, void* stream) {
  if (dtype != B2F_BF16 && dtype != B2F_F16) return B2F_ERR_UNSUPPORTED;
  if (B < 0 || T < 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || Hq % Hkv != 0) return B2F_ERR_INVALID;
  if (D % 8 != 0 || D > 128 || Hq / Hkv > 128 || Hq > 65535 || B > (1 << 20) || T > (int64_t(1) << 30))
    return B2F_ERR_UNSUPPORTED;
  if (T == 0) return B2F_OK;
  if (!q || !k || !v || !cu_seqlens || !out) return B2F_ERR_INVALID;
  if (q_row <= 0 || q_head <= 0 || k_row <= 0 || k_head <= 0 || v_row <= 0 || v_head <= 0) return B2F_ERR_INVALID;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) ||
      (q_row | q_head | k_row | k_head | v_row | v_head) % 8 != 0)
    return B2F_ERR_ALIGN;
  int rc = get_encoder();
  if (rc != B2F_OK) return rc;
  const int64_t G = Hq / Hkv, tpt = 128 / G;
  // items: at most one partial pair of tiles per sequence and one for the rows of none
  const int64_t items = (T / (2 * tpt) + B + 1) * Hkv;
  if (items > 0x7fffffff) return B2F_ERR_UNSUPPORTED;
  const bool bf16 = dtype == B2F_BF16;
  CUtensorMap mq, mk, mv;
  if ((rc = make_rows_map(&mq, q, bf16, D, G, Hkv, T, q_head, q_row, int(G), int(tpt))) != B2F_OK ||
      (rc = make_rows_map(&mk, k, bf16, D, 0, Hkv, T, k_head, k_row, 0, PA_BN)) != B2F_OK ||
      (rc = make_rows_map(&mv, v, bf16, D, 0, Hkv, T, v_head, v_row, 0, PA_BN)) != B2F_OK)
    return rc;
  const float s2 = fabsf(softmax_scale) * kLog2e;
  PromptParams p{cu_seqlens, out, lse, s2 > 1e-30f ? s2 : 1e-30f, softmax_scale < 0.f, int(B), int(T), int(Hq),
                 int(Hkv), int(G), int(D), causal != 0, int(tpt)};
  cudaStream_t st = as_stream(stream);
  const unsigned n = unsigned(items);
  if (bf16) return D <= 64 ? launch_prompt<64, true>(p, mq, mk, mv, n, st) : launch_prompt<128, true>(p, mq, mk, mv, n, st);
  return D <= 64 ? launch_prompt<64, false>(p, mq, mk, mv, n, st) : launch_prompt<128, false>(p, mq, mk, mv, n, st);
}
