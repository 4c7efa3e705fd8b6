// Attention of packed prompts over themselves on the 5th-generation tensor
// cores: for each sequence and query head, softmax(scale * Q K^T) V, causal or
// full, grouped heads, sequences of any length back to back.
//
// Work item = (sequence, 2 tiles of consecutive tokens, KV head).  A tile is
// 128 MMA rows = 128 / G tokens x the G query heads of the KV head, so K and V
// are staged once for all heads that share them, and only the tile's own
// tokens, not 128 of them, see a diagonal block.  Per block of 128 keys:
//   S = Q K^T        tcgen05.mma, Q and K in shared memory (TMA, 128B swizzle)
//   P = 2^(S c - m)  two threads per row, 64 keys each: the scores come out of
//                    TMEM into registers, P goes back to TMEM as 16 bits
//   O += P V         tcgen05.mma with P read from TMEM, V as it lies (MN-major)
// Softmax in base 2, m and l and O in float32; P is rounded to the inputs'
// type because the tensor core takes both operands alike (its relative error
// is that of the output's own rounding).  m moves, and O is rescaled, only
// where a row's new maximum passes it by more than 8 (P stays below 2^8),
// which after the first blocks is rare.  So a row's two threads have to agree
// on one bit per block (a reduction in a barrier of the two warps that share
// 32 rows; each leaves half of its maximum for the other before it), and the
// rescale needs no warps of its own.  Where m moves it is the exact maximum:
// the largest P of a row of up to 128 keys is 1, which 16 bits hold (m rounded
// to 8 bits costs such rows 1.5 to 2.3 times the error of the output's
// rounding, against 1.1 to 1.2, and a row of one key is not its V).
//
// Warps: 0-7 softmax of tile 0, 8-15 of tile 1 (also the epilogue), 16 issues
// the MMAs, 17 plans the items and issues the TMA loads, 18-19 mend value
// tiles (below) and store the output of whole tiles, which the epilogue leaves
// in a ring stage (rows of a tile written by their threads cost a shared-memory
// port cycle per 128-byte line: 4500 cycles a tile).  The two tiles alternate:
// while the tensor core works on one, the other's softmax runs.  One thread
// per row left a warp of each tile on a scheduler, 2400 cycles a block of
// softmax and 1250 of MMA in a chain (1.17 PFLOP/s at 16384 tokens); two
// threads shorten the former.
//
// What bounds it: a block's chain of softmax (2100 cycles: 1536 of them
// exponentials when both tiles compute, the rest loads, the barrier, the
// stores) and MMA (1500), of which the two tiles overlap half; and power when
// it runs for long.  Heads of up to 64 leave TMEM columns for P beside S: the
// next scores are then computed under the softmax, and the tensor core is no
// longer in the chain; there tile 1 begins behind tile 0's first reading of
// its scores, so that their exponentials take turns (53 -> 49 us).  A block of
// two tiles takes 4100 cycles there, of which the exponentials account for
// 1536 (the unit is busy 39 % of the time, issue 51 %, the tensor core 26 %).
// At 128 columns of O per tile P lies over S.  The longest sequences go first
// where a warp holds them all (up to 31): 4 sequences of up to 1500 tokens, 28
// blocks on the busiest SM against 22.
// Measured (kernel): 32 heads of 128, 4 KV heads, causal: 16384 tokens 1.69 to
// 1.75 ms, 1.3 PFLOP/s (2.0 ms back to back, where power holds the clock at
// 1.4 GHz); 16 sequences of 1 to 2047 tokens 185 to 192 us, 0.87 PFLOP/s (an
// item has 6 blocks on average and costs 1.3 more at its ends); 3 of up to 60
// tokens 11 us.
// 16 heads of 64 in full, 4 sequences of 616 to 1500: 50 us, 0.42 PFLOP/s.
//
// A CTA (one per SM) takes item after item from the grid by cancelling CTAs
// that have not been launched; the items' roles overlap: loads and the first
// scores of the next one run under the epilogue of this one.
//
// Rows of V that a tile's rows must not see meet P = 0, and 0 * NaN is NaN.
// So in the blocks in which anything is masked, warps 18-19 zero the rows past
// the item's last key (they belong to other tokens or sequences) and replace
// what is not finite by 0, keeping for each column the first key with a NaN,
// +inf or -inf; the epilogue adds those back to the rows that see them.
#include "attn_tc.cuh"

namespace b2f {

constexpr int PA_THREADS = 640;
constexpr int PA_BN = 128;         // keys per block
constexpr int PA_MEND = 4;         // value tiles being mended (3 fit the ring)
constexpr int PA_STOP = -0x7fffffff - 1;
constexpr uint32_t PA_NO_BAD = 0x3fffffffu;  // 3 x 10 bits: no key

struct PromptParams {
  const int32_t* cu;
  void* out;
  float* lse;
  float scale2;   // |softmax_scale| * log2(e)
  int negate;     // softmax_scale < 0: the MMA negates Q
  int B, T, Hq, Hkv, G, D, causal;
  int tpt;        // tokens per tile
};

// What the planner hands to the other warps, worked out once.
struct __align__(16) PromptItem {
  int row0, len, tok0, hk;  // first row and tokens of the sequence, first token of the item, KV head
  int n0, n1;               // blocks of the tiles
  int mask;                 // first block in which anything is masked: at most 3 from there, as two tiles span <= 256 tokens
  int whole;                // bit i: the rows of tile i are all there; it leaves through a ring stage of its own

  __device__ __forceinline__ int blocks() const { return max(n0, n1); }
  // ring stages of the item: K and V of each block, then those of whole tiles
  __device__ __forceinline__ int stages() const { return 2 * blocks() + (whole & 1) + (whole >> 1); }
  __device__ __forceinline__ void plan(const PromptParams& p) {
    const int t1 = tok0 + p.tpt, e0 = p.causal ? min(len, t1) : len, e1 = t1 >= len ? 0 : p.causal ? min(len, t1 + p.tpt) : len;
    n0 = (e0 + PA_BN - 1) / PA_BN;
    n1 = (e1 + PA_BN - 1) / PA_BN;
    mask = (p.causal ? tok0 : len) / PA_BN;
    whole = int(t1 <= len) | int(t1 + p.tpt <= len) << 1;
  }
};

template <int DP>
struct PromptSmem {
  static constexpr int TILE = 128 * DP * 2;  // bytes of a Q tile, of a K or V block
  static constexpr int STAGES = DP == 128 ? 5 : 8;
  // TMEM columns: scores, P, O.  P lies over the scores where O leaves no other room.
  static constexpr bool APART = DP == 64;
  static constexpr int P_AT = APART ? 256 : 0, P_TILE = APART ? 64 : 128, O_AT = APART ? 384 : 256;
  uint8_t q[2][TILE];
  uint8_t ring[STAGES][TILE];  // K_0 V_0 K_1 V_1 ...
  // Between the two warps of 32 rows.  A thread reads the other's maximum after
  // a block's last barrier.  With P over the scores the next ones need both
  // threads' P, so the word is free by then; with P apart they do not, and the
  // next block's maxima go into words of their own, which that block's barrier
  // orders before the ones after.
  static constexpr int TOPS = APART ? 2 : 1;
  union {
    uint16_t top[TOPS][2][32];
    float sum[32];
  } exchange[8];
  int quit[8][2];              // per pair of warps and parity of the block: a wait gave up
  uint32_t bad[2][DP];         // per column: first key that is NaN | +inf | -inf, from the first masked block on
  int any_bad[2];
  PromptItem item[2];
  uint4 next;  // the answer of next_cta_ask
  uint64_t full[STAGES], empty[STAGES], q_full, q_empty, s_full[2], s_read[2], p_full[2], pv_done[2], v_raw[PA_MEND],
      v_fix[PA_MEND], o_full[2], item_full[2], item_empty[2], asked, drain;
  uint32_t tmem;
  int abort_flag;
};

// Waits with the CTA's abort flag; false once any wait gave up.
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  if (*abort_flag) return false;
  if (mbar_wait_bounded(bar, parity)) return true;
  *abort_flag = 1;
  return false;
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(PA_THREADS, 1) prompt_attn_kernel(const PromptParams p,
                                                                    const __grid_constant__ CUtensorMap tmq,
                                                                    const __grid_constant__ CUtensorMap tmk,
                                                                    const __grid_constant__ CUtensorMap tmv,
                                                                    const __grid_constant__ CUtensorMap tmo) {
  pdl_enter();
  using SM = PromptSmem<DP>;
  constexpr int NST = SM::STAGES, TILE = SM::TILE, HALF = 128 * 128;  // HALF: 64 columns of a tile
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  SM& sm = *reinterpret_cast<SM*>(smem_raw);
  volatile int* abort_flag = &sm.abort_flag;
  // (the shuffles tell the compiler that roles and items are uniform in a warp)
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (smem_u32(smem_raw) & 1023) {  // the swizzled tiles need it; the runtime gives it
    if (tid == 0) report_timeout(nullptr);
    return;
  }

  const bool stall = warp == 17 && producers_stalled();  // test control: stalled producers issue nothing
  if (tid == 0) {
    for (int s = 0; s < NST; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    mbar_init(&sm.q_full, 1);
    mbar_init(&sm.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.s_read[i], 8);
      mbar_init(&sm.p_full[i], 8);
      mbar_init(&sm.pv_done[i], 1);
      mbar_init(&sm.o_full[i], 8);
      mbar_init(&sm.item_full[i], 1);
      mbar_init(&sm.item_empty[i], 19);  // the warps but the planner's
      sm.any_bad[i] = 0;
    }
    for (int i = 0; i < 16; ++i) sm.quit[i >> 1][i & 1] = 0;
    for (int i = 0; i < PA_MEND; ++i) {
      mbar_init(&sm.v_raw[i], 1);
      mbar_init(&sm.v_fix[i], 2);
    }
    mbar_init(&sm.asked, 1);
    mbar_init(&sm.drain, 1);
    sm.abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  for (int i = tid; i < 2 * DP; i += PA_THREADS) sm.bad[i / DP][i % DP] = PA_NO_BAD;
  // Where the heads of a group do not divide 128, no load touches the last rows
  // of a Q tile: zeros, for whatever lay there before could send their warps
  // through the rescale in every block.
  if (const int rows = p.tpt * p.G; rows < 128) {
    for (int i = tid; i < 2 * (DP / 64) * 8 * (128 - rows); i += PA_THREADS) {
      const int part = i / (8 * (128 - rows)), at = i % (8 * (128 - rows));  // tile and 64 columns, 16 bytes
      reinterpret_cast<uint4*>(sm.q[0] + part * HALF + rows * 128)[at] = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);

  if (warp == 17) {
    // ============================ items and TMA loads ===========================
    const int span = 2 * p.tpt;
    int cta = blockIdx.x, asks = 0, items = 0, it = 0, mends = 0, loads = 0;
    int b_from = 0, pairs_before = 0;  // sequences looked through, their pairs: CTAs are taken over in rising order
    // this lane's sequence; sequence B: the rows past the last one
    int b, lo, hi;
    auto look = [&](int from) {
      b = from + lane;
      lo = hi = 0;
      if (b <= p.B) {
        lo = min(max(p.cu[b], 0), p.T);
        hi = b < p.B ? min(max(p.cu[b + 1], lo), p.T) : p.T;
      }
    };
    look(0);
    const bool sorted = p.B < 32;
    if (sorted) {
      const int key = b < p.B ? hi - lo : -1;
      int rank = 0, from = 0;
      for (int o = 0; o < 32; ++o) {
        const int k = __shfl_sync(0xffffffffu, key, o);
        rank += k > key || (k == key && o < lane);
      }
      for (int o = 0; o < 32; ++o)
        if (__shfl_sync(0xffffffffu, rank, o) == lane) from = o;
      b = __shfl_sync(0xffffffffu, b, from);
      lo = __shfl_sync(0xffffffffu, lo, from);
      hi = __shfl_sync(0xffffffffu, hi, from);
    }
    bool ok = true;
    // hands `x` to the other warps
    auto publish = [&](const PromptItem& x) {
      const int slot = items & 1;
      ok = items < 2 || __all_sync(0xffffffffu, wait_or_abort(&sm.item_empty[slot], uint32_t((items / 2 - 1) & 1), abort_flag));
      if (!ok) return;
      if (sm.any_bad[slot]) {  // left by the item before last
        for (int i = lane; i < DP; i += 32) sm.bad[slot][i] = PA_NO_BAD;
        __syncwarp();
        if (lane == 0) sm.any_bad[slot] = 0;
      }
      __syncwarp();
      if (lane == 0) {
        sm.item[slot] = x;
        mbar_arrive(&sm.item_full[slot]);
      }
      ++items;
    };
    while (ok) {
      if (lane == 0) {
        fence_proxy_async_smem();  // the last answer has been read
        mbar_arrive_expect_tx(&sm.asked, 16);
        next_cta_ask(&sm.next, &sm.asked);
      }
      // ---- the item of `cta` ----
      PromptItem x{0, 0, 0, cta % p.Hkv, 0, 0, 0, 0};
      const int want = cta / p.Hkv;  // pair of tiles, over all sequences
      if (want < pairs_before) b_from = pairs_before = 0;
      for (; b_from <= p.B; b_from += 32) {
        if (!sorted) look(b_from);
        const int n = (hi - lo + span - 1) / span;
        int s = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int a = __shfl_up_sync(0xffffffffu, s, o);
          if (lane >= o) s += a;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, s > want - pairs_before);
        if (hit) {
          const int w = __ffs(hit) - 1;
          x.row0 = __shfl_sync(0xffffffffu, lo, w);
          x.len = __shfl_sync(0xffffffffu, b < p.B ? hi - lo : lo - hi, w);  // negative: rows of no sequence
          // the longest sequences, and rows of a sequence, first: they set the tail of the grid
          x.tok0 = (__shfl_sync(0xffffffffu, s, w) - 1 - (want - pairs_before)) * span;
          break;
        }
        pairs_before += __shfl_sync(0xffffffffu, s, 31);
      }
      if (x.len > 0) x.plan(p);
      if (x.len != 0) publish(x);  // 0: a spare CTA of the grid
      if (ok && x.len > 0) {
        const int all = x.blocks(), stages = x.stages();
        if (lane == 0 && !stall) {
          auto load = [&](int i) {  // K (even i) or V of block i / 2; then the stages of whole tiles
            const int n = it + i, s = n % NST;
            if (n >= NST && !wait_or_abort(&sm.empty[s], uint32_t((n / NST - 1) & 1), abort_flag)) return false;
            if (i >= 2 * all) {
              mbar_arrive(&sm.full[s]);
              return true;
            }
            // a value block with masked rows lands on a barrier of its own, for warps 18-19
            const int j = i >> 1;
            const bool mend = (i & 1) && j >= x.mask;
            uint64_t* bar = mend ? &sm.v_raw[(mends + j - x.mask) % PA_MEND] : &sm.full[s];
            if (mend) mbar_arrive(&sm.full[s]);
            mbar_arrive_expect_tx(bar, uint32_t(TILE));
            for (int h = 0; h < DP / 64; ++h)
              tma_load_3d(sm.ring[s] + h * HALF, i & 1 ? &tmv : &tmk, 64 * h, x.hk, x.row0 + j * PA_BN, bar);
            return true;
          };
          int i = 0;
          ok = load(i++) && load(i++);
          ok = ok && (loads == 0 || wait_or_abort(&sm.q_empty, uint32_t((loads - 1) & 1), abort_flag));
          if (ok) {
            const int tiles = x.n1 ? 2 : 1;
            mbar_arrive_expect_tx(&sm.q_full, uint32_t(tiles * (DP / 64) * p.tpt * p.G * 128));
            for (int t = 0; t < tiles; ++t)
              for (int h = 0; h < DP / 64; ++h)
                tma_load_4d(sm.q[t] + h * HALF, &tmq, 64 * h, 0, x.hk, x.row0 + x.tok0 + t * p.tpt, &sm.q_full);
          }
          while (ok && i < stages) ok = load(i++);
          if (!ok) {
            // copies already issued land before the CTA goes away
            mbar_wait_bounded(&sm.q_full, uint32_t(loads & 1), 100000000ull);
            for (int k = 1; k <= NST && it + i - k >= 0; ++k) {
              const int n = it + i - k;
              mbar_wait_bounded(&sm.full[n % NST], uint32_t((n / NST) & 1), 100000000ull);
            }
            for (int j = x.mask; 2 * j + 1 < min(i, 2 * all); ++j) {
              const int m = mends + j - x.mask;
              mbar_wait_bounded(&sm.v_raw[m % PA_MEND], uint32_t((m / PA_MEND) & 1), 100000000ull);
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, int(ok), 0) != 0;
        it += stages;
        mends += max(0, all - x.mask);
        ++loads;
      }
      // the answer lands whatever happened (a bounded wait)
      const bool landed = mbar_wait_bounded(&sm.asked, uint32_t(asks++ & 1));
      if (!__all_sync(0xffffffffu, landed)) {
        if (lane == 0) *abort_flag = 1;
        ok = false;
      }
      if (!ok) break;
      cta = next_cta_answer(&sm.next);
      __syncwarp();
      if (cta < 0) break;
    }
    if (ok) publish(PromptItem{0, PA_STOP, 0, 0, 0, 0, 0, 0});
  } else if (warp >= 18) {
    // ================ value tiles with masked rows; whole tiles' output ==========
    const int tile = warp - 18;
    int stored = 0;
    int it = 0, mends = 0;
    for (int k = 0;; ++k) {
      const int slot = k & 1;
      if (!__all_sync(0xffffffffu, wait_or_abort(&sm.item_full[slot], uint32_t((k / 2) & 1), abort_flag))) break;
      const PromptItem x = sm.item[slot];
      if (x.len == PA_STOP) break;
      bool ok = true;
      if (x.len > 0) {
        const int all = x.blocks();
        const int kend = p.causal ? min(x.len, x.tok0 + 2 * p.tpt) : x.len;  // keys of the item
        for (int j = x.mask; j < all; ++j, ++mends) {
          const int b = mends % PA_MEND;
          ok = __all_sync(0xffffffffu, wait_or_abort(&sm.v_raw[b], uint32_t((mends / PA_MEND) & 1), abort_flag));
          if (!ok) break;
          uint8_t* v = sm.ring[(it + 2 * j + 1) % NST];
          const int valid = min(PA_BN, kend - j * PA_BN);
          // keys up to the item's first token are seen by all its rows
          const int from = p.causal ? max(0, min(PA_BN, x.tok0 + 1 - j * PA_BN)) : valid, n = PA_BN - from;
          // a line = 64 columns of one key; the two warps take four lines each in turn
          for (int line = (warp - 18) * 4 + (lane >> 3); line < n * (DP / 64); line += 8) {
            const int h = line >= n, key = from + line - h * n, c = lane & 7;
            uint4* at = reinterpret_cast<uint4*>(v + h * HALF + key * 128 + ((c ^ (key & 7)) << 4));
            if (key >= valid) {
              *at = make_uint4(0u, 0u, 0u, 0u);
            } else if (p.causal) {
              uint4 w = *at;
              constexpr uint32_t expo = BF16 ? 0x7F80u : 0x7C00u;
              uint32_t* u = reinterpret_cast<uint32_t*>(&w);
              bool any = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) any |= (u[e] & expo) == expo || ((u[e] >> 16) & expo) == expo;
              if (any) {
                for (int e = 0; e < 8; ++e) {
                  const uint32_t y = (u[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
                  if ((y & expo) != expo) continue;
                  const int at10 = (y & ~expo & 0x7FFFu) ? 0 : (y & 0x8000u) ? 20 : 10;  // NaN, +inf, -inf
                  const uint32_t off = uint32_t((j - x.mask) * PA_BN + key);
                  uint32_t* word = &sm.bad[slot][64 * h + 8 * c + e];
                  uint32_t old = *word, seen;
                  do {
                    seen = old;
                    if (((seen >> at10) & 1023u) <= off) break;
                    old = atomicCAS(word, seen, (seen & ~(1023u << at10)) | (off << at10));
                  } while (old != seen);
                  sm.any_bad[slot] = 1;
                  u[e >> 1] &= ~(0xFFFFu << (16 * (e & 1)));
                }
                *at = w;
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.v_fix[b]);
        }
        if (ok && (x.whole >> tile & 1)) {
          const int s = (it + 2 * all + tile) % NST;  // (a whole second tile follows a whole first)
          ok = __all_sync(0xffffffffu, wait_or_abort(&sm.o_full[tile], uint32_t(stored++ & 1), abort_flag));
          if (ok && lane == 0) {
            for (int c = 0; c < DP / 64; ++c)
              if (64 * c < p.D) tma_store_4d(&tmo, sm.ring[s] + c * HALF, 64 * c, 0, x.hk, x.row0 + x.tok0 + tile * p.tpt);
            bulk_s2g_wait();
            mbar_arrive(&sm.empty[s]);
          }
          __syncwarp();
        }
        it += x.stages();
      }
      if (!ok) break;
      if (lane == 0) mbar_arrive(&sm.item_empty[slot]);
    }
    __syncwarp();
  } else if (warp == 16) {
    // ============================ MMA issuer ====================================
    const uint32_t one = elect_lane();
    const uint32_t id_s = mma_idesc(PA_BN, BF16, false, p.negate), id_o = mma_idesc(DP, BF16, true, false);
    auto wait_all = [&](uint64_t* bar, uint32_t parity) {
      return bool(__all_sync(0xffffffffu, wait_or_abort(bar, parity, abort_flag)));
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
    const uint64_t q_desc = sw128_desc(sm.q[0]), k_desc = sw128_desc(sm.ring[0]), v_desc = sw128_mn_desc(sm.ring[0], HALF);
    auto score = [&](int i, int stage) {  // S_i = Q_i K^T
      const uint64_t a = q_desc + uint64_t(i * (TILE >> 4)), b = k_desc + uint64_t(stage * (TILE >> 4));
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        const uint64_t at = (ks >> 2) * (HALF >> 4) + 2 * (ks & 3);
        tc_mma_ss(one, tmem + 128 * i, a + at, b + at, id_s, ks > 0);
      }
      tc_commit_by(one, &sm.s_full[i]);
    };
    Ring ring;
    int mends = 0, loads = 0;
    int done[2] = {0, 0};  // blocks of each tile so far
    bool ok = true;
    for (int k = 0; ok; ++k) {
      const int slot = k & 1;
      ok = wait_all(&sm.item_full[slot], uint32_t((k / 2) & 1));
      if (!ok) break;
      const PromptItem& x = sm.item[slot];
      const int len = __shfl_sync(0xffffffffu, x.len, 0);
      if (len == PA_STOP) break;
      if (len > 0) {
        const int nb[2] = {__shfl_sync(0xffffffffu, x.n0, 0), __shfl_sync(0xffffffffu, x.n1, 0)};
        const int mask = __shfl_sync(0xffffffffu, x.mask, 0), whole = __shfl_sync(0xffffffffu, x.whole, 0);
        const int all = max(nb[0], nb[1]);
        ok = wait_all(&sm.q_full, uint32_t(loads++ & 1)) && full_of(ring);
        if (!ok) break;
        tc_fence_after();
        const int first = ring.s;  // K_0
        score(0, first);
        auto begun = [&]() {
          if (nb[1]) score(1, first);
          tc_commit_by(one, &sm.empty[first]);
          if (all == 1) tc_commit_by(one, &sm.q_empty);
        };
        if (!SM::APART) begun();
        for (int j = 0; ok && j < all; ++j) {
          ring.next();
          const Ring rv = ring;  // V_j
          if (j + 1 < all) {  // K_{j+1} (before the waits for P, which are what takes time)
            ring.next();
            ok = full_of(ring);
          }
          auto scored = [&]() {  // the scores of the next block are issued
            if (j + 1 < all) tc_commit_by(one, &sm.empty[ring.s]);
            if (j + 2 == all) tc_commit_by(one, &sm.q_empty);
          };
          if constexpr (SM::APART) {
            for (int i = 0; ok && i < 2; ++i) {
              if (j >= nb[i]) continue;
              ok = wait_all(&sm.s_read[i], uint32_t(done[i] & 1));
              tc_fence_after();
              if (ok && i == 0 && j == 0) begun();
              if (ok && j + 1 < nb[i]) score(i, ring.s);
            }
            if (!ok) break;
            scored();
          }
          if (j < mask) {
            ok = ok && full_of(rv);
          } else {
            ok = ok && wait_all(&sm.v_fix[mends % PA_MEND], uint32_t((mends / PA_MEND) & 1));
            ++mends;
          }
          for (int i = 0; ok && i < 2; ++i) {
            if (j >= nb[i]) continue;
            const uint64_t v = v_desc + uint64_t(rv.s * (TILE >> 4));
            ok = wait_all(&sm.p_full[i], uint32_t(done[i] & 1));
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)  // O_i += P_i V_j
              tc_mma_ts(one, tmem + SM::O_AT + DP * i, tmem + SM::P_AT + SM::P_TILE * i + 8 * ks,
                        v + ks * (2048 >> 4), id_o, j > 0 || ks > 0);
            ++done[i];
            tc_commit_by(one, &sm.pv_done[i]);
            if (!SM::APART && j + 1 < nb[i]) score(i, ring.s);
          }
          if (!ok) break;
          tc_commit_by(one, &sm.empty[rv.s]);
          if (!SM::APART) scored();
        }
        for (int i = 0; i <= (whole & 1) + (whole >> 1); ++i) ring.next();
      }
      if (ok && lane == 0) mbar_arrive(&sm.item_empty[slot]);
    }
    // all MMAs issued complete before TMEM is released
    tc_commit_by(one, &sm.drain);
    mbar_wait_bounded(&sm.drain, 0u, 100000000ull);
    __syncwarp();
  } else {
    // ============================ softmax and epilogue ==========================
    // The two warps of 32 rows share a barrier and leave the loops together:
    // what a wait that gave up says goes through the barrier first.
    const int i = warp >> 3, h = (warp >> 2) & 1, r = tid & 127;  // tile, half of the keys, MMA row
    const int pair = 4 * i + (warp & 3), bar = 1 + pair;
    auto& exchange = sm.exchange[pair];
    const uint32_t lane_at = uint32_t(32 * (warp & 3)) << 16;
    const uint32_t s_at = tmem + lane_at + 128 * i + 64 * h, o_at = tmem + lane_at + SM::O_AT + DP * i + DP / 2 * h,
                   p_at = tmem + lane_at + SM::P_AT + SM::P_TILE * i + 32 * h;
    auto wait_all = [&](uint64_t* b, uint32_t parity) {
      return bool(__all_sync(0xffffffffu, wait_or_abort(b, parity, abort_flag)));
    };
    // sum over the row's two threads
    auto joined = [&](float v) {
      if (h) exchange.sum[lane] = v;
      bar_all(bar, 64);
      if (!h) exchange.sum[lane] = v += exchange.sum[lane];
      bar_all(bar, 64);
      return h ? exchange.sum[lane] : v;
    };
    const int rt = r / p.G, rh = r - rt * p.G;  // token of the tile, head of the group
    const bool row_of_tile = r < p.tpt * p.G;
    int it = 0;
    int done = 0;  // blocks of this tile so far
    for (int k = 0;; ++k) {
      const int slot = k & 1;
      bool ok = wait_all(&sm.item_full[slot], uint32_t((k / 2) & 1));
      if (bar_or(bar, 64, !ok)) break;
      const PromptItem x = sm.item[slot];
      if (x.len == PA_STOP) break;
      if (x.len < 0) {
        // rows of no sequence: zeros
        const int n = min(2 * p.tpt, -x.len - x.tok0);
        for (int e = tid; e < n * p.G; e += 512) {
          const int64_t row = int64_t(x.row0 + x.tok0 + e / p.G) * p.Hq + x.hk * p.G + e % p.G;
          for (int d = 0; d < p.D; d += 8)
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + row * p.D + d) = make_uint4(0u, 0u, 0u, 0u);
          if (p.lse) p.lse[row] = -INFINITY;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.item_empty[slot]);
        continue;
      }
      const int nb = i ? x.n1 : x.n0;
      const int t = x.tok0 + i * p.tpt + rt;
      const bool live = row_of_tile && t < x.len;
      // last key the row sees (what rows past the sequence hold is not stored)
      const int last = !row_of_tile ? -1 : p.causal ? t : x.len - 1;
      float m = -INFINITY, l = 0.f;  // m: reference of the exponents (scaled scores)
      bool quit = false;
      for (int j = 0; j < nb; ++j, ++done) {
        ok = ok && wait_all(&sm.s_full[i], uint32_t(done & 1));
        tc_fence_after();
        uint32_t s[64];
        tmem_ld64(s_at, s);
        if (SM::APART) {  // the next block's scores may come
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.s_read[i]);
        }
        const int rel = last - j * PA_BN - 64 * h;
        const bool masked = j >= x.mask && !__all_sync(0xffffffffu, rel >= 63);
        if (masked) {
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (c > rel) s[c] = 0xFF800000u;
        }
        const float top = row_max(s) * p.scale2;
        // every score of the 32 rows has been read past this barrier, and what
        // a thread leaves before it can be read by the other: the upper half
        // of its maximum's bits
        auto& tops = exchange.top[j % SM::TOPS];
        tops[h][lane] = uint16_t(__float_as_uint(top) >> 16);
        if (!ok) sm.quit[pair][j & 1] = 1;
        if (bar_or(bar, 64, !ok || j == 0 || !(top <= m + 8.f))) {
          if (*const_cast<volatile int*>(&sm.quit[pair][j & 1])) {
            quit = true;
            break;
          }
          const uint32_t upper = tops[1 - h][lane];
          bar_all(bar, 64);
          tops[h][lane] = uint16_t(__float_as_uint(top));  // then the lower half
          bar_all(bar, 64);
          float both = max2(top, __uint_as_float(upper << 16 | tops[1 - h][lane]));
          if (both == INFINITY) both = __int_as_float(0x7fffffff);  // inf - inf
          const bool move = j == 0 || !(both <= m + 8.f);
          if (j > 0) {
            // O holds blocks up to j - 1 once their product is done
            ok = wait_all(&sm.pv_done[i], uint32_t((done - 1) & 1));
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
        uint64_t sum[2] = {0ull, 0ull};
        uint32_t pk[32];
        if (masked) exp_row<BF16, false>(s, p.scale2, ref, sum, pk);  // exact zeros
        else exp_row<BF16, true>(s, p.scale2, ref, sum, pk);
        // P of the block before has been used up
        if (SM::APART && j > 0) {
          ok = ok && wait_all(&sm.pv_done[i], uint32_t((done - 1) & 1));
          tc_fence_after();
        }
        tmem_st32(p_at, pk);
        const float2 l2 = f32x2_parts(add_x2(sum[0], sum[1]));
        l += l2.x + l2.y;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[i]);
      }
      if (quit) break;
      if (nb) {
        ok = ok && wait_all(&sm.pv_done[i], uint32_t((done - 1) & 1));
        tc_fence_after();
        l = joined(l);  // (the last product needed every thread's P: all maxima have been read)
        const int64_t row = int64_t(x.row0 + t) * p.Hq + x.hk * p.G + rh;
        // NaN where a score is (l is), and where all scores are -inf (a row sees its own key at least)
        const float inv = m == -INFINITY ? __int_as_float(0x7fffffff) : 1.f / l;
        const bool any_bad = *const_cast<volatile int*>(&sm.any_bad[slot]) != 0;
        const int seen = t - x.mask * PA_BN;  // keys up to here, from the first masked block
        // a whole tile leaves through the ring stage that the planner grants it
        const bool staged = x.whole >> i & 1;
        const int n = it + 2 * x.blocks() + i;  // (a whole second tile follows a whole first)
        uint8_t* stage = sm.ring[n % NST];
        if (staged) ok = ok && wait_all(&sm.full[n % NST], uint32_t((n / NST) & 1));
        if (ok) {
#pragma unroll
          for (int c = 0; c < DP / 2; c += 32) {
            uint32_t o[32];
            tmem_ld32(o_at + c, o);
            if (any_bad) {
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const uint32_t w = sm.bad[slot][DP / 2 * h + c + e];
                float y = __uint_as_float(o[e]);
                if (int(w & 1023u) <= seen) y = __int_as_float(0x7fffffff);
                if (int((w >> 10) & 1023u) <= seen) y += INFINITY;
                if (int((w >> 20) & 1023u) <= seen) y -= INFINITY;
                o[e] = __float_as_uint(y);
              }
            }
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float y0 = __uint_as_float(o[2 * e]) * inv, y1 = __uint_as_float(o[2 * e + 1]) * inv;
              w[e] = BF16 ? pack_bf16x2(y0, y1) : pack_f16x2(y0, y1);
            }
            const int d = DP / 2 * h + c;
            if (staged) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int col = d / 8 + e;  // 16-byte column of the row
                *reinterpret_cast<uint4*>(stage + (col >> 3) * HALF + r * 128 + (((col & 7) ^ (r & 7)) << 4)) =
                    make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
              }
            } else if (live) {
              uint16_t* dst = static_cast<uint16_t*>(p.out) + row * p.D + d;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (d + 8 * e < p.D)
                  *reinterpret_cast<uint4*>(dst + 8 * e) = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
            }
            __syncwarp();
          }
          if (staged) fence_proxy_async_smem();
          if (live && p.lse && h == 0)
            p.lse[row] = m == -INFINITY ? m : (m + log2f(l)) * 0.6931471805599453f;
        }
        tc_fence_before();
        __syncwarp();
        if (staged && ok && lane == 0) mbar_arrive(&sm.o_full[i]);  // warp 18 or 19 stores it
      }
      it += x.stages();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.item_empty[slot]);
      // a wait that gave up is told at the next item's barrier (the flag makes that wait fail too)
    }
  }
  __syncthreads();
  if (warp == 16) {
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
                         const CUtensorMap& mo, unsigned grid, cudaStream_t st) {
  constexpr auto kern = prompt_attn_kernel<DP, BF16>;
  const int smem = int(sizeof(PromptSmem<DP>));
  static_assert(sizeof(PromptSmem<DP>) <= 227 * 1024, "one CTA's shared memory");
  const int set = allow_smem<kern>(smem);
  if (set != B2F_OK) return set;
  return launch_kernel(kern, dim3{grid}, dim3{PA_THREADS}, size_t(smem), st, p, mq, mk, mv, mo);
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
  CUtensorMap mq, mk, mv, mo;
  if ((rc = make_rows_map(&mq, q, bf16, D, G, Hkv, T, q_head, q_row, int(G), int(tpt))) != B2F_OK ||
      (rc = make_rows_map(&mk, k, bf16, D, 0, Hkv, T, k_head, k_row, 0, PA_BN)) != B2F_OK ||
      (rc = make_rows_map(&mv, v, bf16, D, 0, Hkv, T, v_head, v_row, 0, PA_BN)) != B2F_OK ||
      (rc = make_rows_map(&mo, out, bf16, D, G, Hkv, T, D, Hq * D, int(G), int(tpt))) != B2F_OK)
    return rc;
  const float s2 = fabsf(softmax_scale) * kLog2e;
  PromptParams p{cu_seqlens, out, lse, s2 <= 1e-30f ? 1e-30f : s2, softmax_scale < 0.f, int(B), int(T), int(Hq),
                 int(Hkv), int(G), int(D), causal != 0, int(tpt)};
  cudaStream_t st = as_stream(stream);
  const unsigned n = unsigned(items);
  if (bf16) return D <= 64 ? launch_prompt<64, true>(p, mq, mk, mv, mo, n, st) : launch_prompt<128, true>(p, mq, mk, mv, mo, n, st);
  return D <= 64 ? launch_prompt<64, false>(p, mq, mk, mv, mo, n, st) : launch_prompt<128, false>(p, mq, mk, mv, mo, n, st);
}
