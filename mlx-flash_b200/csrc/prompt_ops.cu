// What a batch of packed prompts needs before attention: the page plan (block
// tables, slot map, positions) from the requests' lengths, and the per-head
// RMSNorm + rotary position of queries and keys, with the quantized rows
// appended to the planned slots in the same pass.
#include "common.cuh"

#include <type_traits>

namespace b2f {

// ---- page plan --------------------------------------------------------------
// Request b holds ctx[b] tokens and gets n[b] more.  With P tokens a page,
//   have = ceil(ctx / P), need = ceil((ctx + n) / P)
//   cu[b]    = n[0] + ... + n[b-1]          (packed offset of its tokens)
//   first[b] = sum over earlier requests of need - have
//   table[b, have + i] = free[first[b] + i], i < need - have
//   token t of request b: pos = ctx + t - cu[b], slot = table[b, pos / P] * P + pos % P
// The output is 16 bytes a token and 4 a page, so up to 10^5 tokens the launch
// itself is the cost: every CTA scans the lengths for itself (shared memory,
// up to kScanRows requests) instead of waiting for a scan kernel.  More
// requests take the scan in a launch of its own, which leaves both sums in
// global memory for the fill.  Measured: 4.2 us for 3 requests, 6.2 for 509
// with 200003 tokens (3.3 MB), 11.4 for 2048; by two launches 14.5 for 2049.
constexpr int kPlanThreads = 256;
constexpr int kScanRows = 2048;

struct PagePlanParams {
  const int32_t* n;
  const int32_t* ctx;  // or null: nothing held
  const int32_t* free_pages;
  int32_t* table;
  int32_t* cu;
  int32_t* positions;
  int64_t* slots;
  int32_t* rows;
  int32_t* seq_lens;
  int32_t* counts;
  int32_t* first;  // workspace [B + 1], more than kScanRows requests only
  int B, T, F, max_pages, P;
};

__device__ __forceinline__ int pages_for(int tokens, int P) { return (tokens + P - 1) / P; }

// Exclusive sums of the lengths and of the new pages into cu / first [B + 1],
// by the whole CTA.
__device__ void plan_scan(const PagePlanParams& p, int32_t* cu, int32_t* first) {
  __shared__ int2 warp_sum[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  int2 base = make_int2(0, 0);
  for (int b0 = 0; b0 < p.B; b0 += blockDim.x) {
    const int b = b0 + tid;
    int2 v = make_int2(0, 0);
    if (b < p.B) {
      const int c = p.ctx ? max(p.ctx[b], 0) : 0;
      v.x = max(p.n[b], 0);
      v.y = pages_for(c + v.x, p.P) - pages_for(c, p.P);
    }
    int2 s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, s.x, o), c = __shfl_up_sync(0xffffffffu, s.y, o);
      if (lane >= o) s.x += a, s.y += c;
    }
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    int2 before = base, all = make_int2(0, 0);
    for (int w = 0; w < nw; ++w) {
      if (w < warp) before.x += warp_sum[w].x, before.y += warp_sum[w].y;
      all.x += warp_sum[w].x, all.y += warp_sum[w].y;
    }
    if (b < p.B) {
      cu[b] = before.x + s.x - v.x;
      first[b] = before.y + s.y - v.y;
    }
    base.x += all.x, base.y += all.y;
    __syncthreads();
  }
  if (tid == 0) {
    cu[p.B] = base.x;
    first[p.B] = base.y;
  }
  __syncthreads();
}

__global__ void __launch_bounds__(1024) page_plan_scan_kernel(const PagePlanParams p) {
  pdl_enter();
  plan_scan(p, p.cu, p.first);
}

// The largest r in [0, n) with a[r] <= x, where a[0] = 0 <= x (zero-length
// requests share their offset with the next one, which is the one found).
__device__ __forceinline__ int last_at_most(const int32_t* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <bool SCAN>
__global__ void __launch_bounds__(kPlanThreads) page_plan_fill_kernel(const PagePlanParams p) {
  pdl_enter();
  extern __shared__ int32_t plan_smem[];
  const int32_t *cu = p.cu, *first = p.first;
  if constexpr (SCAN) {
    plan_scan(p, plan_smem, plan_smem + p.B + 1);
    cu = plan_smem;
    first = plan_smem + p.B + 1;
  }
  const int gtid = blockIdx.x * blockDim.x + threadIdx.x, nthreads = gridDim.x * blockDim.x;
  const int total = cu[p.B], new_pages = first[p.B];
  if (gtid == 0) {
    p.counts[0] = total;
    p.counts[1] = new_pages;
  }
  for (int b = gtid; b <= p.B; b += nthreads) {
    if constexpr (SCAN) p.cu[b] = cu[b];
    if (b < p.B) p.seq_lens[b] = (p.ctx ? max(p.ctx[b], 0) : 0) + max(p.n[b], 0);
  }
  for (int i = gtid; i < new_pages; i += nthreads) {
    const int b = last_at_most(first, p.B, i);
    const int e = pages_for(p.ctx ? max(p.ctx[b], 0) : 0, p.P) + i - first[b];
    if (e < p.max_pages) p.table[int64_t(b) * p.max_pages + e] = i < p.F ? p.free_pages[i] : -1;
  }
  // four consecutive tokens a thread: one search, then a walk over the requests
  for (int t0 = gtid * 4; t0 < p.T; t0 += nthreads * 4) {
    int pos[4], row[4];
    int64_t slot[4];
    int b = -1, next = 0, off = 0, have = 0, f0 = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = t0 + i;
      pos[i] = 0, row[i] = -1, slot[i] = -1;
      if (t >= total || t >= p.T) continue;
      if (b < 0 || t >= next) {
        if (b < 0) b = last_at_most(cu, p.B, t);
        else
          while (cu[b + 1] <= t) ++b;
        const int c = p.ctx ? max(p.ctx[b], 0) : 0;
        next = cu[b + 1];
        off = c - cu[b];
        have = pages_for(c, p.P);
        f0 = first[b] - have;
      }
      row[i] = b;
      pos[i] = t + off;
      const int e = pos[i] / p.P;
      int page = -1;
      if (e < p.max_pages) {
        if (e < have) page = p.table[int64_t(b) * p.max_pages + e];
        else if (f0 + e < p.F) page = p.free_pages[f0 + e];
      }
      if (page >= 0) slot[i] = int64_t(page) * p.P + (pos[i] - e * p.P);
    }
    if (t0 + 4 <= p.T) {
      *reinterpret_cast<int4*>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<int4*>(p.rows + t0) = make_int4(row[0], row[1], row[2], row[3]);
      reinterpret_cast<longlong2*>(p.slots + t0)[0] = make_longlong2(slot[0], slot[1]);
      reinterpret_cast<longlong2*>(p.slots + t0)[1] = make_longlong2(slot[2], slot[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t0 + i < p.T) {
          p.positions[t0 + i] = pos[i];
          p.rows[t0 + i] = row[i];
          p.slots[t0 + i] = slot[i];
        }
    }
  }
}

// ---- per-head RMSNorm + rotary of packed rows, optional paged append --------
//   y = x * rsqrt(mean(x^2) + eps) * w
//   (y_i, y_{i+R/2}) -> (y_i cos a - y_{i+R/2} sin a, y_{i+R/2} cos a + y_i sin a),
//   a = pos * inv_freq[i], i < R/2 (R = rotary width; dims past R unrotated)
// HBM-bound: q and k are read and written once.  D / 8 lanes hold one head,
// each two pieces of 4 values that rotate into one another (pieces i and
// i + R/8 of the head; past R two neighbours), so the rotation needs no
// shuffles, and a lane keeps one token: w cos and w sin stay in registers for
// all of the token's heads.
// Everything is float32 with one rounding at the end; the angle is formed and
// reduced in double, because pos * inv_freq in float32 is off by 2^-25 * pos
// (0.004 rad at 131072).
// Appended K rows are the rounded k output through the cache's quantizer
// (per 64 values: scale = absmax / max_int, each step rounded to the rows'
// type), V rows are quantized as they are.
struct NormRopeParams {
  const void* qkv;
  int64_t ld;  // elements between rows
  const void* qw;
  const void* kw;
  const double* inv_freq;
  const int32_t* positions;
  void* q_out;
  void* k_out;
  const int64_t* slots;
  uint8_t* k_codes;
  float* k_scales;
  uint8_t* v_codes;
  float* v_scales;
  float eps;
  int T, Hq, Hkv, P, R, bits;
};

template <typename Tag>
__device__ __forceinline__ void unpack4(uint2 w, float (&v)[4]) {
  const typename Tag::T* e = reinterpret_cast<const typename Tag::T*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = Tag::to_f(e[i]);
}
template <typename Tag>
__device__ __forceinline__ uint2 pack4(const float (&v)[4]) {
  typename Tag::T e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = Tag::from_f(v[i]);
  return *reinterpret_cast<uint2*>(e);
}

// One 8-value piece (lane `sub` of a row) of a K or V row through the cache's
// quantizer; 8 neighbouring lanes hold a group of 64.
template <typename Tag, int D>
__device__ __forceinline__ void append_piece(uint4 w, int sub, int64_t row, int bits, uint8_t* codes, float* scales) {
  using T2 = std::conditional_t<Tag::kBits == 8, __nv_bfloat162, __half2>;
  const float mi = bits == 8 ? 127.f : bits == 4 ? 7.f : 1.f;
  const typename Tag::T* e = reinterpret_cast<const typename Tag::T*>(&w);
  const T2* e2 = reinterpret_cast<const T2*>(&w);
  const T2 top = __hmax2(__hmax2(__habs2(e2[0]), __habs2(e2[1])), __hmax2(__habs2(e2[2]), __habs2(e2[3])));
  float m = fmaxf(fmaxf(Tag::to_f(top.x), Tag::to_f(top.y)), 0.f);
#pragma unroll
  for (int k = 1; k < 8; k <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
  if (row < 0) return;
  float scale = Tag::round(__fdiv_rn(m, mi));
  if (scale == 0.f) scale = 1.f;
  // round(v / scale) to the rows' type: the product with the reciprocal is
  // within 2 ulp of the quotient, so both round alike unless the product lies
  // within 8 ulp of a midpoint of the type; there, divide.  Then to the nearest
  // integer (ties to even) by adding 1.5 * 2^23, whose low byte is the code
  // (signed); two values, then four, at a time.
  const float rs = __frcp_rn(scale);
  constexpr uint32_t kLow = (1u << (24 - Tag::kBits)) - 1;  // float bits below the type's last
  float x[8];
  uint32_t near = 0xFFFFFFFFu;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = __fmul_rn(Tag::to_f(e[i]), rs);
    near = min(near, (__float_as_uint(x[i]) & kLow) - (kLow / 2 - 7u));
  }
  if (near <= 0x10u || !isfinite(rs)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fdiv_rn(Tag::to_f(e[i]), scale);
  }
  T2 lo, hi;
  lo.x = lo.y = Tag::from_f(-mi);
  hi.x = hi.y = Tag::from_f(mi);
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    T2 y;
    y.x = Tag::from_f(x[2 * i]);
    y.y = Tag::from_f(x[2 * i + 1]);
    y = __hmin2(__hmax2(y, lo), hi);
    c[2 * i] = __float_as_uint(__fadd_rn(Tag::to_f(y.x), 12582912.f));
    c[2 * i + 1] = __float_as_uint(__fadd_rn(Tag::to_f(y.y), 12582912.f));
  }
  uint32_t b[2];  // a code a byte
#pragma unroll
  for (int i = 0; i < 2; ++i)
    b[i] = (prmt(prmt(c[4 * i], c[4 * i + 1], 0x0040u), prmt(c[4 * i + 2], c[4 * i + 3], 0x0040u), 0x5410u) ^ 0x80808080u) -
           (128u - uint32_t(mi)) * 0x01010101u;
  if (sub % 8 == 0) scales[row * (D / 64) + sub / 8] = scale;
  uint8_t* dst = codes + row * (D * bits / 8) + sub * bits;
  if (bits == 8) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(b[0], b[1]);
  } else if (bits == 4) {
    *reinterpret_cast<uint32_t*>(dst) = prmt(b[0] << 4 | b[0] >> 8, b[1] << 4 | b[1] >> 8, 0x6420u);
  } else {
    *reinterpret_cast<uint16_t*>(dst) =
        uint16_t(prmt(b[0] << 6 | b[0] >> 4 | b[0] >> 14 | b[0] >> 24, b[1] << 6 | b[1] >> 4 | b[1] >> 14 | b[1] >> 24, 0x0040u));
  }
}

// One lane's share of the heads of a token.
template <typename Tag, int D>
struct NormRopeLane {
  using E = typename Tag::T;
  static constexpr int LPH = D / 8;  // lanes a head
  const NormRopeParams& p;
  int sub, ea, eb;  // lane of the head, first values of the lane's two pieces
  bool turns;
  float cs[4], sn[4];
  float ac[4], bs[4], bc[4], as[4];  // (a, b) -> (a * ac - b * bs, b * bc + a * as)

  __device__ __forceinline__ explicit NormRopeLane(const NormRopeParams& q) : p(q) {
    sub = threadIdx.x % LPH;
    turns = sub < p.R / 8;
    ea = turns ? 4 * sub : p.R + 8 * (sub - p.R / 8);
    eb = turns ? ea + p.R / 2 : ea + 4;
  }
  // The angle is within [-pi, pi], where __sincosf is off by at most 2^-20.9.
  __device__ __forceinline__ void angles(int position) {
    constexpr double kTwoPi = 6.283185307179586476925;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double a = turns ? double(position) * p.inv_freq[4 * sub + i] : 0.0;
      __sincosf(float(a - kTwoPi * rint(a * (1.0 / kTwoPi))), &sn[i], &cs[i]);
    }
  }
  __device__ __forceinline__ void weights(const void* w) {
    float wa[4], wb[4];
    unpack4<Tag>(*reinterpret_cast<const uint2*>(static_cast<const E*>(w) + ea), wa);
    unpack4<Tag>(*reinterpret_cast<const uint2*>(static_cast<const E*>(w) + eb), wb);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ac[i] = wa[i] * cs[i];
      as[i] = wa[i] * sn[i];
      bc[i] = wb[i] * cs[i];
      bs[i] = wb[i] * sn[i];
    }
  }
  __device__ __forceinline__ int64_t page_row(int64_t slot) const {  // cache row of head 0, -1: none
    if (slot < 0) return -1;
    const int64_t page = slot >> 32 ? slot / p.P : int64_t(uint32_t(slot) / uint32_t(p.P));
    return page * p.Hkv * p.P + (slot - page * p.P);
  }
  // One head from the lane's two pieces; every lane of the warp calls it
  // (shuffles).  Norm and rotate (unless `raw`); dst: null where nothing is
  // written; QUANT: append to cache row `row` (-1: none).
  template <bool QUANT>
  __device__ __forceinline__ void head(uint2 xa, uint2 xb, bool raw, E* dst, int64_t row, uint8_t* codes,
                                       float* scales) const {
    uint2 ya = xa, yb = xb;
    float a[4], b[4], ss = 0.f;
    unpack4<Tag>(xa, a);
    unpack4<Tag>(xb, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(fmaf(ss, 1.f / float(D), p.eps));
    float c[4], d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = r * (a[i] * ac[i] - b[i] * bs[i]);
      d[i] = r * (b[i] * bc[i] + a[i] * as[i]);
    }
    if (!raw) {
      ya = pack4<Tag>(c);
      yb = pack4<Tag>(d);
    }
    if (dst) {
      *reinterpret_cast<uint2*>(dst + ea) = ya;
      *reinterpret_cast<uint2*>(dst + eb) = yb;
    }
    if constexpr (QUANT) {
      if (!__any_sync(0xffffffffu, row >= 0)) return;
      // 8 consecutive values a lane: 4-value pieces 2 sub and 2 sub + 1 from the lanes that hold them
      uint2 piece[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int j = 2 * sub + k, q8 = p.R / 8;
        const int from = j < q8 ? j : j < 2 * q8 ? j - q8 : q8 + (j - 2 * q8) / 2;
        const bool second = j < q8 ? false : j < 2 * q8 ? true : (j - 2 * q8) & 1;
        const int src = (threadIdx.x & 31 & ~(LPH - 1)) + from;
        const uint2 va = make_uint2(__shfl_sync(0xffffffffu, ya.x, src), __shfl_sync(0xffffffffu, ya.y, src));
        const uint2 vb = make_uint2(__shfl_sync(0xffffffffu, yb.x, src), __shfl_sync(0xffffffffu, yb.y, src));
        piece[k] = second ? vb : va;
      }
      append_piece<Tag, D>(make_uint4(piece[0].x, piece[0].y, piece[1].x, piece[1].y), sub, row, p.bits, codes, scales);
    }
  }
};

// Few tokens: a CTA on each, the heads side by side (latency).
template <typename Tag, int D, bool APPEND>
__global__ void __launch_bounds__(256) qk_norm_rope_few_kernel(const NormRopeParams p) {
  pdl_enter();
  using E = typename Tag::T;
  constexpr int STEP = 256 / (D / 8);  // heads at a time
  NormRopeLane<Tag, D> lane(p);
  const int t = blockIdx.x, NH = p.Hq + p.Hkv * (APPEND ? 2 : 1);
  const E* row = static_cast<const E*>(p.qkv) + int64_t(t) * p.ld;
  int h = threadIdx.x / (D / 8);
  uint2 xa = make_uint2(0u, 0u), xb = xa;
  auto load = [&](int head) {
    if (head >= NH) return;
    xa = *reinterpret_cast<const uint2*>(row + head * D + lane.ea);
    xb = *reinterpret_cast<const uint2*>(row + head * D + lane.eb);
  };
  load(h);
  lane.angles(p.positions[t]);
  bool for_k = h >= p.Hq;
  lane.weights(for_k ? p.kw : p.qw);
  const int64_t row0 = APPEND ? lane.page_row(p.slots[t]) : -1;
  // every lane takes the same number of turns: the shuffles are warp-wide
  for (int h0 = 0; h0 < NH; h0 += STEP, h += STEP) {
    const uint2 a = xa, b = xb;
    load(h + STEP);
    if (!for_k && h >= p.Hq) {
      lane.weights(p.kw);
      for_k = true;
    }
    const bool is_v = h >= p.Hq + p.Hkv;
    E* dst = h < p.Hq ? static_cast<E*>(p.q_out) + (int64_t(t) * p.Hq + h) * D
                      : static_cast<E*>(p.k_out) + (int64_t(t) * p.Hkv + h - p.Hq) * D;
    const int64_t at = row0 < 0 || h < p.Hq || h >= NH ? -1 : row0 + int64_t(h - p.Hq - (is_v ? p.Hkv : 0)) * p.P;
    lane.template head<APPEND>(a, b, is_v, is_v || h >= NH ? nullptr : dst, at, is_v ? p.v_codes : p.k_codes,
                                     is_v ? p.v_scales : p.k_scales);
  }
}

// Many tokens: a warp takes runs of up to 4 KB of a token's q, k or v heads
// from a ring of its own that bulk copies keep filled, so memory has work
// while the warp computes (loads to registers: 4.4 TB/s at 32768 tokens of 40
// heads).  Each warp has the same number of consecutive runs, and forms the
// angles once for those of one token.
// Rows that are appended take more instructions a byte (the quantizer), so
// more warps with less in flight each: 4 CTAs an SM with 3 runs a warp against
// 5 with 2 took 29.4 / 27.5 us for 5003 tokens of 36 heads of 128, 93.1 / 89.5
// for 20000; not appended, 4 x 3 against 6 x 2 took 67.9 / 72.7 us for 20000.
// 32768 tokens of 40 heads (671 MB) take 115 us, 5.8 TB/s.
constexpr int NR_WARPS = 4, NR_CHUNK = 4096;
constexpr int nr_stages(bool append) { return append ? 2 : 3; }
constexpr int nr_ctas(bool append) { return append ? 5 : 4; }

template <typename Tag, int D, bool APPEND>
__global__ void __launch_bounds__(32 * NR_WARPS, nr_ctas(APPEND)) qk_norm_rope_stream_kernel(const NormRopeParams p) {
  pdl_enter();
  using E = typename Tag::T;
  constexpr int NR_STAGES = nr_stages(APPEND);
  constexpr int CH = NR_CHUNK / (2 * D), PER = 32 / (D / 8);  // heads of a run, of a warp's turn
  extern __shared__ __align__(128) uint8_t nr_smem[];
  __shared__ uint64_t full[NR_WARPS][NR_STAGES];
  const int warp = threadIdx.x >> 5, l = threadIdx.x & 31;
  uint8_t* ring = nr_smem + warp * NR_STAGES * NR_CHUNK;
  if (l == 0) {
    for (int s = 0; s < NR_STAGES; ++s) mbar_init(&full[warp][s], 1);
    fence_mbarrier_init();
  }
  __syncwarp();
  // runs of a token: nq of q heads, nk of k heads, as many of v heads
  const int nq = (p.Hq + CH - 1) / CH, nk = (p.Hkv + CH - 1) / CH, NC = nq + nk * (APPEND ? 2 : 1);
  const int64_t runs = int64_t(p.T) * NC;
  const int warps = gridDim.x * NR_WARPS, w = blockIdx.x * NR_WARPS + warp;
  const int64_t begin = runs * w / warps;
  const int count = int(runs * (w + 1) / warps - begin);
  struct Run {
    int t, c;  // token, run of the token
  };
  // first head of the run in the row, number of heads
  auto heads = [&](int c, int& n) {
    const int base = c < nq ? 0 : c < nq + nk ? p.Hq : p.Hq + p.Hkv;
    const int k = (c < nq ? c : c < nq + nk ? c - nq : c - nq - nk) * CH;
    n = min(CH, (c < nq ? p.Hq : p.Hkv) - k);
    return base + k;
  };
  auto advance = [&](Run& r) {
    if (++r.c == NC) r.c = 0, ++r.t;
  };
  const bool stall = producers_stalled();  // test control: nothing is issued
  Run ahead{int(begin / NC), int(begin % NC)}, now = ahead;
  int issued = 0;
  auto issue = [&]() {
    if (issued >= count) return;
    if (l == 0 && !stall) {
      int n;
      const int s = issued % NR_STAGES, h = heads(ahead.c, n);
      const uint32_t bytes = uint32_t(n) * D * 2;
      mbar_arrive_expect_tx(&full[warp][s], bytes);
      bulk_g2s(ring + s * NR_CHUNK, static_cast<const E*>(p.qkv) + ahead.t * p.ld + h * D, bytes, &full[warp][s]);
    }
    ++issued;
    advance(ahead);
  };
  for (int s = 0; s < NR_STAGES; ++s) issue();
  NormRopeLane<Tag, D> lane(p);
  int pos = 0;
  int64_t slot = -1, row0 = -1;
  auto look = [&](int t) {
    if (t >= p.T) return;
    pos = p.positions[t];
    if constexpr (APPEND) slot = p.slots[t];
  };
  look(now.t);
  bool ok = true;
  int n = 0;
  for (; n < count; ++n) {
    const int c = now.c, t = now.t;
    if (n == 0 || c == 0) {
      lane.angles(pos);
      if constexpr (APPEND) row0 = lane.page_row(slot);
      look(t + 1);  // a token ahead
    }
    if (n == 0 || c == 0 || c == nq) lane.weights(c < nq ? p.qw : p.kw);
    const int s = n % NR_STAGES;
    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[warp][s], uint32_t((n / NR_STAGES) & 1)));
    if (!ok) break;
    int hn;
    const int h0 = heads(c, hn), hl = l / (D / 8);
    const uint8_t* src = ring + s * NR_CHUNK + hl * D * 2;
    const bool is_q = c < nq, is_v = APPEND && c >= nq + nk;
    const int kh = h0 - (is_q ? 0 : is_v ? p.Hq + p.Hkv : p.Hq) + hl;  // this lane's first head of its kind
    E* dst = (is_q ? static_cast<E*>(p.q_out) + (int64_t(t) * p.Hq + kh) * D
                   : static_cast<E*>(p.k_out) + (int64_t(t) * p.Hkv + kh) * D);
    int64_t row = row0 + int64_t(kh) * p.P;
    for (int i = hl; i - hl < hn; i += PER) {
      const bool on = i < hn;  // a piece past the run is read from the ring, and dropped
      const uint2 xa = *reinterpret_cast<const uint2*>(src + lane.ea * 2), xb = *reinterpret_cast<const uint2*>(src + lane.eb * 2);
      const int64_t at = on && row0 >= 0 ? row : -1;
      if (is_q) lane.template head<false>(xa, xb, false, on ? dst : nullptr, -1, nullptr, nullptr);
      else if (!is_v) lane.template head<APPEND>(xa, xb, false, on ? dst : nullptr, at, p.k_codes, p.k_scales);
      else if constexpr (APPEND)
        append_piece<Tag, D>(*reinterpret_cast<const uint4*>(src + lane.sub * 16), lane.sub, at, p.bits, p.v_codes, p.v_scales);
      src += PER * D * 2;
      dst += PER * D;
      row += int64_t(PER) * p.P;
    }
    advance(now);
    __syncwarp();  // the run has been read
    issue();
  }
  if (!ok) {
    // copies already issued land before the CTA goes away
    for (int k = n; k < issued && !stall; ++k)
      mbar_wait_bounded(&full[warp][k % NR_STAGES], uint32_t((k / NR_STAGES) & 1), 100000000ull);
    if (l == 0) report_timeout(nullptr);
  }
}

template <typename Tag, int D, bool APPEND>
static int launch_norm_rope(const NormRopeParams& p, cudaStream_t st) {
  // A CTA a token up to 4 per SM, 2 where rows are appended.  Measured for 36
  // heads of 128, a CTA a token against streamed: 3.4 / 4.9 us at 7 tokens,
  // 5.6 / 6.5 at 592, 9.4 / 9.1 at 1184; appended, 5.4 / 6.3 us at 296, 9.0 / 7.4 at 592.
  if (p.T <= (APPEND ? 2 : 4) * 148)
    return launch_kernel(qk_norm_rope_few_kernel<Tag, D, APPEND>, dim3{unsigned(p.T)}, dim3{256}, 0, st, p);
  constexpr auto kern = qk_norm_rope_stream_kernel<Tag, D, APPEND>;
  constexpr int smem = NR_WARPS * nr_stages(APPEND) * NR_CHUNK;
  const int set = allow_smem<kern>(smem);
  if (set != B2F_OK) return set;
  const int want = p.T, most = nr_ctas(APPEND) * 148;
  return launch_kernel(kern, dim3{unsigned(want < most ? want : most)}, dim3{32 * NR_WARPS}, smem, st, p);
}

template <typename Tag, int D>
static int launch_norm_rope_a(const NormRopeParams& p, cudaStream_t st) {
  return p.slots ? launch_norm_rope<Tag, D, true>(p, st) : launch_norm_rope<Tag, D, false>(p, st);
}

template <typename Tag>
static int launch_norm_rope_d(const NormRopeParams& p, int64_t D, cudaStream_t st) {
  if (D == 64) return launch_norm_rope_a<Tag, 64>(p, st);
  if (D == 128) return launch_norm_rope_a<Tag, 128>(p, st);
  return launch_norm_rope_a<Tag, 256>(p, st);
}

B2F_DEFINE_WAIT_CONTROLS(prompt_ops)

}  // namespace b2f

using namespace b2f;

extern "C" {

int64_t b2f_page_plan_workspace_bytes(int64_t B) { return B > kScanRows ? (B + 1) * int64_t(sizeof(int32_t)) : 0; }

int b2f_page_plan(const int32_t* new_lens, const int32_t* context_lens, int64_t B, const int32_t* free_pages,
                  int64_t n_free, int64_t page_size, int32_t* block_table, int64_t max_pages, int64_t T,
                  int32_t* cu_seqlens, int32_t* positions, int64_t* slots, int32_t* rows, int32_t* seq_lens,
                  int32_t* counts, void* workspace, int64_t workspace_bytes, void* stream) {
  constexpr int64_t kMax = int64_t(1) << 30;
  if (B < 0 || n_free < 0 || page_size <= 0 || max_pages <= 0 || T < 0) return B2F_ERR_INVALID;
  if (B > (1 << 20) || n_free > kMax || page_size > kMax || max_pages > kMax || T > kMax) return B2F_ERR_UNSUPPORTED;
  if (!cu_seqlens || !counts || (B > 0 && (!new_lens || !block_table || !seq_lens)) ||
      (T > 0 && (!positions || !slots || !rows)) || (n_free > 0 && !free_pages))
    return B2F_ERR_INVALID;
  if (!aligned(positions, 16) || !aligned(slots, 16) || !aligned(rows, 16)) return B2F_ERR_ALIGN;
  PagePlanParams p{new_lens, context_lens, free_pages, block_table, cu_seqlens, positions, slots, rows, seq_lens,
                   counts, static_cast<int32_t*>(workspace), int(B), int(T), int(n_free), int(max_pages),
                   int(page_size)};
  cudaStream_t st = as_stream(stream);
  const int64_t work = (T + 3) / 4 > B + 1 ? (T + 3) / 4 : B + 1;
  const int64_t want = (work + kPlanThreads - 1) / kPlanThreads;
  const unsigned grid = unsigned(want < 148 * 4 ? want : 148 * 4);
  if (B <= kScanRows)
    return launch_kernel(page_plan_fill_kernel<true>, dim3{grid}, dim3{kPlanThreads}, size_t(B + 1) * 8, st, p);
  if (!workspace || workspace_bytes < b2f_page_plan_workspace_bytes(B)) return B2F_ERR_WORKSPACE;
  const int rc = launch_kernel(page_plan_scan_kernel, dim3{1}, dim3{1024}, 0, st, p);
  if (rc != B2F_OK) return rc;
  return launch_kernel(page_plan_fill_kernel<false>, dim3{grid}, dim3{kPlanThreads}, 0, st, p);
}

int b2f_qk_norm_rope_rows(const void* qkv, int64_t ld, int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                          const void* q_norm, const void* k_norm, float eps, const double* inv_freq,
                          int64_t rotary_dim, const int32_t* positions, void* q_out, void* k_out,
                          const int64_t* slots, uint8_t* k_codes, float* k_scales, uint8_t* v_codes,
                          float* v_scales, int64_t page_size, int bits, void* stream) {
  if (dtype != B2F_BF16 && dtype != B2F_F16) return B2F_ERR_UNSUPPORTED;
  if (!(D == 64 || D == 128 || D == 256)) return B2F_ERR_UNSUPPORTED;
  if (T < 0 || Hq <= 0 || Hkv <= 0 || ld < (Hq + 2 * Hkv) * D) return B2F_ERR_INVALID;
  if (rotary_dim < 0 || rotary_dim > D || rotary_dim % 16 != 0) return B2F_ERR_INVALID;
  if (T > (int64_t(1) << 30) || Hq > 65535 || Hkv > 65535) return B2F_ERR_UNSUPPORTED;
  if (slots) {
    if (!(bits == 2 || bits == 4 || bits == 8)) return B2F_ERR_UNSUPPORTED;
    if (page_size <= 0 || page_size > (1 << 30) || !k_codes || !k_scales || !v_codes || !v_scales)
      return B2F_ERR_INVALID;
    if (!aligned(k_codes, 16) || !aligned(v_codes, 16) || !aligned(k_scales, 4) || !aligned(v_scales, 4) ||
        !aligned(slots, 8))
      return B2F_ERR_ALIGN;
  }
  if (T == 0) return B2F_OK;
  if (!qkv || !q_norm || !k_norm || (rotary_dim > 0 && !inv_freq) || !positions || !q_out || !k_out)
    return B2F_ERR_INVALID;
  if (!aligned(qkv, 16) || ld % 8 != 0 || !aligned(q_norm, 16) || !aligned(k_norm, 16) || !aligned(q_out, 16) ||
      !aligned(k_out, 16) || !aligned(inv_freq, 8) || !aligned(positions, 4))
    return B2F_ERR_ALIGN;
  NormRopeParams p{qkv, ld, q_norm, k_norm, inv_freq, positions, q_out, k_out, slots, k_codes, k_scales, v_codes,
                   v_scales, eps, int(T), int(Hq), int(Hkv), int(page_size), int(rotary_dim), bits};
  cudaStream_t st = as_stream(stream);
  return dtype == B2F_BF16 ? launch_norm_rope_d<TagBF16>(p, D, st) : launch_norm_rope_d<TagF16>(p, D, st);
}

}  // extern "C"
