// What a batch of packed prompts needs before attention: the page plan (block
// tables, slot map, positions) from the requests' lengths, and the per-head
// RMSNorm + rotary position of queries and keys, with the quantized rows
// appended to the planned slots in the same pass.
#include "common.cuh"

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
// global memory for the fill.
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
// D / 8 lanes hold one head, 8 consecutive values each (16-byte loads and
// stores); a rotary pair sits R/16 lanes apart.  Everything is float32 with
// one rounding at the end; the angle is formed and reduced in double, because
// pos * inv_freq in float32 is off by 2^-25 * pos (0.004 rad at 131072).
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

template <typename Tag, int D, bool APPEND>
__global__ void __launch_bounds__(256) qk_norm_rope_rows_kernel(const NormRopeParams p) {
  pdl_enter();
  using E = typename Tag::T;
  constexpr int LPH = D / 8;  // lanes per head
  __shared__ float cs[D / 2], sn[D / 2];
  const int t = blockIdx.x;
  const int half = p.R / 2;
  if (int(threadIdx.x) < half) {
    constexpr double kTwoPi = 6.283185307179586476925;
    const double a = double(p.positions[t]) * p.inv_freq[threadIdx.x];
    sincosf(float(a - kTwoPi * rint(a / kTwoPi)), &sn[threadIdx.x], &cs[threadIdx.x]);
  }
  __syncthreads();
  const int sub = threadIdx.x % LPH;  // this lane's 8 values of the head
  const E* row = static_cast<const E*>(p.qkv) + int64_t(t) * p.ld;
  const int NH = p.Hq + p.Hkv * (APPEND ? 2 : 1);
  const int pair = half / 8;  // lanes between the halves of a rotary pair
  const int lane = threadIdx.x & 31;
  const int partner = sub < pair ? lane + pair : sub < 2 * pair ? lane - pair : lane;
  int64_t slot = -1;
  if constexpr (APPEND) slot = p.slots[t];
  // every lane takes the same number of turns: the shuffles below are warp-wide
  const int per = blockDim.x / LPH;
  for (int h0 = 0; h0 < NH; h0 += per) {
    const int h = h0 + threadIdx.x / LPH;
    const bool on = h < NH;
    float v[8];
    {
      const uint4 w = on ? *reinterpret_cast<const uint4*>(row + int64_t(h) * D + sub * 8) : make_uint4(0, 0, 0, 0);
      const E* e = reinterpret_cast<const E*>(&w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = Tag::to_f(e[i]);
    }
    const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.Hkv;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += v[i] * v[i];
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!is_v) {
      const float r = rsqrtf(ss / float(D) + p.eps);
      const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const E*>(is_q ? p.qw : p.kw) + sub * 8);
      const E* e = reinterpret_cast<const E*>(&w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= r * Tag::to_f(e[i]);
    }
    float u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = __shfl_sync(0xffffffffu, v[i], partner);
    if (!is_v && sub < 2 * pair) {
      const int f = (sub < pair ? sub : sub - pair) * 8;
      const float sign = sub < pair ? -1.f : 1.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] * cs[f + i] + sign * u[i] * sn[f + i];
    }
    E o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = Tag::from_f(v[i]);
    if (on && !is_v) {
      E* dst = is_q ? static_cast<E*>(p.q_out) + (int64_t(t) * p.Hq + h) * D
                    : static_cast<E*>(p.k_out) + (int64_t(t) * p.Hkv + h - p.Hq) * D;
      *reinterpret_cast<uint4*>(dst + sub * 8) = *reinterpret_cast<const uint4*>(o);
    }
    if constexpr (APPEND) {
      const float mi = p.bits == 8 ? 127.f : p.bits == 4 ? 7.f : 1.f;
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = Tag::to_f(o[i]);
        m = fmaxf(m, fabsf(v[i]));
      }
#pragma unroll
      for (int k = 1; k < 8; k <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
      if (!on || is_q || slot < 0) continue;
      float scale = Tag::round(__fdiv_rn(m, mi));
      if (scale == 0.f) scale = 1.f;
      uint32_t c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = Tag::round(rintf(Tag::round(__fdiv_rn(v[i], scale))));
        c[i] = uint32_t(int(Tag::round(fminf(fmaxf(x, -mi), mi) + mi)));
      }
      const int kvh = (h - p.Hq) % p.Hkv;
      const int64_t page = slot / p.P;
      const int64_t r = (page * p.Hkv + kvh) * p.P + (slot - page * p.P);
      if (sub % 8 == 0) (is_v ? p.v_scales : p.k_scales)[r * (D / 64) + sub / 8] = scale;
      uint8_t* dst = (is_v ? p.v_codes : p.k_codes) + r * (D * p.bits / 8) + sub * p.bits;
      if (p.bits == 8) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24,
                                                    c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24);
      } else if (p.bits == 4) {
        *reinterpret_cast<uint32_t*>(dst) = (c[0] << 4 | c[1]) | (c[2] << 4 | c[3]) << 8 |
                                            (c[4] << 4 | c[5]) << 16 | (c[6] << 4 | c[7]) << 24;
      } else {
        *reinterpret_cast<uint16_t*>(dst) = uint16_t((c[0] << 6 | c[1] << 4 | c[2] << 2 | c[3]) |
                                                     (c[4] << 6 | c[5] << 4 | c[6] << 2 | c[7]) << 8);
      }
    }
  }
}

template <typename Tag, int D>
static int launch_norm_rope(const NormRopeParams& p, cudaStream_t st) {
  auto kern = p.slots ? qk_norm_rope_rows_kernel<Tag, D, true> : qk_norm_rope_rows_kernel<Tag, D, false>;
  return launch_kernel(kern, dim3{unsigned(p.T)}, dim3{256}, 0, st, p);
}

template <typename Tag>
static int launch_norm_rope_d(const NormRopeParams& p, int64_t D, cudaStream_t st) {
  if (D == 64) return launch_norm_rope<Tag, 64>(p, st);
  if (D == 128) return launch_norm_rope<Tag, 128>(p, st);
  return launch_norm_rope<Tag, 256>(p, st);
}

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
