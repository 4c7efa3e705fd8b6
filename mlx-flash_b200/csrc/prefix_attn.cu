// Decode attention of rows that share prefixes held once in the paged cache.
#include "common.cuh"

namespace b2f {

// One warp per query row and head; 32 keys at a time: lane j scores key j,
// the online softmax (running maximum m and sum l, base 2) runs across the
// lanes, and each key's value row is added with the lanes over D.
template <int D, typename Rows>
__device__ void attend_row(const float* q, int n, const Rows& rows, float scale2, float (&acc)[D / 32], float& m,
                           float& l) {
  const int lane = threadIdx.x & 31;
  for (int j0 = 0; j0 < n; j0 += 32) {
    const int j = j0 + lane;
    float s = -INFINITY;
    if (j < n) s = rows.dot(j, q) * scale2;
    const float mt = fmaxf(m, warp_max<32>(s));
    const float ref = mt == -INFINITY ? 0.f : mt;
    const float f = exp2f(m - ref), pj = exp2f(s - ref);
    l = l * f + warp_sum<32>(pj);
    m = mt;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] *= f;
    for (int k = 0; k < min(32, n - j0); ++k) {
      const float pk = __shfl_sync(0xffffffffu, pj, k);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] += pk * rows.value(j0 + k, lane + 32 * i);
    }
  }
}

struct PrefixParams {
  const __nv_bfloat16* q;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int32_t *ptable, *plens, *off, *table, *lens;
  __nv_bfloat16* out;
  int64_t pwidth, width;
  float scale2;
  int B, Ng, Hq, Hkv, D, P, bits;
};

struct PagedRows {
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int32_t* pages;
  int hk, Hkv, P, D, bits;
  __device__ int64_t row(int j) const { return (int64_t(pages[j / P]) * Hkv + hk) * P + j % P; }
  __device__ float at(const uint8_t* c, const float* s, int64_t r, int d) const {
    const int per = 8 / bits, top = (1 << (bits - 1)) - 1;
    const int code = (c[r * (D / per) + d / per] >> (bits * (per - 1 - d % per))) & ((1 << bits) - 1);
    return float(code - top) * s[r * (D / 64) + d / 64];
  }
  __device__ float dot(int j, const float* q) const {
    const int64_t r = row(j);
    float s = 0.f;
    for (int d = 0; d < D; ++d) s = fmaf(q[d], at(kc, ks, r, d), s);
    return s;
  }
  __device__ float value(int j, int d) const { return d < D ? at(vc, vs, row(j), d) : 0.f; }
};

__global__ void __launch_bounds__(128) prefix_attn_simple_kernel(const PrefixParams p) {
  pdl_enter();
  __shared__ float qs[4][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x, h = blockIdx.y * 4 + warp;
  if (h >= p.Hq) return;
  for (int d = lane; d < p.D; d += 32) qs[warp][d] = __bfloat162float(p.q[(int64_t(b) * p.Hq + h) * p.D + d]);
  __syncwarp();
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  PagedRows rows{p.kc, p.vc, p.ks, p.vs, nullptr, h / (p.Hq / p.Hkv), p.Hkv, p.P, p.D, p.bits};
  for (int g = 0; g < p.Ng; ++g)
    if (b >= p.off[g] && b < p.off[g + 1]) {
      rows.pages = p.ptable + g * p.pwidth;
      attend_row<128>(qs[warp], p.plens[g], rows, p.scale2, acc, m, l);
    }
  rows.pages = p.table + b * p.width;
  attend_row<128>(qs[warp], p.lens[b], rows, p.scale2, acc, m, l);
  const float inv = l > 0.f ? 1.f / l : l;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < p.D) p.out[(int64_t(b) * p.Hq + h) * p.D + lane + 32 * i] = __float2bfloat16_rn(acc[i] * inv);
}

}  // namespace b2f

using namespace b2f;

extern "C" {

int64_t b2f_shared_prefix_attn_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t n_groups,
                                               int64_t max_prefix, int64_t max_own) {
  return 0;
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
  if (Hq / Hkv > 16 || B > 65535 || Hkv > 65535) return B2F_ERR_UNSUPPORTED;
  if (page_size <= 0 || page_size % 16 != 0 || prefix_pages <= 0 || max_pages <= 0) return B2F_ERR_INVALID;
  if (B == 0) return B2F_OK;
  if (!q || !k_pages || !k_scales || !v_pages || !v_scales || !block_table || !seq_lens || !out ||
      (n_groups > 0 && (!prefix_table || !prefix_lens || !group_offsets)))
    return B2F_ERR_INVALID;
  if (!aligned(q, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(k_scales, 8) ||
      !aligned(v_scales, 8) || !aligned(out, 16))
    return B2F_ERR_ALIGN;
  PrefixParams p{static_cast<const __nv_bfloat16*>(q), k_pages, v_pages, k_scales, v_scales, prefix_table, prefix_lens,
                 group_offsets, block_table, seq_lens, static_cast<__nv_bfloat16*>(out), prefix_pages, max_pages,
                 softmax_scale * 1.4426950408889634f, int(B), int(n_groups), int(Hq), int(Hkv), int(D),
                 int(page_size), bits};
  return launch_kernel(prefix_attn_simple_kernel, dim3{unsigned(B), unsigned((Hq + 3) / 4)}, dim3{128}, 0,
                       as_stream(stream), p);
}

}  // extern "C"
