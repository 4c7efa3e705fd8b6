// Device helpers of the tcgen05 attention kernels (prompt_attn.cu,
// prefix_attn.cu): TMEM row loads and stores, the MMA with its A operand in
// TMEM, the MN-major descriptor of a value tile, higher-rank TMA loads, the
// online softmax of one score row per thread.
#pragma once
#include "tc_common.cuh"

namespace b2f {

constexpr float kLog2e = 1.4426950408889634f;

// ex2.approx.ftz: 2^x (-inf gives +0)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
          "r"(smem_u32(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}

// a box of shared memory into the tensor (part of this thread's bulk group)
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, const void* src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(map), "r"(c0),
               "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(src))
               : "memory");
}

// The warp that issues MMAs runs converged and one elected lane issues: the
// descriptors are then formed in uniform registers, which the instruction
// takes.  From a branch that one lane enters alone an MMA took 82 to 140
// cycles to issue, against 64 to execute.
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t is;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(is));
  return is;
}
// D[tmem] (+)= A[smem] . B[smem], by the elected lane
__device__ __forceinline__ void tc_mma_ss(uint32_t elected, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}
// D[tmem] (+)= A[tmem] . B[smem], by the elected lane
__device__ __forceinline__ void tc_mma_ts(uint32_t elected, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void tc_commit_by(uint32_t elected, uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)),
      "r"(elected)
      : "memory");
}

// MN-major, 128B-swizzled descriptor of a [K rows][64 values] tile: the 64
// values of a row are one 128-byte line, 8 rows an atom of 1024 bytes (the
// stride along K), the next 64 values `next_bytes` further on.
__device__ __forceinline__ uint64_t sw128_mn_desc(const void* tile, uint32_t next_bytes) {
  const uint64_t start = (smem_u32(tile) >> 4) & 0x3FFFu;
  return start | (uint64_t(next_bytes >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// kind::f16 instruction descriptor: fp32 accumulate, M = 128
__host__ __device__ constexpr uint32_t mma_idesc(int n, bool bf16, bool b_mn_major, bool negate_a) {
  return (1u << 4) | (uint32_t(bf16) << 7) | (uint32_t(bf16) << 10) | (uint32_t(negate_a) << 13) |
         (uint32_t(b_mn_major) << 16) | (uint32_t(n >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One thread's row of a TMEM tile: n consecutive columns of its lane (the
// loads have landed on return; the stores after tmem_wait_st).
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&v)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31]),
        "=r"(v[32]), "=r"(v[33]), "=r"(v[34]), "=r"(v[35]), "=r"(v[36]), "=r"(v[37]), "=r"(v[38]), "=r"(v[39]),
        "=r"(v[40]), "=r"(v[41]), "=r"(v[42]), "=r"(v[43]), "=r"(v[44]), "=r"(v[45]), "=r"(v[46]), "=r"(v[47]),
        "=r"(v[48]), "=r"(v[49]), "=r"(v[50]), "=r"(v[51]), "=r"(v[52]), "=r"(v[53]), "=r"(v[54]), "=r"(v[55]),
        "=r"(v[56]), "=r"(v[57]), "=r"(v[58]), "=r"(v[59]), "=r"(v[60]), "=r"(v[61]), "=r"(v[62]), "=r"(v[63])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
      :
      : "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
      :
      : "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
        "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
        "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
      : "memory");
}

// 1-D bulk copy from shared to global memory, and the wait for this thread's
// copies to have read their source.  16-byte aligned, size % 16 == 0.
__device__ __forceinline__ void bulk_s2g(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_s2g_wait() {
  asm volatile("cp.async.bulk.commit_group;\n cp.async.bulk.wait_group.read 0;" ::: "memory");
}

// OR of a predicate over the `n` threads of named barrier `id`
__device__ __forceinline__ bool bar_or(int id, int n, bool v) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n bar.red.or.pred q, %2, %3, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"(uint32_t(v)), "r"(id), "r"(n)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void bar_all(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }

// ---- a running CTA takes over one that has not been launched -----------------
// The answer (16 bytes in shared memory) lands on `bar`.
__device__ __forceinline__ void next_cta_ask(void* answer, uint64_t* bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
          smem_u32(answer)),
      "r"(smem_u32(bar))
      : "memory");
}
// its blockIdx.x, or -1 when none is left
__device__ __forceinline__ int next_cta_answer(const void* answer) {
  uint32_t ok, x;
  asm volatile(
      "{\n .reg .b128 a;\n .reg .pred p;\n ld.shared.b128 a, [%2];\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n selp.u32 %0, 1, 0, p;\n mov.u32 %1, 0;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, _, _, _}, a;\n}\n"
      : "=r"(ok), "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  return ok ? int(x) : -1;
}

// ---- softmax of one score row per thread ------------------------------------
// Two floats in a 64-bit register: the packed FMA, add and multiply issue once
// for both.
__device__ __forceinline__ uint64_t f32x2(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ uint64_t f32x2_bits(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ float2 f32x2_parts(uint64_t v) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
  return d;
}
__device__ __forceinline__ uint64_t fma_x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// maxima that keep NaN
__device__ __forceinline__ float max2(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <int N>
__device__ __forceinline__ float row_max(const uint32_t (&s)[N]) {
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < N; c += 2)
    m[(c >> 1) & 3] = max3(m[(c >> 1) & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
  return max2(max3(m[0], m[1], m[2]), m[3]);
}

// 2^x for a pair on the FMA pipe, for -126 <= x < 128: with n the nearest
// integer, 2^x = 2^n p(x - n), p a polynomial fitted to the least relative
// error on [-1/2, 1/2] (degree 3: 2^-13.7, for bf16 results; degree 4: 2^-18.5,
// for fp16), n added to the exponent bits.  Below -126 the sum falls among the
// subnormals: less than 2^-126, and from just above -127 down below 2^-138,
// which either type rounds to 0 (a value of 2^127 behind it counts for nothing).
// There x is held just above -127, where p is just above 1: at 1 or below, the
// sum would borrow from the sign.  NaN gives the same: a row with one has a
// reference that is NaN, and its other exponentials are NaN.
template <bool BF16>
__device__ __forceinline__ uint64_t exp2_poly_x2(uint64_t x2) {
  const float2 x = f32x2_parts(x2);
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23: the sum's low bits are the nearest integer
  constexpr float kLeast = -126.9998f;  // p is 1.00006 (degree 3), 1.00014 (degree 4) there
  const uint64_t v = f32x2(fmaxf(x.x, kLeast), fmaxf(x.y, kLeast));
  const uint64_t t = add_x2(v, f32x2(kRound, kRound));
  const uint64_t n = add_x2(t, f32x2(-kRound, -kRound));
  const uint64_t r = fma_x2(n, f32x2(-1.f, -1.f), v);
  uint64_t p;
  if constexpr (BF16) {
    p = fma_x2(r, f32x2(0.055171669f, 0.055171669f), f32x2(0.242611122f, 0.242611122f));
    p = fma_x2(p, r, f32x2(0.693260985f, 0.693260985f));
    p = fma_x2(p, r, f32x2(0.999928074f, 0.999928074f));
  } else {
    p = fma_x2(r, f32x2(0.00957010191f, 0.00957010191f), f32x2(0.0559178603f, 0.0559178603f));
    p = fma_x2(p, r, f32x2(0.240247448f, 0.240247448f));
    p = fma_x2(p, r, f32x2(0.693121815f, 0.693121815f));
    p = fma_x2(p, r, f32x2(0.999999261f, 0.999999261f));
  }
  const float2 pf = f32x2_parts(p), tf = f32x2_parts(t);
  return f32x2_bits(__float_as_uint(pf.x) + (__float_as_uint(tf.x) << 23),
                    __float_as_uint(pf.y) + (__float_as_uint(tf.y) << 23));
}

// P = 2^(s * scale - ref) of N scores as packed 16-bit pairs, their sum added
// to sum[0..1] (pairs).  With POLY, one pair of four goes to the FMA pipe: the
// 16 exponentials a cycle of the SM are what bounds a head of 128 otherwise
// (2 * 128 * 128 of them per 2048 cycles of tensor work).
template <bool BF16, bool POLY, int N>
__device__ __forceinline__ void exp_row(const uint32_t (&s)[N], float scale, float ref, uint64_t (&sum)[2],
                                        uint32_t (&out)[N / 2]) {
  const uint64_t k = f32x2(scale, scale), b = f32x2(-ref, -ref);
#pragma unroll
  for (int c = 0; c < N / 2; ++c) {
    const uint64_t x = fma_x2(f32x2_bits(s[2 * c], s[2 * c + 1]), k, b);
    uint64_t p;
    if (POLY && (c & 3) == 3) {
      p = exp2_poly_x2<BF16>(x);
    } else {
      const float2 v = f32x2_parts(x);
      p = f32x2(ex2(v.x), ex2(v.y));
    }
    sum[c & 1] = add_x2(sum[c & 1], p);
    const float2 e = f32x2_parts(p);
    out[c] = BF16 ? pack_bf16x2(e.x, e.y) : pack_f16x2(e.x, e.y);
  }
}

}  // namespace b2f
