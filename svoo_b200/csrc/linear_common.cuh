// Shared by the kernels of the 8-bit matrix product (linear_tc.cu, linear_split.cu).
#pragma once

#include "quant_common.cuh"
#include "tc_common.cuh"

namespace svoo {
namespace tc {


struct LinearArgs {
  const float *sa, *sb;
  int64_t sa_pitch, sb_n, sb_k;                 // sa[kb * sa_pitch + m]; sb[(n / 128) * sb_n + kb * sb_k], kRowScales: sb[kb * sb_k + n]
  const void* bias;
  int bias_type;
  void* out;
  int64_t out_pitch;                            // elements
  float* out_scale;                             // e4m3 output: [n / 128][m]
  int64_t out_scale_pitch;
  int M, N, K;
  int* status;                                  // the device's word: != 0 after a kernel gave up on a bounded wait
  bool box_out;                                 // rows of out are whole 16-byte pieces, each on 16 bytes: they leave by TMA
};

// D[tmem] (+)= A[smem] B[smem]^T, e4m3
template <int CTAS>
__device__ __forceinline__ void umma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrives at the barrier, in both CTAs of the pair, when the issued MMAs have completed.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// TMA load into this CTA's shared memory that signals a barrier of the pair's first CTA.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t first_bar) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(first_bar) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ uint32_t at_cta(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// Instruction descriptor of kind::f8f6f4: D fp32, A and B e4m3, both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// 16 columns of this thread's row: issue, and wait for all that were issued.  The wait takes the registers as operands, so that
// no use of theirs can be moved before it (the kernel must not spill: a register could be saved before it is filled).
__device__ __forceinline__ void wait_columns(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) :: "memory");
}
// acc += {r0, r1} * f
__device__ __forceinline__ void scale_add2(uint64_t& acc, uint32_t r0, uint32_t r1, uint64_t f) {
  asm("{\n\t.reg .b64 a;\n\tmov.b64 a, {%1, %2};\n\tfma.rn.f32x2 %0, a, %3, %0;\n\t}\n" : "+l"(acc) : "r"(r0), "r"(r1), "l"(f));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float half_of(uint64_t v, int i) { return __uint_as_float((uint32_t)(i ? v >> 32 : v)); }

__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// GELU of two values: y / 2 (1 + tanh u) = y / (1 + exp(-2 u)), u = sqrt(2 / pi) (y + 0.044715 y^3).  The special-function unit is
// what it costs most on: the two share a reciprocal (1 / d0 = d1 / (d0 d1)); exponents are cut at 60, so that the product stays
// finite.  Behind the cut, y < -7.47, GELU is below 2^-57: zero here, however large y is (the formula's NaN for minus infinity).
__device__ __forceinline__ uint64_t gelu2(uint64_t y) {
  constexpr float k = -2.f * 0.7978845608028654f * 1.4426950408889634f;
  // constants in scalar operations: a pair of each would take registers that the epilogue does not have
  const uint64_t z = mul2(y, y);
  const uint64_t a = mul2(y, pack2(fmaf(half_of(z, 0), 0.044715f * k, k), fmaf(half_of(z, 1), 0.044715f * k, k)));
  const float d[2] = {1.f + fast_exp2(fminf(half_of(a, 0), 60.f)), 1.f + fast_exp2(fminf(half_of(a, 1), 60.f))};
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d[0] * d[1]));
  return mul2(y, mul2(pack2(d[1], d[0]), pack2(half_of(a, 0) > 60.f ? 0.f : r, half_of(a, 1) > 60.f ? 0.f : r)));
}
// the largest of three magnitudes; NaN if one is
__device__ __forceinline__ float max_magnitude(float top, uint64_t v) {
  asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(fabsf(half_of(v, 0))), "f"(fabsf(half_of(v, 1))));
  return top;
}
// x / s of values that are themselves rounded sums: one correction by the remainder, which leaves half a unit and 2^-22 of
// one (BlockDivide makes it half a unit).  s >= 2^-90, as BlockDivide wants it; the scale as block_scale gives it.
struct BlockDivideOnce {
  float y, ns;
  __device__ __forceinline__ explicit BlockDivideOnce(float s) : y(BlockDivide::reciprocal(s)), ns(s == INFINITY ? -1.f : -s) {}
  __device__ __forceinline__ float quotient(float x) const {
    const float q = x * y;
    return fmaf(fmaf(q, ns, x), y, q);
  }
  __device__ __forceinline__ uint32_t e4m3x4(uint64_t a, uint64_t b) const {
    return e4m3x2(quotient(half_of(a, 0)), quotient(half_of(a, 1))) | e4m3x2(quotient(half_of(b, 0)), quotient(half_of(b, 1))) << 16;
  }
};

// bias of columns n, n + step, ..., zero where there is none; the loads go out together.  Plain loads: the 16-bit forms of __ldg are
// assembly that the compiler may move in front of the condition on a.bias.
template <typename T, int COUNT>
__device__ __forceinline__ void bias_columns_of(const LinearArgs& a, int n, int step, float (&v)[COUNT]) {
  const T* p = static_cast<const T*>(a.bias);
  T raw[COUNT];
#pragma unroll
  for (int i = 0; i < COUNT; ++i)
    if (n + i * step < a.N) raw[i] = p[n + i * step];
#pragma unroll
  for (int i = 0; i < COUNT; ++i) v[i] = n + i * step < a.N ? to_f32(raw[i]) : 0.f;
}
template <int COUNT>
__device__ __forceinline__ void bias_columns(const LinearArgs& a, int n, int step, float (&v)[COUNT]) {
#pragma unroll
  for (int i = 0; i < COUNT; ++i) v[i] = 0.f;
  if (!a.bias) return;
  if (a.bias_type == SVOO_TYPE_FP32) bias_columns_of<float>(a, n, step, v);
  else if (a.bias_type == SVOO_TYPE_BF16) bias_columns_of<__nv_bfloat16>(a, n, step, v);
  else bias_columns_of<__half>(a, n, step, v);
}

}  // namespace tc

struct LinearCall {
  const void *a, *b;
  int64_t a_pitch, b_pitch;
  tc::LinearArgs args;
  cudaStream_t st;
};

}  // namespace svoo
