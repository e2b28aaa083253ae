// A linear layer on at most 16 unquantised rows: quantisation of the rows, product, bias and activation in one kernel.
//
// With so few rows the weights' bytes are all there is to move (N K), and a launch costs as much as they do: 5,120 x 5,120 is 4 us
// at the HBM's rate.  A CTA takes NT x 8 columns, its warps share out the blocks of k; a warp reads its weights
// straight into the fragments of mma.sync (m16n8k16, rows as A, weights as B), so nothing waits for shared memory or for an
// accumulator elsewhere.  The order of k inside a block is free as long as both operands agree on it: lane t of four holds bytes
// 32 t .. 32 t + 31 of its row, and step j multiplies bytes 4 j .. 4 j + 3 of the four lanes.  e4m3 goes to fp16 exactly, a
// product of two is a 32-bit number, sums are in 32 bits; each block is scaled by sa sb as linear_tc.cu does.
// Every warp quantises the rows of its own blocks: again in every CTA, but that is cheaper than a launch.  It is also what bounds the
// kernel at 16 rows of 5,120 columns (12.7 us; 8.7 with one row, 9.3 with 8).
#include "linear_common.cuh"

namespace svoo {

__device__ __forceinline__ uint32_t halves_of(uint32_t word, bool upper) {     // two e4m3 bytes as fp16
  uint32_t r;
  const uint16_t b = (uint16_t)(upper ? word >> 16 : word);
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(b));
  return r;
}
__device__ __forceinline__ void mma_fp16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 bytes of a row of weights of which `left` remain; nothing behind the row is read
__device__ __forceinline__ uint4 load_weights(const uint8_t* p, int left) {
  if (left >= 16) return __ldcs(reinterpret_cast<const uint4*>(p));
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < left) w[i / 4] |= (uint32_t)p[i] << (8 * (i % 4));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 32 values of one row, quantised with the other three lanes of the row: eight words of e4m3; the block's scale
template <typename T, bool kWide>
__device__ __forceinline__ float quantize_lane(const T* p, int k, int K, bool live, uint32_t (&q)[8]) {
  float v[32];
  if constexpr (kWide) {
    constexpr int W = 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < 32; i += W) {
      const bool in = live && k + i < K;                    // rows are whole 16-byte pieces
      Vec<T, W> t = {};
      if (in) t = load_vec<T, W>(p + i);
#pragma unroll
      for (int j = 0; j < W; ++j) v[i + j] = in ? to_f32(t.v[j]) : 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = live && k + i < K ? to_f32(p[i]) : 0.f;
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) m = max(m, magnitude(v[i]));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const float s = block_scale(m);
  const BlockDivide by(s);
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = by.e4m3x4<sizeof(T) == 2>(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  return s;
}

// MT: 8 or 16 rows; NT: column tiles of 8; W: warps
template <typename T, bool kWide, int MT, int NT, int W>
__global__ void __launch_bounds__(W * 32, W == 8 ? 2 : 1)
    linear_few_kernel(const T* __restrict__ x, int64_t x_row, const uint8_t* __restrict__ b, int64_t b_pitch, const tc::LinearArgs a,
                      int out_type, bool gelu) {
  constexpr int NW = NT * 8;
  __shared__ float part[W][MT][NW + 1];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int n0 = blockIdx.x * NW, KB = (a.K + 127) / 128;
  pdl_trigger();
  pdl_wait();
  float sum[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = 0.f;
  const int last = (a.N - 1) / 128;
  for (int kb = warp; kb < KB; kb += W) {
    const int k = kb * 128 + t * 32;
    // the weights first: they are what takes long
    uint4 w[NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int n = n0 + i * 8 + g;
#pragma unroll
      for (int h = 0; h < 2; ++h) w[i][h] = load_weights(b + (int64_t)n * b_pitch + k + h * 16, n < a.N ? a.K - k - h * 16 : 0);
    }
    float fb[NT];                                           // a CTA's columns may lie in two blocks
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int nb = (n0 + i * 8) / 128;
      fb[i] = a.sb[(nb < last ? nb : last) * a.sb_n + kb * a.sb_k];
    }
    uint32_t q0[8], q1[8];
    float s[2] = {0.f, 0.f};
    s[0] = quantize_lane<T, kWide>(x + g * x_row + k, k, a.K, g < a.M, q0);
    if (MT == 16) s[1] = quantize_lane<T, kWide>(x + (g + 8) * x_row + k, k, a.K, g + 8 < a.M, q1);
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t fr[4] = {halves_of(q0[j], false), MT == 16 ? halves_of(q1[j], false) : 0u, halves_of(q0[j], true),
                              MT == 16 ? halves_of(q1[j], true) : 0u};
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint32_t u = reinterpret_cast<const uint32_t*>(w[i])[j];
        mma_fp16(acc[i], fr, halves_of(u, false), halves_of(u, true));
      }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[i][j] = fmaf(acc[i][j], s[j / 2] * fb[i], sum[i][j]);
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
#pragma unroll
    for (int j = 0; j < (MT == 16 ? 4 : 2); ++j) part[warp][g + j / 2 * 8][i * 8 + t * 2 + j % 2] = sum[i][j];
  }
  __syncthreads();
  for (int o = threadIdx.x; o < MT * NW; o += W * 32) {
    const int r = o / NW, n = n0 + o % NW;
    if (r >= a.M || n >= a.N) continue;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) v += part[i][r][o % NW];
    float bias[1];
    tc::bias_columns(a, n, 1, bias);
    v += bias[0];
    if (gelu) v = tc::half_of(tc::gelu2(tc::pack2(v, v)), 0);
    const int64_t at = r * a.out_pitch + n;
    if (out_type == SVOO_TYPE_FP32) static_cast<float*>(a.out)[at] = v;
    else if (out_type == SVOO_TYPE_BF16) static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
    else static_cast<__half*>(a.out)[at] = __float2half_rn(v);
  }
}

template <typename T, bool kWide, int MT, int NT, int W>
static cudaError_t launch_few_nt(const void* x, int64_t x_row, const LinearCall& c, int out_type, bool gelu) {
  count_launches(1);
  return launch_pdl(linear_few_kernel<T, kWide, MT, NT, W>, dim3((unsigned)ceil_div(c.args.N, NT * 8)), dim3(W * 32), 0, c.st, (const T*)x, x_row,
                    (const uint8_t*)c.b, c.b_pitch, c.args, out_type, gelu);
}
// Columns per CTA so that all of them run at once: an SM holds one CTA of sixteen warps or two of eight.  One row, 16 rows of 5,120 x
// 5,120, us: 40 columns by sixteen warps (128 CTAs) 8.7, 12.7; 32 by sixteen (160, two rounds) 14.1, 19.5; 32 by eight 12.1, 18.9.  With 9 to 16
// rows a few of the 128 registers spill: 64 to 120 bytes a thread by type with 40 columns, 56 with 32 columns and 16-bit rows that are not aligned.
template <typename T, bool kWide, int MT>
static cudaError_t launch_few_mt(const void* x, int64_t x_row, const LinearCall& c, int out_type, bool gelu) {
  if (c.args.N <= 148 * 16) return launch_few_nt<T, kWide, MT, 2, 16>(x, x_row, c, out_type, gelu);
  if (c.args.N <= 148 * 40) return launch_few_nt<T, kWide, MT, 5, 16>(x, x_row, c, out_type, gelu);
  return launch_few_nt<T, kWide, MT, 4, 8>(x, x_row, c, out_type, gelu);
}
template <typename T, bool kWide>
static cudaError_t launch_few_t(const void* x, int64_t x_row, const LinearCall& c, int out_type, bool gelu) {
  return c.args.M <= 8 ? launch_few_mt<T, kWide, 8>(x, x_row, c, out_type, gelu) : launch_few_mt<T, kWide, 16>(x, x_row, c, out_type, gelu);
}

// M <= 16, output not e4m3; c.a unused
cudaError_t launch_linear_few(int type, const void* x, int64_t x_row, const LinearCall& c, int out_type, bool gelu) {
  const int e = elem_bytes(type);
  const bool wide = (int64_t)c.args.K * e % 16 == 0 && x_row * e % 16 == 0 && (uintptr_t)x % 16 == 0;
  switch (type) {
    case SVOO_TYPE_BF16: return wide ? launch_few_t<__nv_bfloat16, true>(x, x_row, c, out_type, gelu) : launch_few_t<__nv_bfloat16, false>(x, x_row, c, out_type, gelu);
    case SVOO_TYPE_FP16: return wide ? launch_few_t<__half, true>(x, x_row, c, out_type, gelu) : launch_few_t<__half, false>(x, x_row, c, out_type, gelu);
    default: return wide ? launch_few_t<float, true>(x, x_row, c, out_type, gelu) : launch_few_t<float, false>(x, x_row, c, out_type, gelu);
  }
}

}  // namespace svoo
