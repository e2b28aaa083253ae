// Quantisation to e4m3 with one 32-bit scale per block of 128 values (a stretch of a row, a stretch of a column, or a
// square of 128 x 128):
//
//   scale = max(amax / 448, 2^-126),  q = e4m3(x / scale)         both quotients rounded to 32 bits, q to nearest, ties to even
//
// 448 is the largest e4m3 number.  The largest magnitude is taken over bit patterns, where NaN is above infinity and both
// above every number: a block with a value that is not finite gets a scale that is not, and stands for nothing but NaN.
// All three kernels read x once; they are bound by HBM (2 or 4 bytes in, 1 out per value).
#include <cuda_fp8.h>

#include "rows_common.cuh"

namespace svoo {

constexpr int kBlock = 128;

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ float block_scale(uint32_t amax) {
  const float s = __fdiv_rn(__uint_as_float(amax), 448.f);
  return s < 0x1p-126f ? 0x1p-126f : s;                  // NaN stays
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// One block per half warp, eight values per lane.  V = 8: rows are whole 16-byte pieces, one (fp32: two) wide loads per lane;
// V = 1: any row.  scale[kb * scale_pitch + row]: the product reads the scales of 128 rows and one kb at a time.
template <typename T, int V>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, int64_t row_stride, int M, int K, int KB,
                                                            uint8_t* __restrict__ q, int64_t q_pitch, float* __restrict__ scale,
                                                            int64_t scale_pitch) {
  pdl_trigger();
  pdl_wait();
  const int unit = (int)(blockIdx.x * 16 + threadIdx.x / 16), lane = threadIdx.x % 16;
  const bool live = unit < M * KB;
  const int row = live ? unit / KB : 0, kb = live ? unit - row * KB : 0;
  const int k = kb * kBlock + lane * 8;
  const T* p = x + row * row_stride + k;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  if (live) {
    if constexpr (V == 8) {
      if (k < K) {
        constexpr int W = 16 / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < 8; i += W) {
          const Vec<T, W> t = load_stream<T, W>(p + i);
#pragma unroll
          for (int j = 0; j < W; ++j) v[i + j] = to_f32(t.v[j]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < K) v[i] = to_f32(p[i]);
    }
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, magnitude(v[i]));
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float s = block_scale(m);
  if (!live) return;
  if (lane == 0) scale[kb * scale_pitch + row] = s;
  if (k >= q_pitch) return;                              // q_pitch: K rounded up to 16, the rest of the row is zero
  uint2 out;
  out.x = e4m3x2(__fdiv_rn(v[0], s), __fdiv_rn(v[1], s)) | e4m3x2(__fdiv_rn(v[2], s), __fdiv_rn(v[3], s)) << 16;
  out.y = e4m3x2(__fdiv_rn(v[4], s), __fdiv_rn(v[5], s)) | e4m3x2(__fdiv_rn(v[6], s), __fdiv_rn(v[7], s)) << 16;
  *reinterpret_cast<uint2*>(q + row * q_pitch + k) = out;
}

// x [M, K] -> its transpose [K, M], blocks along M: a CTA takes 128 rows x 32 columns through shared memory.
// qt[c * qt_pitch + m], scale[mb * scale_pitch + c].  column_sum, if given, receives [mb][K] sums of the 128 rows.
template <typename T>
__global__ void __launch_bounds__(256) quantize_columns_kernel(const T* __restrict__ x, int64_t row_stride, int M, int K,
                                                               uint8_t* __restrict__ qt, int64_t qt_pitch, float* __restrict__ scale,
                                                               int64_t scale_pitch, float* __restrict__ column_sum) {
  __shared__ float tile[32][kBlock + 1];                 // [column][row]
  __shared__ uint32_t top[8][32];
  __shared__ float part[8][32];
  const int c0 = blockIdx.x * 32, mb = blockIdx.y, m0 = mb * kBlock;
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  uint32_t m = 0;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = w * 16 + i;
    float v = 0.f;
    if (m0 + r < M && c0 + lane < K) v = to_f32(x[(int64_t)(m0 + r) * row_stride + c0 + lane]);
    tile[lane][r] = v;
    m = max(m, magnitude(v));
    sum += v;
  }
  top[w][lane] = m;
  part[w][lane] = sum;
  __syncthreads();
  // eight threads per column, 16 rows each
  const int c = threadIdx.x / 8, r0 = threadIdx.x % 8 * 16;
  m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, top[i][c]);
  const float s = block_scale(m);
  if (c0 + c >= K) return;
  if (r0 == 0) {
    scale[mb * scale_pitch + c0 + c] = s;
    if (column_sum) {
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += part[i][c];
      column_sum[(int64_t)mb * K + c0 + c] = sum;
    }
  }
  if (m0 + r0 >= qt_pitch) return;
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float* t = &tile[c][r0 + 4 * i];
    o[i] = e4m3x2(__fdiv_rn(t[0], s), __fdiv_rn(t[1], s)) | e4m3x2(__fdiv_rn(t[2], s), __fdiv_rn(t[3], s)) << 16;
  }
  *reinterpret_cast<uint4*>(qt + (int64_t)(c0 + c) * qt_pitch + m0 + r0) = make_uint4(o[0], o[1], o[2], o[3]);
}

// w [N, K] in squares: q [N, q_pitch], scale [NB, KB]; qt [K, qt_pitch], if given, is the same numbers transposed.
template <typename T>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const T* __restrict__ x, int64_t row_stride, int N, int K,
                                                              uint8_t* __restrict__ q, int64_t q_pitch, uint8_t* __restrict__ qt,
                                                              int64_t qt_pitch, float* __restrict__ scale) {
  __shared__ uint32_t top[8];
  __shared__ uint8_t bytes[kBlock][kBlock + 4];          // [column][row] for the transpose
  const int kb = blockIdx.x, nb = blockIdx.y;
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  // thread: 4 columns lane * 4, rows w + 8 i
  float v[16][4];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int n = nb * kBlock + w + 8 * i, k = kb * kBlock + lane * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[i][j] = n < N && k + j < K ? to_f32(x[(int64_t)n * row_stride + k + j]) : 0.f;
      m = max(m, magnitude(v[i][j]));
    }
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) top[w] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, top[i]);
  const float s = block_scale(m);
  if (threadIdx.x == 0) scale[(int64_t)nb * gridDim.x + kb] = s;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = w + 8 * i, n = nb * kBlock + r, k = kb * kBlock + lane * 4;
    const uint32_t o = e4m3x2(__fdiv_rn(v[i][0], s), __fdiv_rn(v[i][1], s)) | e4m3x2(__fdiv_rn(v[i][2], s), __fdiv_rn(v[i][3], s)) << 16;
    if (n < N && k < q_pitch) *reinterpret_cast<uint32_t*>(q + (int64_t)n * q_pitch + k) = o;
    if (qt) {
#pragma unroll
      for (int j = 0; j < 4; ++j) bytes[lane * 4 + j][r] = (uint8_t)(o >> (8 * j));
    }
  }
  if (!qt) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int c = w + 8 * i, k = kb * kBlock + c, n = nb * kBlock + lane * 4;
    if (k < K && n < qt_pitch) *reinterpret_cast<uint32_t*>(qt + (int64_t)k * qt_pitch + n) = *reinterpret_cast<const uint32_t*>(&bytes[c][lane * 4]);
  }
}

template <typename T>
static cudaError_t rows_of(const void* x, int64_t M, int64_t K, int64_t row_stride, void* q, int64_t q_pitch, float* scale,
                           int64_t scale_pitch, cudaStream_t st) {
  const int KB = (int)ceil_div64(K, kBlock);
  const dim3 grid((unsigned)ceil_div64(M * KB, 16));
  const bool wide = K % 8 == 0 && row_stride * sizeof(T) % 16 == 0 && (uintptr_t)x % 16 == 0;
  count_launches(1);
  return launch_pdl(wide ? quantize_rows_kernel<T, 8> : quantize_rows_kernel<T, 1>, grid, dim3(256), 0, st, (const T*)x, row_stride,
                    (int)M, (int)K, KB, (uint8_t*)q, q_pitch, scale, scale_pitch);
}
template <typename T>
static cudaError_t columns_of(const void* x, int64_t M, int64_t K, int64_t row_stride, void* qt, int64_t qt_pitch, float* scale,
                              int64_t scale_pitch, float* column_sum, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div64(K, 32), (unsigned)ceil_div64(M, kBlock));
  quantize_columns_kernel<T><<<grid, 256, 0, st>>>((const T*)x, row_stride, (int)M, (int)K, (uint8_t*)qt, qt_pitch, scale, scale_pitch,
                                                   column_sum);
  count_launches(1);
  return cudaGetLastError();
}
template <typename T>
static cudaError_t blocks_of(const void* w, int64_t N, int64_t K, int64_t row_stride, void* q, int64_t q_pitch, void* qt, int64_t qt_pitch,
                             float* scale, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div64(K, kBlock), (unsigned)ceil_div64(N, kBlock));
  quantize_blocks_kernel<T><<<grid, 256, 0, st>>>((const T*)w, row_stride, (int)N, (int)K, (uint8_t*)q, q_pitch, (uint8_t*)qt, qt_pitch, scale);
  count_launches(1);
  return cudaGetLastError();
}

#define SVOO_BY_TYPE(fn, ...) \
  (type == SVOO_TYPE_BF16 ? fn<__nv_bfloat16>(__VA_ARGS__) : type == SVOO_TYPE_FP16 ? fn<__half>(__VA_ARGS__) : fn<float>(__VA_ARGS__))

cudaError_t launch_quantize_rows(int type, const void* x, int64_t M, int64_t K, int64_t row_stride, void* q, int64_t q_pitch, float* scale,
                                 int64_t scale_pitch, cudaStream_t st) {
  return SVOO_BY_TYPE(rows_of, x, M, K, row_stride, q, q_pitch, scale, scale_pitch, st);
}
cudaError_t launch_quantize_columns(int type, const void* x, int64_t M, int64_t K, int64_t row_stride, void* qt, int64_t qt_pitch,
                                    float* scale, int64_t scale_pitch, float* column_sum, cudaStream_t st) {
  return SVOO_BY_TYPE(columns_of, x, M, K, row_stride, qt, qt_pitch, scale, scale_pitch, column_sum, st);
}
cudaError_t launch_quantize_blocks(int type, const void* w, int64_t N, int64_t K, int64_t row_stride, void* q, int64_t q_pitch, void* qt,
                                   int64_t qt_pitch, float* scale, cudaStream_t st) {
  return SVOO_BY_TYPE(blocks_of, w, N, K, row_stride, q, q_pitch, qt, qt_pitch, scale, st);
}

}  // namespace svoo
