// Quantisation to e4m3 with one 32-bit scale per block of 128 values (a stretch of a row, a stretch of a column, or a
// square of 128 x 128):
//
//   scale = max(amax / 448, 2^-126),  q = e4m3(x / scale)         both quotients rounded to 32 bits, q to nearest, ties to even
//
// 448 is the largest e4m3 number.  The largest magnitude is taken over bit patterns, where NaN is above infinity and both
// above every number: a block with a value that is not finite gets a scale that is not, and stands for nothing but NaN.
// All three kernels read x once; they are bound by HBM (2 or 4 bytes in, 1 out per value).
#include "quant_common.cuh"

namespace svoo {

// A half warp takes one block at a time, kUnits of them with their loads in flight together, eight values per lane.
// kWide: rows are whole 16-byte pieces, one (fp32: two) wide loads per lane; otherwise any row.
// scale[kb * scale_pitch + row]: the product reads the scales of 128 rows and one kb at a time.
template <typename T, bool kWide>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, int64_t row_stride, int M, int K, int KB,
                                                            uint8_t* __restrict__ q, int64_t q_pitch, float* __restrict__ scale,
                                                            int64_t scale_pitch) {
  constexpr int kUnits = sizeof(T) == 2 ? 4 : 2;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x % 16, total = M * KB;
  const int unit0 = (int)(blockIdx.x * (16 * kUnits) + threadIdx.x / 16);
  Vec<T, 8> raw[kUnits];
  int row[kUnits], kb[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int unit = unit0 + u * 16 < total ? unit0 + u * 16 : total - 1;      // the last block again: the same bytes
    row[u] = unit / KB;
    kb[u] = unit - row[u] * KB;
    const int k = kb[u] * kBlock + lane * 8;
    const T* p = x + row[u] * row_stride + k;
    if constexpr (kWide) {
      uint4* r = reinterpret_cast<uint4*>(&raw[u]);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) r[i] = k < K ? __ldcs(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) raw[u].v[i] = k + i < K ? p[i] : from_f32<T>(0.f);
    }
  }
  // the largest magnitudes: 16-bit numbers by their patterns, two at a time
  uint32_t top[kUnits], mine = 0;
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw[u]);
    uint32_t m = 0;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
      m = max(m >> 16, m & 0xffffu);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
    }
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if constexpr (sizeof(T) == 2) {
      const unsigned short h = (unsigned short)m;
      top[u] = __float_as_uint(to_f32(*reinterpret_cast<const T*>(&h)));
    } else {
      top[u] = m;
    }
    if (lane == u) mine = top[u];
  }
  // lane u divides for block u
  const float scale_of = block_scale(mine), reciprocal = BlockDivide::reciprocal(scale_of);
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const float s = __shfl_sync(0xffffffffu, scale_of, u, 16);
    const BlockDivide by(s, __shfl_sync(0xffffffffu, reciprocal, u, 16));
    const int k = kb[u] * kBlock + lane * 8;
    if (lane == u) scale[kb[u] * scale_pitch + row[u]] = s;
    uint2 out;
    out.x = by.e4m3x4(to_f32(raw[u].v[0]), to_f32(raw[u].v[1]), to_f32(raw[u].v[2]), to_f32(raw[u].v[3]));
    out.y = by.e4m3x4(to_f32(raw[u].v[4]), to_f32(raw[u].v[5]), to_f32(raw[u].v[6]), to_f32(raw[u].v[7]));
    if (k < q_pitch) *reinterpret_cast<uint2*>(q + row[u] * q_pitch + k) = out;      // zeros behind the row
  }
}

// x [M, K] -> its transpose [K, M], blocks along M: a CTA takes 128 rows x 64 columns through shared memory.
// qt[c * qt_pitch + m], scale[mb * scale_pitch + c].  column_sum, if given, receives [mb][K] sums of the 128 rows.
template <typename T, bool kWide>
__global__ void __launch_bounds__(256) quantize_columns_kernel(const T* __restrict__ x, int64_t row_stride, int M, int K,
                                                               uint8_t* __restrict__ qt, int64_t qt_pitch, float* __restrict__ scale,
                                                               int64_t scale_pitch, float* __restrict__ column_sum) {
  constexpr int E = 16 / (int)sizeof(T), kPitch = 64 + E;   // a row of the tile is padded by 16 bytes
  __shared__ __align__(16) T tile[kBlock * kPitch];
  __shared__ uint32_t top[4][64];
  __shared__ float part[4][64];
  pdl_trigger();
  pdl_wait();
  const int c0 = blockIdx.x * 64, mb = blockIdx.y, m0 = mb * kBlock;
  if constexpr (kWide) {
    constexpr int P = 64 / E;                               // 16-byte pieces of a row
    uint4 v[kBlock * P / 256];
#pragma unroll
    for (int i = 0; i < kBlock * P / 256; ++i) {
      const int r = (i * 256 + threadIdx.x) / P, p = threadIdx.x % P;
      v[i] = m0 + r < M && c0 + p * E < K ? __ldcs(reinterpret_cast<const uint4*>(x + (int64_t)(m0 + r) * row_stride + c0 + p * E)) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kBlock * P / 256; ++i) {
      const int r = (i * 256 + threadIdx.x) / P, p = threadIdx.x % P;
      *reinterpret_cast<uint4*>(tile + r * kPitch + p * E) = v[i];
    }
  } else {
#pragma unroll 8
    for (int i = 0; i < kBlock / 4; ++i) {
      const int r = i * 4 + threadIdx.x / 64, c = threadIdx.x % 64;
      tile[r * kPitch + c] = m0 + r < M && c0 + c < K ? x[(int64_t)(m0 + r) * row_stride + c0 + c] : from_f32<T>(0.f);
    }
  }
  __syncthreads();
  // thread: 32 rows of one column
  const int c = threadIdx.x % 64, seg = threadIdx.x / 64;
  float v[32], sum = 0.f;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    v[i] = to_f32(tile[(seg * 32 + i) * kPitch + c]);
    m = max(m, magnitude(v[i]));
    sum += v[i];
  }
  top[seg][c] = m;
  part[seg][c] = sum;
  __syncthreads();
  m = max(max(top[0][c], top[1][c]), max(top[2][c], top[3][c]));
  const float s = block_scale(m);
  if (c0 + c >= K) return;
  if (seg == 0) {
    scale[mb * scale_pitch + c0 + c] = s;
    if (column_sum) column_sum[(int64_t)mb * K + c0 + c] = (part[0][c] + part[1][c]) + (part[2][c] + part[3][c]);
  }
  const BlockDivide by(s);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = seg * 32 + h * 16;
    if (m0 + r >= qt_pitch) break;
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = by.e4m3x4(v[h * 16 + 4 * i], v[h * 16 + 4 * i + 1], v[h * 16 + 4 * i + 2], v[h * 16 + 4 * i + 3]);
    *reinterpret_cast<uint4*>(qt + (int64_t)(c0 + c) * qt_pitch + m0 + r) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// w [N, K] in squares: q [N, q_pitch], scale [NB, KB]; qt [K, qt_pitch], if given, is the same numbers transposed.
template <typename T, bool kWide>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const T* __restrict__ x, int64_t row_stride, int N, int K,
                                                              uint8_t* __restrict__ q, int64_t q_pitch, uint8_t* __restrict__ qt,
                                                              int64_t qt_pitch, float* __restrict__ scale) {
  __shared__ uint32_t top[8];
  __shared__ uint8_t bytes[kBlock][kBlock + 4];          // [column][row] for the transpose
  const int kb = blockIdx.x, nb = blockIdx.y;
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  pdl_trigger();
  pdl_wait();
  // thread: 4 columns lane * 4, rows w + 8 i
  Vec<T, 4> v[16];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int n = nb * kBlock + w + 8 * i, k = kb * kBlock + lane * 4;
    const T* p = x + (int64_t)n * row_stride + k;
    if (kWide && n < N && k < K) {
      v[i] = load_vec<T, 4>(p);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i].v[j] = n < N && k + j < K ? p[j] : from_f32<T>(0.f);
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, magnitude(to_f32(v[i].v[j])));
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) top[w] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, top[i]);
  const float s = block_scale(m);
  if (threadIdx.x == 0) scale[(int64_t)nb * gridDim.x + kb] = s;
  const BlockDivide by(s);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = w + 8 * i, n = nb * kBlock + r, k = kb * kBlock + lane * 4;
    const uint32_t o = by.e4m3x4(to_f32(v[i].v[0]), to_f32(v[i].v[1]), to_f32(v[i].v[2]), to_f32(v[i].v[3]));
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
static bool wide_rows(const void* x, int64_t K, int64_t row_stride, int bytes) {
  return K * (int)sizeof(T) % bytes == 0 && row_stride * (int)sizeof(T) % bytes == 0 && (uintptr_t)x % bytes == 0;
}

template <typename T>
static cudaError_t rows_of(const void* x, int64_t M, int64_t K, int64_t row_stride, void* q, int64_t q_pitch, float* scale,
                           int64_t scale_pitch, cudaStream_t st) {
  const int KB = (int)ceil_div64(K, kBlock);
  const dim3 grid((unsigned)ceil_div64(M * KB, 16 * (sizeof(T) == 2 ? 4 : 2)));
  const bool wide = K % 8 == 0 && wide_rows<T>(x, K, row_stride, 16);
  count_launches(1);
  return launch_pdl(wide ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>, grid, dim3(256), 0, st, (const T*)x, row_stride,
                    (int)M, (int)K, KB, (uint8_t*)q, q_pitch, scale, scale_pitch);
}
template <typename T>
static cudaError_t columns_of(const void* x, int64_t M, int64_t K, int64_t row_stride, void* qt, int64_t qt_pitch, float* scale,
                              int64_t scale_pitch, float* column_sum, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div64(K, 64), (unsigned)ceil_div64(M, kBlock));
  count_launches(1);
  return launch_pdl(wide_rows<T>(x, K, row_stride, 16) ? quantize_columns_kernel<T, true> : quantize_columns_kernel<T, false>, grid,
                    dim3(256), 0, st, (const T*)x, row_stride, (int)M, (int)K, (uint8_t*)qt, qt_pitch, scale, scale_pitch, column_sum);
}
template <typename T>
static cudaError_t blocks_of(const void* w, int64_t N, int64_t K, int64_t row_stride, void* q, int64_t q_pitch, void* qt, int64_t qt_pitch,
                             float* scale, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div64(K, kBlock), (unsigned)ceil_div64(N, kBlock));
  count_launches(1);
  return launch_pdl(wide_rows<T>(w, K, row_stride, 4 * sizeof(T)) ? quantize_blocks_kernel<T, true> : quantize_blocks_kernel<T, false>, grid,
                    dim3(256), 0, st, (const T*)w, row_stride, (int)N, (int)K, (uint8_t*)q, q_pitch, (uint8_t*)qt, qt_pitch, scale);
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
