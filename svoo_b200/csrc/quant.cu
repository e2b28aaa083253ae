// Quantisation to e4m3 with one 32-bit scale per block of 128 values (a stretch of a row, a stretch of a column, or a
// square of 128 x 128):
//
//   scale = max(amax / 448, 2^-126),  q = e4m3(x / scale)         both quotients rounded to 32 bits, q to nearest, ties to even
//
// 448 is the largest e4m3 number.  The largest magnitude is taken over bit patterns, where NaN is above infinity and both
// above every number: a block with a value that is not finite gets a scale that is not, and stands for nothing but NaN.
// All kernels read x once (2 or 4 bytes in, 1 out per value); quantize_rows_kernel is bound by HBM, the others by what they do in
// shared memory and registers besides.
#include "quant_common.cuh"

namespace svoo {

// Bytes that a row of n numbers takes: zeros up to the next multiple of 16, whatever the pitch.  What follows may be another's.
__device__ __forceinline__ int written(int n) { return (n + 15) & ~15; }

// The largest magnitude of a half warp's 128 values, as the pattern of a 32-bit number: 16-bit numbers by their own patterns,
// two at a time.
template <typename T>
__device__ __forceinline__ uint32_t block_top(const Vec<T, 8>& v) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
  uint32_t m = 0;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint16_t h = (uint16_t)max(m >> 16, m & 0xffffu);
    return __float_as_uint(to_f32(*reinterpret_cast<const T*>(&h)));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
  }
}

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
  // consecutive blocks; past the end the last one again, the same bytes
  const int unit0 = (int)(blockIdx.x * 16 + threadIdx.x / 16) * kUnits;
  Vec<T, 8> raw[kUnits];
  int row[kUnits], kb[kUnits];
  row[0] = (unit0 < total ? unit0 : total - 1) / KB;
  kb[0] = (unit0 < total ? unit0 : total - 1) - row[0] * KB;
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    if (u > 0) {
      const bool next = kb[u - 1] + 1 == KB, end = next && row[u - 1] + 1 == M;
      row[u] = row[u - 1] + (next && !end);
      kb[u] = end ? kb[u - 1] : next ? 0 : kb[u - 1] + 1;
    }
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
  uint32_t mine = 0;
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const uint32_t m = block_top<T>(raw[u]);
    if (lane == u) mine = m;
  }
  // lane u divides for block u
  const float scale_of = block_scale(mine), reciprocal = BlockDivide::reciprocal(scale_of);
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const float s = __shfl_sync(0xffffffffu, scale_of, u, 16);
    const BlockDivide by(s, __shfl_sync(0xffffffffu, reciprocal, u, 16));
    const int k = kb[u] * kBlock + lane * 8;
    if (lane == u) scale[kb[u] * scale_pitch + row[u]] = s;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(raw[u].v[i]);
    const uint2 out = by.e4m3x8<sizeof(T) == 2>(v);
    if (k < written(K)) *reinterpret_cast<uint2*>(q + row[u] * q_pitch + k) = out;
  }
}

// 4 x 4 bytes transposed: word j of the result holds byte j of the four words
__device__ __forceinline__ void transpose4(uint32_t (&o)[4]) {
  const uint32_t a = __byte_perm(o[0], o[1], 0x5140), b = __byte_perm(o[0], o[1], 0x7362);
  const uint32_t c = __byte_perm(o[2], o[3], 0x5140), d = __byte_perm(o[2], o[3], 0x7362);
  o[0] = __byte_perm(a, c, 0x5410);
  o[1] = __byte_perm(a, c, 0x7632);
  o[2] = __byte_perm(b, d, 0x5410);
  o[3] = __byte_perm(b, d, 0x7632);
}

// w [N, K] in squares: q [N, q_pitch], scale [NB, KB]; qt [K, qt_pitch], if given, is the same numbers transposed, four rows of
// four columns in registers, then by words through shared memory (word r / 4 of column c at (r / 4) ^ (c / 4): no bank conflicts).
// 16-bit types are held to 40 registers, for three CTAs an SM, and spill 36 to 72 bytes a thread.  8,960 x 1,536 bf16 25 us, with qt 27;
// 75,600 x 5,120 408 and 499 (177 and 237 for the bytes).
template <typename T, bool kWide>
__global__ void __launch_bounds__(512, sizeof(T) == 2 ? 3 : 2) quantize_blocks_kernel(const T* __restrict__ x, int64_t row_stride, int N, int K,
                                                              uint8_t* __restrict__ q, int64_t q_pitch, uint8_t* __restrict__ qt,
                                                              int64_t qt_pitch, float* __restrict__ scale) {
  __shared__ uint32_t top[16];
  __shared__ uint32_t words[kBlock][kBlock / 4];
  const int kb = blockIdx.x, nb = blockIdx.y;
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  pdl_trigger();
  pdl_wait();
  // thread: 4 columns lane * 4, 8 rows from w * 8
  Vec<T, 4> v[8];
  uint32_t m = 0;
  const int k = kb * kBlock + lane * 4, n0 = nb * kBlock + w * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const T* p = x + (int64_t)(n0 + i) * row_stride + k;
    if (kWide && n0 + i < N && k < K) {
      v[i] = load_vec<T, 4>(p);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i].v[j] = n0 + i < N && k + j < K ? p[j] : from_f32<T>(0.f);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, magnitude(to_f32(v[i].v[j])));
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) top[w] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, top[i]);
  const float s = block_scale(m);
  if (threadIdx.x == 0) scale[(int64_t)nb * gridDim.x + kb] = s;
  const BlockDivide by(s);
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const Vec<T, 4>& t = v[g * 4 + i];
      o[i] = by.e4m3x4<sizeof(T) == 2>(to_f32(t.v[0]), to_f32(t.v[1]), to_f32(t.v[2]), to_f32(t.v[3]));
      if (n0 + g * 4 + i < N && k < written(K)) *reinterpret_cast<uint32_t*>(q + (int64_t)(n0 + g * 4 + i) * q_pitch + k) = o[i];
    }
    if (qt) {
      transpose4(o);
#pragma unroll
      for (int j = 0; j < 4; ++j) words[lane * 4 + j][(w * 2 + g) ^ lane] = o[j];
    }
  }
  if (!qt) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = w * 8 + i, n = nb * kBlock + lane * 4;
    if (kb * kBlock + c < K && n < written(N))
      *reinterpret_cast<uint32_t*>(qt + (int64_t)(kb * kBlock + c) * qt_pitch + n) = words[c][lane ^ (c / 4)];
  }
}

// x [M, K] transposed, in blocks along its columns, and with kRows also as it is, in blocks along its rows, from one reading: 128 rows
// x 128 columns per CTA.  A half warp holds whole row blocks in registers; the columns go through shared memory.
// qt[c * qt_pitch + m], scale_t[mb * scale_t_pitch + c]; column_sum, if given, receives [mb][K] sums of the 128 rows.
// Three CTAs per SM: 75,600 x 5,120 bf16 397 us both ways, 305 the columns alone (two CTAs: 458 both ways, four: 469).
template <typename T, bool kWide, bool kRows>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2) quantize_tile_kernel(const T* __restrict__ x, int64_t row_stride, int M, int K, uint8_t* __restrict__ q,
                                                            int64_t q_pitch, float* __restrict__ scale, int64_t scale_pitch,
                                                            uint8_t* __restrict__ qt, int64_t qt_pitch, float* __restrict__ scale_t,
                                                            int64_t scale_t_pitch, float* __restrict__ column_sum) {
  constexpr int kPitch = kBlock + 16 / (int)sizeof(T);
  extern __shared__ __align__(16) unsigned char smem[];
  T* tile = reinterpret_cast<T*>(smem);
  __shared__ uint32_t top[4][kBlock / 2];                    // 16-bit patterns of two columns; 32-bit: [2][128]
  __shared__ float part[4][kBlock];
  pdl_trigger();
  pdl_wait();
  const int kb = blockIdx.x, mb = blockIdx.y, m0 = mb * kBlock, lane = threadIdx.x % 16, h = threadIdx.x / 16;
  const int k = kb * kBlock + lane * 8;
  constexpr int U = sizeof(T) == 2 ? 4 : 2;                  // rows of a half warp in flight
  for (int r0 = 0; r0 < kBlock; r0 += 16 * U) {
    Vec<T, 8> raw[U];
    uint32_t mine = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int m = m0 + r0 + u * 16 + h;
      const T* p = x + (int64_t)m * row_stride + k;
      if constexpr (kWide) {
        uint4* r = reinterpret_cast<uint4*>(&raw[u]);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
          r[i] = m < M && k + i * (16 / (int)sizeof(T)) < K ? __ldcs(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0, 0, 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[u].v[i] = m < M && k + i < K ? p[i] : from_f32<T>(0.f);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint4* t = reinterpret_cast<uint4*>(tile + (r0 + u * 16 + h) * kPitch + lane * 8);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) t[i] = reinterpret_cast<const uint4*>(&raw[u])[i];
      if constexpr (kRows) {
        const uint32_t m = block_top<T>(raw[u]);
        if (lane == u) mine = m;
      }
    }
    if constexpr (kRows) {
      const float scale_of = block_scale(mine), reciprocal = BlockDivide::reciprocal(scale_of);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int m = m0 + r0 + u * 16 + h;
        const float s = __shfl_sync(0xffffffffu, scale_of, u, 16);
        const BlockDivide by(s, __shfl_sync(0xffffffffu, reciprocal, u, 16));
        if (m >= M) continue;
        if (lane == u) scale[kb * scale_pitch + m] = s;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32(raw[u].v[i]);
        const uint2 out = by.e4m3x8<sizeof(T) == 2>(v);
        if (k < written(K)) *reinterpret_cast<uint2*>(q + (int64_t)m * q_pitch + k) = out;
      }
    }
  }
  __syncthreads();
  // thread: R rows of C columns, a word each
  constexpr int C = sizeof(T) == 2 ? 2 : 1, kThreadsAcross = kBlock / C, kSegs = 256 / kThreadsAcross, R = kBlock / kSegs;
  static_assert(R * C == 64 && R % 16 == 0);
  const int c = threadIdx.x % kThreadsAcross * C, seg = threadIdx.x / kThreadsAcross;
  uint32_t w[R], m = 0;
  float sum[C] = {};
#pragma unroll
  for (int i = 0; i < R; ++i) {
    w[i] = *reinterpret_cast<const uint32_t*>(tile + (seg * R + i) * kPitch + c);
    if constexpr (C == 2) {
      const Vec<T, 2> v = *reinterpret_cast<const Vec<T, 2>*>(&w[i]);
      m = __vmaxu2(m, w[i] & 0x7fff7fffu);
      sum[0] += to_f32(v.v[0]);
      sum[C - 1] += to_f32(v.v[1]);
    } else {
      m = max(m, w[i] & 0x7fffffffu);
      sum[0] += __uint_as_float(w[i]);
    }
  }
  uint32_t* tops = &top[0][0];
  tops[threadIdx.x] = m;
#pragma unroll
  for (int j = 0; j < C; ++j) part[seg][c + j] = sum[j];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSegs; ++i) {
    const uint32_t o = tops[i * kThreadsAcross + threadIdx.x % kThreadsAcross];
    m = C == 2 ? __vmaxu2(m, o) : max(m, o);
  }
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int col = kb * kBlock + c + j;
    if (col >= K) break;
    const uint16_t half = (uint16_t)(m >> (16 * j));
    const float s = block_scale(C == 2 ? __float_as_uint(to_f32(*reinterpret_cast<const T*>(&half))) : m);
    if (seg == 0) {
      scale_t[mb * scale_t_pitch + col] = s;
      if (column_sum) {
        float all = 0.f;
#pragma unroll
        for (int i = 0; i < kSegs; ++i) all += part[i][c + j];
        column_sum[(int64_t)mb * K + col] = all;
      }
    }
    const BlockDivide by(s);
#pragma unroll
    for (int g = 0; g < R / 16; ++g) {
      const int r = seg * R + g * 16;
      if (m0 + r >= written(M)) break;
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t word = w[g * 16 + i * 4 + e];
          v[e] = C == 2 ? to_f32(reinterpret_cast<const Vec<T, C>*>(&word)->v[j]) : __uint_as_float(word);
        }
        o[i] = by.e4m3x4<sizeof(T) == 2>(v[0], v[1], v[2], v[3]);
      }
      *reinterpret_cast<uint4*>(qt + (int64_t)col * qt_pitch + m0 + r) = make_uint4(o[0], o[1], o[2], o[3]);
    }
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
static cudaError_t blocks_of(const void* w, int64_t N, int64_t K, int64_t row_stride, void* q, int64_t q_pitch, void* qt, int64_t qt_pitch,
                             float* scale, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div64(K, kBlock), (unsigned)ceil_div64(N, kBlock));
  count_launches(1);
  return launch_pdl(wide_rows<T>(w, K, row_stride, 4 * sizeof(T)) ? quantize_blocks_kernel<T, true> : quantize_blocks_kernel<T, false>, grid,
                    dim3(512), 0, st, (const T*)w, row_stride, (int)N, (int)K, (uint8_t*)q, q_pitch, (uint8_t*)qt, qt_pitch, scale);
}

// q null: the columns alone
template <typename T>
static cudaError_t tile_of(const void* x, int64_t M, int64_t K, int64_t row_stride, void* q, int64_t q_pitch, float* scale, int64_t scale_pitch,
                           void* qt, int64_t qt_pitch, float* scale_t, int64_t scale_t_pitch, float* column_sum, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div64(K, kBlock), (unsigned)ceil_div64(M, kBlock));
  const bool wide = wide_rows<T>(x, K, row_stride, 16);
  const int smem = kBlock * (kBlock + 16 / (int)sizeof(T)) * (int)sizeof(T);
  auto* kernel = q ? (wide ? &quantize_tile_kernel<T, true, true> : &quantize_tile_kernel<T, false, true>)
                   : (wide ? &quantize_tile_kernel<T, true, false> : &quantize_tile_kernel<T, false, false>);
  static uint64_t done[4];
  const cudaError_t e = allow_smem(kernel, smem, done[(q ? 2 : 0) + wide]);
  if (e != cudaSuccess) return e;
  count_launches(1);
  return launch_pdl(kernel, grid, dim3(256), smem, st, (const T*)x, row_stride, (int)M, (int)K, (uint8_t*)q, q_pitch, scale, scale_pitch,
                    (uint8_t*)qt, qt_pitch, scale_t, scale_t_pitch, column_sum);
}

#define SVOO_BY_TYPE(fn, ...) \
  (type == SVOO_TYPE_BF16 ? fn<__nv_bfloat16>(__VA_ARGS__) : type == SVOO_TYPE_FP16 ? fn<__half>(__VA_ARGS__) : fn<float>(__VA_ARGS__))

cudaError_t launch_quantize_rows(int type, const void* x, int64_t M, int64_t K, int64_t row_stride, void* q, int64_t q_pitch, float* scale,
                                 int64_t scale_pitch, cudaStream_t st) {
  return SVOO_BY_TYPE(rows_of, x, M, K, row_stride, q, q_pitch, scale, scale_pitch, st);
}
cudaError_t launch_quantize_columns(int type, const void* x, int64_t M, int64_t K, int64_t row_stride, void* qt, int64_t qt_pitch,
                                    float* scale, int64_t scale_pitch, float* column_sum, cudaStream_t st) {
  return SVOO_BY_TYPE(tile_of, x, M, K, row_stride, nullptr, 0, nullptr, 0, qt, qt_pitch, scale, scale_pitch, column_sum, st);
}
cudaError_t launch_quantize_both(int type, const void* x, int64_t M, int64_t K, int64_t row_stride, void* q, int64_t q_pitch, float* scale,
                                 int64_t scale_pitch, void* qt, int64_t qt_pitch, float* scale_t, int64_t scale_t_pitch, float* column_sum,
                                 cudaStream_t st) {
  return SVOO_BY_TYPE(tile_of, x, M, K, row_stride, q, q_pitch, scale, scale_pitch, qt, qt_pitch, scale_t, scale_t_pitch, column_sum, st);
}
cudaError_t launch_quantize_blocks(int type, const void* w, int64_t N, int64_t K, int64_t row_stride, void* q, int64_t q_pitch, void* qt,
                                   int64_t qt_pitch, float* scale, cudaStream_t st) {
  return SVOO_BY_TYPE(blocks_of, w, N, K, row_stride, q, q_pitch, qt, qt_pitch, scale, st);
}

}  // namespace svoo
