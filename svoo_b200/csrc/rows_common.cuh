// Shared by the token-wise kernels (layer norm, 8-bit linear layers): element types, vector loads and stores of
// V elements, reductions.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace svoo {

// Layer norm and its gradient (norm.cu)
struct NormArgs {
  const void *x, *dy, *gain, *offset;
  const void *x_end, *dy_end;                   // the byte behind the last element
  const float *mean_in, *rstd_in;
  void *y, *dx;
  float *mean, *rstd, *partial;
  int64_t x_batch, x_row, dy_batch, dy_row;     // strides in elements
  int64_t gain_batch, offset_batch;             // 0 where all samples share one row
  int64_t batch, rows;                          // rows per sample
  int C;
  bool params_fp32, plus_one;                   // parameters in 32 bits, or in the type of x
  float eps;
  int stages;                                   // rows that a group of the ring kernels has on their way
  int* status;                                  // the device's word: != 0 after a kernel gave up on a bounded wait
};

// SVOO_TYPE_* -> C++ type
template <int TYPE> struct ElemOf;
template <> struct ElemOf<SVOO_TYPE_BF16> { typedef __nv_bfloat16 T; };
template <> struct ElemOf<SVOO_TYPE_FP16> { typedef __half T; };
template <> struct ElemOf<SVOO_TYPE_FP32> { typedef float T; };
__host__ __device__ inline int elem_bytes(int type) { return type == SVOO_TYPE_FP32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// V consecutive elements, moved as one access of V * sizeof(T) <= 16 bytes
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) { return *reinterpret_cast<const Vec<T, V>*>(p); }

__device__ __forceinline__ float warp_sum(float s) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// Sets a kernel's dynamic shared memory limit on the current device, once: `done` is the kernel's own, a bit per device.
template <typename Kernel>
inline cudaError_t allow_smem(Kernel* kernel, int bytes, uint64_t& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (__atomic_load_n(&done, __ATOMIC_ACQUIRE) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) __atomic_fetch_or(&done, bit, __ATOMIC_RELEASE);
  return e;
}

// The status word of the token-wise kernels on the current device; null after a CUDA error.
int* rows_status_word();

}  // namespace svoo
