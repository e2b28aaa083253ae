// Layer norm over the last dimension, affine or with a modulation per sample (AdaLN), and its gradient.
//
//   mean = sum(x) / C, rstd = 1 / sqrt(sum((x - mean)^2) / C + eps), xhat = (x - mean) rstd
//   y  = xhat g + o            g = gain (or 1 + gain), o = offset: one row of C, or one per sample
//   dx = rstd (w - sum(w) / C - xhat sum(w xhat) / C),  w = dy g;    dg = sum_rows dy xhat,  do = sum_rows dy
//
// Everything between the loads and the stores is in 32 bits.  The variance is taken around the mean from the row in
// registers, so a mean far from zero costs no digits.  A row whose values are not all finite comes out NaN.
#include "rows_common.cuh"

namespace svoo {

template <typename T, int V>
__device__ __forceinline__ void load_param(const void* p, bool fp32, int64_t at, float (&out)[V]) {
  if (fp32 || sizeof(T) == 4) {
    const float* q = static_cast<const float*>(p) + at;
    constexpr int W = V < 4 ? V : 4;
#pragma unroll
    for (int i = 0; i < V; i += W) {
      const Vec<float, W> t = load_vec<float, W>(q + i);
#pragma unroll
      for (int k = 0; k < W; ++k) out[i + k] = t.v[k];
    }
  } else {
    const Vec<T, V> t = load_vec<T, V>(static_cast<const T*>(p) + at);
#pragma unroll
    for (int k = 0; k < V; ++k) out[k] = to_f32(t.v[k]);
  }
}

// Sum over the TPR threads of a row, the same in every thread.  `slot`: TPR / 32 floats of the row's own; two calls in a
// row need two slots (a thread may still read the first when another writes the second).
template <int TPR>
__device__ __forceinline__ float row_sum(float s, float* slot, int t) {
  s = warp_sum(s);
  if (TPR == 32) return s;
  if (t % 32 == 0) slot[t / 32] = s;
  __syncthreads();
  s = 0.f;
#pragma unroll
  for (int w = 0; w < TPR / 32; ++w) s += slot[w];
  return s;
}

// TPR threads hold one row, NV vectors of V elements each, vector i of thread t at (i * TPR + t) * V.
template <typename T, int V, int NV, int TPR>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) layer_norm_kernel(const NormArgs a) {
  constexpr int G = TPR < 128 ? 128 / TPR : 1;
  __shared__ float slots[2][G][TPR / 32];
  const int g = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * G + g;
  if (G > 1 && row >= a.batch * a.rows) return;          // whole warps: a row is one warp there
  const int64_t b = a.batch == 1 ? 0 : row / a.rows;
  const T* x = static_cast<const T*>(a.x) + b * a.x_batch + (row - b * a.rows) * a.x_row;
  const int nvec = a.C / V;

  float v[NV][V];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = i * TPR + t;
    if (c < nvec) {
      const Vec<T, V> r = load_stream<T, V>(x + (int64_t)c * V);
#pragma unroll
      for (int k = 0; k < V; ++k) v[i][k] = to_f32(r.v[k]);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) v[i][k] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < V; ++k) s += v[i][k];
  const float mean = row_sum<TPR>(s, slots[0][g], t) / a.C;
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i * TPR + t < nvec) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float d = v[i][k] - mean;
        q += d * d;
      }
    }
  }
  const float rstd = 1.f / sqrtf(row_sum<TPR>(q, slots[1][g], t) / a.C + a.eps);
  if (t == 0 && a.mean) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  T* y = static_cast<T*>(a.y) + row * a.C;
  const float one = a.plus_one ? 1.f : 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = i * TPR + t;
    if (c >= nvec) continue;
    float gain[V], off[V];
#pragma unroll
    for (int k = 0; k < V; ++k) gain[k] = 1.f, off[k] = 0.f;
    if (a.gain) {
      load_param<T, V>(a.gain, a.params_fp32, b * a.gain_batch + c * V, gain);
#pragma unroll
      for (int k = 0; k < V; ++k) gain[k] += one;
    }
    if (a.offset) load_param<T, V>(a.offset, a.params_fp32, b * a.offset_batch + c * V, off);
    Vec<T, V> r;
#pragma unroll
    for (int k = 0; k < V; ++k) r.v[k] = from_f32<T>((v[i][k] - mean) * rstd * gain[k] + off[k]);
    *reinterpret_cast<Vec<T, V>*>(y + (int64_t)c * V) = r;
  }
}

// One CTA of TPR threads walks the rows blockIdx.x, + gridDim.x, ... of group blockIdx.y (a sample where the modulation is
// per sample, otherwise all rows) and keeps the column sums of its rows in registers; they go to `partial`
// [group][CTA][dg, do][C], which column_sum_kernel adds in a fixed order.  The next row is fetched before this one's two
// sums are joined.
template <typename T, int V, int NV, int TPR>
__global__ void __launch_bounds__(TPR) layer_norm_backward_kernel(const NormArgs a) {
  __shared__ float slots[2][2][TPR / 32];
  const int t = threadIdx.x;
  const bool per_sample = gridDim.y > 1;
  const int64_t n = per_sample ? a.rows : a.batch * a.rows;
  const int nvec = a.C / V;
  float dg[NV][V], dof[NV][V], gain[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < V; ++k) dg[i][k] = dof[i][k] = 0.f, gain[i][k] = 1.f;
  if (a.gain) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = i * TPR + t;
      if (c < nvec) load_param<T, V>(a.gain, a.params_fp32, blockIdx.y * a.gain_batch + c * V, gain[i]);
      if (a.plus_one) {
#pragma unroll
        for (int k = 0; k < V; ++k) gain[i][k] += 1.f;
      }
    }
  }
  Vec<T, V> xr[NV], dr[NV];
  float mean = 0.f, rstd = 0.f;
  auto fetch = [&](int64_t r) {
    int64_t b = blockIdx.y, s = r;
    if (!per_sample) b = a.batch == 1 ? 0 : r / a.rows, s = r - b * a.rows;
    const T* x = static_cast<const T*>(a.x) + b * a.x_batch + s * a.x_row;
    const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch + s * a.dy_row;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = i * TPR + t;
      if (c < nvec) {
        xr[i] = load_stream<T, V>(x + (int64_t)c * V);
        dr[i] = load_stream<T, V>(dy + (int64_t)c * V);
      }
    }
    mean = a.mean_in[b * a.rows + s];
    rstd = a.rstd_in[b * a.rows + s];
  };
  if (blockIdx.x < n) fetch(blockIdx.x);
  int buf = 0;
  for (int64_t r = blockIdx.x; r < n; r += gridDim.x, buf ^= 1) {
    float h[NV][V], w[NV][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i * TPR + t < nvec) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float d = to_f32(dr[i].v[k]);
          h[i][k] = (to_f32(xr[i].v[k]) - mean) * rstd;
          dg[i][k] += d * h[i][k];
          dof[i][k] += d;
          w[i][k] = d * gain[i][k];
          s1 += w[i][k];
          s2 += w[i][k] * h[i][k];
        }
      }
    }
    const float rs = rstd;
    if (r + gridDim.x < n) fetch(r + gridDim.x);
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if (TPR > 32) {
      if (t % 32 == 0) slots[buf][0][t / 32] = s1, slots[buf][1][t / 32] = s2;
      __syncthreads();                                   // the other buffer is written only after the next row's barrier
      s1 = s2 = 0.f;
#pragma unroll
      for (int k = 0; k < TPR / 32; ++k) s1 += slots[buf][0][k], s2 += slots[buf][1][k];
    }
    s1 /= a.C;
    s2 /= a.C;
    T* dx = static_cast<T*>(a.dx) + (per_sample ? blockIdx.y * a.rows + r : r) * a.C;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = i * TPR + t;
      if (c >= nvec) continue;
      Vec<T, V> o;
#pragma unroll
      for (int k = 0; k < V; ++k) o.v[k] = from_f32<T>(rs * (w[i][k] - s1 - h[i][k] * s2));
      *reinterpret_cast<Vec<T, V>*>(dx + (int64_t)c * V) = o;
    }
  }
  if (!a.partial) return;
  float* p = a.partial + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * a.C;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = i * TPR + t;
    if (c >= nvec) continue;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      p[(int64_t)c * V + k] = dg[i][k];
      p[a.C + (int64_t)c * V + k] = dof[i][k];
    }
  }
}

// out0[group][c] = sum_p partial[group][p][0][c], out1 the same of [1] (gridDim.z outputs in all): 32 columns per CTA, 32
// warps over the parts.
template <typename T>
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ partial, int parts, int C, void* out0, void* out1,
                                                          bool out_fp32) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  const int c = blockIdx.x * 32 + lane;
  const int64_t row = gridDim.z * (int64_t)C;
  const float* p = partial + (int64_t)blockIdx.y * parts * row + blockIdx.z * (int64_t)C + c;
  float s = 0.f;
  if (c < C)
    for (int i = w; i < parts; i += 32) s += p[i * row];
  sums[w][lane] = s;
  __syncthreads();
  if (w == 0 && c < C) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sums[i][lane];
    void* out = blockIdx.z ? out1 : out0;
    const int64_t at = blockIdx.y * (int64_t)C + c;
    if (out_fp32) static_cast<float*>(out)[at] = s;
    else static_cast<T*>(out)[at] = from_f32<T>(s);
  }
}

namespace {
bool multiple(int64_t v, int64_t of) { return v % of == 0; }

// Elements per access: 16 bytes where every row of every tensor starts on such a boundary, else 4 bytes, else one element.
int norm_vector(const NormArgs& a, int e) {
  for (int bytes : {16, 4}) {
    const int v = bytes / e;
    bool ok = v >= 1;
    for (int64_t stride : {(int64_t)a.C, a.x_batch, a.x_row, a.dy_batch, a.dy_row}) ok = ok && multiple(stride, v);
    for (const void* p : {a.x, a.dy, (const void*)a.y, (const void*)a.dx}) ok = ok && multiple((intptr_t)p, bytes);
    const int pb = a.params_fp32 ? (v < 4 ? v : 4) * 4 : bytes;          // bytes of one parameter access
    for (const void* p : {a.gain, a.offset}) ok = ok && multiple((intptr_t)p, pb);
    for (int64_t stride : {a.gain_batch, a.offset_batch}) ok = ok && multiple(stride * (a.params_fp32 ? 4 : e), pb);
    if (ok) return v;
  }
  return 1;
}

template <typename T, int V, int NF, int TPR>
cudaError_t forward(const NormArgs& a, cudaStream_t st) {
  constexpr int G = TPR < 128 ? 128 / TPR : 1;
  layer_norm_kernel<T, V, NF / V, TPR><<<(unsigned)ceil_div64(a.batch * a.rows, G), TPR < 128 ? 128 : TPR, 0, st>>>(a);
  count_launches(1);
  return cudaGetLastError();
}
template <typename T, int V>
cudaError_t forward_v(const NormArgs& a, cudaStream_t st) {
  if (a.C <= 32 * 16) return forward<T, V, 16, 32>(a, st);
  if (a.C <= 32 * 32) return forward<T, V, 32, 32>(a, st);
  if (a.C <= 32 * 64) return forward<T, V, 64, 32>(a, st);
  if (a.C <= 128 * 64) return forward<T, V, 64, 128>(a, st);
  return forward<T, V, 64, 256>(a, st);
}

constexpr int kBwdCols = 16;                       // columns per thread of the backward kernel
int backward_threads(int C) {
  int t = 32;
  while (t * kBwdCols < C) t *= 2;
  return t;
}
template <typename T, int V, int TPR>
cudaError_t backward(const NormArgs& a, int groups, int parts, cudaStream_t st) {
  layer_norm_backward_kernel<T, V, kBwdCols / V, TPR><<<dim3((unsigned)parts, (unsigned)groups), TPR, 0, st>>>(a);
  count_launches(1);
  return cudaGetLastError();
}
template <typename T, int V>
cudaError_t backward_v(const NormArgs& a, int groups, int parts, cudaStream_t st) {
  switch (backward_threads(a.C)) {
    case 32: return backward<T, V, 32>(a, groups, parts, st);
    case 64: return backward<T, V, 64>(a, groups, parts, st);
    case 128: return backward<T, V, 128>(a, groups, parts, st);
    case 256: return backward<T, V, 256>(a, groups, parts, st);
    case 512: return backward<T, V, 512>(a, groups, parts, st);
    default: return backward<T, V, 1024>(a, groups, parts, st);
  }
}
}  // namespace

// CTAs per group of the backward kernel
int norm_backward_parts(int64_t rows, int groups, int C) {
  const int t = backward_threads(C);
  int64_t parts = (int64_t)148 * (t >= 1024 ? 1 : 1024 / t > 16 ? 16 : 1024 / t) / groups;
  if (parts < 1) parts = 1;
  return (int)(rows < parts ? (rows < 1 ? 1 : rows) : parts);
}

cudaError_t launch_layer_norm(int type, const NormArgs& a, cudaStream_t st) {
  const int v = norm_vector(a, elem_bytes(type));
  switch (type) {
    case SVOO_TYPE_BF16: return v == 8 ? forward_v<__nv_bfloat16, 8>(a, st) : v == 2 ? forward_v<__nv_bfloat16, 2>(a, st) : forward_v<__nv_bfloat16, 1>(a, st);
    case SVOO_TYPE_FP16: return v == 8 ? forward_v<__half, 8>(a, st) : v == 2 ? forward_v<__half, 2>(a, st) : forward_v<__half, 1>(a, st);
    default: return v == 4 ? forward_v<float, 4>(a, st) : forward_v<float, 1>(a, st);
  }
}

cudaError_t launch_layer_norm_backward(int type, const NormArgs& a, int groups, int parts, void* dgain, void* doffset, cudaStream_t st) {
  const int v = norm_vector(a, elem_bytes(type));
  cudaError_t e;
  switch (type) {
    case SVOO_TYPE_BF16: e = v == 8 ? backward_v<__nv_bfloat16, 8>(a, groups, parts, st) : v == 2 ? backward_v<__nv_bfloat16, 2>(a, groups, parts, st) : backward_v<__nv_bfloat16, 1>(a, groups, parts, st); break;
    case SVOO_TYPE_FP16: e = v == 8 ? backward_v<__half, 8>(a, groups, parts, st) : v == 2 ? backward_v<__half, 2>(a, groups, parts, st) : backward_v<__half, 1>(a, groups, parts, st); break;
    default: e = v == 4 ? backward_v<float, 4>(a, groups, parts, st) : backward_v<float, 1>(a, groups, parts, st);
  }
  if (e != cudaSuccess || !a.partial) return e;
  const dim3 grid((unsigned)ceil_div(a.C, 32), (unsigned)groups, 2);
  const bool f32 = a.params_fp32 || type == SVOO_TYPE_FP32;
  if (type == SVOO_TYPE_FP16) column_sum_kernel<__half><<<grid, 1024, 0, st>>>(a.partial, parts, a.C, dgain, doffset, f32);
  else column_sum_kernel<__nv_bfloat16><<<grid, 1024, 0, st>>>(a.partial, parts, a.C, dgain, doffset, f32);
  count_launches(1);
  return cudaGetLastError();
}

cudaError_t launch_column_sum(const float* partial, int64_t parts, int64_t C, void* out, int out_type, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div64(C, 32));
  if (out_type == SVOO_TYPE_FP16) column_sum_kernel<__half><<<grid, 1024, 0, st>>>(partial, (int)parts, (int)C, out, nullptr, false);
  else column_sum_kernel<__nv_bfloat16><<<grid, 1024, 0, st>>>(partial, (int)parts, (int)C, out, nullptr, out_type == SVOO_TYPE_FP32);
  count_launches(1);
  return cudaGetLastError();
}

}  // namespace svoo
