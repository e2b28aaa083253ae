// Layer norm over the last dimension, affine or with a modulation per sample (AdaLN), and its gradient.
//
//   mean = sum(x) / C, rstd = 1 / sqrt(sum((x - mean)^2) / C + eps), xhat = (x - mean) rstd
//   y  = xhat g + o            g = gain (or 1 + gain), o = offset: one row of C, or one per sample
//   dx = rstd (w - sum(w) / C - xhat sum(w xhat) / C),  w = dy g;    dg = sum_rows dy xhat,  do = sum_rows dy
//
// Everything between the loads and the stores is in 32 bits.  The variance is taken around the mean from the row in
// registers, and both directions subtract the mean before they scale, so a mean far from zero costs no digits but those of the mean
// itself (a few 2^-24 of the row's largest magnitude).  A row whose values are not all finite comes out NaN.
#include "rows_common.cuh"
#include "tc_common.cuh"

namespace svoo {

// A group of TPR threads walks rows; cp.async.bulk brings the next rows of every group while one is worked on, so that what is
// in flight does not depend on registers or on where the group is in its arithmetic.  Gain and offset lie in shared memory in 32
// bits for the whole walk.  TPR is small: what a row costs besides its elements (two or three sums over the threads, a
// square root, addresses: some 200 instructions a thread) is paid by every thread of it.  (A thread per eight elements, four rows at
// a time, parameters in registers: 243 instructions per 16 bytes, 2.9 TB/s at 32,760 x 5,120.)
constexpr int kRingThreads = 256;
constexpr int kForwardStages = 1;                  // the row is in registers at once, so its place is free again: three cost 15 %
constexpr int kBackwardStages = 2;                 // the row is read twice; three or four are no faster

// kAligned: every row starts on 16 bytes and is whole 16-byte pieces.  Other rows are fetched with the bytes that share their first and
// last 16 (their neighbours', inside the tensor), and the threads of a group take neighbouring elements, one access each.  (16-byte
// pieces read at the row's shift, written back through shared memory: us against this, forward and backward, 32 bits 2 x 4,097 x 1,001
// 17.8 / 13.0 and 32.7 / 26.3, 4,097 x 5,121 64.9 / 40.3 and 104.8 / 54.5; bf16 16.0 / 12.8 and 25.8 / 26.3, 8,194 x 5,121 71.5 / 79.4 and
// 98.4 / 90.9, 32,760 x 1,537 68.8 / 76.1 and 151.8 / 140.1: long 16-bit rows forward are 10 % slower for it, the rest is faster, and one form
// serves all.)
struct RingLayout {
  int columns, row, ring, bars, total;            // columns rounded up to whole pieces, bytes of a row's place; offsets
  __host__ __device__ RingLayout(int C, int e, int param_rows, int row_tensors, int groups, int stages, bool aligned) {
    columns = (C + 7) & ~7;
    row = aligned ? C * e : ((C * e + 15) & ~15) + 16;
    ring = param_rows * columns * 4;
    bars = ring + groups * stages * row_tensors * row;
    total = bars + groups * stages * 8 + 16;
  }
};

// two 32-bit numbers
__device__ __forceinline__ uint64_t f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float lo2(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi2(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }

// the elements of a 16-byte piece, in pairs
template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, uint64_t (&p)[8 / sizeof(T)]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if constexpr (sizeof(T) == 4) {
    p[0] = (uint64_t)w[1] << 32 | w[0];
    p[1] = (uint64_t)w[3] << 32 | w[2];
  } else {
    const Vec<T, 8>& v = *reinterpret_cast<const Vec<T, 8>*>(w);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = f2(to_f32(v.v[2 * i]), to_f32(v.v[2 * i + 1]));
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const uint64_t (&p)[8 / sizeof(T)]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      w[i] = (uint32_t)(i & 1 ? p[i / 2] >> 32 : p[i / 2]);
    } else {
      Vec<T, 2> v;
      v.v[0] = from_f32<T>(lo2(p[i]));
      v.v[1] = from_f32<T>(hi2(p[i]));
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int TPR>
__device__ __forceinline__ void group_sync(int group) {
  if (TPR == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(TPR) : "memory");
}
// N sums over a group, the same in every thread.  `slot` [warps][N] is written again only behind a barrier that every
// thread reaches when it has read it.
template <int TPR, int N>
__device__ __forceinline__ void group_sums(float (&s)[N], float (*slot)[N], int group) {
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = warp_sum(s[i]);
  if (TPR == 32) return;
  if (threadIdx.x % 32 == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) slot[threadIdx.x % TPR / 32][i] = s[i];
  }
  group_sync<TPR>(group);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i] = slot[0][i];
#pragma unroll
    for (int w = 1; w < TPR / 32; ++w) s[i] += slot[w][i];
  }
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// What a bulk copy brings of a row, to `at` bytes behind its place in shared memory.
struct RowCopy {
  const void* src;
  uint32_t bytes, at;
};
// The copy for a row whose first byte is to lie where it lies in its 16 bytes.  [lo, hi) is the tensor: where the row's outer 16
// bytes reach beyond it, its elements in them are copied here, one by one (the first and the last row of all).
template <typename T, bool kAligned>
__device__ __forceinline__ RowCopy plan_row(unsigned char* place, const T* src, int C, const void* lo, const void* hi) {
  if (kAligned) return {src, (uint32_t)(C * sizeof(T)), 0};
  const uintptr_t first = (uintptr_t)src, last = first + C * sizeof(T);
  uintptr_t from = first & ~(uintptr_t)15, to = (last + 15) & ~(uintptr_t)15;
  const uintptr_t base = from;
  if (from < (uintptr_t)lo) {
    from += 16;
    for (uintptr_t p = first; p < last && p < from; p += sizeof(T)) *reinterpret_cast<T*>(place + (p - base)) = *reinterpret_cast<const T*>(p);
  }
  if (to > (uintptr_t)hi && to > from) {
    to -= 16;
    for (uintptr_t p = first > to ? first : to; p < last; p += sizeof(T)) *reinterpret_cast<T*>(place + (p - base)) = *reinterpret_cast<const T*>(p);
  }
  return {(const void*)from, (uint32_t)(to - from), (uint32_t)(from - base)};
}
__device__ __forceinline__ void start_copy(unsigned char* place, const RowCopy& c, uint32_t bar) {
  if (c.bytes) bulk_load(smem_u32(place) + c.at, c.src, c.bytes, bar);
}
template <typename T>
__device__ __forceinline__ int shift_of(const T* row) { return (int)((uintptr_t)row & 15); }
// Piece i of thread t of TPR: V elements.  kAligned: 16 bytes, piece i TPR + t of the row; else element k is column (V i + k) TPR + t.
template <typename T, int TPR>
__device__ __forceinline__ int column_of(int i, int k, int t) { return (16 / (int)sizeof(T) * i + k) * TPR + t; }
// The pairs of a piece of a row that lies at `shift` in its place; zeros behind the last column.
template <typename T, bool kAligned, int TPR>
__device__ __forceinline__ void read_piece(const unsigned char* place, int shift, int i, int t, int C, uint64_t (&p)[8 / sizeof(T)]) {
  if constexpr (kAligned) {
    unpack<T>(reinterpret_cast<const uint4*>(place)[i * TPR + t], p);
  } else {
    const T* row = reinterpret_cast<const T*>(place + shift);
#pragma unroll
    for (int k = 0; k < 8 / (int)sizeof(T); ++k) {
      const int c = column_of<T, TPR>(i, 2 * k, t);
      p[k] = f2(c < C ? to_f32(row[c]) : 0.f, c + TPR < C ? to_f32(row[c + TPR]) : 0.f);
    }
  }
}
// Pairs 2 j and 2 j + 1 of the parameters of a piece
template <typename T, bool kAligned, int TPR>
__device__ __forceinline__ ulonglong2 read_param(const float* param, int i, int j, int t, int C) {
  if constexpr (kAligned) {
    return reinterpret_cast<const ulonglong2*>(param + (i * TPR + t) * (16 / (int)sizeof(T)))[j];
  } else {
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = column_of<T, TPR>(i, 4 * j + k, t);
      v[k] = c < C ? param[c] : 0.f;
    }
    return make_ulonglong2(f2(v[0], v[1]), f2(v[2], v[3]));
  }
}
template <typename T, bool kAligned, int TPR>
__device__ __forceinline__ void write_piece(T* row, int i, int t, int C, const uint64_t (&p)[8 / sizeof(T)]) {
  if constexpr (kAligned) {
    reinterpret_cast<uint4*>(row)[i * TPR + t] = pack<T>(p);
  } else {
#pragma unroll
    for (int k = 0; k < 16 / (int)sizeof(T); ++k) {
      const int c = column_of<T, TPR>(i, k, t);
      if (c < C) row[c] = from_f32<T>(k & 1 ? hi2(p[k / 2]) : lo2(p[k / 2]));
    }
  }
}

// Row r of the walk of sample `sample` (per_sample) or of all samples: pointer offset in a tensor of these strides
__device__ __forceinline__ int64_t row_offset(const NormArgs& a, bool per_sample, int sample, int r, int64_t batch_stride, int64_t row_stride) {
  if (per_sample) return sample * batch_stride + r * row_stride;
  if (a.batch == 1) return r * row_stride;
  const int b = (int)((unsigned)r / (unsigned)a.rows);
  return b * batch_stride + (r - b * a.rows) * row_stride;
}

// gain (1 + gain, 1) and offset (0) of a sample to shared memory, 32 bits; whole pieces, with `none` behind the last column
template <typename T>
__device__ __forceinline__ void stage_param(const NormArgs& a, int columns, const void* p, int64_t at, float add, float none, float* dst) {
  for (int c = threadIdx.x; c < columns; c += kRingThreads) {
    float v = none;
    if (p && c < a.C) v = add + (a.params_fp32 ? static_cast<const float*>(p)[at + c] : to_f32(static_cast<const T*>(p)[at + c]));
    dst[c] = v;
  }
}

// After a wait that expired, copies in flight land before the CTA ends.
__device__ __forceinline__ void leave(uint32_t bars, int stages, int issued, int t, volatile int* abort_flag, int* status) {
  __syncthreads();
  if (!*abort_flag) return;
  if (t == 0)
    for (int i = 0; i < stages && i < issued; ++i) tc::mbar_drain(bars + 8 * i, ((issued - 1 - i) / stages) & 1);
  if (threadIdx.x == 0) atomicExch(status, 1);
  __syncthreads();
}

template <typename T, int NV, int TPR, bool kAligned>
__global__ void __launch_bounds__(kRingThreads) layer_norm_ring_kernel(const NormArgs a) {
  constexpr int P = 8 / (int)sizeof(T), V = 2 * P, G = kRingThreads / TPR;    // pairs and elements of a piece, groups
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float slots[2][G][TPR / 32][1];
  const int stages = a.stages;
  const RingLayout lay(a.C, sizeof(T), 2, 1, G, stages, kAligned);
  float* gain = reinterpret_cast<float*>(smem);
  float* off = gain + lay.columns;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + lay.bars + G * stages * 8);
  const int group = threadIdx.x / TPR, t = threadIdx.x % TPR, nvec = (a.C + V - 1) / V;
  const bool per_sample = gridDim.y > 1;
  const int n = (int)(per_sample ? a.rows : a.batch * a.rows), step = gridDim.x * G, first = blockIdx.x * G + group;
  unsigned char* ring = smem + lay.ring + group * stages * lay.row;
  const uint32_t bars = smem_u32(smem + lay.bars) + group * stages * 8;
  if (t == 0) {
    for (int i = 0; i < stages; ++i) tc::mbar_init(bars + 8 * i, 1);
    if (threadIdx.x == 0) *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_trigger();
  pdl_wait();
  auto row_of = [&](int r) { return static_cast<const T*>(a.x) + row_offset(a, per_sample, blockIdx.y, r, a.x_batch, a.x_row); };
  auto fetch = [&](int r, int s) {
    const RowCopy c = plan_row<T, kAligned>(ring + s * lay.row, row_of(r), a.C, a.x, a.x_end);
    if (!kAligned) tc::fence_async_proxy();                // elements that plan_row stored here for an earlier row come before this copy
    tc::mbar_expect_tx(bars + 8 * s, c.bytes);
    start_copy(ring + s * lay.row, c, bars + 8 * s);
  };
  int ahead = first, issued = 0;                           // the next row to fetch, fetches so far (thread 0 of the group)
  if (t == 0)
    for (; issued < stages && ahead < n; ++issued, ahead += step) fetch(ahead, issued);
  stage_param<T>(a, lay.columns, a.gain, blockIdx.y * a.gain_batch, a.plus_one ? 1.f : 0.f, 1.f, gain);
  stage_param<T>(a, lay.columns, a.offset, blockIdx.y * a.offset_batch, 0.f, 0.f, off);
  __syncthreads();
  const float inv_c = 1.f / a.C;
  int s = 0, phase = 0;
  bool ok = true;
  for (int r = first; r < n; r += step) {
    // a wait that expires ends the stores and the fetches, not the walk: every thread meets every barrier
    ok = tc::mbar_wait(bars + 8 * s, phase, abort_flag) && ok;
    uint64_t d[NV][P], sum = 0;
    const int shift = kAligned ? 0 : shift_of(row_of(r));
#pragma unroll
    for (int i = 0; i < NV; ++i) {                         // skipping empty pieces costs more here (4,097 x 7,777 in 32 bits: 52.7 -> 67.7 us)
      if (!kAligned || i * TPR + t < nvec) {
        read_piece<T, kAligned, TPR>(ring + s * lay.row, shift, i, t, a.C, d[i]);
#pragma unroll
        for (int k = 0; k < P; ++k) sum = add2(sum, d[i][k]);
      }
    }
    float one[1] = {lo2(sum) + hi2(sum)};
    group_sums<TPR, 1>(one, slots[0][group], group);
    if (TPR == 32) __syncwarp();
    // the row is in everybody's registers: its place takes another
    if (t == 0 && ahead < n && ok) {
      fetch(ahead, s);
      ahead += step;
      ++issued;
    }
    const float mean = one[0] * inv_c;
    const uint64_t minus = f2(-mean, -mean);
    sum = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!kAligned || i * TPR + t < nvec) {
#pragma unroll
        for (int k = 0; k < P; ++k) d[i][k] = add2(d[i][k], minus);
        if constexpr (!kAligned) {
#pragma unroll
          for (int k = 0; k < P; ++k) {
            const int c = column_of<T, TPR>(i, 2 * k, t);
            d[i][k] = f2(c < a.C ? lo2(d[i][k]) : 0.f, c + TPR < a.C ? hi2(d[i][k]) : 0.f);
          }
        }
#pragma unroll
        for (int k = 0; k < P; ++k) sum = fma2(d[i][k], d[i][k], sum);
      }
    }
    one[0] = lo2(sum) + hi2(sum);
    group_sums<TPR, 1>(one, slots[1][group], group);
    const float rstd = 1.f / sqrtf(one[0] * inv_c + a.eps);
    const int64_t row = per_sample ? blockIdx.y * a.rows + r : r;
    if (t == 0 && a.mean && ok) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    const uint64_t rs = f2(rstd, rstd);
    T* y = static_cast<T*>(a.y) + row * a.C;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!kAligned || i * TPR + t < nvec) {
#pragma unroll
        for (int k = 0; k < P; k += 2) {
          const ulonglong2 gv = read_param<T, kAligned, TPR>(gain, i, k / 2, t, a.C), ov = read_param<T, kAligned, TPR>(off, i, k / 2, t, a.C);
          d[i][k] = fma2(mul2(d[i][k], rs), gv.x, ov.x);
          d[i][k + 1] = fma2(mul2(d[i][k + 1], rs), gv.y, ov.y);
        }
        if (ok) write_piece<T, kAligned, TPR>(y, i, t, a.C, d[i]);
      }
    }
    if (++s == stages) s = 0, phase ^= 1;
  }
  leave(bars, stages, issued, t, abort_flag, a.status);
}

// x and dy rows come in together.  A thread's columns are the same in every row: their sums stay in its registers.
template <typename T, int NV, int TPR, bool kAligned>
__global__ void __launch_bounds__(kRingThreads) layer_norm_backward_ring_kernel(const NormArgs a) {
  constexpr int P = 8 / (int)sizeof(T), V = 2 * P, G = kRingThreads / TPR;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float slots[2][G][TPR / 32][2];
  const int stages = a.stages;
  const RingLayout lay(a.C, sizeof(T), 1, 2, G, stages, kAligned);
  float* gain = reinterpret_cast<float*>(smem);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + lay.bars + G * stages * 8);
  const int group = threadIdx.x / TPR, t = threadIdx.x % TPR, nvec = (a.C + V - 1) / V;
  const bool per_sample = gridDim.y > 1;
  const int n = (int)(per_sample ? a.rows : a.batch * a.rows), step = gridDim.x * G, first = blockIdx.x * G + group;
  unsigned char* ring = smem + lay.ring + group * stages * 2 * lay.row;
  const uint32_t bars = smem_u32(smem + lay.bars) + group * stages * 8;
  if (t == 0) {
    for (int i = 0; i < stages; ++i) tc::mbar_init(bars + 8 * i, 1);
    if (threadIdx.x == 0) *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_trigger();
  pdl_wait();
  auto x_of = [&](int r) { return static_cast<const T*>(a.x) + row_offset(a, per_sample, blockIdx.y, r, a.x_batch, a.x_row); };
  auto dy_of = [&](int r) { return static_cast<const T*>(a.dy) + row_offset(a, per_sample, blockIdx.y, r, a.dy_batch, a.dy_row); };
  auto fetch = [&](int r, int s) {
    unsigned char *px = ring + s * 2 * lay.row, *pd = px + lay.row;
    const RowCopy cx = plan_row<T, kAligned>(px, x_of(r), a.C, a.x, a.x_end), cd = plan_row<T, kAligned>(pd, dy_of(r), a.C, a.dy, a.dy_end);
    if (!kAligned) tc::fence_async_proxy();                // as in the forward kernel
    tc::mbar_expect_tx(bars + 8 * s, cx.bytes + cd.bytes);
    start_copy(px, cx, bars + 8 * s);
    start_copy(pd, cd, bars + 8 * s);
  };
  int ahead = first, issued = 0;
  if (t == 0)
    for (; issued < stages && ahead < n; ++issued, ahead += step) fetch(ahead, issued);
  stage_param<T>(a, lay.columns, a.gain, blockIdx.y * a.gain_batch, a.plus_one ? 1.f : 0.f, 1.f, gain);
  __syncthreads();
  const float inv_c = 1.f / a.C;
  uint64_t dg[NV][P], dof[NV][P];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < P; ++k) dg[i][k] = dof[i][k] = 0;
  int s = 0, phase = 0;
  bool ok = true;
  const int64_t sample_row = per_sample ? blockIdx.y * a.rows : 0;
  float mean = 0.f, rstd = 0.f;
  if (first < n) mean = a.mean_in[sample_row + first], rstd = a.rstd_in[sample_row + first];
  for (int r = first, turn = 0; r < n; r += step, turn ^= 1) {
    // a wait that expires ends the stores and the fetches, not the walk: every thread meets every barrier
    ok = tc::mbar_wait(bars + 8 * s, phase, abort_flag) && ok;
    const unsigned char *xs = ring + s * 2 * lay.row, *ds = xs + lay.row;
    const int x_shift = kAligned ? 0 : shift_of(x_of(r)), d_shift = kAligned ? 0 : shift_of(dy_of(r));
    const uint64_t rs = f2(rstd, rstd), minus = f2(-mean, -mean);      // xhat = (x - mean) rstd, as the forward call has it
    uint64_t s1 = 0, s2 = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (kAligned ? i * TPR + t < nvec : i * V * TPR < a.C) {
        uint64_t x[P], d[P];
        read_piece<T, kAligned, TPR>(xs, x_shift, i, t, a.C, x);
        read_piece<T, kAligned, TPR>(ds, d_shift, i, t, a.C, d);
#pragma unroll
        for (int k = 0; k < P; ++k) {
          const ulonglong2 gv = read_param<T, kAligned, TPR>(gain, i, k / 2, t, a.C);
          const uint64_t h = mul2(add2(x[k], minus), rs), w = mul2(d[k], k & 1 ? gv.y : gv.x);
          dg[i][k] = fma2(d[k], h, dg[i][k]);
          dof[i][k] = add2(dof[i][k], d[k]);
          s1 = add2(s1, w);
          s2 = fma2(w, h, s2);
        }
      }
    }
    float sums[2] = {lo2(s1) + hi2(s1), lo2(s2) + hi2(s2)};
    group_sums<TPR, 2>(sums, slots[turn][group], group);
    // dx = rstd (w - s1 - (x - mean) (rstd s2)), s1 and s2 over C
    const float m1 = sums[0] * inv_c, m2 = sums[1] * inv_c * rstd;
    const uint64_t a2 = f2(-m2, -m2), a1 = f2(-m1, -m1);
    T* dx = static_cast<T*>(a.dx) + (sample_row + r) * a.C;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (kAligned ? i * TPR + t < nvec : i * V * TPR < a.C) {
        uint64_t x[P], d[P];
        read_piece<T, kAligned, TPR>(xs, x_shift, i, t, a.C, x);
        read_piece<T, kAligned, TPR>(ds, d_shift, i, t, a.C, d);
#pragma unroll
        for (int k = 0; k < P; ++k) {
          const ulonglong2 gv = read_param<T, kAligned, TPR>(gain, i, k / 2, t, a.C);
          d[k] = mul2(fma2(add2(x[k], minus), a2, fma2(d[k], k & 1 ? gv.y : gv.x, a1)), rs);
        }
        if (ok) write_piece<T, kAligned, TPR>(dx, i, t, a.C, d);
      }
    }
    group_sync<TPR>(group);                                // the row has been read: its place takes another
    if (t == 0 && ahead < n && ok) {
      fetch(ahead, s);
      ahead += step;
      ++issued;
    }
    if (r + step < n) mean = a.mean_in[sample_row + r + step], rstd = a.rstd_in[sample_row + r + step];
    if (++s == stages) s = 0, phase ^= 1;
  }
  if (a.partial) {
    // the groups of the CTA are added in shared memory, in order
    __syncthreads();
    float* acc = reinterpret_cast<float*>(smem);           // [dg, do][columns]: fits the gain's place and the ring behind it
    for (int k = 0; k < G; ++k) {
      if (k == group) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = i * TPR + t;
          if constexpr (!kAligned) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const int col = column_of<T, TPR>(i, j, t);
              const float u = j & 1 ? hi2(dg[i][j / 2]) : lo2(dg[i][j / 2]), w = j & 1 ? hi2(dof[i][j / 2]) : lo2(dof[i][j / 2]);
              if (col < a.C) {
                acc[col] = k > 0 ? acc[col] + u : u;
                acc[lay.columns + col] = k > 0 ? acc[lay.columns + col] + w : w;
              }
            }
          } else if (c < nvec) {
            ulonglong2* p = reinterpret_cast<ulonglong2*>(acc + c * V);
            ulonglong2* q = reinterpret_cast<ulonglong2*>(acc + lay.columns + c * V);
#pragma unroll
            for (int j = 0; j < P; j += 2) {
              ulonglong2 u = make_ulonglong2(dg[i][j], dg[i][j + 1]), w = make_ulonglong2(dof[i][j], dof[i][j + 1]);
              if (k > 0) {
                const ulonglong2 pu = p[j / 2], qw = q[j / 2];
                u = make_ulonglong2(add2(pu.x, u.x), add2(pu.y, u.y));
                w = make_ulonglong2(add2(qw.x, w.x), add2(qw.y, w.y));
              }
              p[j / 2] = u;
              q[j / 2] = w;
            }
          }
        }
      }
      __syncthreads();
    }
    float* out = a.partial + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * a.C;
    const bool whole = !*abort_flag;                       // rows are missing after a wait that expired
    for (int c = threadIdx.x; c < 2 * a.C; c += kRingThreads) out[c] = whole ? acc[c < a.C ? c : c - a.C + lay.columns] : NAN;
  }
  leave(bars, stages, issued, t, abort_flag, a.status);
}

// out0[group][c] = sum_p partial[group][p][0][c], out1 the same of [1] (gridDim.z outputs in all): 32 columns per CTA, 32
// warps over the parts.
template <typename T>
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ partial, int parts, int C, void* out0, void* out1,
                                                          bool out_fp32) {
  pdl_trigger();
  pdl_wait();
  __shared__ float sums[32][33];
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  const int c = blockIdx.x * 32 + lane;
  const int64_t row = gridDim.z * (int64_t)C;
  const float* p = partial + (int64_t)blockIdx.y * parts * row + blockIdx.z * (int64_t)C + c;
  float s = 0.f;
  if (c < C) {
#pragma unroll 4
    for (int i = w; i < parts; i += 32) s += p[i * row];
  }
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
// Threads per row of the ring kernels: at most 80 elements a thread forward (75,600 x 5,120: 128 threads 306 us, 64 threads
// 284); backward 80 bytes a thread and tensor (40 elements with two sums each; 32-bit rows take twice the place in the ring, and
// twice the threads keep two CTAs on an SM: 2 x 4,097 x 1,000 22.5 us, with half the threads 35.1; rows that are not aligned count as 32-bit ones, bf16 2 x 4,097 x 1,001 26.3, half 58.7).
// More than 8,192 columns: 256 threads a row (a CTA per row straight from global memory, backward with 1,024 threads that walk rows:
// 8,194 x 16,384 167 us forward, here 158, backward 587, here 211; 4,097 x 10,001 335 and 301, here 72 and 133).
int ring_threads_forward(int C) { return C <= 32 * 64 ? 32 : C <= 64 * 80 ? 64 : C <= 128 * 64 ? 128 : 256; }
int ring_threads_backward(int C, int e) { return C * e <= 32 * 80 ? 32 : C * e <= 64 * 80 ? 64 : C * e <= 128 * 80 ? 128 : 256; }
// CTAs of a kernel that the SMs hold at this much shared memory; the answer for the last size is kept.
constexpr int kRingSmem = 230000;                  // above what any layout needs (197,000: 16,384 columns)
template <typename Kernel>
cudaError_t resident(Kernel* kernel, int smem, int64_t& kept, int& ctas) {
  const int64_t known = __atomic_load_n(&kept, __ATOMIC_RELAXED);
  if (known >> 8 == smem) {
    ctas = (int)(known & 255) * 148;
    return cudaSuccess;
  }
  int per_sm = 0;
  cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kRingThreads, smem);
  if (e != cudaSuccess) return e;
  if (per_sm < 1) return cudaErrorInvalidConfiguration;
  ctas = per_sm * 148;
  __atomic_store_n(&kept, (int64_t)smem << 8 | per_sm, __ATOMIC_RELAXED);
  return cudaSuccess;
}
template <typename Kernel>
cudaError_t launch_ring(Kernel* kernel, const NormArgs& a, int64_t ctas, int groups, int smem, cudaStream_t st) {
  count_launches(1);
  return launch_pdl(kernel, dim3((unsigned)ctas, (unsigned)groups), dim3(kRingThreads), smem, st, a);
}
template <typename T, bool kAligned, int NV, int TPR>
cudaError_t forward_ring(NormArgs a, cudaStream_t st) {
  constexpr int G = kRingThreads / TPR;
  static int64_t kept;
  const int samples = a.gain_batch || a.offset_batch ? (int)a.batch : 1;
  a.stages = kForwardStages;
  // where an SM holds one CTA of one row anyway, the next row is fetched a row earlier: 4,097 x 12,288 in 32 bits 85.7 -> 75.2 us (two
  // CTAs with one row each are better: bf16 4,097 x 10,001 72 against 90)
  if (G == 1 && RingLayout(a.C, sizeof(T), 2, 1, G, 1, kAligned).total > 113000 && RingLayout(a.C, sizeof(T), 2, 1, G, 2, kAligned).total <= kRingSmem)
    a.stages = 2;
  const int smem = RingLayout(a.C, sizeof(T), 2, 1, G, a.stages, kAligned).total;
  int fit = 0;
  static uint64_t done;
  cudaError_t e = allow_smem(&layer_norm_ring_kernel<T, NV, TPR, kAligned>, kRingSmem, done);
  if (e == cudaSuccess) e = resident(&layer_norm_ring_kernel<T, NV, TPR, kAligned>, smem, kept, fit);
  if (e != cudaSuccess) return e;
  const int64_t jobs = ceil_div64(samples > 1 ? a.rows : a.batch * a.rows, G), ctas = ceil_div64(fit, samples);
  return launch_ring(&layer_norm_ring_kernel<T, NV, TPR, kAligned>, a, jobs < ctas ? jobs : ctas, samples, smem, st);
}
template <typename T, bool kAligned>
cudaError_t forward_ring_t(const NormArgs& a, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T), Q = 8 / V;          // pieces per 8 elements
  const int tpr = ring_threads_forward(a.C), nv = ceil_div(ceil_div(a.C, V), tpr);
  if (tpr == 32) {
    if (nv <= 2 * Q) return forward_ring<T, kAligned, 2 * Q, 32>(a, st);
    if (nv <= 4 * Q) return forward_ring<T, kAligned, 4 * Q, 32>(a, st);
    if (nv <= 6 * Q) return forward_ring<T, kAligned, 6 * Q, 32>(a, st);
    return forward_ring<T, kAligned, 8 * Q, 32>(a, st);
  }
  if (tpr == 64) return nv <= 6 * Q ? forward_ring<T, kAligned, 6 * Q, 64>(a, st) : forward_ring<T, kAligned, 10 * Q, 64>(a, st);
  return tpr == 128 ? forward_ring<T, kAligned, 8 * Q, 128>(a, st) : forward_ring<T, kAligned, 8 * Q, 256>(a, st);
}
template <typename T, bool kAligned, int NV, int TPR>
cudaError_t backward_ring(NormArgs a, int groups, int parts, cudaStream_t st) {
  constexpr int G = kRingThreads / TPR;
  a.stages = kBackwardStages;
  if (RingLayout(a.C, sizeof(T), 1, 2, G, a.stages, kAligned).total > kRingSmem) a.stages = 1;       // 32-bit rows of more than 11,490 columns
  static uint64_t done;
  const cudaError_t e = allow_smem(&layer_norm_backward_ring_kernel<T, NV, TPR, kAligned>, kRingSmem, done);
  if (e != cudaSuccess) return e;
  return launch_ring(&layer_norm_backward_ring_kernel<T, NV, TPR, kAligned>, a, parts, groups, RingLayout(a.C, sizeof(T), 1, 2, G, a.stages, kAligned).total, st);
}
template <typename T, bool kAligned>
cudaError_t backward_ring_t(const NormArgs& a, int groups, int parts, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T), Q = 8 / V;
  const int tpr = ring_threads_backward(a.C, kAligned ? sizeof(T) : 4);
  const int nv = ceil_div(ceil_div(a.C, V), tpr);
  // up to 128 threads a row, 80 bytes a thread: 32-bit rows and those that count as such stay within 3 Q pieces
  if constexpr (kAligned && sizeof(T) == 2) {
    if (nv > 3 * Q) {
      switch (tpr) {
        case 32: return backward_ring<T, kAligned, 5 * Q, 32>(a, groups, parts, st);
        case 64: return backward_ring<T, kAligned, 5 * Q, 64>(a, groups, parts, st);
        case 128: return backward_ring<T, kAligned, 5 * Q, 128>(a, groups, parts, st);
        default: break;
      }
    }
  }
  switch (tpr) {
    case 32: return backward_ring<T, kAligned, 3 * Q, 32>(a, groups, parts, st);
    case 64: return backward_ring<T, kAligned, 3 * Q, 64>(a, groups, parts, st);
    case 128: return backward_ring<T, kAligned, 3 * Q, 128>(a, groups, parts, st);
    default: break;
  }
  if (nv <= 3 * Q) return backward_ring<T, kAligned, 3 * Q, 256>(a, groups, parts, st);
  return nv <= 5 * Q ? backward_ring<T, kAligned, 5 * Q, 256>(a, groups, parts, st) : backward_ring<T, kAligned, 8 * Q, 256>(a, groups, parts, st);
}
// Whether all rows are whole 16-byte pieces.  (The strides of parameters do not matter to the ring kernels.)
bool ring_aligned(const NormArgs& a, int e) {
  for (int64_t stride : {(int64_t)a.C, a.x_batch, a.x_row, a.dy_batch, a.dy_row})
    if (stride * e % 16) return false;
  for (const void* p : {a.x, a.dy, (const void*)a.y, (const void*)a.dx})
    if ((uintptr_t)p % 16) return false;
  return true;
}
#define SVOO_RING(fn, aligned, ...) \
  (type == SVOO_TYPE_BF16 ? (aligned ? fn<__nv_bfloat16, true>(__VA_ARGS__) : fn<__nv_bfloat16, false>(__VA_ARGS__)) \
   : type == SVOO_TYPE_FP16 ? (aligned ? fn<__half, true>(__VA_ARGS__) : fn<__half, false>(__VA_ARGS__))             \
                            : (aligned ? fn<float, true>(__VA_ARGS__) : fn<float, false>(__VA_ARGS__)))
}  // namespace

// CTAs per group of the backward kernel: what the SMs hold at once, at most one per row of every group, as many as for 32-bit rows
// whatever the type, so that the workspace does not depend on it.
int norm_backward_parts(int64_t rows, int groups, int C) {
  int64_t parts = (int64_t)148 * (C <= 8192 ? 2 : 1) / groups, jobs = ceil_div64(rows, kRingThreads / ring_threads_backward(C, 4));
  if (parts > jobs) parts = jobs;
  return parts < 1 ? 1 : (int)parts;
}
int64_t norm_backward_bytes(int64_t batch, int64_t rows, int groups, int C) {
  return (int64_t)groups * norm_backward_parts(groups > 1 ? rows : batch * rows, groups, C) * 2 * C * 4;
}

cudaError_t launch_layer_norm(int type, const NormArgs& a, cudaStream_t st) {
  const int e = elem_bytes(type);
  return SVOO_RING(forward_ring_t, ring_aligned(a, e), a, st);
}

cudaError_t launch_layer_norm_backward(int type, const NormArgs& a, int groups, void* dgain, void* doffset, cudaStream_t st) {
  const bool aligned = ring_aligned(a, elem_bytes(type));
  const int parts = norm_backward_parts(groups > 1 ? a.rows : a.batch * a.rows, groups, a.C);
  const cudaError_t e = SVOO_RING(backward_ring_t, aligned, a, groups, parts, st);
  if (e != cudaSuccess || !a.partial) return e;
  const dim3 grid((unsigned)ceil_div(a.C, 32), (unsigned)groups, 2);
  const bool f32 = a.params_fp32 || type == SVOO_TYPE_FP32;
  count_launches(1);
  return launch_pdl(type == SVOO_TYPE_FP16 ? column_sum_kernel<__half> : column_sum_kernel<__nv_bfloat16>, grid, dim3(1024), 0, st,
                    (const float*)a.partial, parts, a.C, dgain, doffset, f32);
}

cudaError_t launch_column_sum(const float* partial, int64_t parts, int64_t C, void* out, int out_type, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div64(C, 32));
  count_launches(1);
  return launch_pdl(out_type == SVOO_TYPE_FP16 ? column_sum_kernel<__half> : column_sum_kernel<__nv_bfloat16>, grid, dim3(1024), 0, st,
                    partial, (int)parts, (int)C, out, (void*)nullptr, out_type == SVOO_TYPE_FP32);
}

}  // namespace svoo
