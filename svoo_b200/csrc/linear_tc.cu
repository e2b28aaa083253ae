// Matrix product of e4m3 operands with 32-bit block scales:
//
//   y[m, n] = act( sum_kb sa[kb, m] sb[n, kb] ( sum_{k in kb} a[m, k] b[n, k] ) + bias[n] ),     kb: 128 consecutive k
//
// a [M, K], b [N, K] row-major.  sb has one scale per 128 x 128 block of b (weights), or one per row and kb (kRowScales:
// the product of two token-major operands in the gradient of a weight).
//
// The tensor core sums the 128 products of a block (four K = 32 steps of tcgen05.mma kind::f8f6f4, 32-bit accumulators in
// TMEM); a scale that changes from block to block cannot be applied there, so every block starts a fresh accumulator and
// the epilogue threads add it to their running sums in registers, times sa sb.  Two accumulators alternate.
//
//   warp 0       TMA producer: 128 x 128 bytes of a, 256 x 128 of b per stage (128-byte swizzle), four stages
//   warp 1       MMA issuer: M 128, N 256, K 32
//   warps 4-11   thread r of each group of four warps owns row r (TMEM lane r) and 128 columns, one scale block of b: the
//                factor sa sb is one number per thread and block.  The sums (128 registers) are moved between warpgroups by
//                setmaxnreg.  Rows leave through shared memory, so that stores are whole 128-byte lines.
//
// Every mbarrier wait is bounded; on expiry the CTA sets the status word of the device and leaves.
#include <cuda_fp8.h>

#include "rows_common.cuh"
#include "tc_common.cuh"

namespace svoo {
namespace tc {

constexpr int kLinThreads = 384;
constexpr int kLinRegsSums = 216, kLinRegsService = 72;       // 2 x 128 x 216 + 128 x 72 = 384 x 168
constexpr int kLinM = 128, kLinN = 256;
constexpr int kLinStages = 4;
constexpr int kLinABytes = kLinM * 128, kLinBBytes = kLinN * 128, kLinStageBytes = kLinABytes + kLinBBytes;
constexpr int kLinOutBytes = 32 * 128;                        // staging of one warp: 32 rows x 128 bytes
constexpr int kLinSmemData = kLinStages * kLinStageBytes + 8 * kLinOutBytes;
constexpr int kLinSmemBytes = kLinSmemData + 256 + 1024;
enum { LIN_FULL = 0, LIN_EMPTY = LIN_FULL + kLinStages, LIN_ACC_FULL = LIN_EMPTY + kLinStages, LIN_ACC_EMPTY = LIN_ACC_FULL + 2,
       LIN_BARS = LIN_ACC_EMPTY + 2 };
constexpr int kLinGroupM = 16;                                // row tiles that sweep the columns together

__device__ int g_linear_status;                               // != 0 after a kernel gave up on a bounded wait

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
};

// D[tmem] (+)= A[smem] B[smem]^T, e4m3
__device__ __forceinline__ void umma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Instruction descriptor of kind::f8f6f4: D fp32, A and B e4m3, both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// 32 columns of this thread's row.  Load and wait are one statement: the registers are never live between the two.
__device__ __forceinline__ void load_columns(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
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

// y / 2 (1 + tanh u) = y / (1 + exp(-2 u)), u = sqrt(2 / pi) (y + 0.044715 y^3)
__device__ __forceinline__ float gelu_tanh(float y) {
  const float u = 0.7978845608028654f * (y + 0.044715f * y * y * y);
  return __fdividef(y, 1.f + fast_exp2(-2.f * 1.4426950408889634f * u));
}

__device__ __forceinline__ float load_bias(const LinearArgs& a, int n) {
  if (n >= a.N) return 0.f;
  if (a.bias_type == SVOO_TYPE_FP32) return __ldg(static_cast<const float*>(a.bias) + n);
  if (a.bias_type == SVOO_TYPE_BF16) return to_f32(__ldg(static_cast<const __nv_bfloat16*>(a.bias) + n));
  return to_f32(__ldg(static_cast<const __half*>(a.bias) + n));
}

struct LinTile {
  int tm, tn;
  // tiles in groups of kLinGroupM row tiles; a group goes through the column tiles, its row tiles fastest
  __device__ __forceinline__ LinTile(int t, int tiles_m, int tiles_n) {
    const int group = t / (kLinGroupM * tiles_n), first = group * kLinGroupM;
    const int rows = tiles_m - first < kLinGroupM ? tiles_m - first : kLinGroupM;
    const int in = t - group * kLinGroupM * tiles_n;
    tn = in / rows;
    tm = first + in - tn * rows;
  }
};

// 32 rows x 128 bytes of one warp, staged swizzled (16-byte piece p of row r at p ^ (r & 7)), to out rows row0 + r,
// elements [n0, n0 + 128 / sizeof(T)) of which those below `limit` exist.
template <typename T>
__device__ __forceinline__ void store_rows(const unsigned char* stage, T* out, int64_t pitch, int row0, int M, int n0, int limit, int lane) {
  constexpr int E = 16 / (int)sizeof(T), COLS = 128 / (int)sizeof(T);
  const bool wide = (pitch * (int)sizeof(T)) % 16 == 0 && (uintptr_t)out % 16 == 0;
  if (wide) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = i * 4 + lane / 8, p = lane % 8, n = n0 + p * E;
      if (row0 + r >= M) continue;
      const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + ((p ^ (r & 7)) << 4));
      T* dst = out + (int64_t)(row0 + r) * pitch + n;
      if (n + E <= limit) {
        *reinterpret_cast<uint4*>(dst) = v;
      } else {
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (n + j < limit) dst[j] = e[j];
      }
    }
  } else {
    for (int r = 0; r < 32 && row0 + r < M; ++r) {
#pragma unroll
      for (int c = lane; c < COLS; c += 32) {
        if (n0 + c < limit)
          out[(int64_t)(row0 + r) * pitch + n0 + c] = *reinterpret_cast<const T*>(stage + r * 128 + (((c / E) ^ (r & 7)) << 4) + c % E * sizeof(T));
      }
    }
  }
}

// OUT: SVOO_TYPE_* of the output, SVOO_TYPE_E4M3 with scales
template <int OUT, bool kGelu, bool kRowScales>
__global__ void __launch_bounds__(kLinThreads, 1) linear_tc_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                                                                   const LinearArgs a) {
  extern __shared__ unsigned char smem_raw[];
  const int tiles_m = (a.M + kLinM - 1) / kLinM, tiles_n = (a.N + kLinN - 1) / kLinN, tiles = tiles_m * tiles_n;
  const int KB = (a.K + 127) / 128;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + kLinSmemData;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gen + kLinSmemData + LIN_BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + kLinSmemData + LIN_BARS * 8 + 8);
  auto bar = [&](int i) { return bars + 8u * i; };
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 0) {
    for (int i = 0; i < LIN_BARS; ++i) mbar_init(bar(i), i >= LIN_ACC_EMPTY ? 256 : 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLinRegsService));
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------------------ TMA producer
      int it = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const LinTile tile(t, tiles_m, tiles_n);
        for (int kb = 0; kb < KB; ++kb, ++it) {
          const int s = it % kLinStages;
          if (!(ok = mbar_wait(bar(LIN_EMPTY + s), ((it / kLinStages) & 1) ^ 1, abort_flag))) break;
          mbar_expect_tx(bar(LIN_FULL + s), kLinStageBytes);
          const uint32_t dst = base + s * kLinStageBytes;
          tma_load_2d(dst, &tm_a, kb * 128, tile.tm * kLinM, bar(LIN_FULL + s));
          tma_load_2d(dst + kLinABytes, &tm_b, kb * 128, tile.tn * kLinN, bar(LIN_FULL + s));
        }
      }
      // copies in flight land before the CTA ends
      if (!ok)
        for (int s = 0; s < kLinStages; ++s)
          if (it > s) mbar_drain(bar(LIN_FULL + s), ((it - 1 - s) / kLinStages) & 1);
    } else if (warp == 1 && lane == 0) {
      // ------------------------------------------------------------------ MMA issuer
      int it = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        for (int kb = 0; kb < KB; ++kb, ++it) {
          const int s = it % kLinStages, b = it & 1;
          if (!(ok = mbar_wait(bar(LIN_FULL + s), (it / kLinStages) & 1, abort_flag))) break;
          if (!(ok = mbar_wait(bar(LIN_ACC_EMPTY + b), ((it >> 1) & 1) ^ 1, abort_flag))) break;
          tc_fence_after();
          const uint32_t as = base + s * kLinStageBytes, bs = as + kLinABytes;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma_e4m3(tmem + b * 256, smem_desc_sw128(as + ks * 32, 16, 1024), smem_desc_sw128(bs + ks * 32, 16, 1024),
                      idesc_e4m3(kLinM, kLinN), ks > 0);
          tc_commit(bar(LIN_EMPTY + s));
          tc_commit(bar(LIN_ACC_FULL + b));
        }
      }
    }
  } else {
    // -------------------------------------------------------------------- sums and epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kLinRegsSums));
    const int quad = warp & 3, half = (warp - 4) >> 2;
    const uint32_t acc_addr = tmem + ((uint32_t)(quad * 32) << 16) + half * 128;
    unsigned char* stage = gen + kLinStages * kLinStageBytes + (warp - 4) * kLinOutBytes;
    int it = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const LinTile tile(t, tiles_m, tiles_n);
      const int row0 = tile.tm * kLinM + quad * 32, row = row0 + lane, n0 = tile.tn * kLinN + half * 128;
      const float* sa = a.sa + (row < a.M ? row : a.M - 1);
      const int last = (a.N - 1) / 128;
      const float* sb = kRowScales ? a.sb + n0 : a.sb + (int64_t)(n0 / 128 < last ? n0 / 128 : last) * a.sb_n;
      uint64_t sum[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) sum[i] = 0;
      // the factors of two blocks ahead are on their way
      float fa = sa[0], fa1 = KB > 1 ? sa[a.sa_pitch] : 0.f;
      float fb = kRowScales ? 1.f : sb[0], fb1 = !kRowScales && KB > 1 ? sb[a.sb_k] : 1.f;
      for (int kb = 0; kb < KB; ++kb, ++it) {
        const float fa2 = kb + 2 < KB ? sa[(kb + 2) * a.sa_pitch] : 0.f;
        const float fb2 = !kRowScales && kb + 2 < KB ? sb[(kb + 2) * a.sb_k] : 1.f;
        const int b = it & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(bar(LIN_ACC_FULL + b), (it >> 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const float f = fa * fb;
        const uint64_t f2 = pack2(f, f);
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          uint32_t r[32];
          load_columns(acc_addr + b * 256 + ch * 32, r);
          if (kRowScales) {
            const float4* cs = reinterpret_cast<const float4*>(sb + kb * a.sb_k + ch * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 c = n0 + ch * 32 + i * 4 < a.N ? __ldg(cs + i) : make_float4(0.f, 0.f, 0.f, 0.f);
              scale_add2(sum[ch * 16 + 2 * i], r[4 * i], r[4 * i + 1], mul2(pack2(c.x, c.y), f2));
              scale_add2(sum[ch * 16 + 2 * i + 1], r[4 * i + 2], r[4 * i + 3], mul2(pack2(c.z, c.w), f2));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) scale_add2(sum[ch * 16 + i], r[2 * i], r[2 * i + 1], f2);
          }
        }
        tc_fence_before();
        mbar_arrive(bar(LIN_ACC_EMPTY + b));
        fa = fa1, fa1 = fa2, fb = fb1, fb1 = fb2;
      }
      if (!ok) break;
      if (n0 >= a.N) continue;
      if (a.bias) {
#pragma unroll
        for (int i = 0; i < 64; ++i)
          sum[i] = pack2(half_of(sum[i], 0) + load_bias(a, n0 + 2 * i), half_of(sum[i], 1) + load_bias(a, n0 + 2 * i + 1));
      }
      if (kGelu) {
#pragma unroll
        for (int i = 0; i < 64; ++i) sum[i] = pack2(gelu_tanh(half_of(sum[i], 0)), gelu_tanh(half_of(sum[i], 1)));
      }
      if constexpr (OUT == SVOO_TYPE_E4M3) {
        // the thread's 128 columns are one block of its row; columns behind N are zero
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 64; ++i)
          top = max(top, max((uint32_t)sum[i] & 0x7fffffffu, (uint32_t)(sum[i] >> 32) & 0x7fffffffu));
        float s = __fdiv_rn(__uint_as_float(top), 448.f);
        s = s < 0x1p-126f ? 0x1p-126f : s;
        if (row < a.M) a.out_scale[(n0 / 128) * a.out_scale_pitch + row] = s;
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint64_t u = sum[p * 8 + 2 * i], v = sum[p * 8 + 2 * i + 1];
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(half_of(u, 0), s), __fdiv_rn(half_of(u, 1), s)), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(half_of(v, 0), s), __fdiv_rn(half_of(v, 1), s)), __NV_SATFINITE, __NV_E4M3);
            w[i] = lo | hi << 16;
          }
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((p ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        store_rows<uint8_t>(stage, (uint8_t*)a.out, a.out_pitch, row0, a.M, n0, (int)a.out_pitch, lane);
        __syncwarp();
      } else {
        typedef typename ElemOf<OUT>::T T;
        constexpr int COLS = 128 / (int)sizeof(T), E = 16 / (int)sizeof(T);
#pragma unroll
        for (int pass = 0; pass < 128 / COLS; ++pass) {
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            Vec<T, E> o;
#pragma unroll
            for (int i = 0; i < E; ++i) o.v[i] = from_f32<T>(half_of(sum[(pass * COLS + p * E + i) / 2], i & 1));
            *reinterpret_cast<Vec<T, E>*>(stage + lane * 128 + ((p ^ (lane & 7)) << 4)) = o;
          }
          __syncwarp();
          store_rows<T>(stage, (T*)a.out, a.out_pitch, row0, a.M, n0 + pass * COLS, a.N, lane);
          __syncwarp();
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicExch(&g_linear_status, 1);
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

}  // namespace tc

template <int OUT, bool kGelu, bool kRowScales>
static cudaError_t launch_one(const CUtensorMap& ma, const CUtensorMap& mb, const tc::LinearArgs& args, cudaStream_t st) {
  auto* kernel = &tc::linear_tc_kernel<OUT, kGelu, kRowScales>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, tc::kLinSmemBytes);
  if (e != cudaSuccess) return e;
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t tiles = ceil_div64(args.M, tc::kLinM) * ceil_div64(args.N, tc::kLinN);
  count_launches(1);
  return launch_pdl(kernel, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(tc::kLinThreads), (size_t)tc::kLinSmemBytes, st, ma, mb, args);
}

cudaError_t launch_linear_tc(const void* a, int64_t a_pitch, const float* sa, int64_t sa_pitch, const void* b, int64_t b_pitch, const float* sb,
                             int64_t sb_n, int64_t sb_k, bool row_scales, const void* bias, int bias_type, int64_t M, int64_t N, int64_t K,
                             bool gelu, int out_type, void* out, int64_t out_pitch, float* out_scale, int64_t out_scale_pitch, cudaStream_t st) {
  alignas(64) CUtensorMap ma, mb;
  if (!tc::make_byte_tensor_map(&ma, a, M, K, a_pitch, tc::kLinM) || !tc::make_byte_tensor_map(&mb, b, N, K, b_pitch, tc::kLinN))
    return cudaErrorInvalidValue;
  const tc::LinearArgs args{sa, sb, sa_pitch, sb_n, sb_k, bias, bias_type, out, out_pitch, out_scale, out_scale_pitch, (int)M, (int)N, (int)K};
  if (row_scales) {
    switch (out_type) {
      case SVOO_TYPE_BF16: return launch_one<SVOO_TYPE_BF16, false, true>(ma, mb, args, st);
      case SVOO_TYPE_FP16: return launch_one<SVOO_TYPE_FP16, false, true>(ma, mb, args, st);
      default: return launch_one<SVOO_TYPE_FP32, false, true>(ma, mb, args, st);
    }
  }
  if (gelu) {
    switch (out_type) {
      case SVOO_TYPE_BF16: return launch_one<SVOO_TYPE_BF16, true, false>(ma, mb, args, st);
      case SVOO_TYPE_FP16: return launch_one<SVOO_TYPE_FP16, true, false>(ma, mb, args, st);
      case SVOO_TYPE_FP32: return launch_one<SVOO_TYPE_FP32, true, false>(ma, mb, args, st);
      default: return launch_one<SVOO_TYPE_E4M3, true, false>(ma, mb, args, st);
    }
  }
  switch (out_type) {
    case SVOO_TYPE_BF16: return launch_one<SVOO_TYPE_BF16, false, false>(ma, mb, args, st);
    case SVOO_TYPE_FP16: return launch_one<SVOO_TYPE_FP16, false, false>(ma, mb, args, st);
    case SVOO_TYPE_FP32: return launch_one<SVOO_TYPE_FP32, false, false>(ma, mb, args, st);
    default: return launch_one<SVOO_TYPE_E4M3, false, false>(ma, mb, args, st);
  }
}

cudaError_t read_linear_status(int32_t* out, cudaStream_t st) {
  void* p = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&p, tc::g_linear_status);
  return e == cudaSuccess ? cudaMemcpyAsync(out, p, 4, cudaMemcpyDeviceToDevice, st) : e;
}

}  // namespace svoo
