// The product of linear_tc.cu where it has few tiles: the blocks of k of one 128 x 128 tile are shared out among the CTAs of a
// cluster, which join their sums through distributed shared memory.
//
// With few rows the product reads its weights once and does little else; what bounds it is how many SMs work on it: a block of k takes
// a CTA 0.45 us (300 x 300 x 8,000 on one CTA a tile 28.7), some 800 cycles, most of them the latency of four 16-column loads from TMEM, one
// behind the other, and of the hand-over of the accumulator; the tensor pipe needs 128.  A 128 x 128 tile has N / 128 of them to offer (5,120 columns: 40), a cluster of up to eight
// CTAs per tile up to eight times as many.  Every CTA sums its blocks of k as linear_tc.cu does, leaves the sums in its
// shared memory, and takes a share of the tile's rows, a warp per row: the cluster's sums of that row are added in rank order
// (the same bits on every call), then bias, activation and the store or the quantisation of the row's 128 columns, which are
// one block.
#include "linear_common.cuh"

namespace svoo {
namespace tc {

constexpr int kSplitThreads = 384;
constexpr int kSplitM = 128, kSplitN = 128;
constexpr int kSplitStages = 6;
constexpr int kSplitScales = 8;
constexpr int kSplitStageBytes = (kSplitM + kSplitN) * 128;
constexpr int kSplitScaleFloats = kSplitM + 4;
constexpr int kSplitData = kSplitStages * kSplitStageBytes, kSplitBars = kSplitData + kSplitScales * kSplitScaleFloats * 4;
constexpr int kSplitSmem = kSplitBars + 512 + 1024;
static_assert(kSplitM * kSplitN * 4 <= kSplitData, "the sums of the tile take the place of the operands");
constexpr int kSplitAcc = 2;                                  // accumulators (four are no faster)
enum { SPL_FULL = 0, SPL_EMPTY = SPL_FULL + kSplitStages, SPL_ACC_FULL = SPL_EMPTY + kSplitStages, SPL_ACC_EMPTY = SPL_ACC_FULL + kSplitAcc,
       SPL_SC_FULL = SPL_ACC_EMPTY + kSplitAcc, SPL_SC_EMPTY = SPL_SC_FULL + kSplitScales, SPL_BARS = SPL_SC_EMPTY + kSplitScales };

__device__ __forceinline__ float4 load_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void store_cluster(uint32_t addr, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

template <int OUT, bool kGelu>
__global__ void __launch_bounds__(kSplitThreads, 1) linear_split_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                                                                     const LinearArgs a) {
  extern __shared__ unsigned char smem_raw[];
  const int ranks = gridDim.x, rank = blockIdx.x;            // the cluster is a row of the grid
  const int tiles_m = (a.M + kSplitM - 1) / kSplitM;
  const int tn = blockIdx.y / tiles_m, tm = blockIdx.y - tn * tiles_m;
  const int KB = (a.K + 127) / 128, kb0 = (int)((int64_t)KB * rank / ranks), kb1 = (int)((int64_t)KB * (rank + 1) / ranks);
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;      // the same in every CTA of the cluster
  unsigned char* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + kSplitBars;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gen + kSplitBars + SPL_BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + kSplitBars + SPL_BARS * 8 + 8);
  auto bar = [&](int i) { return bars + 8u * i; };
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int row0 = tm * kSplitM, n0 = tn * kSplitN;
  if (tid == 32) {
    prefetch_map(&tm_a);
    prefetch_map(&tm_b);
  }
  if (tid == 0) {
    for (int i = 0; i < SPL_BARS; ++i) mbar_init(bar(i), i >= SPL_SC_EMPTY ? 8 : i >= SPL_SC_FULL ? 32 : i >= SPL_ACC_EMPTY ? 8 : 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kSplitAcc * kSplitN) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  if (warp == 0 && lane == 0) {
    bool ok = true;
    int it = 0;
    for (; it < kb1 - kb0; ++it) {
      const int s = it % kSplitStages;
      if (!(ok = mbar_wait(bar(SPL_EMPTY + s), ((it / kSplitStages) & 1) ^ 1, abort_flag))) break;
      mbar_expect_tx(bar(SPL_FULL + s), kSplitStageBytes);
      const uint32_t dst = base + s * kSplitStageBytes;
      tma_load_2d(dst, &tm_a, (kb0 + it) * 128, row0, bar(SPL_FULL + s));
      tma_load_2d(dst + kSplitM * 128, &tm_b, (kb0 + it) * 128, n0, bar(SPL_FULL + s));
    }
    if (!ok)
      for (int s = 0; s < kSplitStages; ++s)
        if (it > s) mbar_drain(bar(SPL_FULL + s), ((it - 1 - s) / kSplitStages) & 1);
  } else if (warp == 1 && lane == 0) {
    for (int it = 0; it < kb1 - kb0; ++it) {
      const int s = it % kSplitStages, b = it % kSplitAcc;
      if (!mbar_wait(bar(SPL_FULL + s), (it / kSplitStages) & 1, abort_flag)) break;
      if (!mbar_wait(bar(SPL_ACC_EMPTY + b), ((it / kSplitAcc) & 1) ^ 1, abort_flag)) break;
      tc_fence_after();
      const uint32_t as = base + s * kSplitStageBytes, bs = as + kSplitM * 128;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        umma_e4m3<1>(tmem + b * kSplitN, smem_desc_sw128(as + ks * 32, 16, 1024), smem_desc_sw128(bs + ks * 32, 16, 1024),
                     idesc_e4m3(kSplitM, kSplitN), ks > 0);
      tc_commit(bar(SPL_EMPTY + s));
      tc_commit(bar(SPL_ACC_FULL + b));
    }
  } else if (warp == 2) {
    for (int it = 0; it < kb1 - kb0; ++it) {
      const int s = it % kSplitScales, kb = kb0 + it;
      if (!__all_sync(0xffffffffu, mbar_wait(bar(SPL_SC_EMPTY + s), ((it / kSplitScales) & 1) ^ 1, abort_flag))) break;
      const uint32_t dst = base + kSplitData + s * kSplitScaleFloats * 4;
#pragma unroll
      for (int i = 0; i < kSplitM / 32; ++i) {
        const int r = i * 32 + lane;
        copy4(dst + r * 4, a.sa + kb * a.sa_pitch + (row0 + r < a.M ? row0 + r : a.M - 1));
      }
      if (lane == 0) copy4(dst + kSplitM * 4, a.sb + tn * a.sb_n + kb * a.sb_k);
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar(SPL_SC_FULL + s)) : "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp >= 4) {
    const int quad = warp & 3, half = (warp - 4) >> 2;
    const uint32_t acc_addr = tmem + ((uint32_t)(quad * 32) << 16) + half * 64;
    const int r = quad * 32 + lane;
    uint64_t sum[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) sum[i] = 0;
#pragma unroll 1
    for (int it = 0; it < kb1 - kb0; ++it) {
      const int b = it % kSplitAcc, sl = it % kSplitScales;
      if (!__all_sync(0xffffffffu, mbar_wait(bar(SPL_SC_FULL + sl), (it / kSplitScales) & 1, abort_flag) &&
                                       mbar_wait(bar(SPL_ACC_FULL + b), (it / kSplitAcc) & 1, abort_flag)))
        break;
      tc_fence_after();
      const float* sc = reinterpret_cast<const float*>(gen + kSplitData) + sl * kSplitScaleFloats;
      const float f = sc[r] * sc[kSplitM];
      const uint64_t f2 = pack2(f, f);
      const uint32_t at = acc_addr + b * kSplitN;
      uint32_t v[2][16];
      tmem_ld16_nowait(at, v[0]);
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {
        wait_columns(v[ch & 1]);
        if (ch < 3) tmem_ld16_nowait(at + (ch + 1) * 16, v[(ch + 1) & 1]);
#pragma unroll
        for (int i = 0; i < 8; ++i) scale_add2(sum[ch * 8 + i], v[ch & 1][2 * i], v[ch & 1][2 * i + 1], f2);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(SPL_ACC_EMPTY + b));
        mbar_arrive(bar(SPL_SC_EMPTY + sl));
      }
    }
    // the last sums are here, so the operands have been read: row r of the tile, 16-byte piece p at p ^ (r & 31)
    float4* row = reinterpret_cast<float4*>(gen + r * kSplitN * 4);
    if (!*abort_flag) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        row[(half * 16 + i) ^ lane] = make_float4(half_of(sum[2 * i], 0), half_of(sum[2 * i], 1), half_of(sum[2 * i + 1], 0), half_of(sum[2 * i + 1], 1));
    }
  }
  __syncthreads();
  // a CTA that gave up on a wait has left no sums: the others learn of it, and the tile stays unwritten
  if (warp == 0) {
    if (lane < ranks && *abort_flag) store_cluster(at_cta(bars + SPL_BARS * 8 + 8, lane), 1);
    __syncwarp();
  }
  cluster_sync();
  // rows of this CTA; a lane holds four columns
  const int rows = *abort_flag ? 0 : a.M - row0 < kSplitM ? a.M - row0 : kSplitM;
  const int n = n0 + lane * 4;
  float bias[4];
  bias_columns(a, n, 1, bias);
  const int r1 = rows * (rank + 1) / ranks;
  for (int r = rows * rank / ranks + warp; r < r1; r += kSplitThreads / 32) {
    const uint32_t at = base + r * kSplitN * 4 + ((lane ^ (r & 31)) << 4);
    float4 part[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < ranks) part[k] = load_cluster(at_cta(at, k));
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < ranks) v[0] += part[k].x, v[1] += part[k].y, v[2] += part[k].z, v[3] += part[k].w;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += bias[i];
    if (kGelu) {
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const uint64_t g = gelu2(pack2(v[i], v[i + 1]));
        v[i] = half_of(g, 0), v[i + 1] = half_of(g, 1);
      }
    }
    if constexpr (OUT == SVOO_TYPE_E4M3) {
      uint32_t top = max(max(magnitude(v[0]), magnitude(v[1])), max(magnitude(v[2]), magnitude(v[3])));
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float s = block_scale(top);
      if (lane == 0) a.out_scale[tn * a.out_scale_pitch + row0 + r] = s;
      if (n < ((a.N + 15) & ~15))
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.out) + (int64_t)(row0 + r) * a.out_pitch + n) = BlockDivide(s).e4m3x4(v[0], v[1], v[2], v[3]);
    } else {
      typedef typename ElemOf<OUT>::T T;
      T* dst = static_cast<T*>(a.out) + (int64_t)(row0 + r) * a.out_pitch + n;
      Vec<T, 4> o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o.v[i] = from_f32<T>(v[i]);
      if (a.box_out && n + 4 <= a.N) {
        *reinterpret_cast<Vec<T, 4>*>(dst) = o;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < a.N) dst[i] = o.v[i];
      }
    }
  }
  __syncwarp();
  cluster_sync();                                            // nobody reads this CTA's sums any more
  if (tid == 0 && *abort_flag) atomicExch(a.status, 1);
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kSplitAcc * kSplitN) : "memory");
  }
}

}  // namespace tc

template <int OUT, bool kGelu>
static cudaError_t launch_split_one(const LinearCall& c, int ranks) {
  alignas(64) CUtensorMap ma, mb;
  if (!tc::make_byte_tensor_map(&ma, c.a, c.args.M, c.args.K, c.a_pitch, tc::kSplitM) ||
      !tc::make_byte_tensor_map(&mb, c.b, c.args.N, c.args.K, c.b_pitch, tc::kSplitN))
    return cudaErrorInvalidValue;
  auto* kernel = &tc::linear_split_kernel<OUT, kGelu>;
  static uint64_t done;
  const cudaError_t e = allow_smem(kernel, tc::kSplitSmem, done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ranks, (unsigned)(ceil_div(c.args.M, tc::kSplitM) * ceil_div(c.args.N, tc::kSplitN)));
  cfg.blockDim = dim3(tc::kSplitThreads);
  cfg.dynamicSmemBytes = tc::kSplitSmem;
  cfg.stream = c.st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ranks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  count_launches(1);
  return cudaLaunchKernelEx(&cfg, kernel, ma, mb, c.args);
}

// Clusters of each size that the device holds at once (a cluster stays inside one GPC, so sizes that do not divide one leave SMs
// idle); asked for once per device.
static int clusters_of(int ranks) {
  static int known[64][9];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return 0;
  int n = __atomic_load_n(&known[dev][ranks], __ATOMIC_RELAXED);
  if (n == 0) {
    auto* kernel = &tc::linear_split_kernel<SVOO_TYPE_BF16, false>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, tc::kSplitSmem) != cudaSuccess) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ranks, 148);
    cfg.blockDim = dim3(tc::kSplitThreads);
    cfg.dynamicSmemBytes = tc::kSplitSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) return 0;
    __atomic_store_n(&known[dev][ranks], n < 1 ? -1 : n, __ATOMIC_RELAXED);
  }
  return n < 0 ? 0 : n;
}

// CTAs per tile: as many as run at once, each with two blocks of k or more; 0 where the tiles alone fill the device.
// us for 40 tiles of 5,120 columns, 40 blocks: 18.2 / 12.3 / 11.3 with 1 / 2 / 3 CTAs, 15.3 with 4 (two rounds);
// 21 tiles, 8 blocks (333 x 777 x 1,000): 9.4 / 7.4 / 7.1 / 6.5 with 1 / 2 / 3 / 4, 13.9 with 7;
// 9 tiles, 63 blocks (300 x 300 x 8,000): 28.7 / 17.1 / 13.2 / 11.2 / 10.0 / 9.0 with 1 / 2 / 3 / 4 / 6 / 8.
int linear_split_ranks(int64_t tiles, int64_t blocks) {
  if (tiles > 148) return 0;
  int ranks = 8;
  while (ranks > 1 && (ranks * 2 > blocks || tiles > clusters_of(ranks))) --ranks;
  return ranks;
}

cudaError_t launch_linear_split(const LinearCall& c, int out_type, bool gelu, int ranks) {
  switch (out_type) {
    case SVOO_TYPE_BF16: return gelu ? launch_split_one<SVOO_TYPE_BF16, true>(c, ranks) : launch_split_one<SVOO_TYPE_BF16, false>(c, ranks);
    case SVOO_TYPE_FP16: return gelu ? launch_split_one<SVOO_TYPE_FP16, true>(c, ranks) : launch_split_one<SVOO_TYPE_FP16, false>(c, ranks);
    case SVOO_TYPE_FP32: return gelu ? launch_split_one<SVOO_TYPE_FP32, true>(c, ranks) : launch_split_one<SVOO_TYPE_FP32, false>(c, ranks);
    default: return gelu ? launch_split_one<SVOO_TYPE_E4M3, true>(c, ranks) : launch_split_one<SVOO_TYPE_E4M3, false>(c, ranks);
  }
}

}  // namespace svoo
