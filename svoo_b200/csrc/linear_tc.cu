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
// A tile is 256 rows x 256 columns and belongs to a pair of SMs (cta_group::2), each with its half of a's and of b's rows in
// shared memory, so that a byte that was fetched feeds twice the products.
//
//   warp 0       TMA producer: 128 x 128 bytes of a, 128 x 128 of b per stage (128-byte swizzle)
//   warp 1       MMA issuer (of the pair's first CTA): M 256, N 256, K 32
//   warp 2       copies the scales of a block of k into a ring of their own (cp.async)
//   warp 3       brings the bias of a tile's columns to 32 bits
//   warps 4-11   thread r of each group of four warps owns row r (TMEM lane r) and 128 columns, which are one scale block
//                of b: the factor sa sb is one number per thread and block.  The registers for the 128 sums come from the
//                other warps (setmaxnreg).  Rows leave by TMA (boxes of 32 rows x 128 bytes) while the next tile runs.
//
// Every mbarrier wait is bounded; on expiry the CTA sets the status word of the device and leaves.
#include "linear_common.cuh"

namespace svoo {
namespace tc {

constexpr int kLinThreads = 384;
constexpr int kLinM = 128, TM = 2 * kLinM, TN = 256;          // rows of a CTA; a pair's tile
constexpr int HC = TN / 2;                                    // columns of a warpgroup of sums
constexpr int kLinBox = 32 * 128;                             // rows leave in boxes of 32 rows x 128 bytes, two per warp in flight
constexpr int kLinScales = 8;                                 // scale blocks in flight

template <bool kRowScales>
struct LinCfg {
  static constexpr int kABytes = kLinM * 128, kBRows = TN / 2, kBBytes = kBRows * 128, kStageBytes = kABytes + kBBytes;
  static constexpr int kScaleFloats = kLinM + (kRowScales ? TN : 4);       // sa of the rows, sb of the columns (or of two blocks)
  static constexpr int kFixed = 16 * kLinBox + kLinScales * kScaleFloats * 4 + 2 * TN * 4 + 512 + 1024;
  static constexpr int kStages = (232448 - kFixed) / kStageBytes < 8 ? (232448 - kFixed) / kStageBytes : 8;
  static constexpr int kOut = kStages * kStageBytes, kScale = kOut + 16 * kLinBox, kBias = kScale + kLinScales * kScaleFloats * 4,
                       kBars = kBias + 2 * TN * 4;
  static constexpr int kSmemBytes = kBars + 512 + 1024;
  static constexpr int FULL = 0, EMPTY = FULL + kStages, ACC_FULL = EMPTY + kStages, ACC_EMPTY = ACC_FULL + 2, SC_FULL = ACC_EMPTY + 2,
                       SC_EMPTY = SC_FULL + kLinScales, BIAS_FULL = SC_EMPTY + kLinScales, BIAS_EMPTY = BIAS_FULL + 2, BARS = BIAS_EMPTY + 2;
  static constexpr int kTmemColumns = 2 * TN;
  // registers after setmaxnreg: without spills in the warps that read TMEM (a register could be saved before it is filled)
  static constexpr int kRegsSums = kRowScales ? 216 : 232, kRegsService = kRowScales ? 72 : 40;
  static_assert(256 * kRegsSums + 128 * kRegsService <= kLinThreads * 168);
  static_assert(BARS * 8 + 16 <= 512 && kSmemBytes <= 232448 && kStages >= 3);
};
__device__ int g_linear_status;

constexpr int kLinGroupM = 16;                                // row tiles that sweep the columns together

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

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(src) : "memory");
}

// One warp's staged box of 32 rows x 128 bytes (16-byte piece p of row r at p ^ (r & 7): the 128-byte swizzle) to out rows
// row0 + r, elements [n0, n0 + 128 / sizeof(T)) of which those below N exist: rows that TMA cannot address, whose 16-byte pieces
// are not aligned.
template <typename T>
__device__ __forceinline__ void store_ragged(const unsigned char* box, const LinearArgs& a, int row0, int n0, int lane) {
  constexpr int E = 16 / (int)sizeof(T), COLS = 128 / (int)sizeof(T);
  for (int r = 0; r < 32 && row0 + r < a.M; ++r) {
#pragma unroll
    for (int c = lane; c < COLS; c += 32) {
      if (n0 + c < a.N)
        static_cast<T*>(a.out)[(int64_t)(row0 + r) * a.out_pitch + n0 + c] =
            *reinterpret_cast<const T*>(box + r * 128 + (((c / E) ^ (r & 7)) << 4) + c % E * sizeof(T));
    }
  }
}

// OUT: SVOO_TYPE_* of the output, SVOO_TYPE_E4M3 with scales
template <int OUT, bool kGelu, bool kRowScales>
__global__ void __launch_bounds__(kLinThreads, 1) linear_tc_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                                                                   const __grid_constant__ CUtensorMap tm_out, const LinearArgs a) {
  using C = LinCfg<kRowScales>;
  extern __shared__ unsigned char smem_raw[];
  const int tiles_m = (a.M + TM - 1) / TM, tiles_n = (a.N + TN - 1) / TN, tiles = tiles_m * tiles_n;
  const int KB = (a.K + 127) / 128;
  const int rank = (int)(blockIdx.x & 1), worker = blockIdx.x / 2, workers = gridDim.x / 2;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + C::kBars;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gen + C::kBars + C::BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + C::kBars + C::BARS * 8 + 8);
  auto bar = [&](int i) { return bars + 8u * i; };
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 32) {
    prefetch_map(&tm_a);
    prefetch_map(&tm_b);
    if (a.box_out) prefetch_map(&tm_out);
  }
  if (tid == 0) {
    for (int i = 0; i < C::BARS; ++i)
      mbar_init(bar(i), i >= C::BIAS_EMPTY ? 8 : i >= C::BIAS_FULL ? 32 : i >= C::SC_EMPTY ? 8 : i >= C::SC_FULL ? 32 : i >= C::ACC_EMPTY ? 16 : 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(C::kTmemColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  cluster_sync();                                          // the other CTA's barriers are set up before they are signalled
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsService));
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------------------ TMA producer
      // The first CTA's FULL barrier counts the bytes of both.
      int it = 0;
      bool ok = true;
      for (int t = worker; t < tiles && ok; t += workers) {
        const LinTile tile(t, tiles_m, tiles_n);
        for (int kb = 0; kb < KB; ++kb, ++it) {
          const int s = it % C::kStages;
          if (!(ok = mbar_wait(bar(C::EMPTY + s), ((it / C::kStages) & 1) ^ 1, abort_flag))) break;
          const uint32_t dst = base + s * C::kStageBytes;
          if (rank == 0) mbar_expect_tx(bar(C::FULL + s), 2 * C::kStageBytes);
          const uint32_t full = at_cta(bar(C::FULL + s), 0);
          tma_load_pair(dst, &tm_a, kb * 128, tile.tm * TM + rank * kLinM, full);
          tma_load_pair(dst + C::kABytes, &tm_b, kb * 128, tile.tn * TN + rank * C::kBRows, full);
        }
      }
      // copies in flight land before the CTA ends (the pair leaves together)
      if (!ok && rank == 0)
        for (int s = 0; s < C::kStages; ++s)
          if (it > s) mbar_drain(bar(C::FULL + s), ((it - 1 - s) / C::kStages) & 1);
    } else if (warp == 1 && lane == 0 && rank == 0) {
      // ------------------------------------------------------------------ MMA issuer
      int it = 0;
      bool ok = true;
      for (int t = worker; t < tiles && ok; t += workers) {
        for (int kb = 0; kb < KB; ++kb, ++it) {
          const int s = it % C::kStages, b = it & 1;
          if (!(ok = mbar_wait(bar(C::FULL + s), (it / C::kStages) & 1, abort_flag))) break;
          if (!(ok = mbar_wait(bar(C::ACC_EMPTY + b), ((it >> 1) & 1) ^ 1, abort_flag))) break;
          tc_fence_after();
          const uint32_t as = base + s * C::kStageBytes, bs = as + C::kABytes;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma_e4m3<2>(tmem + b * TN, smem_desc_sw128(as + ks * 32, 16, 1024), smem_desc_sw128(bs + ks * 32, 16, 1024),
                            idesc_e4m3(TM, TN), ks > 0);
          commit_pair(bar(C::EMPTY + s));
          commit_pair(bar(C::ACC_FULL + b));
        }
      }
    } else if (warp == 2) {
      // ------------------------------------------------------------------ scales
      int it = 0;
      bool ok = true;
      const int last = (a.N - 1) / 128;
      for (int t = worker; t < tiles && ok; t += workers) {
        const LinTile tile(t, tiles_m, tiles_n);
        const int row0 = tile.tm * TM + rank * kLinM, n0 = tile.tn * TN;
        for (int kb = 0; kb < KB; ++kb, ++it) {
          const int s = it % kLinScales;
          ok = __all_sync(0xffffffffu, mbar_wait(bar(C::SC_EMPTY + s), ((it / kLinScales) & 1) ^ 1, abort_flag));
          if (!ok) break;
          const uint32_t dst = base + C::kScale + s * C::kScaleFloats * 4;
          const float* sa = a.sa + kb * a.sa_pitch;
#pragma unroll
          for (int i = 0; i < kLinM / 32; ++i) {
            const int r = i * 32 + lane;
            copy4(dst + r * 4, sa + (row0 + r < a.M ? row0 + r : a.M - 1));
          }
          if (kRowScales) {
#pragma unroll
            for (int i = 0; i < TN / 32; ++i) {
              const int n = i * 32 + lane;
              copy4(dst + (kLinM + n) * 4, a.sb + kb * a.sb_k + (n0 + n < a.N ? n0 + n : a.N - 1));
            }
          } else if (lane < 2) {
            const int nb = (n0 + lane * HC) / 128;
            copy4(dst + (kLinM + lane) * 4, a.sb + (int64_t)(nb < last ? nb : last) * a.sb_n + kb * a.sb_k);
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar(C::SC_FULL + s)) : "memory");
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (!kRowScales && warp == 3 && a.bias) {
      // ------------------------------------------------------------------ bias
      int i = 0;
      for (int t = worker; t < tiles; t += workers, ++i) {
        const LinTile tile(t, tiles_m, tiles_n);
        if (!__all_sync(0xffffffffu, mbar_wait(bar(C::BIAS_EMPTY + (i & 1)), ((i >> 1) & 1) ^ 1, abort_flag))) break;
        float* dst = reinterpret_cast<float*>(gen + C::kBias) + (i & 1) * TN + lane;
#pragma unroll 1
        for (int k = 0; k < TN; k += 128) {                // four loads at a time: these warps have few registers
          float v[4];
          bias_columns(a, tile.tn * TN + k + lane, 32, v);
#pragma unroll
          for (int j = 0; j < 4; ++j) dst[k + j * 32] = v[j];
        }
        mbar_arrive(bar(C::BIAS_FULL + (i & 1)));
      }
    }
  } else {
    // -------------------------------------------------------------------- sums and epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsSums));
    const int quad = warp & 3, half = (warp - 4) >> 2;
    const uint32_t acc_addr = tmem + ((uint32_t)(quad * 32) << 16) + half * HC;
    const float* scales = reinterpret_cast<const float*>(gen + C::kScale);
    unsigned char* box = gen + C::kOut + (warp - 4) * 2 * kLinBox;
    const bool has_bias = !kRowScales && a.bias;
    int n_tile = 0;
    const uint32_t acc_empty = at_cta(bar(C::ACC_EMPTY), 0);
    int it = 0;
    bool ok = true;
    for (int t = worker; t < tiles && ok; t += workers, ++n_tile) {
      uint64_t sum[HC / 2];
#pragma unroll
      for (int i = 0; i < HC / 2; ++i) sum[i] = 0;
#pragma unroll 1
      for (int kb = 0; kb < KB; ++kb, ++it) {
        const int b = it & 1, sl = it % kLinScales;
        ok = __all_sync(0xffffffffu, mbar_wait(bar(C::SC_FULL + sl), (it / kLinScales) & 1, abort_flag) &&
                                         mbar_wait(bar(C::ACC_FULL + b), (it >> 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const float* sc = scales + sl * C::kScaleFloats;
        const float f = sc[quad * 32 + lane] * (kRowScales ? 1.f : sc[kLinM + half]);
        const uint64_t f2 = pack2(f, f);
        const uint32_t at = acc_addr + b * TN;
        uint32_t r[2][16];
        tmem_ld16_nowait(at, r[0]);
#pragma unroll
        for (int ch = 0; ch < HC / 16; ++ch) {
          wait_columns(r[ch & 1]);
          if (ch + 1 < HC / 16) {
            tmem_ld16_nowait(at + (ch + 1) * 16, r[(ch + 1) & 1]);
          } else {                                         // all columns are here: the next block may be summed over them
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_cluster(acc_empty + 8 * b);
          }
          const uint32_t(&v)[16] = r[ch & 1];
          if (kRowScales) {
            const float4* cs = reinterpret_cast<const float4*>(sc + kLinM + half * HC + ch * 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 c = cs[i];
              scale_add2(sum[ch * 8 + 2 * i], v[4 * i], v[4 * i + 1], mul2(pack2(c.x, c.y), f2));
              scale_add2(sum[ch * 8 + 2 * i + 1], v[4 * i + 2], v[4 * i + 3], mul2(pack2(c.z, c.w), f2));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) scale_add2(sum[ch * 8 + i], v[2 * i], v[2 * i + 1], f2);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::SC_EMPTY + sl));
      }
      if (!ok) break;
      const LinTile tile(t, tiles_m, tiles_n);
      const int row0 = tile.tm * TM + rank * kLinM + quad * 32, row = row0 + lane, n0 = tile.tn * TN + half * HC;
      const uint32_t bias = base + C::kBias + ((n_tile & 1) * TN + half * HC) * 4;
      if (has_bias) ok = __all_sync(0xffffffffu, mbar_wait(bar(C::BIAS_FULL + (n_tile & 1)), (n_tile >> 1) & 1, abort_flag));
      if (!ok) break;
      const bool skip = n0 >= a.N || row0 >= a.M;
      // four columns at a time, the bias of the next four on its way (volatile: all of it at once would not fit the registers)
      uint64_t ahead[2] = {0, 0};
      auto bias4 = [&](int c) {
        if (has_bias && c < HC)
          asm volatile("ld.volatile.shared.v2.b64 {%0, %1}, [%2];" : "=l"(ahead[0]), "=l"(ahead[1]) : "r"(bias + c * 4));
      };
      bias4(0);
      auto finish4 = [&](int c) {
        uint64_t v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) v[i] = has_bias ? add2(sum[c / 2 + i], ahead[i]) : sum[c / 2 + i];
        bias4(c + 4);
#pragma unroll
        for (int i = 0; i < 2; ++i) sum[c / 2 + i] = kGelu ? gelu2(v[i]) : v[i];
      };
      // A box is written again when the store before the last, its own, has read it.  Every box is a group, an empty one where all of it
      // lies outside the result: otherwise the wait would count a store that is one box older.
      auto begin_box = [&](int i) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        __syncwarp();
        return box + (i & 1) * kLinBox;
      };
      auto end_box = [&](const unsigned char* at, int n) {
        fence_async_proxy();
        __syncwarp();
        if (lane == 0) {
          if (!skip) tma_store_2d(&tm_out, n, row0, smem_u32(at));
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      };
      if constexpr (OUT == SVOO_TYPE_E4M3) {
        // the thread's 128 columns are one block of its row; columns behind N are zero
        static_assert(HC == 128);
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < HC; c += 4) {
          finish4(c);
#pragma unroll
          for (int i = 0; i < 2; ++i) top = max_magnitude(top, sum[c / 2 + i]);
        }
        const float s = block_scale(__float_as_uint(top) & 0x7fffffffu);
        if (row < a.M && !skip) a.out_scale[(n0 / 128) * a.out_scale_pitch + row] = s;
        const bool tiny = s < 0x1p-90f;
        if (tiny) {
#pragma unroll
          for (int i = 0; i < HC / 2; ++i) sum[i] = mul2(sum[i], pack2(0x1p64f, 0x1p64f));
        }
        const BlockDivideOnce by(tiny ? s * 0x1p64f : s);
        unsigned char* at = begin_box(n_tile);
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[i] = by.e4m3x4(sum[p * 8 + 2 * i], sum[p * 8 + 2 * i + 1]);
          }
          *reinterpret_cast<uint4*>(at + lane * 128 + ((p ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        end_box(at, n0);
      } else {
        typedef typename ElemOf<OUT>::T T;
        constexpr int COLS = 128 / (int)sizeof(T), E = 16 / (int)sizeof(T);
#pragma unroll
        for (int pass = 0; pass < HC / COLS; ++pass) {
          unsigned char* at = begin_box(pass);
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            const int c = pass * COLS + p * E;
            Vec<T, E> o;
#pragma unroll
            for (int i = 0; i < E; i += 4) finish4(c + i);
#pragma unroll
            for (int i = 0; i < E; ++i) o.v[i] = from_f32<T>(half_of(sum[(c + i) / 2], i & 1));
            *reinterpret_cast<Vec<T, E>*>(at + lane * 128 + ((p ^ (lane & 7)) << 4)) = o;
          }
          if (a.box_out) {
            end_box(at, n0 + pass * COLS);
          } else {
            __syncwarp();
            if (!skip) store_ragged<T>(at, a, row0, n0 + pass * COLS, lane);
          }
        }
      }
      if (has_bias) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::BIAS_EMPTY + (n_tile & 1)));
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (tid == 0 && *abort_flag) atomicExch(a.status, 1);
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmemColumns) : "memory");
  }
}

}  // namespace tc

template <int OUT, bool kGelu, bool kRowScales>
static cudaError_t launch_one(const LinearCall& c) {
  using C = tc::LinCfg<kRowScales>;
  alignas(64) CUtensorMap ma, mb, mo = {};
  if (!tc::make_byte_tensor_map(&ma, c.a, c.args.M, c.args.K, c.a_pitch, tc::kLinM) ||
      !tc::make_byte_tensor_map(&mb, c.b, c.args.N, c.args.K, c.b_pitch, C::kBRows) ||
      (c.args.box_out && !tc::make_out_tensor_map(&mo, OUT, c.args.out, c.args.M, c.args.N, c.args.out_pitch)))
    return cudaErrorInvalidValue;
  auto* kernel = &tc::linear_tc_kernel<OUT, kGelu, kRowScales>;
  static uint64_t done;
  const cudaError_t e = allow_smem(kernel, C::kSmemBytes, done);
  if (e != cudaSuccess) return e;
  const int64_t tiles = ceil_div64(c.args.M, tc::TM) * ceil_div64(c.args.N, tc::TN);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (unsigned)(tiles < 74 ? tiles : 74));      // a pair per two SMs
  cfg.blockDim = dim3(tc::kLinThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = c.st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  count_launches(1);
  return cudaLaunchKernelEx(&cfg, kernel, ma, mb, mo, c.args);
}

cudaError_t launch_linear_few(int type, const void* x, int64_t x_row, const LinearCall& c, int out_type, bool gelu);
int linear_split_ranks(int64_t tiles, int64_t blocks);
cudaError_t launch_linear_split(const LinearCall& c, int out_type, bool gelu, int ranks);

cudaError_t launch_linear(const void* a, int64_t a_pitch, const float* sa, int64_t sa_pitch, const void* b, int64_t b_pitch, const float* sb,
                             int64_t sb_n, int64_t sb_k, bool row_scales, const void* bias, int bias_type, int64_t M, int64_t N, int64_t K,
                             bool gelu, int out_type, void* out, int64_t out_pitch, float* out_scale, int64_t out_scale_pitch, cudaStream_t st) {
  const int e = out_type == SVOO_TYPE_E4M3 ? 1 : elem_bytes(out_type);
  // a box that reaches behind a row is cut at 16 bytes, not at the row's last number: a row that ends inside 16 bytes of a wider
  // pitch leaves element by element (e4m3 rows end at 16 bytes by their contract)
  const bool box_out = out_pitch * e % 16 == 0 && (uintptr_t)out % 16 == 0 && (e == 1 || N * e % 16 == 0);
  const LinearCall c{a, b, a_pitch, b_pitch,
                     {sa, sb, sa_pitch, sb_n, sb_k, bias, bias_type, out, out_pitch, out_scale, out_scale_pitch, (int)M, (int)N, (int)K, rows_status_word(), box_out}, st};
  if (!c.args.status) return cudaErrorInvalidDevice;
  if (!row_scales) {
    const int ranks = linear_split_ranks(ceil_div64(M, 128) * ceil_div64(N, 128), ceil_div64(K, 128));
    if (ranks) return launch_linear_split(c, out_type, gelu, ranks);
  }
  if (row_scales) {
    switch (out_type) {
      case SVOO_TYPE_BF16: return launch_one<SVOO_TYPE_BF16, false, true>(c);
      case SVOO_TYPE_FP16: return launch_one<SVOO_TYPE_FP16, false, true>(c);
      default: return launch_one<SVOO_TYPE_FP32, false, true>(c);
    }
  }
  if (gelu) {
    switch (out_type) {
      case SVOO_TYPE_BF16: return launch_one<SVOO_TYPE_BF16, true, false>(c);
      case SVOO_TYPE_FP16: return launch_one<SVOO_TYPE_FP16, true, false>(c);
      case SVOO_TYPE_FP32: return launch_one<SVOO_TYPE_FP32, true, false>(c);
      default: return launch_one<SVOO_TYPE_E4M3, true, false>(c);
    }
  }
  switch (out_type) {
    case SVOO_TYPE_BF16: return launch_one<SVOO_TYPE_BF16, false, false>(c);
    case SVOO_TYPE_FP16: return launch_one<SVOO_TYPE_FP16, false, false>(c);
    case SVOO_TYPE_FP32: return launch_one<SVOO_TYPE_FP32, false, false>(c);
    default: return launch_one<SVOO_TYPE_E4M3, false, false>(c);
  }
}

// The product on few rows that are not quantised yet, in one launch.  us on the GPU, this / quantisation and split product:
// 1 x 5,120 x 5,120 8.7 / 12.5, 1 x 1,536 x 1,536 2.6 / 6.8, 1 x 8,960 x 1,536 4.8 / 9.2, 1 x 1,536 x 8,960 9.1 / 9.9; 16 rows 12.7 / 12.5,
// 4.0 / 6.8, 7.2 / 9.2, 13.5 / 9.9.  The second launch and its workspace cost the host another 4 us (13.6 and 17.7 a call).
bool linear_few_rows(int64_t M, int64_t K, int out_type) { return (M <= 8 || (M <= 16 && K <= 4096)) && out_type != SVOO_TYPE_E4M3; }
cudaError_t launch_linear_few_rows(int x_type, const void* x, int64_t x_row, const void* b, int64_t b_pitch, const float* sb, int64_t sb_n,
                                   int64_t sb_k, const void* bias, int bias_type, int64_t M, int64_t N, int64_t K, bool gelu, int out_type,
                                   void* out, int64_t out_pitch, cudaStream_t st) {
  const LinearCall c{nullptr, b, 0, b_pitch, {nullptr, sb, 0, sb_n, sb_k, bias, bias_type, out, out_pitch, nullptr, 0, (int)M, (int)N, (int)K, nullptr, false}, st};
  return launch_linear_few(x_type, x, x_row, c, out_type, gelu);
}

int* rows_status_word() {
  static int* words[64];                                 // per device; every thread finds the same address
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  int* p = __atomic_load_n(&words[dev], __ATOMIC_RELAXED);
  if (!p) {
    if (cudaGetSymbolAddress(reinterpret_cast<void**>(&p), tc::g_linear_status) != cudaSuccess) return nullptr;
    __atomic_store_n(&words[dev], p, __ATOMIC_RELAXED);
  }
  return p;
}

cudaError_t read_linear_status(int32_t* out, cudaStream_t st) {
  int* p = rows_status_word();
  return p ? cudaMemcpyAsync(out, p, 4, cudaMemcpyDeviceToDevice, st) : cudaErrorInvalidDevice;
}

}  // namespace svoo
