// Product of 8-bit activations and 8-bit weights on the tcgen05 tensor cores:
//
//   y[m, n] = (sum_k x[m, k] w[n, k]) * xs[m] * ws[n] + b[n]
//
// x [M, K] with a scale a token, w [N, K] with a scale an output channel, the sum exact in
// 32-bit integers (K is at most 2^17 - 1, so that it cannot overflow), the scales and the
// bias applied in f32 with one rounding at the store.
//
// Weights are the A operand (128 channels a tile, one TMEM lane each) and tokens the B
// operand (BN a tile, one TMEM column each), for every M: a thread of the epilogue then
// owns one channel, its scale and bias stay in registers, and a warp stores 32
// consecutive channels of a token at a time, whatever N and its alignment are.  Both
// operands are staged by TMA as 128-byte rows (K = 128) in the 128-byte swizzle; rows
// and k beyond the tensors are filled with zeros.
//
// Two forms:
//  * persistent: one CTA an SM walks the tiles; two TMEM accumulators, so that the
//    epilogue of one tile runs under the products of the next.
//  * split: with few tiles (small M) a cluster of up to 8 CTAs shares one tile, each
//    takes a part of K, and the 32-bit partial sums are added over distributed shared
//    memory (integer sums: the order does not matter).
//
// Warps 0-3 epilogue (TMEM lanes 32 w), warp 4 TMA producer, warp 5 UMMA issuer and TMEM
// owner.  Every wait is bounded; on a timeout the CTA drains and the status word is set.
#include <cuda.h>

#include <atomic>
#include <cstring>

#include "common.cuh"
#include "internal.h"
#include "umma.cuh"
#include "vec_types.cuh"

namespace fpk {
namespace lin8 {

using namespace umma;

constexpr int kBM = 128;       // channels per tile (UMMA M)
constexpr int kBK = 128;       // bytes of K per stage: one swizzle row
constexpr int kThreads = 192;
constexpr int kTmaWarp = 4, kMmaWarp = 5;
constexpr int kMaxSplit = 8;   // portable cluster size

template <int BN>
struct Cfg {
  static constexpr int kABytes = kBM * kBK;
  static constexpr int kBBytes = BN * kBK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // BN >= 128: one CTA an SM, as deep as shared memory goes; below: two CTAs an SM
  static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 6 : BN == 64 ? 4 : BN == 32 ? 5 : 6;
  static constexpr int kSmem = kStages * kStageBytes + 1024;
  static constexpr int kAccs = 2;
  static constexpr uint32_t kTmemCols = kAccs * BN < 32 ? 32 : kAccs * BN;
};

struct Params {
  int* status;
  const float* xs;
  const float* ws;
  const void* bias;  // null: none
  void* y;
  int64_t y_stride;
  int32_t m, n;
  int32_t kblocks;   // of kBK bytes
  int32_t tiles_n, tiles_m;
  int32_t split;     // CTAs sharing a tile (the cluster size)
};

struct Bars {
  uint64_t full[8], empty[8];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};

// signed 8-bit A and B (both K-major), 32-bit integer accumulator
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void mma_i8_l(uint32_t leader, uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc,
                                         uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 e, %5, 0;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader));
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int ld_dsmem(uint32_t saddr, uint32_t rank) {
  uint32_t a;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// tiles in groups of 8 channel tiles, token tiles inside: the group's weights stay in L2
__device__ __forceinline__ void tile_of(const Params& p, int t, int* tn, int* tm) {
  constexpr int kGroup = 8;
  const int per = kGroup * p.tiles_m;
  const int g = t / per, r = t % per;
  const int wide = min(kGroup, p.tiles_n - g * kGroup);
  *tn = g * kGroup + r % wide;
  *tm = r / wide;
}

template <typename T>
__device__ __forceinline__ void store_y(const Params& p, int m, int n, int acc, float ws, float b) {
  if (m < p.m) {
    const float v = __fmaf_rn(__fmul_rn(__int2float_rn(acc), __ldg(p.xs + m)), ws, b);
    static_cast<T*>(p.y)[static_cast<int64_t>(m) * p.y_stride + n] = from_f32<T>(v);
  }
}

template <typename T, int BN, bool SPLIT>
__global__ void __launch_bounds__(kThreads, BN >= 128 ? 1 : 2)
    linear_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx,
                  const __grid_constant__ Params p) {
  using C = Cfg<BN>;
  constexpr int NS = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort = &bars.abort;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&bars.full[s], 1);
      mbar_init(&bars.empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.acc_full[i], 1);
      mbar_init(&bars.acc_empty[i], 4);
    }
    mbar_init(&bars.drain, 1);
    bars.abort = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_base)),
                 "r"(C::kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = bars.tmem_base;

  const int tiles = p.tiles_n * p.tiles_m;
  const int split = SPLIT ? p.split : 1;
  const int rank = SPLIT ? static_cast<int>(blockIdx.x) % split : 0;
  const int first = static_cast<int>(blockIdx.x) / split;
  const int step = static_cast<int>(gridDim.x) / split;
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.kblocks) * rank / split);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.kblocks) * (rank + 1) / split);

  if (warp == kTmaWarp) {
    if (lane == 0) {
      uint32_t it = 0;  // stages filled so far
      bool ok = true;
      for (int t = first; ok && t < tiles; t += step) {
        int tn, tm;
        tile_of(p, t, &tn, &tm);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = static_cast<int>(it % NS);
          if (!mbar_wait(&bars.empty[s], ((it / NS) & 1u) ^ 1u, abort, p.status, kWaitLimitNs)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * C::kStageBytes;
          mbar_arrive_expect_tx(&bars.full[s], C::kStageBytes);
          tma_load_2d(st, &tw, kb * kBK, tn * kBM, &bars.full[s]);
          tma_load_2d(st + C::kABytes, &tx, kb * kBK, tm * BN, &bars.full[s]);
        }
      }
      // no TMA write may land after the CTA has gone
      for (uint32_t k = it > NS ? it - NS : 0; k < it; ++k)
        drain_wait(&bars.full[k % NS], (k / NS) & 1u, p.status);
    }
  } else if (warp == kMmaWarp) {
    const uint32_t leader = elect_one();
    constexpr uint32_t idesc = idesc_i8(kBM, BN);
    const uint64_t a_desc = sdesc(smem_u32(smem), 16, 8 * kBK, 2u);
    const uint64_t b_desc = sdesc(smem_u32(smem + C::kABytes), 16, 8 * kBK, 2u);
    uint32_t it = 0, na = 0;
    bool ok = true;
    for (int t = first; ok && t < tiles; t += step, ++na) {
      const uint32_t acc = na & 1u;
      if (!mbar_wait_w(&bars.acc_empty[acc], ((na >> 1) & 1u) ^ 1u, abort, p.status, kWaitLimitNs)) break;
      tc_fence_after();
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const uint32_t s = it % NS;
        if (!mbar_wait_w(&bars.full[s], (it / NS) & 1u, abort, p.status, kWaitLimitNs)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t off = static_cast<uint64_t>(s) * (C::kStageBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < kBK / 32; ++kk)
          mma_i8_l(leader, tbase + acc * BN, a_desc + off + kk * 2, b_desc + off + kk * 2, idesc,
                   (kb > kb0 || kk > 0) ? 1u : 0u);
        mma_commit_l(leader, &bars.empty[s]);
      }
      if (ok) mma_commit_l(leader, &bars.acc_full[acc]);
    }
    // every UMMA issued so far must finish before TMEM is freed
    mma_commit_l(leader, &bars.drain);
    drain_wait_w(&bars.drain, 0, p.status);
  } else {
    uint32_t na = 0;
    for (int t = first; t < tiles; t += step, ++na) {
      int tn, tm;
      tile_of(p, t, &tn, &tm);
      const uint32_t acc = na & 1u;
      const int n = tn * kBM + warp * 32 + lane;
      const bool in = n < p.n;
      const float ws = in ? __ldg(p.ws + n) : 0.0f;
      const float b = in && p.bias ? to_f32(static_cast<const T*>(p.bias)[n]) : 0.0f;
      if (!mbar_wait(&bars.acc_full[acc], (na >> 1) & 1u, abort, p.status, kWaitLimitNs)) break;
      tc_fence_after();
      const uint32_t taddr = tbase + acc * BN + (static_cast<uint32_t>(warp * 32) << 16);
      constexpr int kChunk = BN < 32 ? BN : 32;
#pragma unroll 1
      for (int c0 = 0; c0 < BN; c0 += kChunk) {
        if (!SPLIT && tm * BN + c0 >= p.m) break;
        uint32_t r[kChunk];
        __syncwarp();
        tmem_ld<kChunk>(taddr + c0, r);
        if constexpr (SPLIT) {
          int* part = reinterpret_cast<int*>(smem);
#pragma unroll
          for (int c = 0; c < kChunk; ++c) part[(c0 + c) * kBM + warp * 32 + lane] = static_cast<int>(r[c]);
        } else if (in) {
#pragma unroll
          for (int c = 0; c < kChunk; ++c) store_y<T>(p, tm * BN + c0 + c, n, static_cast<int>(r[c]), ws, b);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.acc_empty[acc]);
    }
  }
  if constexpr (SPLIT) {
    // the ring is drained (acc_full follows every product of this CTA): its memory held the partial sums
    __syncwarp();
    cluster_sync();
    if (warp < 4) {
      int tn, tm;
      tile_of(p, first, &tn, &tm);
      const int n = tn * kBM + warp * 32 + lane;
      if (n < p.n && !*abort) {
        const float ws = __ldg(p.ws + n);
        const float b = p.bias ? to_f32(static_cast<const T*>(p.bias)[n]) : 0.0f;
        for (int c = rank; c < BN && tm * BN + c < p.m; c += split) {
          const uint32_t at = smem_u32(smem) + static_cast<uint32_t>(c * kBM + warp * 32 + lane) * 4u;
          int sum = 0;
          for (int r = 0; r < split; ++r) sum += ld_dsmem(at, r);
          store_y<T>(p, tm * BN + c, n, sum, ws, b);
        }
      }
    }
    cluster_sync();  // no CTA leaves while another reads its memory
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(C::kTmemCols));
  }
}

static int make_map(CUtensorMap* m, const void* base, int64_t rows, int64_t k, int64_t stride, int box_rows) {
  EncodeTiledFn enc = encoder();
  if (!enc) return FPK_ERR_CUDA;
  if (reinterpret_cast<uintptr_t>(base) % 16 || stride % 16) return FPK_ERR_ALIGN;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
  const cuuint32_t box[2] = {kBK, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1u, 1u};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FPK_OK : FPK_ERR_INVALID;
}

template <typename T, int BN, bool SPLIT>
static int launch(const fpk_linear_desc* d, const void* x, const void* w, Params p, int num_sms, cudaStream_t s) {
  static std::atomic<int> opted[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return FPK_ERR_CUDA;
  auto kern = linear_kernel<T, BN, SPLIT>;
  if (!opted[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<BN>::kSmem) != cudaSuccess)
      return FPK_ERR_CUDA;
    opted[dev].store(1, std::memory_order_release);
  }
  p.tiles_n = static_cast<int32_t>((d->n + kBM - 1) / kBM);
  p.tiles_m = static_cast<int32_t>((d->m + BN - 1) / BN);
  const int64_t tiles = static_cast<int64_t>(p.tiles_n) * p.tiles_m;
  if (tiles * kMaxSplit > 0x7fffffffLL) return FPK_ERR_UNSUPPORTED;
  CUtensorMap mw, mx;
  int rc = make_map(&mw, w, d->n, d->k, d->w_stride, kBM);
  if (rc == FPK_OK) rc = make_map(&mx, x, d->m, d->k, d->x_stride, BN);
  if (rc != FPK_OK) return rc;
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg<BN>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  const int per_sm = BN >= 128 ? 1 : 2;
  if constexpr (SPLIT) {
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * p.split));
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  } else {
    p.split = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(tiles < num_sms * per_sm ? tiles : num_sms * per_sm));
  }
  return cudaLaunchKernelEx(&cfg, kern, mw, mx, p) == cudaSuccess ? FPK_OK : FPK_ERR_CUDA;
}

template <typename T>
static int launch_t(const fpk_linear_desc* d, const void* x, const void* w, Params p, int num_sms, cudaStream_t s) {
  const int64_t tn = (d->n + kBM - 1) / kBM;
  // few tokens: the narrowest token tile that holds them, K split until about two CTAs an SM are busy
  if (d->m <= 128) {
    int split = 1;
    while (split < kMaxSplit && tn * split < num_sms && p.kblocks >= 4 * split) split *= 2;
    p.split = split;
    if (split > 1) {
      if (d->m <= 16) return launch<T, 16, true>(d, x, w, p, num_sms, s);
      if (d->m <= 32) return launch<T, 32, true>(d, x, w, p, num_sms, s);
      if (d->m <= 64) return launch<T, 64, true>(d, x, w, p, num_sms, s);
      return launch<T, 128, true>(d, x, w, p, num_sms, s);
    }
    if (d->m <= 16) return launch<T, 16, false>(d, x, w, p, num_sms, s);
    if (d->m <= 32) return launch<T, 32, false>(d, x, w, p, num_sms, s);
    if (d->m <= 64) return launch<T, 64, false>(d, x, w, p, num_sms, s);
    return launch<T, 128, false>(d, x, w, p, num_sms, s);
  }
  if (tn * ((d->m + 255) / 256) < num_sms) return launch<T, 128, false>(d, x, w, p, num_sms, s);
  return launch<T, 256, false>(d, x, w, p, num_sms, s);
}

}  // namespace lin8

int launch_linear_int8(const fpk_linear_desc* d, const void* x, const float* xs, const void* w, const float* ws,
                       const void* bias, void* y, cudaStream_t stream, const DeviceInfo& dev) {
  using namespace lin8;
  Params p;
  std::memset(&p, 0, sizeof(p));
  p.status = dev.status;
  p.xs = xs;
  p.ws = ws;
  p.bias = bias;
  p.y = y;
  p.y_stride = d->y_stride;
  p.m = static_cast<int32_t>(d->m);
  p.n = static_cast<int32_t>(d->n);
  p.kblocks = static_cast<int32_t>((d->k + kBK - 1) / kBK);
  const int sms = dev.num_sms > 0 ? dev.num_sms : 148;
  if (d->out_dtype == FPK_F16) return launch_t<__half>(d, x, w, p, sms, stream);
  if (d->out_dtype == FPK_BF16) return launch_t<__nv_bfloat16>(d, x, w, p, sms, stream);
  return launch_t<float>(d, x, w, p, sms, stream);
}

}  // namespace fpk
