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
// Three forms (launch_t says which runs when):
//  * persistent: one CTA an SM walks the tiles; two TMEM accumulators, so that the
//    epilogue of one tile runs under the products of the next.
//  * pairs: the same with two CTAs on one tile (below), for many tokens.
//  * split: with few tiles (small M) a cluster of up to 8 CTAs shares one tile, each
//    takes a part of K, and the 32-bit partial sums are added over distributed shared
//    memory (integer sums: the order does not matter).
//
// Warps 0-7 epilogue (TMEM lanes 32 (w mod 4)), warp 8 TMA producer, warp 9 UMMA issuer and
// TMEM owner.  Every wait is bounded; on a timeout the CTA drains and the status word is set.
#include <cuda.h>

#include <algorithm>
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
constexpr int kEpiWarps = 8;   // two a quarter of the TMEM lanes, half of the tokens each
constexpr int kThreads = 32 * (kEpiWarps + 2);
constexpr int kTmaWarp = kEpiWarps, kMmaWarp = kEpiWarps + 1;
constexpr int kMaxSplit = 8;   // portable cluster size

template <int BN>
struct Cfg {
  static constexpr int kABytes = kBM * kBK;
  static constexpr int kBBytes = BN * kBK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // BN = 128: one CTA an SM, as deep as shared memory goes; below: two CTAs an SM
  static constexpr int kStages = BN == 128 ? 6 : BN == 64 ? 4 : BN == 32 ? 5 : 6;
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

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t saddr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
  return a;
}
__device__ __forceinline__ int ld_dsmem(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
// stream order towards the kernel before (programmatic dependent launch): everything ahead of
// this, barriers and TMEM, may run while that kernel finishes
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// tiles in groups of 8 channel tiles, token tiles inside: the group's weights stay in L2
__device__ __forceinline__ void tile_of(const Params& p, int t, int* tn, int* tm) {
  constexpr int kGroup = 8;
  const int per = kGroup * p.tiles_m;
  const int g = t / per, r = t % per;
  const int wide = min(kGroup, p.tiles_n - g * kGroup);
  *tn = g * kGroup + r % wide;
  *tm = r / wide;
}

__device__ __forceinline__ float value(int acc, float xs, float ws, float b) {
  return __fmaf_rn(__fmul_rn(__int2float_rn(acc), xs), ws, b);
}

// The scales of BN tokens from m0, one a lane in chunks of 32 (or BN); asked for before the
// wait for the products.
template <int BN>
struct TokenScales {
  static constexpr int kChunk = BN < 32 ? BN : 32, kN = BN / kChunk;
  float s[kN];
  __device__ __forceinline__ void load(const Params& p, int m0, int lane) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int m = m0 + i * kChunk + lane;
      s[i] = lane < kChunk && m < p.m ? __ldg(p.xs + m) : 0.0f;
    }
  }
};

// BN columns of a CTA's accumulator to y: 128 channels (a TMEM lane each) x BN tokens from m0.
// Lane c holds the scale of token c of a chunk and hands it round, so that nothing but the
// stores is left in the loop over the tokens.
template <typename T, int BN>
__device__ __forceinline__ void store_tile(const Params& p, const TokenScales<BN>& xs, uint32_t taddr, int m0, int n,
                                           float ws, float b) {
  constexpr int kChunk = TokenScales<BN>::kChunk;
  const bool in = n < p.n;
#pragma unroll
  for (int i = 0; i < TokenScales<BN>::kN; ++i) {
    const int c0 = i * kChunk;
    if (m0 + c0 >= p.m) break;
    uint32_t r[kChunk];
    __syncwarp();
    tmem_ld<kChunk>(taddr + c0, r);
    T* y = static_cast<T*>(p.y) + static_cast<int64_t>(m0 + c0) * p.y_stride + n;
    const int left = p.m - m0 - c0;
    T v[kChunk];
#pragma unroll
    for (int c = 0; c < kChunk; ++c)
      v[c] = from_f32<T>(value(static_cast<int>(r[c]), __shfl_sync(0xffffffffu, xs.s[i], c), ws, b));
    if (in) {
      // one epilogue warp a scheduler: a test and a branch a token cost as much as the rest
      if (left >= kChunk) {
#pragma unroll
        for (int c = 0; c < kChunk; ++c, y += p.y_stride) *y = v[c];
      } else {
#pragma unroll
        for (int c = 0; c < kChunk; ++c, y += p.y_stride)
          if (c < left) *y = v[c];
      }
    }
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
      mbar_init(&bars.acc_empty[i], kEpiWarps);
    }
    mbar_init(&bars.drain, 1);
    bars.abort = 0;
    fence_mbar_init();
  }
  if (warp == kTmaWarp && lane == 0) {
    prefetch_map(&tw);
    prefetch_map(&tx);
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
  grid_wait();

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
    const int quarter = warp & 3, half = warp >> 2;
    uint32_t na = 0;
    for (int t = first; t < tiles; t += step, ++na) {
      int tn, tm;
      tile_of(p, t, &tn, &tm);
      const uint32_t acc = na & 1u;
      const int n = tn * kBM + quarter * 32 + lane;
      const bool in = n < p.n;
      const float ws = in ? __ldg(p.ws + n) : 0.0f;
      const float b = in && p.bias ? to_f32(static_cast<const T*>(p.bias)[n]) : 0.0f;
      TokenScales<BN / 2> xs;
      if constexpr (!SPLIT) xs.load(p, tm * BN + half * (BN / 2), lane);
      if (!__all_sync(0xffffffffu, mbar_wait(&bars.acc_full[acc], (na >> 1) & 1u, abort, p.status, kWaitLimitNs))) break;
      tc_fence_after();
      const uint32_t taddr = tbase + acc * BN + (static_cast<uint32_t>(quarter * 32) << 16);
      if constexpr (SPLIT) {
        constexpr int kChunk = BN / 2 < 32 ? BN / 2 : 32;
        int* part = reinterpret_cast<int*>(smem);
#pragma unroll 1
        for (int c0 = half * (BN / 2); c0 < (half + 1) * (BN / 2); c0 += kChunk) {
          uint32_t r[kChunk];
          __syncwarp();
          tmem_ld<kChunk>(taddr + c0, r);
#pragma unroll
          for (int c = 0; c < kChunk; ++c) part[(c0 + c) * kBM + quarter * 32 + lane] = static_cast<int>(r[c]);
        }
      } else {
        store_tile<T, BN / 2>(p, xs, taddr + half * (BN / 2), tm * BN + half * (BN / 2), n, ws, b);
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
    if (warp < kEpiWarps) {
      int tn, tm;
      tile_of(p, first, &tn, &tm);
      const int n = tn * kBM + (warp & 3) * 32 + lane;
      if (n < p.n && !*abort) {
        const float ws = __ldg(p.ws + n);
        const float b = p.bias ? to_f32(static_cast<const T*>(p.bias)[n]) : 0.0f;
        // this CTA's share of the tokens, half of it a warp, four sums at a time
        const int share = BN / split, each = (share + 1) / 2;
        const int c0 = rank * share + (warp >> 2) * each;
        const int c1 = min(min(c0 + each, (rank + 1) * share), p.m - tm * BN);
        const uint32_t base = smem_u32(smem) + static_cast<uint32_t>((warp & 3) * 32 + lane) * 4u;
        for (int c = c0; c < c1; c += 4) {
          int sum[4] = {0, 0, 0, 0};
          for (int r = 0; r < split; ++r) {
            const uint32_t at = map_rank(base, r);
#pragma unroll
            for (int i = 0; i < 4; ++i)  // the last of a short group reads a token again
              sum[i] += ld_dsmem(at + static_cast<uint32_t>(min(c + i, c1 - 1) * kBM) * 4u);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int m = tm * BN + c + i;
            if (c + i < c1)
              static_cast<T*>(p.y)[static_cast<int64_t>(m) * p.y_stride + n] =
                  from_f32<T>(value(sum[i], __ldg(p.xs + m), ws, b));
          }
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

// ------------------------------------------------------- two CTAs on one tile ---
// A pair of CTAs (a cluster of two, on neighbouring SMs) shares a tile of 256 channels x BN
// tokens with cta_group::2 products: each CTA stages its own 128 channels and half of the
// tokens, and the tensor cores read the other half from the neighbour, so an operand byte
// is fetched from L2 once a pair.  One CTA alone asks L2 for 48 KB in the time of 512 cycles
// of products (128 x 256 x 128), a pair for 32 KB each: 8192^3 ran at 2868 TOPS with single
// CTAs (L2 bound, about 16 TB/s).
//
// The even CTA issues the products and owns the `full` barriers (both CTAs' copies count on
// them) and `acc_empty` (both epilogues arrive); commits signal `empty` and `acc_full` in both.
template <int BN>
struct PairCfg {
  static constexpr int kABytes = kBM * kBK;
  static constexpr int kBBytes = BN / 2 * kBK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = BN == 256 ? 6 : 8;
  static constexpr int kSmem = kStages * kStageBytes + 1024;
};

__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mma_i8_pair_l(uint32_t leader, uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc,
                                              uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 e, %5, 0;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader));
}
__device__ __forceinline__ void mma_commit_pair_l(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b16 m;\n\tmov.b16 m, 3;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}" ::"r"(
          smem_u32(bar)),
      "r"(leader)
      : "memory");
}

template <typename T, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx,
                       const __grid_constant__ Params p) {
  using C = PairCfg<BN>;
  constexpr int NS = C::kStages;
  constexpr uint32_t kCols = 2 * BN;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x & 1);
  volatile int* abort = &bars.abort;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&bars.full[s], 1);
      mbar_init(&bars.empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.acc_full[i], 1);
      mbar_init(&bars.acc_empty[i], 2 * kEpiWarps);
    }
    mbar_init(&bars.drain, 1);
    bars.abort = 0;
    fence_mbar_init();
  }
  if (warp == kTmaWarp && lane == 0) {
    prefetch_map(&tw);
    prefetch_map(&tx);
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_base)),
                 "r"(kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  cluster_sync();  // both CTAs' barriers are ready before anyone signals across
  tc_fence_after();
  const uint32_t tbase = bars.tmem_base;
  grid_wait();
  const int tiles = p.tiles_n * p.tiles_m;
  const int first = static_cast<int>(blockIdx.x >> 1);
  const int step = static_cast<int>(gridDim.x >> 1);

  if (warp == kTmaWarp) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += step) {
        int tn, tm;
        tile_of(p, t, &tn, &tm);
        for (int kb = 0; kb < p.kblocks; ++kb, ++it) {
          const int s = static_cast<int>(it % NS);
          if (!mbar_wait(&bars.empty[s], ((it / NS) & 1u) ^ 1u, abort, p.status, kWaitLimitNs)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * C::kStageBytes;
          if (rank == 0) mbar_arrive_expect_tx(&bars.full[s], 2 * C::kStageBytes);
          const uint32_t bar = map_rank(smem_u32(&bars.full[s]), 0);
          tma_load_2d_pair(st, &tw, kb * kBK, (tn * 2 + rank) * kBM, bar);
          tma_load_2d_pair(st + C::kABytes, &tx, kb * kBK, tm * BN + rank * (BN / 2), bar);
        }
      }
      // no TMA write may land after the CTA has gone: the even CTA's barriers count both CTAs' bytes
      if (rank == 0)
        for (uint32_t k = it > NS ? it - NS : 0; k < it; ++k)
          drain_wait(&bars.full[k % NS], (k / NS) & 1u, p.status);
    }
  } else if (warp == kMmaWarp) {
    if (rank == 0) {
      const uint32_t leader = elect_one();
      constexpr uint32_t idesc = idesc_i8(2 * kBM, BN);
      const uint64_t a_desc = sdesc(smem_u32(smem), 16, 8 * kBK, 2u);
      const uint64_t b_desc = sdesc(smem_u32(smem + C::kABytes), 16, 8 * kBK, 2u);
      uint32_t it = 0, na = 0;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += step, ++na) {
        const uint32_t acc = na & 1u;
        if (!mbar_wait_w(&bars.acc_empty[acc], ((na >> 1) & 1u) ^ 1u, abort, p.status, kWaitLimitNs)) break;
        asm volatile("fence.acq_rel.cluster;" ::: "memory");  // the other CTA's epilogue has read it
        tc_fence_after();
        for (int kb = 0; kb < p.kblocks; ++kb, ++it) {
          const uint32_t s = it % NS;
          if (!mbar_wait_w(&bars.full[s], (it / NS) & 1u, abort, p.status, kWaitLimitNs)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t off = static_cast<uint64_t>(s) * (C::kStageBytes >> 4);
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            mma_i8_pair_l(leader, tbase + acc * BN, a_desc + off + kk * 2, b_desc + off + kk * 2, idesc,
                          (kb > 0 || kk > 0) ? 1u : 0u);
          mma_commit_pair_l(leader, &bars.empty[s]);
        }
        if (ok) mma_commit_pair_l(leader, &bars.acc_full[acc]);
      }
      // every UMMA issued so far must finish before TMEM is freed (in both CTAs: cluster_sync below)
      mma_commit_pair_l(leader, &bars.drain);
      drain_wait_w(&bars.drain, 0, p.status);
    }
  } else {
    const int quarter = warp & 3, half = warp >> 2;
    uint32_t na = 0;
    for (int t = first; t < tiles; t += step, ++na) {
      int tn, tm;
      tile_of(p, t, &tn, &tm);
      const uint32_t acc = na & 1u;
      const int n = (tn * 2 + rank) * kBM + quarter * 32 + lane;
      const float ws = n < p.n ? __ldg(p.ws + n) : 0.0f;
      const float b = n < p.n && p.bias ? to_f32(static_cast<const T*>(p.bias)[n]) : 0.0f;
      TokenScales<BN / 2> xs;
      xs.load(p, tm * BN + half * (BN / 2), lane);
      if (!__all_sync(0xffffffffu, mbar_wait(&bars.acc_full[acc], (na >> 1) & 1u, abort, p.status, kWaitLimitNs))) break;
      tc_fence_after();
      store_tile<T, BN / 2>(p, xs, tbase + acc * BN + half * (BN / 2) + (static_cast<uint32_t>(quarter * 32) << 16),
                            tm * BN + half * (BN / 2), n, ws, b);
      tc_fence_before();
      __syncwarp();
      if (lane == 0)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                         map_rank(smem_u32(&bars.acc_empty[acc]), 0))
                     : "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  // the last commit signals the odd CTA too: it must not leave before that has arrived
  if (rank == 1 && warp == kMmaWarp) drain_wait_w(&bars.drain, 0, p.status);
  __syncwarp();
  cluster_sync();  // no CTA leaves, or frees its TMEM, while the other may still use it
  tc_fence_after();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(kCols));
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
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int per_sm = BN >= 128 ? 1 : 2;
  if constexpr (SPLIT) {
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * p.split));
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.split;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  } else {
    p.split = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(tiles < num_sms * per_sm ? tiles : num_sms * per_sm));
  }
  return cudaLaunchKernelEx(&cfg, kern, mw, mx, p) == cudaSuccess ? FPK_OK : FPK_ERR_CUDA;
}

template <typename T, int BN>
static int launch_pair(const fpk_linear_desc* d, const void* x, const void* w, Params p, int num_sms, cudaStream_t s) {
  static std::atomic<int> opted[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return FPK_ERR_CUDA;
  auto kern = linear_pair_kernel<T, BN>;
  if (!opted[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg<BN>::kSmem) != cudaSuccess)
      return FPK_ERR_CUDA;
    opted[dev].store(1, std::memory_order_release);
  }
  p.tiles_n = static_cast<int32_t>((d->n + 2 * kBM - 1) / (2 * kBM));
  p.tiles_m = static_cast<int32_t>((d->m + BN - 1) / BN);
  p.split = 1;
  const int64_t tiles = static_cast<int64_t>(p.tiles_n) * p.tiles_m;
  if (tiles > 0x3fffffffLL) return FPK_ERR_UNSUPPORTED;
  CUtensorMap mw, mx;
  int rc = make_map(&mw, w, d->n, d->k, d->w_stride, kBM);
  if (rc == FPK_OK) rc = make_map(&mx, x, d->m, d->k, d->x_stride, BN / 2);
  if (rc != FPK_OK) return rc;
  const int64_t pairs = tiles < num_sms / 2 ? tiles : num_sms / 2;
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = PairCfg<BN>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, mw, mx, p) == cudaSuccess ? FPK_OK : FPK_ERR_CUDA;
}

// The form with the least estimated time, in cycles of one SM.  A step of K takes the longer
// of its products (8192 multiply-adds a cycle) and its copies (about 64 bytes a cycle and SM
// from L2; never below 400 cycles, a ring's bytes over the latency), the tiles come in rounds
// over the SMs, and sharing a tile's K costs 3500 + 65 cycles a token for joining.  Measured,
// in us, K shared by 1 / 2 / 4 / 8 CTAs:
//   8 x 4096 x 4096: 10.0 / 9.0 / 8.0 / 8.9     8 x 1024 x 8192: 16.5 / 11.5 / 8.3 / 7.0
//   64 x 4096 x 4096: 11.9 / 11.7 / 9.8 / 10.4  256 x 4096 x 4096: 11.8 / 13.5 / 19.8 / 41.3
// and pairs of CTAs (256, 128 tokens) against single CTAs (128 tokens): 1024 x 4096 x 4096
// 18.0, 20.3, 20.4; 8192^3 346, 452, 481.
template <typename T>
static int launch_t(const fpk_linear_desc* d, const void* x, const void* w, Params p, int num_sms, cudaStream_t s) {
  const int64_t kb = p.kblocks;
  const int64_t tn = (d->n + kBM - 1) / kBM, tn2 = (d->n + 2 * kBM - 1) / (2 * kBM);
  const int bn = d->m <= 16 ? 16 : d->m <= 32 ? 32 : d->m <= 64 ? 64 : 128;
  const int64_t tm = (d->m + bn - 1) / bn;
  const int64_t slots = bn < 128 ? 2 * num_sms : num_sms;  // CTAs that run at once
  const int64_t step = std::max<int64_t>(400, (kBM + bn) * kBK / 64);
  const auto rounds = [](int64_t tiles, int64_t at_once) { return (tiles + at_once - 1) / at_once; };
  int best = 1;
  int64_t least = kb * step * rounds(tn * tm, slots);
  for (int split = 2; split <= kMaxSplit && kb >= 2 * split && tn * tm * split <= slots; split *= 2) {
    const int64_t t = (kb + split - 1) / split * step + 3500 + 65 * bn;
    if (t < least) {
      least = t;
      best = split;
    }
  }
  const int64_t pair128 = kb * 400 * rounds(tn2 * ((d->m + 127) / 128), num_sms / 2);
  const int64_t pair256 = kb * 512 * rounds(tn2 * ((d->m + 255) / 256), num_sms / 2);
  if (d->m > 128 && least > std::min(pair128, pair256))
    return pair256 <= pair128 ? launch_pair<T, 256>(d, x, w, p, num_sms, s) : launch_pair<T, 128>(d, x, w, p, num_sms, s);
  p.split = best;
  if (best > 1) {
    if (bn == 16) return launch<T, 16, true>(d, x, w, p, num_sms, s);
    if (bn == 32) return launch<T, 32, true>(d, x, w, p, num_sms, s);
    if (bn == 64) return launch<T, 64, true>(d, x, w, p, num_sms, s);
    return launch<T, 128, true>(d, x, w, p, num_sms, s);
  }
  if (bn == 16) return launch<T, 16, false>(d, x, w, p, num_sms, s);
  if (bn == 32) return launch<T, 32, false>(d, x, w, p, num_sms, s);
  if (bn == 64) return launch<T, 64, false>(d, x, w, p, num_sms, s);
  return launch<T, 128, false>(d, x, w, p, num_sms, s);
}

// ------------------------------------------------ rows that TMA cannot read ---
// Rows whose stride is not a multiple of 16 bytes (or whose base is off 16 bytes) are laid
// out again, one launch for both operands.  A thread writes 16 bytes of a row from the 32-bit
// words that hold them, shifted into place; a word that reaches outside of the row's bytes is
// read a byte at a time.
struct PadArgs {
  const uint8_t* src[2];
  uint8_t* dst[2];
  int64_t rows[2], stride[2];  // of the source, in bytes; rows 0: nothing to do
  int64_t k, pitch;
};
__device__ __forceinline__ uint32_t word_of(const uint8_t* row, int64_t at, int64_t k) {
  uint32_t v = 0;
  for (int i = 0; i < 4; ++i)
    if (at + i < k) v |= static_cast<uint32_t>(row[at + i]) << (8 * i);
  return v;
}
__global__ void __launch_bounds__(256) pad_rows_kernel(const __grid_constant__ PadArgs a) {
  grid_wait();
  const int64_t units = a.pitch / 16;
  const int64_t total = (a.rows[0] + a.rows[1]) * units;
  for (int64_t x = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; x < total; x += static_cast<int64_t>(gridDim.x) * 256) {
    int64_t r = x / units;
    const int64_t c = x % units * 16;
    const int o = r >= a.rows[0];
    if (o) r -= a.rows[0];
    const uint8_t* row = a.src[o] + r * a.stride[o];
    uint32_t w[4];
    const uint32_t mis = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row + c) & 3u);
    if (c + 20 <= a.k && (mis == 0 || c >= 4)) {  // all words lie within the row
      const uint32_t* p = reinterpret_cast<const uint32_t*>(row + c - mis);
      uint32_t v[5];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __ldg(p + i);
      v[4] = mis ? __ldg(p + 4) : 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(v[i], v[i + 1], mis * 8);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = word_of(row, c + 4 * i, a.k);
    }
    *reinterpret_cast<uint4*>(a.dst[o] + r * a.pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace lin8

static bool needs_rows(const void* p, int64_t stride) {
  return reinterpret_cast<uintptr_t>(p) % 16 != 0 || stride % 16 != 0;
}

int64_t linear_int8_workspace(const fpk_linear_desc* d, const void* x, const void* w) {
  const int64_t pitch = (d->k + 15) / 16 * 16;
  return (needs_rows(x, d->x_stride) ? (d->m * pitch + 255) / 256 * 256 : 0) +
         (needs_rows(w, d->w_stride) ? (d->n * pitch + 255) / 256 * 256 : 0);
}

int launch_linear_int8(const fpk_linear_desc* d, const void* x, const float* xs, const void* w, const float* ws,
                       const void* bias, void* y, void* workspace, cudaStream_t stream, const DeviceInfo& dev) {
  using namespace lin8;
  fpk_linear_desc laid = *d;  // with rows as TMA reads them
  const bool pad_x = needs_rows(x, d->x_stride), pad_w = needs_rows(w, d->w_stride);
  const int sms = dev.num_sms > 0 ? dev.num_sms : 148;
  if (pad_x || pad_w) {
    PadArgs a{};
    a.k = d->k;
    a.pitch = (d->k + 15) / 16 * 16;
    uint8_t* at = static_cast<uint8_t*>(workspace);
    int64_t units = 0;
    if (pad_x) {
      a.src[0] = static_cast<const uint8_t*>(x);
      a.rows[0] = d->m;
      a.stride[0] = d->x_stride;
      a.dst[0] = at;
      x = at;
      laid.x_stride = a.pitch;
      at += (d->m * a.pitch + 255) / 256 * 256;
      units += d->m * (a.pitch / 16);
    }
    if (pad_w) {
      a.src[1] = static_cast<const uint8_t*>(w);
      a.rows[1] = d->n;
      a.stride[1] = d->w_stride;
      a.dst[1] = at;
      w = at;
      laid.w_stride = a.pitch;
      units += d->n * (a.pitch / 16);
    }
    const int64_t blocks = std::min<int64_t>((units + 255) / 256, 16 * sms);
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, pad_rows_kernel, a) != cudaSuccess) return FPK_ERR_CUDA;
    d = &laid;
  }
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
  if (d->out_dtype == FPK_F16) return launch_t<__half>(d, x, w, p, sms, stream);
  if (d->out_dtype == FPK_BF16) return launch_t<__nv_bfloat16>(d, x, w, p, sms, stream);
  return launch_t<float>(d, x, w, p, sms, stream);
}

}  // namespace fpk
