// Tree attention on the 5th-generation tensor cores (f16 and bf16, caches of that type or in 8
// bits), for more rows than mma.sync's kernel takes.
//
//   S = Q K^T;  x = S * (scale, and the key's scale);  P = exp2(x - m);  O += (P * the value's scale) V
//
// The rows are the nodes of all heads of a group (row r: head r / nodes, node r % nodes), in tiles
// of 128; a CTA takes its part of the blocks' 128-key tiles (tree_common.cuh).  Two warpgroups do the
// softmax, one thread a row: with more than 128 rows each has its own row tile and both take every
// key tile; with up to 128 they take every other key tile of the same rows, each with its own
// maximum, sum and result, which are joined in TMEM at the block's end.  Either way one's
// exponentials run beside the other's waits.  Roles:
//   warps 0-3, 4-7  softmax of row tile, or key tiles, 0 and 1
//   warps 8-11      K and V from memory into the tensor cores' layout
//   warp  12        UMMA issuer, TMEM owner
// TMEM: S_t at column 128 t, P_t over its first half, O_t at 256 + 128 t.
//
// 8-bit caches: the loaders hold a tile's bytes in registers while it is on its way, and write them as
// 16-bit numbers (exact) in the layout that a TMA load would give; K V in shared memory is then as
// for a 16-bit cache.  Scales go with the scores and the weights, 128 f32 of each a tile.  In f16 the
// weights are divided by a power of two near the largest value's scale so far (tree_dec.cu).
//
// Only tiles with rows from `all` on look at masks.  There what is not finite in a 16-bit V becomes
// zero and its node is noted; in the epilogue a row that sees a noted node looks at the values again
// and adds those that are not finite (a note of another block's node finds none, or the row's own).
#pragma once

#include <cmath>
#include <type_traits>

#include "internal.h"
#include "tree_common.cuh"
#include "umma.cuh"
#include "vec_types.cuh"

namespace fpk {
namespace tree {
namespace tc {

using namespace umma;

constexpr int kBM = 128, kBN = kUnit;
constexpr int kStages = 2;      // of K, and of V
constexpr int kScaleSlots = 4;  // tiles whose scales are held
constexpr int kSoftWarps = 8, kLoadWarps = 4, kLoadWarp = 8, kMmaWarp = 12;
constexpr int kLoadThreads = 32 * kLoadWarps;
constexpr int kThreads = 512;
// setmaxnreg split of 512 x 128: 256 x 176 softmax, 128 x 112 loaders, 128 x 48 the rest
constexpr int kRegsSoft = 176, kRegsLoad = 112, kRegsCtl = 48;
static_assert(256 * kRegsSoft + 128 * kRegsLoad + 128 * kRegsCtl <= kThreads * 128, "setmaxnreg split exceeds the launch");
constexpr float kRescaleLog2 = 8.0f;
constexpr uint32_t kTmemCols = 512, kOCol = 256;

template <int D>
struct Cfg {
  static constexpr int kBoxCols = D >= 64 ? 64 : D;
  static constexpr int kRowBytes = kBoxCols * 2;
  static constexpr int kBoxes = D / kBoxCols;
  static constexpr int kBoxBytes = 128 * kRowBytes;
  static constexpr int kTileBytes = kBoxes * kBoxBytes;
  static constexpr uint32_t kLayout = D >= 64 ? 2u : (D == 32 ? 4u : 6u);
  static constexpr uint32_t kSwzMask = D >= 64 ? 7u : (D == 32 ? 3u : 1u);
  static constexpr int kKStepsPerBox = kRowBytes / 32;
  static constexpr int kTiles = 2 + 2 * kStages;  // Q of two row tiles, K, V
  static constexpr int kSmem = kTiles * kTileBytes + 1024;
  static constexpr int kMinSmem = 116 * 1024;  // one CTA an SM: it has all of TMEM
  static constexpr int kLaunchSmem = kSmem > kMinSmem ? kSmem : kMinSmem;
};
// where the 16 bytes `chunk` (8 elements) of a row lie in a tile
template <int D>
__device__ __forceinline__ uint32_t chunk_at(int row, int chunk) {
  using C = Cfg<D>;
  constexpr int kPerBox = C::kRowBytes / 16;
  const uint32_t off = static_cast<uint32_t>(row * C::kRowBytes + (chunk % kPerBox) * 16);
  return static_cast<uint32_t>(chunk / kPerBox) * C::kBoxBytes + (off ^ (((off >> 7) & C::kSwzMask) << 4));
}

template <typename T>
struct Elem;
template <>
struct Elem<__half> {
  static constexpr uint32_t kFormat = 0, kExpMask = 0x7c007c00u, kExpLsb = 0x04000400u;
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr uint32_t kFormat = 1, kExpMask = 0x7f807f80u, kExpLsb = 0x00800080u;
};
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t u) {
  return ((u & Elem<T>::kExpMask) + Elem<T>::kExpLsb) & 0x80008000u;
}
template <typename T, int M, int N, bool BMN>
__host__ __device__ constexpr uint32_t idesc16() {
  return idesc_f16(M, N, BMN) | (Elem<T>::kFormat << 7) | (Elem<T>::kFormat << 10);
}
__device__ __forceinline__ float max3n(float a, float b, float c) {  // a NaN is kept
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ void mul2v(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
// 4 bytes as 4 numbers of T (tree_dec.cu)
template <typename T>
__device__ __forceinline__ uint2 four_of(uint32_t u) {
  uint2 r;
  if constexpr (std::is_same<T, __half>::value) {
    u ^= 0x80808080u;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r.x) : "r"(__byte_perm(u, 0x64646464u, 0x4140u)), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r.y) : "r"(__byte_perm(u, 0x64646464u, 0x4342u)), "r"(0x64806480u));
  } else {
    const uint32_t a = __byte_perm(u, 0x43434343u, 0x4140u), b = __byte_perm(u, 0x43434343u, 0x4342u);
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r.x) : "r"(a & 0xff7fff7fu), "r"(a & 0xff80ff80u));
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r.y) : "r"(b & 0xff7fff7fu), "r"(b & 0xff80ff80u));
  }
  return r;
}
// mbar_wait by every lane, with one answer for the warp
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, volatile int* abort, int* status) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status, kWaitLimitNs));
}

struct Ctl {
  uint64_t q_full;
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[2], p_half[2], p_full[2], o_done[2];
  uint64_t c_full[kScaleSlots];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  uint32_t bad[kWords];              // nodes whose V was not finite, of this CTA's blocks so far
  alignas(16) float kscale[kScaleSlots][kBN];
  alignas(16) float vscale[kScaleSlots][kBN];
  float vref[kScaleSlots];           // f16: the power of two that the tile's weights are divided by
  float2 ml[256];                    // both warpgroups' (m, l)
  int parent[kMaxNodes];
  uint32_t bits[256][kWords + 1];    // what each row sees of the tree; the last word is 0
};

// The key tiles of a block that warpgroup t takes: n-th of them, and how many of `tiles`
struct Turns {
  int step, first;
  __device__ __forceinline__ Turns(bool by_rows, int t) : step(by_rows ? 1 : 2), first(by_rows ? 0 : t) {}
  __device__ __forceinline__ int tile(int n) const { return first + n * step; }
  __device__ __forceinline__ int count(int tiles) const { return tiles > first ? (tiles - first + step - 1) / step : 0; }
};

// A loader's part of one operand of a key tile on its way: 8-bit rows in registers
template <int D>
struct Bytes {
  static constexpr int kUnits = D / 16;                                    // 16 bytes of a row
  static constexpr int kN = 128 * kUnits / kLoadThreads;  // a thread
  uint4 w[kN];
  __device__ __forceinline__ void load(const uint8_t* src, int64_t stride, int64_t j0, int n, int tid) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int x = tid + i * kLoadThreads, r = x / kUnits, u = x % kUnits;
      w[i] = r < n ? __ldg(reinterpret_cast<const uint4*>(src + (j0 + r) * stride + u * 16)) : make_uint4(0u, 0u, 0u, 0u);
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(uint8_t* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int x = tid + i * kLoadThreads, r = x / kUnits, u = x % kUnits;
      const uint2 a = four_of<T>(w[i].x), b = four_of<T>(w[i].y), c = four_of<T>(w[i].z), d = four_of<T>(w[i].w);
      const uint4 lo = make_uint4(a.x, a.y, b.x, b.y), hi = make_uint4(c.x, c.y, d.x, d.y);
      // D = 128: eight lanes write even chunks of one box and odd ones of the other, no bank conflict
      const bool odd = D == 128 && (u & 4);
      *reinterpret_cast<uint4*>(tile + chunk_at<D>(r, 2 * u + (odd ? 1 : 0))) = odd ? hi : lo;
      *reinterpret_cast<uint4*>(tile + chunk_at<D>(r, 2 * u + (odd ? 0 : 1))) = odd ? lo : hi;
    }
  }
};

template <typename T, int D, bool Q8>
__global__ void __launch_bounds__(kThreads, 1) tree_tc_kernel(const __grid_constant__ Params p) {
  using C = Cfg<D>;
  constexpr int NS = kStages;
  constexpr bool kNorm = Q8 && std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Ctl ctl;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * C::kTileBytes;
  uint8_t* sV = sK + NS * C::kTileBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = static_cast<int>(blockIdx.x);
  volatile int* abort = &ctl.abort;
  if (threadIdx.x == 0) {
    mbar_init(&ctl.q_full, kSoftWarps);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&ctl.k_full[s], kLoadWarps);
      mbar_init(&ctl.k_empty[s], 1);
      mbar_init(&ctl.v_full[s], kLoadWarps);
      mbar_init(&ctl.v_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&ctl.s_full[t], 1);
      mbar_init(&ctl.p_half[t], 4);
      mbar_init(&ctl.p_full[t], 4);
      mbar_init(&ctl.o_done[t], 1);
    }
    for (int s = 0; s < kScaleSlots; ++s) mbar_init(&ctl.c_full[s], kLoadWarps);
    mbar_init(&ctl.drain, 1);
    ctl.abort = 0;
    fence_mbar_init();
  }
  if (threadIdx.x < kWords) ctl.bad[threadIdx.x] = 0u;
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem_base)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = ctl.tmem_base;
  grid_wait();
  const int rows = p.group * p.nodes;
  const bool by_rows = p.by_rows != 0;
  // a scale that is not positive goes with Q, so that the largest product is the largest score
  const float factor = p.scale_log2 == 0.0f ? 1.0f : fabsf(p.scale_log2);
  Walk walk(p, cta);

  if (warp >= kMmaWarp) {
    setmaxnreg_dec<kRegsCtl>();
    if (warp == kMmaWarp) {
      // ------------------------------------------------ UMMA issuer (whole warp)
      constexpr uint32_t idesc_qk = idesc16<T, kBM, kBN, false>();
      constexpr uint32_t idesc_pv = idesc16<T, kBM, D, true>();
      constexpr uint64_t kTileStep = static_cast<uint64_t>(C::kTileBytes >> 4);
      const uint32_t leader = elect_one();
      const uint64_t q_desc = sdesc(smem_u32(sQ), 16, 8 * C::kRowBytes, C::kLayout);
      const uint64_t k_desc = sdesc(smem_u32(sK), 16, 8 * C::kRowBytes, C::kLayout);
      const uint64_t v_desc = sdesc(smem_u32(sV), C::kBoxBytes, 8 * C::kRowBytes, C::kLayout);
      bool ok = true;
      uint32_t it = 0;               // tiles of the blocks before
      uint32_t steps[2] = {0u, 0u};  // of each warpgroup
      uint32_t blocks = 0;
      auto issue_qk = [&](int t, uint32_t tile) {
        const uint32_t s = tile % NS;
        if (!mbar_wait_w(&ctl.k_full[s], (tile / NS) & 1u, abort, p.status, kWaitLimitNs)) return false;
        tc_fence_after();
        const uint64_t a0 = q_desc + static_cast<uint64_t>(by_rows ? t : 0) * kTileStep;
        const uint64_t b0 = k_desc + static_cast<uint64_t>(s) * kTileStep;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          constexpr int kSteps = C::kKStepsPerBox;
          const uint64_t off = static_cast<uint64_t>((kk / kSteps) * (C::kBoxBytes >> 4) + (kk % kSteps) * 2);
          mma_ss_l(leader, tbase + static_cast<uint32_t>(t * 128), a0 + off, b0 + off, idesc_qk, kk > 0 ? 1u : 0u);
        }
        mma_commit_l(leader, &ctl.s_full[t]);
        if (!by_rows || t == 1) mma_commit_l(leader, &ctl.k_empty[s]);
        return true;
      };
      auto issue_pv = [&](int t, uint32_t tile, bool accumulate, int half) {
        const uint32_t d_tmem = tbase + kOCol + static_cast<uint32_t>(t) * 128u;
        const uint32_t a_tmem = tbase + static_cast<uint32_t>(t) * 128u;
        const uint64_t b0 = v_desc + static_cast<uint64_t>(tile % NS) * kTileStep;
#pragma unroll
        for (int k2 = 0; k2 < kBN / 32; ++k2) {
          const int kk = half * (kBN / 32) + k2;
          mma_ts_l(leader, d_tmem, a_tmem + static_cast<uint32_t>(kk * 8), b0 + static_cast<uint64_t>(kk * C::kRowBytes),
                   idesc_pv, (accumulate || kk > 0) ? 1u : 0u);
        }
      };
      while (walk.more()) {
        const Block blk = next_block(p, walk);
        const int tiles = blk.t1 - blk.t0;
        const Turns turns[2] = {Turns(by_rows, 0), Turns(by_rows, 1)};
        ok = ok && mbar_wait_w(&ctl.q_full, blocks & 1u, abort, p.status, kWaitLimitNs);
        ++blocks;
        for (int t = 0; ok && t < 2; ++t)
          if (turns[t].count(tiles) > 0) ok = issue_qk(t, it + turns[t].tile(0));
        const int most = turns[0].count(tiles);
        for (int n = 0; ok && n < most; ++n) {
          for (int t = 0; ok && t < 2; ++t) {
            const int mine = turns[t].count(tiles);
            if (n >= mine) continue;
            const uint32_t tile = it + turns[t].tile(n), par = (steps[t] + n) & 1u;
            ok = mbar_wait_w(&ctl.v_full[tile % NS], (tile / NS) & 1u, abort, p.status, kWaitLimitNs) &&
                 mbar_wait_w(&ctl.p_half[t], par, abort, p.status, kWaitLimitNs);
            if (!ok) break;
            tc_fence_after();
            issue_pv(t, tile, n > 0, 0);
            ok = mbar_wait_w(&ctl.p_full[t], par, abort, p.status, kWaitLimitNs);
            if (!ok) break;
            tc_fence_after();
            issue_pv(t, tile, n > 0, 1);
            mma_commit_l(leader, &ctl.o_done[t]);
            if (!by_rows || t == 1) mma_commit_l(leader, &ctl.v_empty[tile % NS]);
            if (n + 1 < mine) ok = issue_qk(t, it + turns[t].tile(n + 1));
          }
        }
        it += tiles;
        for (int t = 0; t < 2; ++t) steps[t] += turns[t].count(tiles);
      }
      // every UMMA issued so far must finish before TMEM is freed
      mma_commit_l(leader, &ctl.drain);
      drain_wait_w(&ctl.drain, 0, p.status);
    }
  } else if (warp >= kLoadWarp) {
    setmaxnreg_dec<kRegsLoad>();
    // ------------------------------------------------------------- loaders
    const int tid = static_cast<int>(threadIdx.x) - kLoadWarp * 32;
    uint32_t it = 0;
    bool ok = true;
    [[maybe_unused]] float vref = 0.0f;
    auto arrive = [&](uint64_t* bar) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    if constexpr (Q8) {
      // the tile after the one that is written is in registers, asked for when its place got free
      struct Next {
        bool any;
        const uint8_t *k, *v;
        const float *ks, *vs;
        int64_t j0;
        int n;
        bool first;  // of its block
      };
      Bytes<D> kw, vw;
      float ks = 0.0f, vs[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      Block blk;
      int at = 0, tiles = 0;
      auto next = [&]() {
        Next x;
        x.first = false;
        while (at == tiles) {
          if (!walk.more()) {
            x.any = false;
            return x;
          }
          blk = next_block(p, walk);
          at = 0;
          tiles = blk.t1 - blk.t0;
          x.first = true;
        }
        x.any = true;
        x.k = static_cast<const uint8_t*>(p.k) + blk.b * p.k_st[0] + blk.kvh * p.k_st[1];
        x.v = static_cast<const uint8_t*>(p.v) + blk.b * p.v_st[0] + blk.kvh * p.v_st[1];
        x.ks = p.ks + blk.b * p.ks_st[0] + blk.kvh * p.ks_st[1];
        x.vs = p.vs + blk.b * p.vs_st[0] + blk.kvh * p.vs_st[1];
        x.j0 = static_cast<int64_t>(blk.t0 + at) * kBN;
        x.n = blk.sq.len - (blk.t0 + at) * kBN;
        ++at;
        return x;
      };
      auto load_k = [&](const Next& x) {
        kw.load(x.k, p.k_st[2], x.j0, x.n, tid);
        ks = tid < x.n ? __ldg(x.ks + (x.j0 + tid) * p.ks_st[2]) : 0.0f;
        if constexpr (kNorm) {
#pragma unroll
          for (int i = 0; i < 4; ++i) vs[i] = lane + 32 * i < x.n ? __ldg(x.vs + (x.j0 + lane + 32 * i) * p.vs_st[2]) : 0.0f;
        } else {
          vs[0] = tid < x.n ? __ldg(x.vs + (x.j0 + tid) * p.vs_st[2]) : 0.0f;
        }
      };
      Next cur = next();
      if (cur.any) {
        load_k(cur);
        vw.load(cur.v, p.v_st[2], cur.j0, cur.n, tid);
      }
      while (ok && cur.any) {
        const uint32_t s = it % NS, par = ((it / NS) & 1u) ^ 1u;
        const int slot = static_cast<int>(it % kScaleSlots);
        const Next nx = next();
        // the scales' slot is free with the K stage: the tile of four before has been weighed
        if (!wait_all(&ctl.k_empty[s], par, abort, p.status)) break;
        ctl.kscale[slot][tid] = ks * factor;
        if constexpr (kNorm) {
          if (cur.first) vref = 0.0f;
          uint32_t top = 0u;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t u = __float_as_uint(vs[i]) & 0x7fffffffu;
            top = max(top, u < 0x7f800000u ? u : 0u);
          }
          top = __reduce_max_sync(0xffffffffu, top);
          if (__uint_as_float(top) > vref || vref == 0.0f) {  // at least the largest scale, within 2^-126 .. 2^126
            const uint32_t u = min(max((top + 0x007fffffu) & 0x7f800000u, 1u << 23), 253u << 23);
            vref = __uint_as_float(u);
          }
          const float inv = __uint_as_float((254u << 23) - __float_as_uint(vref));
          const int w = warp - kLoadWarp;
          ctl.vscale[slot][tid] = (w == 0 ? vs[0] : w == 1 ? vs[1] : w == 2 ? vs[2] : vs[3]) * inv;
          if (tid == 0) ctl.vref[slot] = vref;
        } else {
          ctl.vscale[slot][tid] = vs[0];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.c_full[slot]);
        kw.template store<T>(sK + s * C::kTileBytes, tid);
        arrive(&ctl.k_full[s]);
        if (nx.any) load_k(nx);
        if (!wait_all(&ctl.v_empty[s], par, abort, p.status)) break;
        vw.template store<T>(sV + s * C::kTileBytes, tid);
        arrive(&ctl.v_full[s]);
        if (nx.any) vw.load(nx.v, p.v_st[2], nx.j0, nx.n, tid);
        cur = nx;
        ++it;
      }
    } else {
      // asynchronous copies, a tile ahead of the one whose arrival is signalled
      constexpr int kUnits = D / 8, kN = 128 * kUnits / kLoadThreads;
      auto copy = [&](uint8_t* tile, const uint8_t* src, int64_t stride, int64_t j0, int n) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          const int x = tid + i * kLoadThreads, r = x / kUnits, u = x % kUnits;
          const bool in = r < n;  // beyond the length: zeros, nothing read
          asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(smem_u32(tile + chunk_at<D>(r, u))),
                       "l"(src + (j0 + (in ? r : 0)) * stride + u * 16), "r"(in ? 16 : 0)
                       : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      // V of a tile with keys that some row may not see: what is not finite becomes zero
      auto clean = [&](uint8_t* tile, int j0, const Seq& sq) {
#pragma unroll 1
        for (int i = 0; i < kN; ++i) {
          const int x = tid + i * kLoadThreads, r = x / kUnits, u = x % kUnits;
          if (j0 + r < sq.all || j0 + r >= sq.len) continue;
          uint4* at = reinterpret_cast<uint4*>(tile + chunk_at<D>(r, u));
          uint4 w = *at;
          uint32_t* e = reinterpret_cast<uint32_t*>(&w);
          bool hit = false;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t nf = not_finite<T>(e[q]);
            if (nf & 0x8000u) e[q] &= 0xffff0000u;
            if (nf & 0x80000000u) e[q] &= 0x0000ffffu;
            hit |= nf != 0u;
          }
          if (hit) {
            *at = w;
            const int node = j0 + r - sq.past;
            atomicOr(&ctl.bad[node >> 5], 1u << (node & 31));
          }
        }
      };
      uint32_t done = 0;  // tiles signalled
      int j_of[NS] = {};  // of the tiles on their way
      Seq sq_of[NS] = {};
      auto signal = [&]() {
        const uint32_t s = done % NS;
        asm volatile("cp.async.wait_group 1;" ::: "memory");  // the tile's K, ahead of its V
        arrive(&ctl.k_full[s]);
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        uint8_t* v = sV + s * C::kTileBytes;
        const int j0 = s == 0 ? j_of[0] : j_of[1];
        const Seq sq = s == 0 ? sq_of[0] : sq_of[1];
        if (j0 + kBN > sq.all) clean(v, j0, sq);
        arrive(&ctl.v_full[s]);
        ++done;
      };
      while (ok && walk.more()) {
        const Block blk = next_block(p, walk);
        const uint8_t* k = static_cast<const uint8_t*>(p.k) + (blk.b * p.k_st[0] + blk.kvh * p.k_st[1]) * 2;
        const uint8_t* v = static_cast<const uint8_t*>(p.v) + (blk.b * p.v_st[0] + blk.kvh * p.v_st[1]) * 2;
        for (int t = blk.t0; t < blk.t1; ++t) {
          const uint32_t s = it % NS, par = ((it / NS) & 1u) ^ 1u;
          const int n = blk.sq.len - t * kBN;
          if (!wait_all(&ctl.k_empty[s], par, abort, p.status)) {
            ok = false;
            break;
          }
          copy(sK + s * C::kTileBytes, k, p.k_st[2] * 2, static_cast<int64_t>(t) * kBN, n);
          if (it > done) {  // the tile before: its K and V are the groups ahead of this one
            const uint32_t o = done % NS;
            asm volatile("cp.async.wait_group 2;" ::: "memory");
            arrive(&ctl.k_full[o]);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            const int j0 = o == 0 ? j_of[0] : j_of[1];
            const Seq sq = o == 0 ? sq_of[0] : sq_of[1];
            if (j0 + kBN > sq.all) clean(sV + o * C::kTileBytes, j0, sq);
            arrive(&ctl.v_full[o]);
            ++done;
          }
          if (!wait_all(&ctl.v_empty[s], par, abort, p.status)) {
            ok = false;
            break;
          }
          copy(sV + s * C::kTileBytes, v, p.v_st[2] * 2, static_cast<int64_t>(t) * kBN, n);
          if (s == 0) {
            j_of[0] = t * kBN;
            sq_of[0] = blk.sq;
          } else {
            j_of[1] = t * kBN;
            sq_of[1] = blk.sq;
          }
          ++it;
        }
      }
      if (ok && it > done) signal();
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
  } else {
    // ------------------------------------------------------ softmax + epilogue
    setmaxnreg_inc<kRegsSoft>();
    const int t = warp >> 2, row = static_cast<int>(threadIdx.x) & (kBM - 1);
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tbase + lane_off + static_cast<uint32_t>(t * 128);
    const uint32_t tO = tbase + lane_off + kOCol + static_cast<uint32_t>(t) * 128u;
    const uint32_t tP = tS;
    const Turns turns(by_rows, t);
    const int slot_row = by_rows ? t * kBM + row : row;  // of the block
    bool ok = true;
    uint32_t it = 0, steps = 0;
    while (walk.more()) {
      const Block blk = next_block(p, walk);
      const Seq sq = blk.sq;
      const int r0 = blk.mb * p.block_rows, tiles = blk.t1 - blk.t0, mine = turns.count(tiles);
      // the block's queries (rows from the last on are zeros) and what its rows see of the tree
      named_bar_sync(1, 256);  // the block before is through
      {
        constexpr int kUnits = D / 8;
        const int n = by_rows ? 256 : 128;
        const float turn = p.scale_log2 < 0.0f ? -1.0f : (p.scale_log2 == 0.0f ? 0.0f : 1.0f);
        for (int x = threadIdx.x; x < n * kUnits; x += 256) {
          const int r = x / kUnits, u = x % kUnits, g = r0 + r;
          uint4 w = make_uint4(0u, 0u, 0u, 0u);
          if (g < rows)
            w = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + blk.b * p.q_st[0] +
                                                     (blk.kvh * p.group + g / p.nodes) * p.q_st[1] +
                                                     (g % p.nodes) * p.q_st[2]) + u);
          if (turn != 1.0f) {
            uint32_t* e = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = turn < 0.0f ? e[i] ^ 0x80008000u : 0u;
          }
          *reinterpret_cast<uint4*>(sQ + (r >> 7) * C::kTileBytes + chunk_at<D>(r & 127, u)) = w;
        }
      }
      const bool tail = blk.t1 * kBN > sq.all;
      if (tail) {
        load_parents(p, sq, blk.b, ctl.parent, 256);
        named_bar_sync(1, 256);
        if (by_rows || t == 0) {
          uint32_t* bits = ctl.bits[slot_row];
          walk_up(sq, ctl.parent, r0 + slot_row < rows ? (r0 + slot_row) % p.nodes : kMaxNodes, bits);
          bits[kWords] = 0u;
        }
      }
      fence_proxy_async_smem();
      named_bar_sync(1, 256);
      if (lane == 0) mbar_arrive(&ctl.q_full);
      const bool active = r0 + (by_rows ? t * kBM : 0) + (warp & 3) * 32 < rows;  // else no row of this warp is real
      float m_run = -INFINITY, l = 0.0f;
      float vref = 0.0f;
      for (int n = 0; ok && n < mine; ++n) {
        const int i = turns.tile(n), j0 = (blk.t0 + i) * kBN;
        const uint32_t par = (steps + n) & 1u;
        const bool all = j0 + kBN <= sq.all;
        [[maybe_unused]] const int slot = static_cast<int>((it + i) % kScaleSlots);
        if (!wait_all(&ctl.s_full[t], par, abort, p.status)) {
          ok = false;
          break;
        }
        if (!active) {
          if (lane == 0) {
            mbar_arrive(&ctl.p_half[t]);
            mbar_arrive(&ctl.p_full[t]);
          }
          continue;
        }
        if constexpr (Q8) {
          if (!wait_all(&ctl.c_full[slot], ((it + i) / kScaleSlots) & 1u, abort, p.status)) {
            ok = false;
            break;
          }
        }
        tc_fence_after();
        uint32_t sr[kBN];
        tmem_ld_x64(tS, sr);
        tmem_ld_x64(tS + 64u, sr + 64);
        if constexpr (Q8) {
          const float4* kf = reinterpret_cast<const float4*>(ctl.kscale[slot]);
#pragma unroll
          for (int c = 0; c < kBN; c += 4) {
            const float4 f = kf[c / 4];
            float x[4];
            mul2v(x[0], x[1], __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]), f.x, f.y);
            mul2v(x[2], x[3], __uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3]), f.z, f.w);
#pragma unroll
            for (int e = 0; e < 4; ++e) sr[c + e] = __float_as_uint(x[e]);
          }
        }
        if (!all) {
          uint32_t vis[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int jq = j0 + 32 * q, a = jq - sq.past;  // node of its first key
            uint32_t u = 0u;
            if (a >= 0 && a < kMaxNodes) {
              const uint32_t* w = &ctl.bits[slot_row][a >> 5];
              u = __funnelshift_r(w[0], w[1], static_cast<uint32_t>(a & 31));
            } else if (a < 0 && a > -32) {
              u = ctl.bits[slot_row][0] << (-a);
            }
            vis[q] = (u & score::span_bits(0, sq.len, jq)) | score::span_bits(0, sq.all, jq);
          }
#pragma unroll
          for (int c = 0; c < kBN; ++c)
            if (!((vis[c >> 5] >> (c & 31)) & 1u)) sr[c] = __float_as_uint(-INFINITY);
        }
        float m8[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) m8[q] = -INFINITY;
#pragma unroll
        for (int c = 0; c < kBN; c += 2)
          m8[(c >> 1) & 7] = max3n(m8[(c >> 1) & 7], __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
        float mx = max3n(max3n(m8[0], m8[1], m8[2]), max3n(m8[3], m8[4], m8[5]), max3n(m8[6], m8[6], m8[7]));
        if constexpr (!Q8) mx *= factor;
        if (!(mx < INFINITY)) l = __uint_as_float(0x7fc00000u);  // a NaN or an infinite score: the row is NaN
        float shrink = 1.0f;
        if constexpr (kNorm) {
          const float to = ctl.vref[slot];
          if (n == 0) vref = to;
          // a warpgroup may have passed over a tile: the power's own ratio
          shrink = vref * __uint_as_float((254u << 23) - __float_as_uint(to));
          vref = to;
        }
        if (n == 0) {
          m_run = mx;
        } else {
          const bool need = mx > m_run + kRescaleLog2;
          if (__any_sync(0xffffffffu, need || shrink != 1.0f)) {
            // S_t followed the earlier P V, so that O_t stands
            const float alpha = need ? ex2(m_run - mx) : 1.0f;
            if (need) m_run = mx;
            l *= alpha;
            const float by = alpha * shrink;
            constexpr int kChunk = D < 32 ? D : 32;
#pragma unroll
            for (int c0 = 0; c0 < D; c0 += kChunk) {
              // in small pieces: the scores stay in registers
              uint32_t orow[8];
#pragma unroll
              for (int c1 = 0; c1 < kChunk; c1 += 8) {
                tmem_ld<8>(tO + static_cast<uint32_t>(c0 + c1), orow);
#pragma unroll
                for (int c = 0; c < 8; ++c) orow[c] = __float_as_uint(__uint_as_float(orow[c]) * by);
                tmem_st<8>(tO + static_cast<uint32_t>(c0 + c1), orow);
              }
            }
          }
        }
        const float neg_m = m_run == -INFINITY ? 0.0f : -m_run;
        const float by = Q8 ? 1.0f : factor;
        float la[4] = {0.0f, 0.0f, 0.0f, 0.0f}, lb[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < kBN; c += 2) {
          float x0 = __uint_as_float(sr[c]), x1 = __uint_as_float(sr[c + 1]), p0, p1;
          fma2(x0, x1, x0, x1, by, neg_m);
          p0 = ex2(x0);
          p1 = ex2(x1);
          add2(la[(c >> 1) & 3], lb[(c >> 1) & 3], p0, p1);
          if constexpr (Q8) {
            const float2 f = *reinterpret_cast<const float2*>(&ctl.vscale[slot][c]);
            float w0, w1;
            mul2v(w0, w1, p0, p1, f.x, f.y);
            // a masked weight is 0 whatever the scale
            p0 = all || p0 != 0.0f ? w0 : 0.0f;
            p1 = all || p1 != 0.0f ? w1 : 0.0f;
          }
          sr[c >> 1] = pack2<T>(p0, p1);
          if (c == kBN / 2 - 2) tmem_st_x32(tP, sr);
          if (c == 78) {
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl.p_half[t]);
          }
        }
        l += ((la[0] + lb[0]) + (la[1] + lb[1])) + ((la[2] + lb[2]) + (la[3] + lb[3]));
        tmem_st_x32(tP + 32u, sr + 32);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.p_full[t]);
      }
      // ---- epilogue
      if (ok && mine > 0) ok = wait_all(&ctl.o_done[t], (steps + mine - 1) & 1u, abort, p.status);
      if (!by_rows) {
        ctl.ml[threadIdx.x & 255] = make_float2(m_run, l);
        tc_fence_before();
        named_bar_sync(1, 256);  // the other warpgroup's last P V is done, too
        tc_fence_after();
      }
      const int head = blk.kvh * p.group + (r0 + slot_row) / p.nodes, node = (r0 + slot_row) % p.nodes;
      const bool real = r0 + slot_row < rows;
      if (ok && active) {
        float2 a = make_float2(m_run, l), z = make_float2(-INFINITY, 0.0f);
        if (!by_rows) {
          a = ctl.ml[row];
          z = ctl.ml[128 + row];
        }
        const int na = by_rows ? mine : Turns(false, 0).count(tiles), nz = by_rows ? 0 : Turns(false, 1).count(tiles);
        const float top = fmaxf(a.x, z.x), ref = top == -INFINITY ? 0.0f : top;
        float fa = na > 0 && !(a.x == -INFINITY && a.y == 0.0f) ? (by_rows ? 1.0f : ex2(a.x - ref)) : 0.0f;
        float fz = nz > 0 && !(z.x == -INFINITY && z.y == 0.0f) ? ex2(z.x - ref) : 0.0f;
        const float sum = (fa != 0.0f ? a.y * fa : 0.0f) + (fz != 0.0f ? z.y * fz : 0.0f);
        if constexpr (kNorm) {
          // each warpgroup's result is in parts of the power at its last tile
          fa *= na > 0 ? ctl.vref[(it + Turns(by_rows, by_rows ? t : 0).tile(na - 1)) % kScaleSlots] : 1.0f;
          fz *= nz > 0 ? ctl.vref[(it + Turns(false, 1).tile(nz - 1)) % kScaleSlots] : 1.0f;
        }
        const float rl = blk.whole ? (sum == 0.0f ? 0.0f : __frcp_rn(sum)) : 1.0f;
        const int64_t to = blk.whole ? 0 : part_row(p, cta, blk.slot, slot_row);
        T* out = blk.whole && real ? static_cast<T*>(p.o) + blk.b * p.o_st[0] + head * p.o_st[1] + node * p.o_st[2] : nullptr;
        // rows of the block's own columns: all, or with joined results half of them a warpgroup
        constexpr int kChunk = D < 32 ? 8 : 16;
        const int c_from = by_rows ? 0 : t * (D / 2), c_to = by_rows ? D : c_from + D / 2;
        const uint32_t tA = tbase + lane_off + kOCol + (by_rows ? static_cast<uint32_t>(t) * 128u : 0u);
        const uint32_t tZ = tbase + lane_off + kOCol + 128u;
        bool any_bad = false;
        if constexpr (!Q8) {
          if (tail)
            for (int w = 0; w < kWords; ++w) any_bad |= *const_cast<volatile uint32_t*>(&ctl.bad[w]) != 0u;
        }
#pragma unroll 1
        for (int c0 = c_from; c0 < c_to; c0 += kChunk) {
          __syncwarp();
          float o[kChunk];
          uint32_t u[kChunk];
#pragma unroll
          for (int c = 0; c < kChunk; ++c) o[c] = 0.0f;
          if (na > 0) {
            tmem_ld<kChunk>(tA + static_cast<uint32_t>(c0), u);
            if (fa != 0.0f) {
#pragma unroll
              for (int c = 0; c < kChunk; ++c) o[c] = __uint_as_float(u[c]) * fa;
            }
          }
          if (nz > 0) {
            tmem_ld<kChunk>(tZ + static_cast<uint32_t>(c0), u);
            if (fz != 0.0f) {
#pragma unroll
              for (int c = 0; c < kChunk; ++c) o[c] = __fmaf_rn(__uint_as_float(u[c]), fz, o[c]);
            }
          }
          if (any_bad && real) {
            for (int x = 0; x < sq.n; ++x) {
              const int j = sq.past + x;
              if (!((*const_cast<volatile uint32_t*>(&ctl.bad[x >> 5]) >> (x & 31)) & 1u)) continue;
              if (!((ctl.bits[slot_row][x >> 5] >> (x & 31)) & 1u) || j < blk.t0 * kBN || j >= blk.t1 * kBN) continue;
              const T* v = static_cast<const T*>(p.v) + blk.b * p.v_st[0] + blk.kvh * p.v_st[1] + j * p.v_st[2] + c0;
#pragma unroll
              for (int c = 0; c < kChunk; ++c) {
                const float f = to_f32(v[c]);
                if (!(fabsf(f) < INFINITY)) o[c] += f;
              }
            }
          }
          if (!real) continue;
          if (!blk.whole) {
#pragma unroll
            for (int c = 0; c < kChunk; c += 4)
              *reinterpret_cast<float4*>(p.part_o + to * D + c0 + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
          } else {
            const bool seen = node < sq.n;
            uint32_t h[kChunk / 2];
#pragma unroll
            for (int c = 0; c < kChunk; c += 2) h[c / 2] = seen ? pack2<T>(o[c] * rl, o[c + 1] * rl) : 0u;
#pragma unroll
            for (int c = 0; c < kChunk; c += 8)
              *reinterpret_cast<uint4*>(out + c0 + c) = make_uint4(h[c / 2], h[c / 2 + 1], h[c / 2 + 2], h[c / 2 + 3]);
          }
        }
        if (!blk.whole && real && (by_rows || t == 0)) p.part_ml[to] = make_float2(top, sum);
      }
      tc_fence_before();
      it += tiles;
      steps += mine;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(kTmemCols));
  }
}

template <typename T, int D, bool Q8>
int launch(const Params& p, cudaStream_t s) {
  using C = Cfg<D>;
  static OptIn opted;
  if (!opted.shared(tree_tc_kernel<T, D, Q8>, C::kLaunchSmem)) return FPK_ERR_CUDA;
  return launch_dependent(tree_tc_kernel<T, D, Q8>, dim3(static_cast<unsigned>(p.ctas)), kThreads, C::kLaunchSmem, s, p);
}
template <typename T>
int launch_type(const Params& p, int D, cudaStream_t s) {
  switch (D) {
    case 16: return p.ks ? launch<T, 16, true>(p, s) : launch<T, 16, false>(p, s);
    case 32: return p.ks ? launch<T, 32, true>(p, s) : launch<T, 32, false>(p, s);
    case 64: return p.ks ? launch<T, 64, true>(p, s) : launch<T, 64, false>(p, s);
    default: return p.ks ? launch<T, 128, true>(p, s) : launch<T, 128, false>(p, s);
  }
}

}  // namespace tc
}  // namespace tree
}  // namespace fpk
