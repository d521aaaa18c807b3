// Tree attention on the 5th-generation tensor cores (f16 and bf16, caches of that type or in 8
// bits), for more rows than mma.sync's kernel takes.
//
//   S = Q K^T;  x = S * (scale, and the key's scale);  P = exp2(x - m);  O += (P * the value's scale) V
//
// The rows are the nodes of all heads of a group (row r: head r / nodes, node r % nodes), in tiles
// of 128; a CTA takes its part of the blocks' 128-key tiles (tree_common.cuh).  Two warpgroups do the
// softmax, four threads a row: with more than 128 rows each has its own row tile and both take every
// key tile; with up to 128 they take every other key tile of the same rows, each with its own
// maximum, sum and result, which are joined at the block's end.  Either way one's exponentials run
// beside the other's waits.  Roles:
//   warps 0-3, 4-7  softmax of row tile, or key tiles, 0 and 1
//   warps 8-11      K and V from memory into the tensor cores' layout
//   warps 12, 13    UMMA issuers for warpgroup 0 and 1 (12 owns TMEM)
// TMEM: S_t at column 128 t, in halves of 64 keys, each with its P over its first half; O_t at
// 256 + 128 t.  A half is a step of the softmax (its scores fit a thread's registers, and are read once):
// while one is weighed, P V and the next tile's Q K^T of the other run.
//
// 8-bit caches: the loaders hold a tile's bytes in registers while it is on its way, and write them as
// 16-bit numbers (exact) in the layout that a TMA load would give; K V in shared memory is then as
// for a 16-bit cache.  Scales go with the scores and the weights, 128 f32 of each a tile, and in f16 the
// power of two of a value's scale with the score (tree_common.cuh).
//
// Only tiles with rows from `all` on look at masks.  There what is not finite in a 16-bit V becomes
// zero and its node is noted; in the epilogue a row that sees a noted node looks at it again and adds what
// is not finite (a note of another block's node finds nothing, or the row's own).
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

constexpr int kBM = 128, kBN = kUnit, kHalf = kBN / 2;
constexpr int kStages = 2;      // of K, and of V
constexpr int kScaleSlots = 4;  // tiles whose scales are held
constexpr int kSoftWarps = 8, kLoadWarps = 4, kLoadWarp = 8, kMmaWarp = 12;
constexpr int kLoadThreads = 32 * kLoadWarps;
constexpr int kThreads = 512;
// setmaxnreg split of 512 x 128: 256 x 144 softmax, 128 x 136 loaders, 128 x 88 the rest
constexpr int kRegsSoft = 144, kRegsLoad = 136, kRegsCtl = 88;
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
// d = a b + c
__device__ __forceinline__ void fma2p(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0, float c1) {
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
// 4 bytes as 4 numbers of T (tree_dec.cu); in order, so that a tile's are not all made before the first is stored
template <typename T>
__device__ __forceinline__ uint2 four_of(uint32_t u) {
  uint2 r;
  if constexpr (std::is_same<T, __half>::value) {
    u ^= 0x80808080u;
    asm volatile("sub.rn.f16x2 %0, %1, %2;" : "=r"(r.x) : "r"(__byte_perm(u, 0x64646464u, 0x4140u)), "r"(0x64806480u));
    asm volatile("sub.rn.f16x2 %0, %1, %2;" : "=r"(r.y) : "r"(__byte_perm(u, 0x64646464u, 0x4342u)), "r"(0x64806480u));
  } else {
    const uint32_t a = __byte_perm(u, 0x43434343u, 0x4140u), b = __byte_perm(u, 0x43434343u, 0x4342u);
    asm volatile("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r.x) : "r"(a & 0xff7fff7fu), "r"(a & 0xff80ff80u));
    asm volatile("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r.y) : "r"(b & 0xff7fff7fu), "r"(b & 0xff80ff80u));
  }
  return r;
}
// mbar_wait by every lane, with one answer for the warp
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, volatile int* abort, int* status) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status, kWaitLimitNs));
}

// what a thread takes of two keys' scales
template <bool NORM>
using ScaleOf = std::conditional_t<NORM, float4, float2>;

struct Ctl {
  uint64_t q_full[2];                // of a warpgroup's issuer: a phase a block in which it has key tiles
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[2][2], p_full[2][2], o_done[2][2];  // of a warpgroup's half tiles: a phase a tile
  uint64_t c_full[kScaleSlots];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  uint32_t bad[kWords];              // nodes whose V was not finite, of this CTA's blocks so far
  // of two neighbouring keys: what their scores are multiplied by (x, y), and in f16 what is added (z, w)
  float4 kscale[kScaleSlots][kBN / 2];
  // what their weights are multiplied by (x, y), and in f16 what counts for the sum (z, w)
  float4 vscale[kScaleSlots][kBN / 2];
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

// 16 bytes, zeros where !in (nothing is read then), into registers that hold something already: a load whose
// result is moved, or that stands where the bytes are used, is waited for one by one.
__device__ __forceinline__ void load16(uint4& w, const void* src, bool in) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\t@!p mov.b32 %0, 0;\n\t@!p mov.b32 %1, 0;\n\t@!p mov.b32 %2, 0;\n\t"
      "@!p mov.b32 %3, 0;\n\t@p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "+r"(w.x), "+r"(w.y), "+r"(w.z), "+r"(w.w)
      : "l"(src), "r"(in ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void load4(float& w, const float* src, bool in) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@!p mov.b32 %0, 0;\n\t@p ld.global.b32 %0, [%1];\n\t}"
               : "+f"(w)
               : "l"(src), "r"(in ? 1 : 0)
               : "memory");
}

// A loader's part of one operand of a key tile on its way: 8-bit rows in registers.  A thread's rows lie
// 128 / kUnits apart, a multiple of the swizzle's period.
template <int D>
struct Bytes {
  static constexpr int kUnits = D / 16;                    // 16 bytes of a row
  static constexpr int kN = 128 * kUnits / kLoadThreads;   // a thread
  static constexpr int kApart = kLoadThreads / kUnits;     // rows
  uint4 w[kN];
  // `src`: the tile's first row; n: its rows that are there
  __device__ __forceinline__ void load(const uint8_t* src, int64_t stride, int n, int tid) {
    const int r = tid / kUnits;
    src += r * stride + (tid % kUnits) * 16;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      load16(w[i], src, r + i * kApart < n);
      src += kApart * stride;
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(uint8_t* tile, int tid) const {
    const int r = tid / kUnits, u = tid % kUnits;
    // D = 128: eight lanes write even chunks of one box and odd ones of the other, no bank conflict
    const bool odd = D == 128 && (u & 4);
    uint8_t* first = tile + chunk_at<D>(r, 2 * u + (odd ? 1 : 0));
    uint8_t* second = tile + chunk_at<D>(r, 2 * u + (odd ? 0 : 1));
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const uint2 a = four_of<T>(w[i].x), b = four_of<T>(w[i].y), c = four_of<T>(w[i].z), d = four_of<T>(w[i].w);
      const uint4 lo = make_uint4(a.x, a.y, b.x, b.y), hi = make_uint4(c.x, c.y, d.x, d.y);
      *reinterpret_cast<uint4*>(first + i * kApart * Cfg<D>::kRowBytes) = odd ? hi : lo;
      *reinterpret_cast<uint4*>(second + i * kApart * Cfg<D>::kRowBytes) = odd ? lo : hi;
    }
  }
};
// TMEM in the layout of a matrix fragment: 16 lanes, each thread rows lane / 4 and lane / 4 + 8, of each
// 8 columns 2 (lane % 4) and the next (f32), of each 4 words word lane % 4 (pairs of 16 bits)
__device__ __forceinline__ void frag_ld_32(uint32_t taddr, uint32_t* r) {  // 32 columns
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void frag_ld_8(uint32_t taddr, uint32_t* r) {  // 8 columns
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void frag_st_8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x1.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3])
               : "memory");
}
__device__ __forceinline__ void frag_st_words(uint32_t taddr, const uint32_t* r) {  // 32 words: 64 pairs' columns
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// N columns of a thread's row
template <int N>
__device__ __forceinline__ void row_ld(uint32_t taddr, uint32_t* r) {
  if constexpr (N >= 8)
    tmem_ld<N>(taddr, r);
  else
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(taddr)
                 : "memory");
}
// the loads so far have arrived; the values pass through so that no use is moved ahead
template <int N>
__device__ __forceinline__ void frag_wait(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

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
    const uint32_t readers = p.by_rows ? 2 : 1;  // issuers that read a K or V tile
    for (int s = 0; s < NS; ++s) {
      mbar_init(&ctl.k_full[s], kLoadWarps);
      mbar_init(&ctl.k_empty[s], readers);
      mbar_init(&ctl.v_full[s], kLoadWarps);
      mbar_init(&ctl.v_empty[s], readers);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&ctl.q_full[t], kSoftWarps);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&ctl.s_full[t][h], 1);
        mbar_init(&ctl.p_full[t][h], 4);
        mbar_init(&ctl.o_done[t][h], 1);
      }
    }
    for (int s = 0; s < kScaleSlots; ++s) mbar_init(&ctl.c_full[s], kLoadWarps);
    mbar_init(&ctl.drain, 2);
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
    if (warp < kMmaWarp + 2) {
      // ----------------------------------- UMMA issuers (whole warps), one a warpgroup of the softmax
      constexpr uint32_t idesc_qk = idesc16<T, kBM, kHalf, false>();
      constexpr uint32_t idesc_pv = idesc16<T, kBM, D, true>();
      constexpr uint64_t kTileStep = static_cast<uint64_t>(C::kTileBytes >> 4);
      const uint32_t leader = elect_one();
      const uint64_t q_desc = sdesc(smem_u32(sQ), 16, 8 * C::kRowBytes, C::kLayout);
      const uint64_t k_desc = sdesc(smem_u32(sK), 16, 8 * C::kRowBytes, C::kLayout);
      const uint64_t v_desc = sdesc(smem_u32(sV), C::kBoxBytes, 8 * C::kRowBytes, C::kLayout);
      // What one waits for per step is kept to the one barrier that the step needs: a wait costs it some 200
      // cycles even where the phase is over.  (One issuer for both warpgroups, four steps a tile, us when it was
      // tried: 8 caches of 16384 with 64 nodes of D 128, 8-bit 226, two 225; 16 ragged ones of 4096 with 16 nodes
      // 86, two 78; 8 ragged ones of 8192 with 49 nodes of D 64, 16-bit 74, two 72.)
      const int t = warp - kMmaWarp;
      bool ok = true;
      uint32_t it = 0;     // tiles of the blocks before
      uint32_t steps = 0;  // of the warpgroup
      uint32_t blocks = 0; // with key tiles of the warpgroup
      auto issue_qk = [&](uint32_t tile, int half) {
        const uint32_t s = tile % NS;
        if (half == 0) {
          if (!mbar_wait_w(&ctl.k_full[s], (tile / NS) & 1u, abort, p.status, kWaitLimitNs)) return false;
          tc_fence_after();
        }
        const uint64_t a0 = q_desc + static_cast<uint64_t>(by_rows ? t : 0) * kTileStep;
        const uint64_t b0 = k_desc + static_cast<uint64_t>(s) * kTileStep + static_cast<uint64_t>(half * ((kHalf * C::kRowBytes) >> 4));
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          constexpr int kSteps = C::kKStepsPerBox;
          const uint64_t off = static_cast<uint64_t>((kk / kSteps) * (C::kBoxBytes >> 4) + (kk % kSteps) * 2);
          mma_ss_l(leader, tbase + static_cast<uint32_t>(t * 128 + half * kHalf), a0 + off, b0 + off, idesc_qk, kk > 0 ? 1u : 0u);
        }
        mma_commit_l(leader, &ctl.s_full[t][half]);
        if (half == 1) mma_commit_l(leader, &ctl.k_empty[s]);
        return true;
      };
      while (walk.more()) {
        const Block blk = next_block(p, walk);
        const int tiles = blk.t1 - blk.t0, mine = Turns(by_rows, t).count(tiles);
        const auto tile_of = [&](int n) { return it + static_cast<uint32_t>(by_rows ? n : 2 * n + t); };
        // Only where the softmax then waits for this issuer: one that fell two blocks behind would take the
        // barrier's phase for the one before.
        if (mine > 0) {
          ok = ok && mbar_wait_w(&ctl.q_full[t], blocks & 1u, abort, p.status, kWaitLimitNs);
          ++blocks;
          ok = ok && issue_qk(tile_of(0), 0) && issue_qk(tile_of(0), 1);
        }
#pragma unroll 1
        for (int x = 0; ok && x < 2 * mine; ++x) {
          const int half = x & 1, n = x >> 1;
          const uint32_t tile = tile_of(n), s = tile % NS;
          if (half == 0) ok = mbar_wait_w(&ctl.v_full[s], (tile / NS) & 1u, abort, p.status, kWaitLimitNs);
          ok = ok && mbar_wait_w(&ctl.p_full[t][half], (steps + n) & 1u, abort, p.status, kWaitLimitNs);
          if (!ok) break;
          tc_fence_after();
          const uint32_t d_tmem = tbase + kOCol + static_cast<uint32_t>(t) * 128u;
          const uint32_t a_tmem = tbase + static_cast<uint32_t>(t * 128 + half * kHalf);
          const uint64_t b0 = v_desc + static_cast<uint64_t>(s) * kTileStep + static_cast<uint64_t>(half * ((kHalf * C::kRowBytes) >> 4));
#pragma unroll
          for (int kk = 0; kk < kHalf / 16; ++kk)
            mma_ts_l(leader, d_tmem, a_tmem + static_cast<uint32_t>(kk * 8), b0 + static_cast<uint64_t>(kk * C::kRowBytes),
                     idesc_pv, (x > 0 || kk > 0) ? 1u : 0u);
          mma_commit_l(leader, &ctl.o_done[t][half]);
          if (half == 1) mma_commit_l(leader, &ctl.v_empty[s]);
          if (n + 1 < mine) ok = issue_qk(tile_of(n + 1), half);
        }
        it += tiles;
        steps += mine;
      }
      // every UMMA issued so far must finish before TMEM is freed
      mma_commit_l(leader, &ctl.drain);
      drain_wait_w(&ctl.drain, 0, p.status);
    }
  } else if (warp >= kLoadWarp) {
    setmaxnreg_inc<kRegsLoad>();
    // ------------------------------------------------------------- loaders
    // K runs a tile ahead of V: K0 K1 V0 K2 V1 ...  The issuer takes them in an order in which nothing
    // that it waits for comes behind a place that only its later steps set free.
    const int tid = static_cast<int>(threadIdx.x) - kLoadWarp * 32;
    constexpr int kSize = Q8 ? 1 : 2;
    struct Tile {
      const uint8_t *k, *v;  // first rows
      int n, j0;             // rows from the first on, its number
      int all, past;
    };
    Tile kt{}, vt{};
    [[maybe_unused]] const float *ksp = nullptr, *vsp = nullptr;
    int left = 0;
    auto next = [&]() {
      if (left == 0) {
        if (!walk.more()) {
          kt.n = 0;
          return false;
        }
        const Block blk = next_block(p, walk);
        kt.j0 = blk.t0 * kBN;
        kt.n = blk.sq.len - kt.j0;
        kt.all = blk.sq.all;
        kt.past = blk.sq.past;
        kt.k = static_cast<const uint8_t*>(p.k) + (blk.b * p.k_st[0] + blk.kvh * p.k_st[1] + kt.j0 * p.k_st[2]) * kSize;
        kt.v = static_cast<const uint8_t*>(p.v) + (blk.b * p.v_st[0] + blk.kvh * p.v_st[1] + kt.j0 * p.v_st[2]) * kSize;
        if constexpr (Q8) {
          ksp = p.ks + blk.b * p.ks_st[0] + blk.kvh * p.ks_st[1] + kt.j0 * p.ks_st[2];
          vsp = p.vs + blk.b * p.vs_st[0] + blk.kvh * p.vs_st[1] + kt.j0 * p.vs_st[2];
        }
        left = blk.t1 - blk.t0;
      } else {
        kt.k += kBN * p.k_st[2] * kSize;
        kt.v += kBN * p.v_st[2] * kSize;
        if constexpr (Q8) {
          ksp += kBN * p.ks_st[2];
          vsp += kBN * p.vs_st[2];
        }
        kt.n -= kBN;
        kt.j0 += kBN;
      }
      --left;
      return true;
    };
    auto arrive = [&](uint64_t* bar) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    const auto empty = [](uint32_t tile) { return ((tile / NS) & 1u) ^ 1u; };
    uint32_t ik = 0, iv = 0;  // tiles of K, V
    bool have_k = next(), have_v = false;
    if constexpr (Q8) {
      Bytes<D> kw{}, vw{};  // on their way, asked for when the registers got free (nothing, behind the last tile)
      float ks = 0.0f, vs = 0.0f;
      auto load_k = [&]() {
        kw.load(kt.k, p.k_st[2], kt.n, tid);
        load4(ks, ksp + tid * p.ks_st[2], tid < kt.n);
        load4(vs, vsp + tid * p.vs_st[2], tid < kt.n);
      };
      load_k();
      while (have_k || have_v) {
        const bool ahead = have_k;
        const Tile now = kt;
        if (have_k) {
          const int slot = static_cast<int>(ik % kScaleSlots);
          // the scales' slot is free with the K stage: the tile of four before has been weighed
          if (!wait_all(&ctl.k_empty[ik % NS], empty(ik), abort, p.status)) break;
          float* kf = reinterpret_cast<float*>(&ctl.kscale[slot][tid >> 1]) + (tid & 1);
          float* vf = reinterpret_cast<float*>(&ctl.vscale[slot][tid >> 1]) + (tid & 1);
          const ValueScale x = value_scale<kNorm>(vs);
          const bool odd = !(fabsf(vs) < INFINITY);
          kf[0] = odd ? __uint_as_float(0x7fc00000u) : ks * factor;
          vf[0] = odd ? 0.0f : x.rest;
          if constexpr (kNorm) {
            kf[2] = x.lift;
            vf[2] = x.lower;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl.c_full[slot]);
          kw.template store<T>(sK + (ik % NS) * C::kTileBytes, tid);
          arrive(&ctl.k_full[ik % NS]);
          ++ik;
          have_k = next();
        }
        load_k();
        if (have_v) {
          if (!wait_all(&ctl.v_empty[iv % NS], empty(iv), abort, p.status)) break;
          vw.template store<T>(sV + (iv % NS) * C::kTileBytes, tid);
          arrive(&ctl.v_full[iv % NS]);
          ++iv;
        }
        have_v = ahead;
        vw.load(now.v, p.v_st[2], ahead ? now.n : 0, tid);
      }
    } else {
      // asynchronous copies, up to three operands on their way
      constexpr int kUnits = D / 8, kN = 128 * kUnits / kLoadThreads;
      constexpr int kApart = kLoadThreads / kUnits;  // a thread's rows: a multiple of the swizzle's period
      auto copy = [&](uint8_t* tile, const uint8_t* src, int64_t stride, int n) {
        const int r = tid / kUnits;
        const uint32_t to = smem_u32(tile + chunk_at<D>(r, tid % kUnits));
        src += (tid % kUnits) * 16;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          const bool in = r + i * kApart < n;  // beyond the length: zeros, nothing read
          asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(to + i * kApart * C::kRowBytes),
                       "l"(src + (in ? r + i * kApart : 0) * stride), "r"(in ? 16 : 0)
                       : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      // V of a tile with keys that some row may not see: what is not finite becomes zero
      auto clean = [&](uint8_t* tile, int j0, int all, int past, int n) {
#pragma unroll 1
        for (int i = 0; i < kN; ++i) {
          const int x = tid + i * kLoadThreads, r = x / kUnits, u = x % kUnits;
          if (j0 + r < all || r >= n) continue;
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
            const int node = j0 + r - past;
            atomicOr(&ctl.bad[node >> 5], 1u << (node & 31));
          }
        }
      };
      uint32_t dk = 0, dv = 0;   // tiles signalled
      int way = 0;               // operands on their way, the oldest first in the order above
      int4 of[NS] = {};          // of V's stages: j0, all, past, n
      // the oldest, which has arrived
      auto signal = [&]() {
        if (dk < ik && dk < dv + 2) {
          arrive(&ctl.k_full[dk % NS]);
          ++dk;
        } else {
          const int4 x = dv % NS == 0 ? of[0] : of[1];
          if (x.x + kBN > x.y) clean(sV + (dv % NS) * C::kTileBytes, x.x, x.y, x.z, x.w);
          arrive(&ctl.v_full[dv % NS]);
          ++dv;
        }
        --way;
      };
      // a place for the next: what is on its way is signalled ahead of a wait that may need it
      auto place = [&](uint64_t* bar, uint32_t par) {
        if (__all_sync(0xffffffffu, mbar_test(bar, par))) return true;
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        while (way > 0) signal();
        return wait_all(bar, par, abort, p.status);
      };
      auto sent = [&]() {
        if (++way > 2) {
          asm volatile("cp.async.wait_group 2;" ::: "memory");
          signal();
        }
      };
      while (have_k || have_v) {
        const bool ahead = have_k;
        const Tile now = kt;
        if (have_k) {
          if (!place(&ctl.k_empty[ik % NS], empty(ik))) break;
          copy(sK + (ik % NS) * C::kTileBytes, kt.k, p.k_st[2] * 2, kt.n);
          ++ik;
          sent();
          have_k = next();
        }
        if (have_v) {
          if (!place(&ctl.v_empty[iv % NS], empty(iv))) break;
          copy(sV + (iv % NS) * C::kTileBytes, vt.v, p.v_st[2] * 2, vt.n);
          const int4 x = make_int4(vt.j0, vt.all, vt.past, vt.n);
          if (iv % NS == 0) of[0] = x;
          else of[1] = x;
          ++iv;
          sent();
        }
        have_v = ahead;
        if (ahead) vt = now;
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      while (way > 0) signal();
    }
  } else {
    // ------------------------------------------------------ softmax + epilogue
    setmaxnreg_inc<kRegsSoft>();
    const int t = warp >> 2, row = static_cast<int>(threadIdx.x) & (kBM - 1);
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tbase + lane_off + static_cast<uint32_t>(t * 128);
    const uint32_t tO = tbase + lane_off + kOCol + static_cast<uint32_t>(t) * 128u;
    const uint32_t tP = tS;  // a lane offset of 16 << 16 has the warp's other 16 lanes
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
      const bool tail = blk.t1 * kBN > sq.all;
      if (tail) load_parents(p, sq, blk.b, ctl.parent, 256);
      {
        constexpr int kUnits = D / 8, kAtOnce = 8;
        const int n = (by_rows ? 256 : 128) * kUnits;
        const float turn = p.scale_log2 < 0.0f ? -1.0f : (p.scale_log2 == 0.0f ? 0.0f : 1.0f);
        const T* qb = static_cast<const T*>(p.q) + blk.b * p.q_st[0] + blk.kvh * p.group * p.q_st[1];
        for (int x0 = static_cast<int>(threadIdx.x); x0 < n; x0 += 256 * kAtOnce) {
          uint4 w[kAtOnce] = {};
#pragma unroll
          for (int i = 0; i < kAtOnce; ++i) {
            const int x = x0 + 256 * i, g = r0 + x / kUnits;
            const bool in = x < n && g < rows;
            load16(w[i], qb + (in ? g / p.nodes * p.q_st[1] + g % p.nodes * p.q_st[2] + x % kUnits * 8 : 0), in);
          }
#pragma unroll
          for (int i = 0; i < kAtOnce; ++i) {
            const int x = x0 + 256 * i, r = x / kUnits;
            if (x >= n) continue;
            if (turn != 1.0f) {
              uint32_t* e = reinterpret_cast<uint32_t*>(&w[i]);
#pragma unroll
              for (int j = 0; j < 4; ++j) e[j] = turn < 0.0f ? e[j] ^ 0x80008000u : 0u;
            }
            *reinterpret_cast<uint4*>(sQ + (r >> 7) * C::kTileBytes + chunk_at<D>(r & 127, x % kUnits)) = w[i];
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        for (int w = 0; w < 2; ++w)
          if (Turns(by_rows, w).count(tiles) > 0) mbar_arrive(&ctl.q_full[w]);
      }
      if (tail) {  // beside the first Q K^T
        named_bar_sync(1, 256);
        if (by_rows || t == 0) {
          uint32_t* bits = ctl.bits[slot_row];
          walk_up(sq, ctl.parent, r0 + slot_row < rows ? (r0 + slot_row) % p.nodes : kMaxNodes, bits);
          bits[kWords] = 0u;
        }
        named_bar_sync(1, 256);
      }
      const bool active = r0 + (by_rows ? t * kBM : 0) + (warp & 3) * 32 < rows;  // else no row of this warp is real
      // this thread's part of 4 rows of the warp's 32, lane / 4 and 8, 16 and 24 more: of each 8 keys two,
      // so that one scale serves four scores (a thread a row reads as many scales as scores from
      // shared memory, whose bandwidth that took: 6 us a tile).  A quad shares a row.
      const int g = lane >> 2, q4 = lane & 3, bits_row = slot_row - lane;
      float m_run[4], l[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        m_run[h] = -INFINITY;
        l[h] = 0.0f;
      }
#pragma unroll 1
      for (int x = 0; x < 2 * mine; ++x) {
        const int n = x >> 1, half = x & 1, i = turns.tile(n), j0 = (blk.t0 + i) * kBN + half * kHalf;
        const bool all = j0 + kHalf <= sq.all;
        [[maybe_unused]] const int slot = static_cast<int>((it + i) % kScaleSlots);
        if (!wait_all(&ctl.s_full[t][half], (steps + n) & 1u, abort, p.status)) {
          ok = false;
          break;
        }
        if (!active) {
          if (lane == 0) mbar_arrive(&ctl.p_full[t][half]);
          continue;
        }
        if constexpr (Q8) {
          if (half == 0 && !wait_all(&ctl.c_full[slot], ((it + i) / kScaleSlots) & 1u, abort, p.status)) {
            ok = false;
            break;
          }
        }
        tc_fence_after();
        uint32_t sr[64];  // [2][8 key groups][4]: lanes 0-15 and 16-31 of the warp's
        {
          const uint32_t from = tS + static_cast<uint32_t>(half * kHalf);
          frag_ld_32(from, sr);
          frag_ld_32(from + 32u, sr + 16);
          frag_ld_32(from + (16u << 16), sr + 32);
          frag_ld_32(from + (16u << 16) + 32u, sr + 48);
          [[maybe_unused]] ScaleOf<kNorm> f[8];
          if constexpr (Q8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = *reinterpret_cast<const ScaleOf<kNorm>*>(&ctl.kscale[slot][half * (kHalf / 2) + j * 4 + q4]);
          }
          frag_wait<64>(sr);
          if constexpr (Q8) {
#pragma unroll
            for (int c = 0; c < 64; c += 2) {
              float x0, x1;
              const auto& k = f[(c >> 2) & 7];
              if constexpr (kNorm) fma2p(x0, x1, __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]), k.x, k.y, k.z, k.w);
              else mul2v(x0, x1, __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]), k.x, k.y);
              sr[c] = __float_as_uint(x0);
              sr[c + 1] = __float_as_uint(x1);
            }
          }
        }
        if (__builtin_expect(!all, 0)) {  // out of the loop's way
#pragma unroll
          for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int word = 0; word < 2; ++word) {
              const int jq = j0 + word * 32, a = jq - sq.past;  // node of its first key
              const uint32_t* row_bits = ctl.bits[bits_row + g + 8 * h];
              uint32_t u = 0u;
              if (a >= 0 && a < kMaxNodes) u = __funnelshift_r(row_bits[a >> 5], row_bits[(a >> 5) + 1], static_cast<uint32_t>(a & 31));
              else if (a < 0 && a > -32) u = row_bits[0] << (-a);
              u = (u & score::span_bits(0, sq.len, jq)) | score::span_bits(0, sq.all, jq);
              u >>= q4 * 2;
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (!((u >> (j * 8 + e)) & 1u))
                    sr[(h >> 1) * 32 + (word * 4 + j) * 4 + (h & 1) * 2 + e] = __float_as_uint(-INFINITY);
            }
        }
        float mx[4];
        bool any_need = false;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int at = (h >> 1) * 32 + (h & 1) * 2;
          float m2 = max3n(__uint_as_float(sr[at]), __uint_as_float(sr[at + 1]), __uint_as_float(sr[at + 4]));
          mx[h] = max3n(__uint_as_float(sr[at + 5]), __uint_as_float(sr[at + 8]), __uint_as_float(sr[at + 9]));
#pragma unroll
          for (int j = 3; j < 8; ++j) {
            if (j & 1) mx[h] = max3n(mx[h], __uint_as_float(sr[at + 4 * j]), __uint_as_float(sr[at + 4 * j + 1]));
            else m2 = max3n(m2, __uint_as_float(sr[at + 4 * j]), __uint_as_float(sr[at + 4 * j + 1]));
          }
          mx[h] = max3n(mx[h], m2, m2);
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) mx[h] = max3n(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1), mx[h]);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          mx[h] = max3n(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2), mx[h]);
          if constexpr (!Q8) mx[h] *= factor;
          if (!(mx[h] < INFINITY)) l[h] = __uint_as_float(0x7fc00000u);  // a NaN or an infinite score: the row is NaN
          any_need |= mx[h] > m_run[h] + kRescaleLog2;
        }
        if (x == 0) {
#pragma unroll
          for (int h = 0; h < 4; ++h) m_run[h] = mx[h];
        } else if (__builtin_expect(__any_sync(0xffffffffu, any_need), 0)) {
          // the half before may still be on its way into O_t
          if (!wait_all(&ctl.o_done[t][half ^ 1], (steps + n - (half ^ 1)) & 1u, abort, p.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          float by[4];
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            float alpha = 1.0f;
            if (mx[h] > m_run[h] + kRescaleLog2) {
              alpha = ex2(m_run[h] - mx[h]);
              m_run[h] = mx[h];
              l[h] *= alpha;
            }
            by[h] = alpha;
          }
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += 8) {
            uint32_t o[8];
            const uint32_t at = tO + static_cast<uint32_t>(c0);
            frag_ld_8(at, o);
            frag_ld_8(at + (16u << 16), o + 4);
            frag_wait<8>(o);
#pragma unroll
            for (int c = 0; c < 8; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * by[c >> 1]);
            frag_st_8(at, o);
            frag_st_8(at + (16u << 16), o + 4);
          }
        }
        float neg_m[4], la[4][2];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          neg_m[h] = m_run[h] == -INFINITY ? 0.0f : -m_run[h];
          la[h][0] = la[h][1] = 0.0f;
        }
        uint32_t w[32];  // [2][8 key groups][2]
        [[maybe_unused]] ScaleOf<kNorm> f[8];
        if constexpr (Q8) {
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = *reinterpret_cast<const ScaleOf<kNorm>*>(&ctl.vscale[slot][half * (kHalf / 2) + j * 4 + q4]);
        }
#pragma unroll
        for (int c = 0; c < 32; ++c) {  // pairs of keys
          const int h = (c >> 4) * 2 + (c & 1), j = (c >> 1) & 7, at = (h >> 1) * 32 + j * 4 + (h & 1) * 2;
          float x0, x1, p0, p1;
          fma2(x0, x1, __uint_as_float(sr[at]), __uint_as_float(sr[at + 1]), Q8 ? 1.0f : factor, neg_m[h]);
          p0 = ex2(x0);
          p1 = ex2(x1);
          if constexpr (kNorm) fma2p(la[h][0], la[h][1], p0, p1, f[j].z, f[j].w, la[h][0], la[h][1]);
          else add2(la[h][0], la[h][1], p0, p1);
          if constexpr (Q8) mul2v(p0, p1, p0, p1, f[j].x, f[j].y);
          w[(c >> 4) * 16 + j * 2 + (c & 1)] = pack2<T>(p0, p1);
        }
        const uint32_t to = tP + static_cast<uint32_t>(half * kHalf);
        frag_st_words(to, w);
        frag_st_words(to + (16u << 16), w + 16);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.p_full[t][half]);
#pragma unroll
        for (int h = 0; h < 4; ++h) l[h] += la[h][0] + la[h][1];
      }
      // ---- epilogue
      if (ok && mine > 0) ok = wait_all(&ctl.o_done[t][1], (steps + mine - 1) & 1u, abort, p.status);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if (q4 == 0) ctl.ml[(threadIdx.x & ~31u) + g + 8 * h] = make_float2(m_run[h], l[h]);
      }
      __syncwarp();
      if (!by_rows) {
        tc_fence_before();
        named_bar_sync(1, 256);  // the other warpgroup's last P V is done, too
        tc_fence_after();
      }
      const int node = (r0 + slot_row) % p.nodes;
      const bool real = r0 + slot_row < rows;
      if (ok && active) {
        // from here on a thread a row
        const float2 a = ctl.ml[slot_row], z = by_rows ? make_float2(-INFINITY, 0.0f) : ctl.ml[128 + row];
        const int na = by_rows ? mine : Turns(false, 0).count(tiles), nz = by_rows ? 0 : Turns(false, 1).count(tiles);
        const float top = fmaxf(a.x, z.x), ref = top == -INFINITY ? 0.0f : top;
        const bool some_a = na > 0 && !(a.x == -INFINITY && a.y == 0.0f), some_z = nz > 0 && !(z.x == -INFINITY && z.y == 0.0f);
        const float fa = some_a ? (by_rows ? 1.0f : ex2(a.x - ref)) : 0.0f, fz = some_z ? ex2(z.x - ref) : 0.0f;
        const float sum = a.y * fa + z.y * fz;  // a NaN stays, also where the weight is 0
        const float rl = blk.whole ? (sum == 0.0f ? 0.0f : __frcp_rn(sum)) : 1.0f;
        bool any_bad = false;
        if (!Q8 && tail)
          for (int w = 0; w < kWords; ++w) any_bad |= *const_cast<volatile uint32_t*>(&ctl.bad[w]) != 0u;
        // The block's columns of the warp's rows: all, or with joined results half of them a warpgroup.  A
        // thread a row makes them, and they go through shared memory (over the queries, which are read no
        // more), so that a warp writes whole rows: sixteen bytes a row and store took 11700 cycles a block of 256 rows.
        constexpr int kChunk = D / 4, kVecs = kChunk / 4;  // columns at a time, and 16-byte vectors of f32
        float4* room = reinterpret_cast<float4*>(sQ + warp * (2 * C::kTileBytes / kSoftWarps));  // [32][kVecs]
        const int c_from = by_rows ? 0 : t * (D / 2), c_to = by_rows ? D : c_from + D / 2;
        const uint32_t tA = tbase + lane_off + kOCol + (by_rows ? static_cast<uint32_t>(t) * 128u : 0u);
        const uint32_t tZ = tbase + lane_off + kOCol + 128u;
        const int first_row = slot_row - lane;
        constexpr int kSwap = kVecs - 1;  // of the vectors of a row by its number: no bank conflicts
#pragma unroll 1
        for (int c0 = c_from; c0 < c_to; c0 += kChunk) {
          __syncwarp();
          float o[kChunk];
          uint32_t u[kChunk < 8 ? 8 : kChunk];
#pragma unroll
          for (int c = 0; c < kChunk; ++c) o[c] = 0.0f;
          if (na > 0) {
            row_ld<kChunk>(tA + static_cast<uint32_t>(c0), u);
            if (some_a) {  // also where the weight is 0: what is not finite in a value that was seen stays so
#pragma unroll
              for (int c = 0; c < kChunk; ++c) o[c] = __uint_as_float(u[c]) * fa;
            }
          }
          if (nz > 0) {
            row_ld<kChunk>(tZ + static_cast<uint32_t>(c0), u);
            if (some_z) {
#pragma unroll
              for (int c = 0; c < kChunk; ++c) o[c] = __fmaf_rn(__uint_as_float(u[c]), fz, o[c]);
            }
          }
          if (!Q8 && any_bad && real) {
            for (int x = 0; x < sq.n; ++x) {
              const int j = sq.past + x;
              if (!((*const_cast<volatile uint32_t*>(&ctl.bad[x >> 5]) >> (x & 31)) & 1u)) continue;
              // of this part, and held: a tree may end behind the cache, where the last tile goes on
              if (!((ctl.bits[slot_row][x >> 5] >> (x & 31)) & 1u) || j < blk.t0 * kBN || j >= min(blk.t1 * kBN, sq.len)) continue;
              const T* v = static_cast<const T*>(p.v) + blk.b * p.v_st[0] + blk.kvh * p.v_st[1] + j * p.v_st[2] + c0;
#pragma unroll
              for (int c = 0; c < kChunk; ++c) {
                const float f = to_f32(v[c]);
                if (!(fabsf(f) < INFINITY)) o[c] += f;
              }
            }
          }
          const float by = node < sq.n ? rl : 0.0f;
#pragma unroll
          for (int v = 0; v < kVecs; ++v) {
            float4 x = make_float4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
            if (blk.whole)  // a node behind the tree: zeros, whatever its row holds
              x = by == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : make_float4(x.x * by, x.y * by, x.z * by, x.w * by);
            room[lane * kVecs + (v ^ (lane & kSwap))] = x;
          }
          __syncwarp();
          for (int x = lane; x < 32 * kVecs; x += 32) {
            const int r = x / kVecs, v = x % kVecs, rb = first_row + r, g = r0 + rb;
            if (g >= rows) continue;
            const float4 y = room[r * kVecs + (v ^ (r & kSwap))];
            const int col = c0 + v * 4;
            if (blk.whole) {
              T* out = static_cast<T*>(p.o) + blk.b * p.o_st[0] + (blk.kvh * p.group + g / p.nodes) * p.o_st[1] +
                       g % p.nodes * p.o_st[2] + col;
              *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(y.x, y.y), pack2<T>(y.z, y.w));
            } else {
              *reinterpret_cast<float4*>(p.part_o + part_row(p, cta, blk.slot, rb) * D + col) = y;
            }
          }
        }
        if (!blk.whole && real && (by_rows || t == 0)) p.part_ml[part_row(p, cta, blk.slot, slot_row)] = make_float2(top, sum);
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
