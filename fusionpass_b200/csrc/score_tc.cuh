// Score attention on the 5th-generation tensor cores (f16 and bf16): softmax attention
// with grouped heads whose scores may be capped by a tanh, get a bias that falls with the
// distance, and are masked (score_common.cuh says which key a query sees).
//
//   x = scale q.k;  x = cap tanh(x / cap);  x -= slope_h |p - j|;  O = softmax(x) V
//
// A CTA takes tiles of 128 query rows that read the same keys (D = 128: two, neighbouring tiles of
// one head, or one tile of each of two heads of a group when the queries fit in one tile; D <= 64:
// one), walks the 128-key tiles that its rows see and keeps the running maximum and sum of the
// softmax; scores never leave the SM.  Roles, for two tiles (for one the last four follow warp 3):
//   warps 0-3, 4-7  softmax of tile 0, 1 (one thread a query row)
//   warp  8         TMA producer          warp 9  UMMA issuer, TMEM owner
//   warps 10-11     keep the V tiles that some row sees in part finite (below)
//
// TMEM, D <= 64: S at columns 0, O at 128, P at 192, so Q K^T of the next tile is issued once the
// scores are in registers and runs under the softmax.  D = 128: S_t at 128 t, O_t at 256 + 128 t
// and P_t over the first half of S_t, so Q K^T of the next tile follows P V.  P_t is handed over
// in two halves of the keys.  With a cap the two softmax warpgroups take turns at the
// exponentials, so that one's cap and maximum run beside the other's exponentials.  Without a cap
// the distance's bias is part of Q K^T where it can be (side_of).
//
// Masks are decided a tile at a time: a key tile that every row of a query tile sees runs
// the unmasked loop; any other gets 128 bits of visibility a row, made from the row's
// intervals (and by a ballot for each document id among the warp's rows).  A row that has
// seen no key yet keeps the maximum -inf and exponents taken against 0, so that it ends
// with l = 0 and the result 0.
//
// A masked key has p = 0, but 0 * inf and 0 * NaN are NaN inside the tensor core: what
// lies behind a cache's length or in another document must not reach a row that does not
// see it.  So for each partly seen tile the two spare warps look through V, replace what is
// not finite by zeros and note the keys; a row that does see such a key adds its values in
// the epilogue.
//
// Few CTAs and many keys: the key tiles of a CTA are split over several, which write
// unnormalised rows (f32) with their maximum and sum; score_combine_kernel joins them.
#pragma once

#include <cuda.h>

#include <atomic>
#include <cmath>
#include <cstring>

#include "internal.h"
#include "score_common.cuh"
#include "umma.cuh"
#include "vec_types.cuh"

namespace fpk {
namespace score {

using namespace umma;

constexpr int kBM = 128;
constexpr int kBN = kKeyTile;
constexpr int kTiles = 2;
constexpr int kStages = 2;  // of K, and of V
constexpr int kTileWarps = 4;
constexpr int kTurnAt = 88;         // score column after which the turn at the exponentials passes
constexpr int kHalfSignalAt = 78;   // score column at which the first half of P_t is signalled
constexpr float kRescaleLog2 = 8.0f;
constexpr float kMaxSlope = 1e28f;    // times a distance it is finite: the row's and the key's part may be apart
constexpr int kMaxBad = 32;           // partly seen tiles with values that are not finite, noted by key (a lane each)

// D = 128: two query tiles a CTA, one CTA an SM, which owns all of TMEM.  D <= 64: one tile a CTA
// and two CTAs an SM with half of TMEM each, which run apart, so that one's start, end and partly
// seen tiles lie under the other's work.  (us with two tiles / one: D 64, 2 x 16 heads, 4096
// keys: 228 / 209, 32 x 100 keys 26.1 / 13.9, documents 114 / 113; D 128, where one tile leaves
// room for single K and V stages: 8192 keys causal 472 / 500, with bias 583 / 818, 2048 91 / 82.)
template <int D>
struct Cfg {
  static constexpr int TILES = D == 128 ? 2 : 1;
  static constexpr int kBoxCols = D >= 64 ? 64 : D;
  static constexpr int kRowBytes = kBoxCols * 2;
  static constexpr int kBoxes = D / kBoxCols;
  static constexpr int kBoxBytes = 128 * kRowBytes;
  static constexpr int kTileBytes = kBoxes * kBoxBytes;
  static constexpr uint32_t kLayout = D >= 64 ? 2u : (D == 32 ? 4u : 6u);
  static constexpr uint32_t kSwzMask = D >= 64 ? 7u : (D == 32 ? 3u : 1u);
  static constexpr int kKStepsPerBox = kRowBytes / 32;
  static constexpr int kSlopeBytes = 128 * 32;  // 128 rows of 16 bf16
  static constexpr int kSmemBytes = (TILES + 2 * kStages) * kTileBytes + (TILES + 2) * kSlopeBytes + 1024;
  static constexpr int kMinSmem = (TILES == 2 ? 116 : 77) * 1024;  // no more CTAs an SM than TMEM holds
  static constexpr int kLaunchSmem = kSmemBytes > kMinSmem ? kSmemBytes : kMinSmem;
  // TMEM columns
  static constexpr uint32_t kTmemCols = 256 * TILES;
  static constexpr bool kAlias = D == 128;  // P_t over S_t
  static constexpr uint32_t kOCol = 128 * TILES, kOStride = kAlias ? 128 : 64;
  static constexpr uint32_t kPCol = kAlias ? 0 : 192 * TILES, kPStride = kAlias ? 128 : 64;
  // warps
  static constexpr int kTmaWarp = TILES * kTileWarps, kMmaWarp = kTmaWarp + 1, kCleanWarp = kTmaWarp + 2;
  static constexpr int kThreads = 32 * (kTmaWarp + 4);
  // setmaxnreg split of what the CTA is launched with: 384 x 168 (256 x 216 for the softmax, 128 x
  // 72 for the control warpgroup) or 256 x 128 (128 x 192, 128 x 64)
  static constexpr int kRegs = TILES == 2 ? 168 : 128, kRegsSoftmax = TILES == 2 ? 216 : 192,
                       kRegsCtl = TILES == 2 ? 72 : 64;
  static_assert(TILES * 128 * kRegsSoftmax + 128 * kRegsCtl <= kThreads * kRegs, "setmaxnreg split exceeds the launch");
};

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
// nonzero where a 16-bit half of u has an all-ones exponent (infinity or NaN)
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t u) {
  return ((u & Elem<T>::kExpMask) + Elem<T>::kExpLsb) & 0x80008000u;
}

// Keys of a partly seen tile with values that are not finite.  The entry is there once its tile is
// written, after the keys: a query tile may look while the spare warps note a step that only the
// other one takes.  The entries of its own steps are complete (v_ok, then o_done, follow them).
struct Bad {
  int j;  // key tile; -1: not there (yet)
  uint32_t keys[4];
};

struct Ctl {
  uint64_t q_full;
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], v_ok[kStages];
  uint64_t s_full[kTiles], s_free[kTiles], p_half[kTiles], p_full[kTiles], o_done[kTiles], turn[kTiles], epi[kTiles];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  int from[kTiles], to[kTiles];  // the part of the tile list with each query tile's ids
  int qlo[kTiles], qhi[kTiles];  // document ids of each query tile
  int n_bad;
  Bad bad[kMaxBad];
};

struct Where {
  int b, ntiles, kvh, sp;
  int h0, h1;        // head of tile 0, 1
  int row0, row1;    // first query of tile 0, 1
  __device__ __forceinline__ int h(int t) const { return t ? h1 : h0; }
  __device__ __forceinline__ int row(int t) const { return t ? row1 : row0; }
};
template <int TILES>
__device__ __forceinline__ Where where_of(const Params& p) {
  Where w;
  int item = static_cast<int>(blockIdx.x);
  w.sp = item % p.splits;
  item /= p.splits;
  // the last query blocks first: under a causal mask they have the most keys
  const int mb = p.mblocks - 1 - item / (p.items / p.mblocks);
  const int bh = item % (p.items / p.mblocks);
  if (TILES == 2 && p.pair_heads) {
    const int pairs = p.heads / 2;
    w.b = bh / pairs;
    w.h0 = (bh % pairs) * 2;
    w.h1 = w.h0 + 1;
    w.row0 = w.row1 = 0;
    w.ntiles = 2;
  } else {
    w.b = bh / p.heads;
    w.h0 = w.h1 = bh % p.heads;
    w.row0 = mb * TILES * kBM;
    w.row1 = w.row0 + kBM;
    w.ntiles = TILES == 2 && w.row1 < p.q_len ? 2 : 1;
  }
  w.kvh = w.h0 / p.group;
  return w;
}

// every row of query tile t sees every key of tile j
struct TileSight {
  int lo, hi, pre;  // lo of the last row, hi of the first
  int id;           // the rows' one document id; -2: no ids, -1: none for all
  const IdRange* ranges;
};
__device__ __forceinline__ TileSight sight_of(const Params& p, const Seq& s, const Where& w, int t, const Ctl& c) {
  TileSight r;
  const int first = s.base + w.row(t), last = s.base + min(w.row(t) + kBM, p.q_len) - 1;
  r.lo = span_of(p, s, last).lo;
  r.hi = span_of(p, s, first).hi;
  r.pre = s.pre;
  r.id = -2;
  r.ranges = nullptr;
  if (p.ids) {
    r.id = c.qlo[t] == c.qhi[t] && c.qlo[t] >= 0 ? c.qlo[t] : -1;
    r.ranges = p.ranges + static_cast<int64_t>(w.b) * p.k_tiles;
  }
  return r;
}
__device__ __forceinline__ bool sees_all(const TileSight& r, int j) {
  const int j0 = j * kBN;
  bool all = j0 + kBN <= r.pre || (j0 >= r.lo && j0 + kBN <= r.hi);
  if (r.id != -2 && all) {
    const IdRange k = r.ranges[j];
    all = r.id >= 0 && k.same && k.lo == r.id;
  }
  return all;
}

// mbar_wait by every lane, with one answer for the warp
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, volatile int* abort, int* status) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status, kWaitLimitNs));
}

// max of three that keeps a NaN
__device__ __forceinline__ float max3n(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

template <typename T, int M, int N, bool BMN>
__host__ __device__ constexpr uint32_t idesc16() {
  return idesc_f16(M, N, BMN) | (Elem<T>::kFormat << 7) | (Elem<T>::kFormat << 10);
}

__device__ __forceinline__ void mul2(float& d0, float& d1, float a0, float a1, float b) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\t"
      "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b));
}

__device__ __forceinline__ void mul2v(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

// d = a * s + c per lane, s broadcast
__device__ __forceinline__ void fma2s(float& d0, float& d1, float a0, float a1, float s, float c0, float c1) {
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%5, %6};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(s), "f"(c0), "f"(c1));
}
// min that keeps a NaN
__device__ __forceinline__ float min_nan(float x, float c) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(c));
  return y;
}

// The cap, of 8 scores: s -> 1 / (1 + 2^(in s)) with in = -2 log2(e) scale / cap, so that
//   cap tanh(scale q.k / cap) = 2 cap / (1 + e^(-2 scale q.k / cap)) - cap
// is a product and a shift that the softmax takes anyway.  It is off by 1.1e-6 cap at most, in
// steps of 2^-24 cap: 14 by seven roundings of a value up to 1, twice (1 + e, two products, the
// reciprocal within an ulp, two products; the factors' own errors cancel), 2 by the ex2 (2^-22, at
// most a quarter of it, twice) and 1.8 by its argument (four roundings, x / cosh^2 x <= 0.448); 5.1e-7
// is the worst of 240 million with exact functions.  Four scores take four ex2 and one shared
// reciprocal, 1 / (a b c d), on the MUFU (a pair a reciprocal: 870 us, four 838; f16
// [1, 32, 8192, 128], 8 key/value heads, causal).  A rational function of degree 7 / 8 on the FMA
// pipe, alone or for half of the pairs, was slower (1093 and 965 us against 945 of a pair a
// reciprocal at that time): it has more to issue.  A NaN in one of the four makes all NaN.
__device__ __forceinline__ void cap4(uint32_t* s, float in) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) mul2(x[i], x[i + 1], __uint_as_float(s[i]), __uint_as_float(s[i + 1]), in);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = ex2(min_nan(x[i], 24.0f));  // four times 24 bits are in range; 2^-24 is 0 to the cap
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    add2(x[i], x[i + 1], 1.0f, 1.0f);
    add2(x[i + 2], x[i + 3], 1.0f, 1.0f);
    float a, b, y[4];
    mul2v(a, b, x[i], x[i + 1], x[i + 2], x[i + 3]);
    const float r = rcp_approx(a * b), ra = r * b, rb = r * a;
    mul2v(y[0], y[1], x[i + 2], x[i + 3], ra, rb);
    mul2v(y[2], y[3], x[i], x[i + 1], ra, rb);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i + e] = __float_as_uint(y[e]);
  }
}

// The part of the tile list that query tile t needs, by its rows' intervals.
__device__ __forceinline__ void part_of(const Params& p, const Seq& s, const Where& w, const Tiles& tl, int t, int* a,
                                        int* b) {
  const int lo = span_of(p, s, s.base + w.row(t)).lo;
  const int hi = span_of(p, s, s.base + min(w.row(t) + kBM, p.q_len) - 1).hi;
  *a = tl.pre > 0 ? 0 : min(max(lo / kBN - tl.from, 0), tl.n);
  *b = hi > lo ? min(max(tl.pre + (hi + kBN - 1) / kBN - tl.from, tl.pre), tl.n) : tl.pre;
}

// The bias on the tensor core.  For a key tile that lies before, or behind, all rows of a query
// tile the bias is +-slope (j - p), a term of the row and slope times a whole number of the key:
//   before: slope (j0 + 127 - p) + slope (c - 127)      behind: slope (p - j0) - slope c
// The row's term goes with the maximum; the key's is one more product of K = 16, in bf16 whatever
// the type: slope / scale as a sum of three bf16 (24 bits) in the rows' operand, c - 127 or -c
// (exact, and 0 at the key that is nearest) in the keys'.  (us with the bias in the softmax loop / here, causal, 8192: D 128 577 / 535, D 64 275 / 243;
// documents 113 / 101.)  With a cap, which comes before the bias, it stays in the loop.
__device__ __forceinline__ int side_of(int j0, int first, int last) {
  return j0 + kBN - 1 <= first ? -1 : (j0 >= last ? 1 : 0);
}
// one row of 16 bf16 (a, b, c, 0, ...) in the 32-byte swizzle
__device__ __forceinline__ void put_row(uint8_t* tile, int row, uint32_t ab, uint32_t c) {
  const uint32_t off = static_cast<uint32_t>(row * 32), flip = ((off >> 7) & 1u) << 4;
  *reinterpret_cast<uint4*>(tile + (off ^ flip)) = make_uint4(ab, c, 0u, 0u);
  *reinterpret_cast<uint4*>(tile + ((off + 16u) ^ flip)) = make_uint4(0u, 0u, 0u, 0u);
}

// CAP: scores are capped.  BIAS: they get the distance's bias, or the scale is not positive, so
// that the largest product is not the largest score.  Where the bias is not in the product the
// scores are turned into exponents before the maximum; otherwise the maximum is taken of the
// values and the factor folds into the exponent's FFMA.
template <typename T, int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__(Cfg<D>::kThreads, Cfg<D>::TILES == 2 ? 1 : 2)
    score_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                    const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap to,
                    const __grid_constant__ Params p) {
  using C = Cfg<D>;
  constexpr int TILES = C::TILES;
  constexpr int NS = kStages;
  // turns at the exponentials, us with / without (f16, causal, 8192): plain 485 / 467, biased 604 /
  // 578, capped 868 / 894, both 949 / 1047; the turn passes after column 72, 88, 104, 120: capped 865, 832,
  // 836, 870, both 920, 909, 915, 900
  constexpr bool kTurns = TILES == 2 && CAP;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Ctl ctl;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + TILES * C::kTileBytes;
  uint8_t* sV = sK + NS * C::kTileBytes;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const Where w = where_of<TILES>(p);
  volatile int* abort = &ctl.abort;
  if (threadIdx.x == 0) {
    mbar_init(&ctl.q_full, 1);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&ctl.k_full[s], 1);
      mbar_init(&ctl.k_empty[s], 1);
      mbar_init(&ctl.v_full[s], 1);
      mbar_init(&ctl.v_empty[s], 1);
      mbar_init(&ctl.v_ok[s], 2);
    }
    for (int t = 0; t < kTiles; ++t) {
      mbar_init(&ctl.s_full[t], 1);
      mbar_init(&ctl.s_free[t], kTileWarps);
      mbar_init(&ctl.p_half[t], kTileWarps);
      mbar_init(&ctl.p_full[t], kTileWarps);
      mbar_init(&ctl.turn[t], kTileWarps);
      mbar_init(&ctl.o_done[t], 1);
      mbar_init(&ctl.epi[t], kTileWarps);
    }
    mbar_init(&ctl.drain, 1);
    ctl.abort = 0;
    ctl.n_bad = 0;
    for (int t = 0; t < kTiles; ++t) {
      ctl.qlo[t] = 0x7fffffff;
      ctl.qhi[t] = -0x7fffffff;
    }
    fence_mbar_init();
  }
  if (warp == 1) ctl.bad[lane].j = -1;
  if (warp == C::kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&ctl.tmem_base)),
                 "r"(C::kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = ctl.tmem_base;
  grid_wait();
  uint8_t* sSlope = sV + NS * C::kTileBytes;  // the rows' operand of each query tile, then the keys' two
  bool fold = false;                          // the same for the whole CTA
  if constexpr (BIAS && !CAP) {
    if (p.slopes && p.scale_log2 >= 1.17549435e-38f) {
      const float b0 = __ldg(p.slopes + w.h0), b1 = __ldg(p.slopes + w.h1);
      const float v0 = __fdiv_rn(b0, p.scale), v1 = __fdiv_rn(b1, p.scale);
      fold = fabsf(v0) < 1e30f && fabsf(v1) < 1e30f && fabsf(b0) < kMaxSlope && fabsf(b1) < kMaxSlope;
      if (fold && warp < TILES * kTileWarps) {
        const int t = warp / kTileWarps, r = static_cast<int>(threadIdx.x & (kBM - 1));
        const float v = t ? v1 : v0;
        const __nv_bfloat16 hi = __float2bfloat16_rn(v);
        const float rest = v - __bfloat162float(hi);
        const __nv_bfloat16 mid = __float2bfloat16_rn(rest), lo = __float2bfloat16_rn(rest - __bfloat162float(mid));
        put_row(sSlope + t * C::kSlopeBytes, r,
                __bfloat16_as_ushort(hi) | static_cast<uint32_t>(__bfloat16_as_ushort(mid)) << 16, __bfloat16_as_ushort(lo));
        if (t == 0)
          for (int side = 0; side < 2; ++side) {
            const uint32_t c = __bfloat16_as_ushort(__int2bfloat16_rn(side ? -r : r - (kBN - 1)));
            put_row(sSlope + (TILES + side) * C::kSlopeBytes, r, c | c << 16, c);
          }
        fence_proxy_async_smem();
      }
      __syncthreads();
    }
  }
  const Seq sq = seq_of(p, w.b);
  const Tiles tl = tiles_of(p, sq, sq.base + w.row0, sq.base + min(w.row(w.ntiles - 1) + kBM, p.q_len) - 1);
  // each query tile's own part [ta, tb) of the list: the other tile's keys beyond it (the end of
  // a causal block, a neighbouring document) are not its work
  int ta0, tb0, ta1, tb1;
  part_of(p, sq, w, tl, 0, &ta0, &tb0);
  part_of(p, sq, w, tl, w.ntiles - 1, &ta1, &tb1);
  int my_id = -1;
  if (p.ids) {
    // the query tiles' ids, then the ends of the parts that share none of them
    const int t = warp / kTileWarps;
    const int row = w.row(t & 1) + static_cast<int>(threadIdx.x & (kBM - 1));
    if (t < w.ntiles && row < p.q_len) {
      my_id = id_at(p, w.b, sq.base + row, sq.len);
      atomicMin(&ctl.qlo[t], my_id);
      atomicMax(&ctl.qhi[t], my_id);
    }
    __syncthreads();
    if (warp >= C::kCleanWarp && warp < C::kCleanWarp + w.ntiles) {
      const int u = warp - C::kCleanWarp;
      const int lo = max(ctl.qlo[u], 0), hi = ctl.qhi[u];
      const IdRange* rg = p.ranges + static_cast<int64_t>(w.b) * p.k_tiles;
      int a = u ? tb1 : tb0, b = 0;
      for (int i = (u ? ta1 : ta0) + lane; i < (u ? tb1 : tb0); i += 32) {
        const IdRange r = rg[tl.at(i)];
        if (r.hi >= lo && r.lo <= hi) {
          a = min(a, i);
          b = max(b, i + 1);
        }
      }
      a = __reduce_min_sync(0xffffffffu, a);
      b = __reduce_max_sync(0xffffffffu, b);
      if (lane == 0) {
        ctl.from[u] = a;
        ctl.to[u] = b;
      }
    }
    __syncthreads();
    ta0 = ctl.from[0];
    tb0 = ctl.to[0];
    ta1 = ctl.from[w.ntiles - 1];
    tb1 = ctl.to[w.ntiles - 1];
  }
  // the CTA walks [i0, i1): both parts, or its share of them
  int i0 = tb0 > ta0 ? (tb1 > ta1 ? min(ta0, ta1) : ta0) : ta1;
  int i1 = max(i0, tb0 > ta0 ? (tb1 > ta1 ? max(tb0, tb1) : tb0) : tb1);
  if (p.splits > 1) {
    const int n = i1 - i0;
    const int from = i0;
    i0 = from + static_cast<int>(static_cast<int64_t>(n) * w.sp / p.splits);
    i1 = from + static_cast<int>(static_cast<int64_t>(n) * (w.sp + 1) / p.splits);
  }
  const int nkv = i1 - i0;
  // from here on relative to i0
  ta0 = min(max(ta0 - i0, 0), nkv);
  tb0 = max(min(tb0 - i0, nkv), ta0);
  ta1 = min(max(ta1 - i0, 0), nkv);
  tb1 = max(min(tb1 - i0, nkv), ta1);
  // with a bias under a causal mask the nearest tiles first: the maximum then stays and O is not
  // scaled again at each step (8192 keys, D 128 536 -> 470 us, with the cap 955 -> 903; plain 464 -> 466,
  // capped 869 -> 898, so not there)
  const bool back = BIAS && p.causal;
  if (back) {
    const int a0 = nkv - tb0, a1 = nkv - tb1;
    tb0 = nkv - ta0;
    tb1 = nkv - ta1;
    ta0 = a0;
    ta1 = a1;
  }
  const auto tile_at = [&](int i) { return tl.at(back ? i1 - 1 - i : i0 + i); };

  if (warp >= TILES * kTileWarps) {
    setmaxnreg_dec<C::kRegsCtl>();
    if (warp == C::kTmaWarp) {
      // --------------------------------------------------------- TMA producer
      if (lane == 0 && nkv > 0) {
        int last_k[NS], last_v[NS];
        for (int s = 0; s < NS; ++s) last_k[s] = last_v[s] = -1;
        // no load where a tile has no step: its zeros are staged there, and nothing waits for the load
        // (waiting for it there cost 1 % with a cap at D 128, 843 us against 836)
        const bool some0 = tb0 > ta0, some1 = w.ntiles == 2 && tb1 > ta1;
        mbar_arrive_expect_tx(&ctl.q_full, static_cast<uint32_t>((some0 + some1) * C::kTileBytes));
        for (int t = 0; t < w.ntiles; ++t) {
          if (!(t ? some1 : some0)) continue;
          for (int bx = 0; bx < C::kBoxes; ++bx)
            tma_load_4d(sQ + t * C::kTileBytes + bx * C::kBoxBytes, &tq, bx * C::kBoxCols, w.row(t), w.h(t), w.b,
                        &ctl.q_full);
        }
        for (int i = 0; i < nkv; ++i) {
          const int s = i % NS;
          const uint32_t r = static_cast<uint32_t>(i / NS);
          const int j0 = tile_at(i) * kBN;
          if (!mbar_wait(&ctl.k_empty[s], (r & 1u) ^ 1u, abort, p.status, kWaitLimitNs)) break;
          mbar_arrive_expect_tx(&ctl.k_full[s], C::kTileBytes);
          for (int bx = 0; bx < C::kBoxes; ++bx)
            tma_load_4d(sK + s * C::kTileBytes + bx * C::kBoxBytes, &tk, bx * C::kBoxCols, j0, w.kvh, w.b,
                        &ctl.k_full[s]);
          last_k[s] = i;
          if (!mbar_wait(&ctl.v_empty[s], (r & 1u) ^ 1u, abort, p.status, kWaitLimitNs)) break;
          mbar_arrive_expect_tx(&ctl.v_full[s], C::kTileBytes);
          for (int bx = 0; bx < C::kBoxes; ++bx)
            tma_load_4d(sV + s * C::kTileBytes + bx * C::kBoxBytes, &tv, bx * C::kBoxCols, j0, w.kvh, w.b,
                        &ctl.v_full[s]);
          last_v[s] = i;
        }
        // no TMA write may land after the CTA has gone
        drain_wait(&ctl.q_full, 0, p.status);
        for (int s = 0; s < NS; ++s) {
          if (last_k[s] >= 0) drain_wait(&ctl.k_full[s], static_cast<uint32_t>(last_k[s] / NS) & 1u, p.status);
          if (last_v[s] >= 0) drain_wait(&ctl.v_full[s], static_cast<uint32_t>(last_v[s] / NS) & 1u, p.status);
        }
      }
    } else if (warp == C::kMmaWarp) {
      // ------------------------------------------------ UMMA issuer (whole warp)
      constexpr uint32_t idesc_qk = idesc16<T, kBM, kBN, false>();
      constexpr uint32_t idesc_pv = idesc16<T, kBM, D, true>();
      constexpr uint64_t kTileStep = static_cast<uint64_t>(C::kTileBytes >> 4);
      const uint32_t leader = elect_one();
      const uint64_t q_desc = sdesc(smem_u32(sQ), 16, 8 * C::kRowBytes, C::kLayout);
      const uint64_t k_desc = sdesc(smem_u32(sK), 16, 8 * C::kRowBytes, C::kLayout);
      const uint64_t v_desc = sdesc(smem_u32(sV), C::kBoxBytes, 8 * C::kRowBytes, C::kLayout);
      constexpr uint32_t idesc_slope = idesc16<__nv_bfloat16, kBM, kBN, false>();
      const uint64_t slope_desc = sdesc(smem_u32(sSlope), 16, 8 * 32, 6u);
      // i: the step whose tile is in stage s
      auto issue_qk = [&](int t, int s, int i) {
        const uint32_t d_tmem = tbase + static_cast<uint32_t>(t * 128);
        const uint64_t a0 = q_desc + static_cast<uint64_t>(t) * kTileStep;
        const uint64_t b0 = k_desc + static_cast<uint64_t>(s) * kTileStep;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          constexpr int kSteps = C::kKStepsPerBox;
          const uint64_t off = static_cast<uint64_t>((kk / kSteps) * (C::kBoxBytes >> 4) + (kk % kSteps) * 2);
          mma_ss_l(leader, d_tmem, a0 + off, b0 + off, idesc_qk, kk > 0 ? 1u : 0u);
        }
        if constexpr (BIAS && !CAP) {
          const int first = sq.base + w.row(t);
          const int side = fold ? side_of(tile_at(i) * kBN, first, sq.base + min(w.row(t) + kBM, p.q_len) - 1) : 0;
          if (side != 0)
            mma_ss_l(leader, d_tmem, slope_desc + static_cast<uint64_t>(t * (C::kSlopeBytes >> 4)),
                     slope_desc + static_cast<uint64_t>((TILES + (side > 0)) * (C::kSlopeBytes >> 4)), idesc_slope, 1u);
        }
      };
      auto issue_pv = [&](int t, int s, bool accumulate, int half) {
        const uint32_t d_tmem = tbase + C::kOCol + static_cast<uint32_t>(t) * C::kOStride;
        const uint32_t a_tmem = tbase + C::kPCol + static_cast<uint32_t>(t) * C::kPStride;
        const uint64_t b0 = v_desc + static_cast<uint64_t>(s) * kTileStep;
#pragma unroll
        for (int k2 = 0; k2 < kBN / 32; ++k2) {
          const int kk = half * (kBN / 32) + k2;
          mma_ts_l(leader, d_tmem, a_tmem + static_cast<uint32_t>(kk * 8),
                   b0 + static_cast<uint64_t>(kk * C::kRowBytes), idesc_pv, (accumulate || kk > 0) ? 1u : 0u);
        }
      };
      const auto in_part = [&](int t, int i) { return t ? i >= ta1 && i < tb1 : i >= ta0 && i < tb0; };
      bool ok = nkv > 0 && mbar_wait_w(&ctl.q_full, 0, abort, p.status, kWaitLimitNs) &&
                mbar_wait_w(&ctl.k_full[0], 0, abort, p.status, kWaitLimitNs);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < w.ntiles; ++t) {
          if (!in_part(t, 0)) continue;
          issue_qk(t, 0, 0);
          mma_commit_l(leader, &ctl.s_full[t]);
        }
        mma_commit_l(leader, &ctl.k_empty[0]);
      }
      int s = 0, s1 = 1;
      uint32_t r = 0u, r1 = 0u;
      for (int i = 0; ok && i < nkv; ++i) {
        const bool more = i + 1 < nkv;
        if (!C::kAlias && more) {
          // the next scores, as soon as these are in registers
          if (!mbar_wait_w(&ctl.k_full[s1], r1, abort, p.status, kWaitLimitNs)) break;
          for (int t = 0; ok && t < w.ntiles; ++t) {
            if (!in_part(t, i + 1)) continue;
            if (in_part(t, i))
              ok = mbar_wait_w(&ctl.s_free[t], static_cast<uint32_t>(i - (t ? ta1 : ta0)) & 1u, abort, p.status,
                               kWaitLimitNs);
            if (!ok) break;
            tc_fence_after();
            issue_qk(t, s1, i + 1);
            mma_commit_l(leader, &ctl.s_full[t]);
          }
          if (!ok) break;
          mma_commit_l(leader, &ctl.k_empty[s1]);
        }
        if (!mbar_wait_w(&ctl.v_ok[s], r, abort, p.status, kWaitLimitNs)) break;
        bool k_ready = false;
        for (int t = 0; ok && t < w.ntiles; ++t) {
          if (in_part(t, i)) {
            const int n = i - (t ? ta1 : ta0);  // this tile's step
            const uint32_t par = static_cast<uint32_t>(n) & 1u;
            ok = mbar_wait_w(&ctl.p_half[t], par, abort, p.status, kWaitLimitNs);
            if (!ok) break;
            tc_fence_after();
            issue_pv(t, s, n > 0, 0);
            ok = mbar_wait_w(&ctl.p_full[t], par, abort, p.status, kWaitLimitNs);
            if (!ok) break;
            tc_fence_after();
            issue_pv(t, s, n > 0, 1);
            mma_commit_l(leader, &ctl.o_done[t]);
          }
          if (C::kAlias && more && in_part(t, i + 1)) {
            ok = k_ready || mbar_wait_w(&ctl.k_full[s1], r1, abort, p.status, kWaitLimitNs);
            if (!ok) break;
            k_ready = true;
            tc_fence_after();
            issue_qk(t, s1, i + 1);
            mma_commit_l(leader, &ctl.s_full[t]);
          }
        }
        if (!ok) break;
        mma_commit_l(leader, &ctl.v_empty[s]);
        if (C::kAlias && more) {
          if (!k_ready && !mbar_wait_w(&ctl.k_full[s1], r1, abort, p.status, kWaitLimitNs)) break;
          mma_commit_l(leader, &ctl.k_empty[s1]);
        }
        s = s1;
        r = r1;
        if (++s1 == NS) {
          s1 = 0;
          r1 ^= 1u;
        }
      }
      // every UMMA issued so far must finish before TMEM is freed
      mma_commit_l(leader, &ctl.drain);
      drain_wait_w(&ctl.drain, 0, p.status);
    } else {
      // -------------------- V of partly seen tiles: what is not finite becomes zero
      const TileSight s0 = sight_of(p, sq, w, 0, ctl), s1 = sight_of(p, sq, w, w.ntiles - 1, ctl);
      const int tid = static_cast<int>(threadIdx.x) - C::kCleanWarp * 32;  // 0..63
      for (int i = 0; i < nkv; ++i) {
        const int s = i % NS;
        if (!wait_all(&ctl.v_full[s], static_cast<uint32_t>(i / NS) & 1u, abort, p.status)) break;
        const int j = tile_at(i);
        if (!(sees_all(s0, j) && sees_all(s1, j))) {
          uint4* v = reinterpret_cast<uint4*>(sV + s * C::kTileBytes);
          constexpr int kVecs = C::kTileBytes / 16, kRowVecs = C::kRowBytes / 16;
          bool any = false;
#pragma unroll 4
          for (int x = tid; x < kVecs; x += 64) {
            uint4 u = v[x];
            const uint32_t bits = not_finite<T>(u.x) | not_finite<T>(u.y) | not_finite<T>(u.z) | not_finite<T>(u.w);
            any |= bits != 0u;
          }
          if (__any_sync(0xffffffffu, any)) {
            // note the tile's keys (the swizzle moves vectors within a row only)
            uint32_t keys[4] = {0u, 0u, 0u, 0u};
            for (int x = tid; x < kVecs; x += 64) {
              uint4 u = v[x];
              uint32_t* e = reinterpret_cast<uint32_t*>(&u);
              bool hit = false;
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const uint32_t nf = not_finite<T>(e[q]);
                if (nf & 0x8000u) e[q] &= 0xffff0000u;
                if (nf & 0x80000000u) e[q] &= 0x0000ffffu;
                hit |= nf != 0u;
              }
              if (hit) {
                v[x] = u;
                const int key = (x / kRowVecs) & 127;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  if (q == key >> 5) keys[q] |= 1u << (key & 31);
              }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) keys[q] = __reduce_or_sync(0xffffffffu, keys[q]);
            if (lane == 0) {
              const int at = atomicAdd(&ctl.n_bad, 1);
              if (at < kMaxBad) {
                for (int q = 0; q < 4; ++q) ctl.bad[at].keys[q] = keys[q];
                __threadfence_block();
                *const_cast<volatile int*>(&ctl.bad[at].j) = j;
              }
            }
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.v_ok[s]);
      }
    }
  } else {
    // ------------------------------------------------------ softmax + epilogue
    setmaxnreg_inc<C::kRegsSoftmax>();
    const int t = warp / kTileWarps;
    const int row = threadIdx.x & (kBM - 1);
    if (t < w.ntiles) {
      const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t tS = tbase + lane_off + static_cast<uint32_t>(t * 128);
      const uint32_t tO = tbase + lane_off + C::kOCol + static_cast<uint32_t>(t) * C::kOStride;
      const uint32_t tP = tbase + lane_off + C::kPCol + static_cast<uint32_t>(t) * C::kPStride;
      const TileSight sight = sight_of(p, sq, w, t, ctl);
      const int in_seq = min(w.row(t) + row, p.q_len - 1);
      const int pos = sq.base + in_seq;
      const Span span = span_of(p, sq, pos);
      // a score's exponent of base 2 is value * factor + offset (+ the bias): the value is the
      // product q.k, or what cap4 makes of it
      const float factor = CAP ? 2.0f * 1.4426950408889634f * p.cap : p.scale_log2;
      const float offset = CAP ? -1.4426950408889634f * p.cap : 0.0f;
      const float cap_in = CAP ? -2.0f * 1.4426950408889634f * p.scale / p.cap : 0.0f;
      const bool biased = BIAS && p.slopes != nullptr;
      const float slope2 = biased ? __ldg(p.slopes + w.h(t)) * 1.4426950408889634f : 0.0f;
      const bool apart = CAP && biased && fabsf(slope2) < kMaxSlope;
      float m_run = -INFINITY;
      float l = 0.0f;
      bool ok = true;
      const int first = t ? ta1 : ta0;
      const int steps = (t ? tb1 : tb0) - first;
      // the steps that both tiles take, in which their warpgroups take turns
      const int both0 = max(ta0, ta1) - first, both1 = min(tb0, tb1) - first;
      for (int i = 0; i < steps; ++i) {
        const int j = tile_at(first + i);
        const int j0 = j * kBN;
        // what does not need the scores, ahead of the wait for them: its loads are on the way meanwhile
        const bool all = sees_all(sight, j);
        float shift = offset;  // what every score of the row is still to get
        float sl = -slope2;    // bias a key, on one side of the row
        bool one_side = false;
        int side = 0;  // not 0: the product has the key's part of the bias
        if constexpr (BIAS && !CAP) {
          if (fold) {
            side = side_of(j0, sq.base + w.row(t), sq.base + min(w.row(t) + kBM, p.q_len) - 1);
            if (side != 0) shift += side < 0 ? slope2 * static_cast<float>(j0 + kBN - 1 - pos) : sl * static_cast<float>(j0 - pos);
          }
        }
        if (apart) {
          // -slope |p - j|: with all of the warp's rows at or after the tile, or before it, it
          // is +-slope (j0 - p), one value a row, and +-slope c
          const int w_first = sq.base + min(w.row(t) + (row & ~31), p.q_len - 1);
          const int w_last = sq.base + min(w.row(t) + (row | 31), p.q_len - 1);
          one_side = j0 + kBN - 1 <= w_first || j0 >= w_last;
          if (one_side) {
            sl = j0 >= w_last ? -slope2 : slope2;
            shift += sl * static_cast<float>(j0 - pos);
          }
        }
        uint32_t vis[4];
        if (!all) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            vis[q] = span_bits(span.lo, span.hi, j0 + 32 * q) | span_bits(0, sq.pre, j0 + 32 * q);
          if (p.ids) {
            // ids of the tile's keys, four a lane; one ballot for each id among the warp's rows
            uint32_t same[4] = {0u, 0u, 0u, 0u};
            int kid[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) kid[q] = id_at(p, w.b, j0 + 32 * q + lane, sq.len);
            uint32_t todo = __ballot_sync(0xffffffffu, my_id >= 0);
            while (todo) {
              const int id = __shfl_sync(0xffffffffu, my_id, __ffs(todo) - 1);
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const uint32_t eq = __ballot_sync(0xffffffffu, kid[q] == id);
                if (my_id == id) same[q] = eq;
              }
              todo &= ~__ballot_sync(0xffffffffu, my_id == id);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) vis[q] &= same[q];
          }
        }
        if (!wait_all(&ctl.s_full[t], static_cast<uint32_t>(i) & 1u, abort, p.status)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t sr[kBN];
        if constexpr (TILES == 2) {
          tmem_ld_x128(tS, sr);
        } else {
          tmem_ld_x64(tS, sr);
          tmem_ld_x64(tS + 64u, sr + 64);
        }
        if constexpr (!C::kAlias) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl.s_free[t]);
        }
        if (!all) {
          // with a cap a masked value is 0 until the cap is through: four share a reciprocal there
          if (CAP || !BIAS) {
            constexpr float kNone = CAP ? 0.0f : -INFINITY;
#pragma unroll
            for (int c = 0; c < kBN; ++c)
              if (!((vis[c >> 5] >> (c & 31)) & 1u)) sr[c] = __float_as_uint(kNone);
          }
        }
        if constexpr (CAP) {
#pragma unroll
          for (int c = 0; c < kBN; c += 8) cap4(sr + c, cap_in);
        }
        const float by = BIAS && side == 0 ? 1.0f : factor;  // what is left to multiply by
        if (BIAS && side == 0) {
          if (CAP && one_side) {
            // the bias of eight keys once, and of each eighth key
            float d[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) d[c] = sl * static_cast<float>(c);
#pragma unroll
            for (int c8 = 0; c8 < kBN; c8 += 8) {
              const float far = sl * static_cast<float>(c8);
#pragma unroll
              for (int c = 0; c < 8; c += 2) {
                float x0, x1;
                fma2s(x0, x1, __uint_as_float(sr[c8 + c]), __uint_as_float(sr[c8 + c + 1]), factor, d[c], d[c + 1]);
                add2(x0, x1, far, far);
                sr[c8 + c] = __float_as_uint(x0);
                sr[c8 + c + 1] = __float_as_uint(x1);
              }
            }
          } else {
            const float d0 = static_cast<float>(j0 - pos);
#pragma unroll
            for (int c = 0; c < kBN; ++c)
              sr[c] = __float_as_uint(
                  __fmaf_rn(-slope2, fabsf(d0 + static_cast<float>(c)), __uint_as_float(sr[c]) * factor));
          }
        }
        // after the cap, and where the scale is not positive (-inf times it is not -inf)
        if (!all && (CAP || BIAS)) {
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
        mx = __fmaf_rn(mx, by, shift);
        if (!(mx < INFINITY)) l = __uint_as_float(0x7fc00000u);  // a NaN or an infinite score: the row is NaN
        bool pv_done = C::kAlias || i == 0;  // the earlier P V is complete: aliased, S_t follows it
        if (i == 0) {
          m_run = mx;
        } else {
          const bool need = mx > m_run + kRescaleLog2;
          if (__any_sync(0xffffffffu, need)) {
            if (!pv_done && !wait_all(&ctl.o_done[t], static_cast<uint32_t>(i - 1) & 1u, abort, p.status)) {
              ok = false;
              break;
            }
            pv_done = true;
            tc_fence_after();
            const float alpha = need ? ex2(m_run - mx) : 1.0f;
            if (need) m_run = mx;
            l *= alpha;
            constexpr int kChunk = D < 32 ? D : 32;
#pragma unroll
            for (int c0 = 0; c0 < D; c0 += kChunk) {
              uint32_t orow[kChunk];
              tmem_ld<kChunk>(tO + static_cast<uint32_t>(c0), orow);
#pragma unroll
              for (int c = 0; c < kChunk; ++c) orow[c] = __float_as_uint(__uint_as_float(orow[c]) * alpha);
              tmem_st<kChunk>(tO + static_cast<uint32_t>(c0), orow);
            }
          }
        }
        if (!pv_done) {  // P_t has been read
          if (!wait_all(&ctl.o_done[t], static_cast<uint32_t>(i - 1) & 1u, abort, p.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
        }
        // the two warpgroups take turns at the exponentials
        const bool shared = kTurns && w.ntiles == 2 && i >= both0 && i < both1;
        if (shared && (t == 1 || i > both0)) {
          const uint32_t par = static_cast<uint32_t>(t == 1 ? i - both0 : i - both0 - 1) & 1u;
          if (!wait_all(&ctl.turn[t], par, abort, p.status)) {
            ok = false;
            break;
          }
        }
        const float neg_m = m_run == -INFINITY ? 0.0f : shift - m_run;
        float la[4] = {0.0f, 0.0f, 0.0f, 0.0f}, lb[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < kBN; c += 2) {
          float x0 = __uint_as_float(sr[c]), x1 = __uint_as_float(sr[c + 1]), p0, p1;
          fma2(x0, x1, x0, x1, by, neg_m);
          // all on the MUFU: with a quarter of the pairs on an FMA polynomial, which pays in a kernel
          // without masks and NaN rules, this loop has more to issue (f16, D 128, causal, us: plain
          // 504 -> 484, bias 690 -> 654, cap 971 -> 950; D 64 217 -> 205)
          p0 = ex2(x0);
          p1 = ex2(x1);
          add2(la[(c >> 1) & 3], lb[(c >> 1) & 3], p0, p1);
          sr[c >> 1] = pack2<T>(p0, p1);
          if (c == kBN / 2 - 2) tmem_st_x32(tP, sr);
          if (c == kHalfSignalAt) {
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl.p_half[t]);
          }
          if (c == kTurnAt && shared) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl.turn[1 - t]);
          }
        }
        l += ((la[0] + lb[0]) + (la[1] + lb[1])) + ((la[2] + lb[2]) + (la[3] + lb[3]));
        tmem_st_x32(tP + 32u, sr + 32);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.p_full[t]);
      }
      // epilogue.  The result is staged over this tile's Q: the last P V follows its load, and with
      // no step it is not loaded
      if (ok && steps > 0) ok = wait_all(&ctl.o_done[t], static_cast<uint32_t>(steps - 1) & 1u, abort, p.status);
      if (ok) {
        tc_fence_after();
        const int n_bad = steps > 0 ? *const_cast<volatile int*>(&ctl.n_bad) : 0;
        const bool whole = n_bad > kMaxBad;  // too many to note: look through every partly seen tile again
        const TileSight other = sight_of(p, sq, w, w.ntiles - 1 - t, ctl);
        const T* vb = static_cast<const T*>(p.v) + w.b * p.v_st[0] + w.kvh * p.v_st[1];
        const float rl = p.splits > 1 ? 1.0f : (l == 0.0f ? 0.0f : __frcp_rn(l));
        uint8_t* stage = sQ + t * C::kTileBytes;
        const int64_t grow = (static_cast<int64_t>(w.b) * p.heads + w.h(t)) * p.q_len + w.row(t) + row;
        const bool real = w.row(t) + row < p.q_len;
        float* po = p.splits > 1 ? p.part_o + (grow * p.splits + w.sp) * D : nullptr;
        constexpr int kChunk = D < 32 ? D : 32;
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += kChunk) {
          uint32_t orow[kChunk];
          if (steps > 0) {
            __syncwarp();
            tmem_ld<kChunk>(tO + static_cast<uint32_t>(c0), orow);
          } else {
#pragma unroll
            for (int c = 0; c < kChunk; ++c) orow[c] = 0u;
          }
          if (n_bad > 0 && real) {
            const int entries = whole ? nkv : n_bad;
            for (int e = 0; e < entries; ++e) {
              const int j = whole ? tl.at(i0 + e) : *const_cast<volatile int*>(&ctl.bad[e].j);
              if (j < 0) continue;  // being noted: not a tile of these rows
              if (whole && sees_all(sight, j) && sees_all(other, j)) continue;  // V was left as it is
              if (!whole) __threadfence_block();  // the keys after the tile
              for (int key = 0; key < kBN; ++key) {
                if (!whole && !((ctl.bad[e].keys[key >> 5] >> (key & 31)) & 1u)) continue;
                const int kp = j * kBN + key;
                if (!(kp < sq.pre || (kp >= span.lo && kp < span.hi))) continue;
                if (p.ids && (my_id < 0 || id_at(p, w.b, kp, sq.len) != my_id)) continue;
                const T* vr = vb + kp * p.v_st[2] + c0;
#pragma unroll
                for (int c = 0; c < kChunk; ++c) {
                  const float f = to_f32(vr[c]);
                  if (!(fabsf(f) < INFINITY)) orow[c] = __float_as_uint(__uint_as_float(orow[c]) + f);
                }
              }
            }
          }
          if (p.splits > 1) {
            if (real) {
#pragma unroll
              for (int c = 0; c < kChunk; c += 4)
                *reinterpret_cast<float4*>(po + c0 + c) =
                    make_float4(__uint_as_float(orow[c]), __uint_as_float(orow[c + 1]), __uint_as_float(orow[c + 2]),
                                __uint_as_float(orow[c + 3]));
            }
          } else {
            uint32_t h2[kChunk / 2];
#pragma unroll
            for (int c = 0; c < kChunk; c += 2)
              h2[c / 2] = pack2<T>(__fmul_rn(__uint_as_float(orow[c]), rl), __fmul_rn(__uint_as_float(orow[c + 1]), rl));
#pragma unroll
            for (int q = 0; q < kChunk / 8; ++q) {
              const int col = c0 + q * 8;
              const int bx = col / C::kBoxCols;
              const uint32_t off = static_cast<uint32_t>(row * C::kRowBytes + (col % C::kBoxCols) * 2);
              const uint32_t phys = off ^ (((off >> 7) & C::kSwzMask) << 4);
              *reinterpret_cast<uint4*>(stage + bx * C::kBoxBytes + phys) =
                  make_uint4(h2[q * 4], h2[q * 4 + 1], h2[q * 4 + 2], h2[q * 4 + 3]);
            }
          }
        }
        if (p.splits > 1) {
          if (real) p.part_ml[grow * p.splits + w.sp] = make_float2(m_run, l);
        } else {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl.epi[t]);
          if (wait_all(&ctl.epi[t], 0, abort, p.status) && row == 0) {
            for (int bx = 0; bx < C::kBoxes; ++bx)
              tma_store_4d(&to, stage + bx * C::kBoxBytes, bx * C::kBoxCols, w.row(t), w.h(t), w.b);
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == C::kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(C::kTmemCols));
  }
}

// ------------------------------------------------------------- host side ---
template <typename T>
static int make_map(CUtensorMap* m, const void* base, const int64_t* st, int D, int64_t rows, int64_t heads,
                    int64_t batch) {
  EncodeTiledFn enc = encoder();
  if (!enc) return FPK_ERR_CUDA;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(rows),
                              static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(batch)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(st[2] * 2), static_cast<cuuint64_t>(st[1] * 2),
                                 static_cast<cuuint64_t>(st[0] * 2)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(D >= 64 ? 64 : D), 128u, 1u, 1u};
  const cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  const CUtensorMapSwizzle swz = D >= 64 ? CU_TENSOR_MAP_SWIZZLE_128B
                                         : (D == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B);
  const CUresult r = enc(m, Elem<T>::kFormat ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                         const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swz,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FPK_OK : FPK_ERR_INVALID;
}

template <typename T, int D, bool CAP, bool BIAS>
static int launch(const CUtensorMap* maps, const Params& p, cudaStream_t s) {
  using C = Cfg<D>;
  static OptIn opted;
  if (!opted.shared(score_tc_kernel<T, D, CAP, BIAS>, C::kLaunchSmem)) return FPK_ERR_CUDA;
  const int64_t grid = static_cast<int64_t>(p.items) * p.splits;
  if (grid > 0x7fffffffLL) return FPK_ERR_UNSUPPORTED;
  return launch_dependent(score_tc_kernel<T, D, CAP, BIAS>, dim3(static_cast<unsigned>(grid)), C::kThreads,
                          C::kLaunchSmem, s, maps[0], maps[1], maps[2], maps[3], p);
}

template <typename T, int D>
static int launch_d(const CUtensorMap* maps, const Params& p, cudaStream_t s) {
  // a factor that is not a positive normal number would not keep the order of the products, nor -inf
  const bool bias = p.slopes != nullptr || (p.cap == 0.0f && !(p.scale_log2 >= 1.17549435e-38f));
  if (p.cap > 0.0f) return bias ? launch<T, D, true, true>(maps, p, s) : launch<T, D, true, false>(maps, p, s);
  return bias ? launch<T, D, false, true>(maps, p, s) : launch<T, D, false, false>(maps, p, s);
}

template <typename T>
static int launch_tc_type(const Params& p, int D, cudaStream_t s) {
  CUtensorMap maps[4];
  int rc;
  if ((rc = make_map<T>(&maps[0], p.q, p.q_st, D, p.q_len, p.heads, p.batch)) != FPK_OK) return rc;
  if ((rc = make_map<T>(&maps[1], p.k, p.k_st, D, p.k_len, p.kv_heads, p.batch)) != FPK_OK) return rc;
  if ((rc = make_map<T>(&maps[2], p.v, p.v_st, D, p.k_len, p.kv_heads, p.batch)) != FPK_OK) return rc;
  if ((rc = make_map<T>(&maps[3], p.o, p.o_st, D, p.q_len, p.heads, p.batch)) != FPK_OK) return rc;
  switch (D) {
    case 16: return launch_d<T, 16>(maps, p, s);
    case 32: return launch_d<T, 32>(maps, p, s);
    case 64: return launch_d<T, 64>(maps, p, s);
    case 128: return launch_d<T, 128>(maps, p, s);
    default: return FPK_ERR_UNSUPPORTED;
  }
}

}  // namespace score
}  // namespace fpk
