// Tree attention for few rows (f16 and bf16, caches of that type or in 8 bits), single tokens
// among them.
//
// The nodes of all heads of a group read the same keys and values, so 16 rows (row r: head
// r / nodes of the group, node r % nodes) are one m16 operand of the mma.sync matrix instruction.
// A CTA takes its part of the blocks' keys (tree_common.cuh); its 4 warps take 16 keys at a time in
// turn, each with its own ring of cp.async stages (no barrier between warps), its own running maximum
// and sum and its own 16 x D result in registers, joined through shared memory at a block's end.
// Bound by reading the cache.
//
// 8-bit caches.  A whole number of 8 bits is exact in f16 and in bf16, so the products run on the
// numbers themselves, and the scales go where they cost least: the key's with the score, the
// value's with the weight.  The numbers reach the matrix instruction's layout without a shuffle:
// * Q K^T sums over the head dim in any order.  A thread takes the bytes that lie together in a key's
//   row as its k indices, and loads Q by the same order.
// * P V needs pairs of keys.  ldmatrix.trans moves pairs of bytes, that is two neighbouring columns; of
//   the four bytes a thread gets the even ones are a pair of keys of one column, the odd ones of the
//   next: two operands, for even and odd columns of the result.
// A byte becomes f16 as 0x6400 | (byte ^ 0x80), which is 1152 + the number, less 1152; and bf16 as
// (0x4300 | low 7 bits) - (0x4300 | sign bit), 128 + low 7 bits less 128 or 256.  Both are exact.
// In f16 the power of two of a value's scale goes with the score (tree_common.cuh).
//
// Values behind a node's mask must not reach it: in the last chunks what is not finite in a 16-bit V
// is replaced by zeros before the product and added for the rows that see it.  (8-bit values are
// finite, and a scale that is not is in the score.)
#include <cuda_runtime.h>

#include <cmath>
#include <type_traits>

#include "internal.h"
#include "mma_sync.cuh"
#include "tree_common.cuh"
#include "vec_types.cuh"

namespace fpk {
namespace tree {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 16;

template <int D, bool Q8, bool FEW>
struct Cfg {
  // keys a warp takes at a time: 8-bit ones of up to 8 rows, where each step's instructions bound the kernel, two
  // operands' worth
  static constexpr int kChunk = Q8 && FEW ? 32 : 16;
  static constexpr int kRowBytes = Q8 ? D : D * 2;
  // 16-bit rows: an odd number of 16-byte units apart, no bank conflicts; 8-bit rows: swizzled
  static constexpr int kPitch = Q8 ? D : D * 2 + 16;
  static constexpr int kHalf = kChunk * kPitch;
  static constexpr int kScales = Q8 ? 2 * kChunk * 4 : 0;
  static constexpr int kStage = 2 * kHalf + kScales;  // K, V, their scales
  static constexpr int kStages = Q8 ? (D == 128 ? (FEW ? 3 : 4) : (FEW ? 4 : 6)) : (D == 128 ? 3 : 4);
  static constexpr int kWarpBytes = kStages * kStage;
  static constexpr int kJoin = kWarps * kRows * (D + 2) * 4;
  static constexpr int kSmem = kWarps * kWarpBytes > kJoin ? kWarps * kWarpBytes : kJoin;
};

// the 16-byte unit of an 8-bit row where unit u is held: 8 rows' equal units fall on distinct banks
// (ldmatrix), and so do the units 0 .. 3 of two rows (16-byte loads by a quarter of a warp)
template <int D>
__device__ __forceinline__ int unit_at(int row, int u) {
  if constexpr (D == 128) return u ^ (((row & 1) << 2) | ((row >> 1) & 3));
  else if constexpr (D == 64) return u ^ ((row >> 1) & 3);
  else if constexpr (D == 32) return u ^ ((row >> 2) & 1);
  else return u;
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}
// two bytes of u, selected as for prmt by (0, 4, ...) nibbles, as two numbers of T; u has its sign
// bits flipped for f16
template <typename T, uint32_t SEL>
__device__ __forceinline__ uint32_t two_of(uint32_t u) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) {
    const uint32_t y = __byte_perm(u, 0x64646464u, SEL);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(y), "r"(0x64806480u));
  } else {
    const uint32_t y = __byte_perm(u, 0x43434343u, SEL);
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(y & 0xff7fff7fu), "r"(y & 0xff80ff80u));
  }
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t flipped(uint32_t u) {
  return std::is_same<T, __half>::value ? u ^ 0x80808080u : u;
}
constexpr uint32_t kLow = 0x4140u, kHigh = 0x4342u, kEven = 0x4240u, kOdd = 0x4341u;

// FEW: no block has more than 8 rows, so that the operand's rows 8 .. 15 are nothing
template <typename T, int D, bool Q8, bool FEW>
__global__ void __launch_bounds__(kThreads) tree_dec_kernel(const __grid_constant__ Params p) {
  using C = Cfg<D, Q8, FEW>;
  constexpr int kChunk = C::kChunk, KN = kChunk / 8;  // n-tiles of 8 keys
  constexpr int R2 = FEW ? 1 : 2;  // of this thread's rows g and g + 8
  constexpr int NS = C::kStages;
  constexpr bool kNorm = Q8 && std::is_same<T, __half>::value;
  constexpr int kBytes = D >= 64 ? 16 : D / 4;  // of an 8-bit key's row that a thread takes together
  constexpr int kBlocks = D / (4 * kBytes);
  extern __shared__ __align__(16) uint8_t dec_smem[];
  __shared__ int parent[kMaxNodes];
  __shared__ uint32_t bits[kRows][kWords + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q4 = lane & 3;
  const int cta = static_cast<int>(blockIdx.x), rows = p.group * p.nodes;
  grid_wait();
  Walk walk(p, cta);
  while (walk.more()) {
  const Block blk = next_block(p, walk);
  const Seq sq = blk.sq;
  const int b = blk.b, kvh = blk.kvh, r0 = blk.mb * kRows;
  // this CTA's chunks, shared by its warps in turn
  const int c0 = blk.t0 * (kUnit / kChunk), c1 = min(blk.t1 * (kUnit / kChunk), (sq.len + kChunk - 1) / kChunk);

  const uint32_t ring = smem_u32(dec_smem) + warp * C::kWarpBytes;
  const uint8_t* kb = static_cast<const uint8_t*>(p.k) + (b * p.k_st[0] + kvh * p.k_st[1]) * (Q8 ? 1 : 2);
  const uint8_t* vb = static_cast<const uint8_t*>(p.v) + (b * p.v_st[0] + kvh * p.v_st[1]) * (Q8 ? 1 : 2);
  const int64_t krow = p.k_st[2] * (Q8 ? 1 : 2), vrow = p.v_st[2] * (Q8 ? 1 : 2);
  const float* ksb = Q8 ? p.ks + b * p.ks_st[0] + kvh * p.ks_st[1] : nullptr;
  const float* vsb = Q8 ? p.vs + b * p.vs_st[0] + kvh * p.vs_st[1] : nullptr;
  // this lane's 16-byte unit and its first row; its rows are kApart apart, where the swizzle's period allows
  constexpr int kUnits = C::kRowBytes / 16, kApart = 32 / kUnits, kCopies = (kChunk + kApart - 1) / kApart;
  const int fr = lane / kUnits, fu = lane % kUnits;
  const uint8_t *kp = kb + fu * 16 + fr * krow, *vp = vb + fu * 16 + fr * vrow;
  auto fetch = [&](int c, int stage) {
    if (c < c1) {
      const int j0 = c * kChunk;
      const uint32_t at = ring + stage * C::kStage;
      const int64_t ko = j0 * krow, vo = j0 * vrow;
      if (j0 + kChunk <= sq.len) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int r = fr + i * kApart, to = r * C::kPitch + (Q8 ? unit_at<D>(r, fu) : fu) * 16;
          if (kChunk % kApart && r >= kChunk) break;  // 16 rows of 16 bytes: half of the lanes
          cp16(at + to, kp + ko + i * kApart * krow, true);
          cp16(at + C::kHalf + to, vp + vo + i * kApart * vrow, true);
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < kCopies; ++i) {
          const int r = fr + i * kApart, to = r * C::kPitch + (Q8 ? unit_at<D>(r, fu) : fu) * 16;
          if (kChunk % kApart && r >= kChunk) break;
          const bool in = j0 + r < sq.len;  // beyond the length: zeros, nothing read
          cp16(at + to, in ? kp + ko + i * kApart * krow : kb, in);
          cp16(at + C::kHalf + to, in ? vp + vo + i * kApart * vrow : vb, in);
        }
      }
      if constexpr (Q8) {
#pragma unroll
        for (int i = 0; i < 2 * kChunk; i += 32) {  // the keys' scales, then the values'
          const int r = (lane + i) % kChunk;
          const bool in = j0 + r < sq.len;
          const int64_t row = in ? j0 + r : 0;
          cp4(at + 2 * C::kHalf + (lane + i) * 4, lane + i < kChunk ? ksb + row * p.ks_st[2] : vsb + row * p.vs_st[2], in);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int first = c0 + warp;
#pragma unroll
  for (int s = 0; s < NS - 1; ++s) fetch(first + s * kWarps, s);

  // Q as A fragments: k-step s, rows g / g + 8; columns 16 s + 2 q4 (+8), or for 8-bit keys the
  // columns of the bytes that the thread takes
  uint32_t qa[D / 16][4] = {};
#pragma unroll
  for (int h = 0; h < R2; ++h) {
    const int r = min(r0 + g + 8 * h, rows - 1);
    const T* qr = static_cast<const T*>(p.q) + b * p.q_st[0] + (kvh * p.group + r / p.nodes) * p.q_st[1] +
                  (r % p.nodes) * p.q_st[2];
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const int at = Q8 ? (s / (kBytes / 4)) * 4 * kBytes + q4 * kBytes + (s % (kBytes / 4)) * 4 : 16 * s + 2 * q4;
      qa[s][h] = __ldg(reinterpret_cast<const uint32_t*>(qr + at));
      qa[s][2 + h] = __ldg(reinterpret_cast<const uint32_t*>(qr + at + (Q8 ? 2 : 8)));
    }
  }
  if (c1 * kChunk > sq.all) {  // some of this CTA's keys are the tree's
    load_parents(p, sq, b, parent, kThreads);
    __syncthreads();
    if (threadIdx.x < kRows) walk_up(sq, parent, min(r0 + static_cast<int>(threadIdx.x), rows - 1) % p.nodes, bits[threadIdx.x]);
    __syncthreads();
  }
  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

  int stage = 0;
  for (int c = first; c < c1; c += kWarps) {
    asm volatile("cp.async.wait_group %0;" ::"n"(NS - 2) : "memory");
    __syncwarp();
    const int j0 = c * kChunk;
    const uint32_t sk = ring + stage * C::kStage, sv = sk + C::kHalf;
    const uint8_t* at = dec_smem + (sk - smem_u32(dec_smem));
    // S = Q K^T, 8 keys an n-tile
    float s[KN][4] = {};
    float kscale[KN][2];
    ValueScale vscale[KN][2];
    if constexpr (Q8) {
#pragma unroll
      for (int n = 0; n < KN; ++n) {
        const int r = n * 8 + g;
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
          uint32_t w[kBytes / 4];
          const uint8_t* row = at + r * C::kPitch;
          if constexpr (kBytes == 16) {
            const uint4 x = *reinterpret_cast<const uint4*>(row + unit_at<D>(r, 4 * i + q4) * 16);
            w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
          } else if constexpr (kBytes == 8) {
            const uint2 x = *reinterpret_cast<const uint2*>(row + unit_at<D>(r, q4 >> 1) * 16 + (q4 & 1) * 8);
            w[0] = x.x; w[1] = x.y;
          } else {
            w[0] = *reinterpret_cast<const uint32_t*>(row + q4 * 4);
          }
#pragma unroll
          for (int x = 0; x < kBytes / 4; ++x) {
            const uint32_t u = flipped<T>(w[x]);
            mma16816<T>(s[n], qa[i * (kBytes / 4) + x], two_of<T, kLow>(u), two_of<T, kHigh>(u));
          }
        }
        const float2 a = *reinterpret_cast<const float2*>(at + 2 * C::kHalf + (n * 8 + q4 * 2) * 4);
        const float2 z = *reinterpret_cast<const float2*>(at + 2 * C::kHalf + (kChunk + n * 8 + q4 * 2) * 4);
        vscale[n][0] = value_scale<kNorm>(z.x);
        vscale[n][1] = value_scale<kNorm>(z.y);
        kscale[n][0] = a.x * p.scale_log2;
        kscale[n][1] = a.y * p.scale_log2;
      }
    } else {
      const uint32_t from = sk + ((lane & 7) + ((lane >> 4) << 3)) * C::kPitch + ((lane >> 3) & 1) * 16;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t r[4];  // keys 0-7: k 0-7, k 8-15; keys 8-15: k 0-7, k 8-15
        ldsm4(r, from + ks * 32);
        mma16816<T>(s[0], qa[ks], r[0], r[1]);
        mma16816<T>(s[1], qa[ks], r[2], r[3]);
      }
    }
    // exponents of base 2
    const bool inside = j0 + kChunk <= sq.all;
    if constexpr (Q8) {
      if (!inside) {
#pragma unroll
        for (int n = 0; n < KN; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!(fabsf(vscale[n][e].rest) < INFINITY)) {
              kscale[n][e] = __uint_as_float(0x7fc00000u);
              vscale[n][e].rest = 0.0f;
            }
      }
    }
#pragma unroll
    for (int n = 0; n < KN; ++n)
#pragma unroll
      for (int e = 0; e < 2 * R2; ++e) {
        float x;
        if constexpr (kNorm) x = __fmaf_rn(s[n][e], kscale[n][e & 1], vscale[n][e & 1].lift);
        else x = s[n][e] * (Q8 ? kscale[n][e & 1] : p.scale_log2);
        s[n][e] = inside || sees(sq, bits[g + 8 * (e >> 1)], j0 + n * 8 + q4 * 2 + (e & 1)) ? x : -INFINITY;
      }
    float alpha[2];
#pragma unroll
    for (int h = 0; h < R2; ++h) {
      float mx = s[0][2 * h];
#pragma unroll
      for (int n = 0; n < KN; ++n)
        asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(mx) : "f"(mx), "f"(s[n][2 * h]), "f"(s[n][2 * h + 1]));
      mx = quad_max(mx);
      if (!(mx < INFINITY)) l[h] = __uint_as_float(0x7fc00000u);  // a NaN or an infinite score
      const float mn = fmaxf(m[h], mx);
      const float ref = mn == -INFINITY ? 0.0f : mn;
      alpha[h] = ex2_approx(m[h] - ref);
      m[h] = mn;
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < KN; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[n][2 * h + e] = ex2_approx(s[n][2 * h + e] - ref);
          if constexpr (kNorm) sum = __fmaf_rn(s[n][2 * h + e], vscale[n][e].lower, sum);
          else sum += s[n][2 * h + e];
        }
      l[h] = __fmaf_rn(l[h], alpha[h], sum);  // this thread's columns; joined over the quad at the end
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[R2 - 1] != 1.0f)) {
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2 * R2; ++e) o[n][e] *= alpha[e >> 1];
    }
    if constexpr (Q8) {
      // the value's scale with the weight
#pragma unroll
      for (int n = 0; n < KN; ++n)
#pragma unroll
        for (int e = 0; e < 2 * R2; ++e) s[n][e] *= vscale[n][e & 1].rest;
    } else if (!inside) {
      bool bad = false;
      for (int x = lane; x < kChunk * (D / 8); x += 32) {
        uint4* v = reinterpret_cast<uint4*>(dec_smem + (sv - smem_u32(dec_smem)) + (x / (D / 8)) * C::kPitch +
                                            (x % (D / 8)) * 16);
        uint4 u = *v;
        uint32_t* e = reinterpret_cast<uint32_t*>(&u);
        bool hit = false;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t nf = bad_bits<T>(e[q]);
          if (nf & 0x8000u) e[q] &= 0xffff0000u;
          if (nf & 0x80000000u) e[q] &= 0x0000ffffu;
          hit |= nf != 0u;
        }
        if (hit) *v = u;
        bad |= hit;
      }
      __syncwarp();
      if (__any_sync(0xffffffffu, bad)) {
        for (int j = j0; j < min(j0 + kChunk, sq.len); ++j) {
          const T* vr = reinterpret_cast<const T*>(vb + j * vrow);
#pragma unroll
          for (int h = 0; h < R2; ++h) {
            if (!sees(sq, bits[g + 8 * h], j)) continue;
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float f = to_f32(vr[n * 8 + q4 * 2 + e]);
                if (!(fabsf(f) < INFINITY)) o[n][2 * h + e] += f;
              }
          }
        }
      }
    }
    // O += P V, 16 keys an operand
    uint32_t pa[KN / 2][4];
#pragma unroll
    for (int k = 0; k < KN / 2; ++k) {
      pa[k][0] = pack2<T>(s[2 * k][0], s[2 * k][1]);
      pa[k][1] = FEW ? 0u : pack2<T>(s[2 * k][2], s[2 * k][3]);
      pa[k][2] = pack2<T>(s[2 * k + 1][0], s[2 * k + 1][1]);
      pa[k][3] = FEW ? 0u : pack2<T>(s[2 * k + 1][2], s[2 * k + 1][3]);
    }
    if constexpr (Q8) {
#pragma unroll
      for (int u = 0; u < D / 16; u += 2) {
        const int x = D == 16 ? 0 : u + (lane >> 4);
#pragma unroll
        for (int k = 0; k < KN / 2; ++k) {
          uint32_t r[4];  // bytes 16 u: keys 0-7, 8-15; bytes 16 u + 16: keys 0-7, 8-15
          const int row = k * 16 + (lane & 15);
          ldsm4t(r, sv + row * C::kPitch + unit_at<D>(row, x) * 16);
#pragma unroll
          for (int e = 0; e < (D == 16 ? 1 : 2); ++e) {
            const uint32_t a = flipped<T>(r[2 * e]), z = flipped<T>(r[2 * e + 1]);
            mma16816<T>(o[2 * (u + e)], pa[k], two_of<T, kEven>(a), two_of<T, kEven>(z));
            mma16816<T>(o[2 * (u + e) + 1], pa[k], two_of<T, kOdd>(a), two_of<T, kOdd>(z));
          }
        }
      }
    } else {
      const uint32_t from = sv + (lane & 15) * C::kPitch + (lane >> 4) * 16;
#pragma unroll
      for (int n = 0; n < D / 8; n += 2) {
        uint32_t r[4];  // columns 8 n: keys 0-7, 8-15; columns 8 n + 8: keys 0-7, 8-15
        ldsm4t(r, from + n * 16);
        mma16816<T>(o[n], pa[0], r[0], r[1]);
        mma16816<T>(o[n + 1], pa[0], r[2], r[3]);
      }
    }
    __syncwarp();  // every lane has read the stage that is filled next
    const int ahead = stage + NS - 1 >= NS ? stage - 1 : stage + NS - 1;
    fetch(c + (NS - 1) * kWarps, ahead);
    stage = stage + 1 == NS ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int h = 0; h < R2; ++h)
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], off);

  // join the warps
  __syncthreads();
  float* jo = reinterpret_cast<float*>(dec_smem);         // [warp][row][D]
  float* jm = jo + kWarps * kRows * D;                    // [warp][row]
  float* jl = jm + kWarps * kRows;
#pragma unroll
  for (int h = 0; h < R2; ++h) {
    const int r = g + 8 * h;
    float* to = jo + (warp * kRows + r) * D;
#pragma unroll
    for (int n = 0; n < D / 8; n += 2) {
      if constexpr (Q8) {  // the columns of tile n are 8 n + 0, 2, 4, ..., those of n + 1 lie between them
        *reinterpret_cast<float4*>(to + n * 8 + q4 * 4) =
            make_float4(o[n][2 * h], o[n + 1][2 * h], o[n][2 * h + 1], o[n + 1][2 * h + 1]);
      } else {
        *reinterpret_cast<float2*>(to + n * 8 + q4 * 2) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        *reinterpret_cast<float2*>(to + n * 8 + 8 + q4 * 2) = make_float2(o[n + 1][2 * h], o[n + 1][2 * h + 1]);
      }
    }
    if (q4 == 0) {
      jm[warp * kRows + r] = m[h];
      jl[warp * kRows + r] = l[h];
    }
  }
  __syncthreads();
  const int here = min(kRows, rows - r0);
  for (int x = threadIdx.x; x < here * (D / 2); x += kThreads) {
    const int r = x / (D / 2), d = (x % (D / 2)) * 2;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, jm[w * kRows + r]);
    const float ref = mm == -INFINITY ? 0.0f : mm;
    float a0 = 0.0f, a1 = 0.0f, ll = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (jm[w * kRows + r] == -INFINITY && jl[w * kRows + r] == 0.0f) continue;  // saw no key
      const float f = ex2_approx(jm[w * kRows + r] - ref);
      const float2 v = *reinterpret_cast<const float2*>(jo + (w * kRows + r) * D + d);
      a0 = __fmaf_rn(v.x, f, a0);
      a1 = __fmaf_rn(v.y, f, a1);
      ll = __fmaf_rn(jl[w * kRows + r], f, ll);
    }
    const int head = kvh * p.group + (r0 + r) / p.nodes, node = (r0 + r) % p.nodes;
    if (!blk.whole) {
      const int64_t to = part_row(p, cta, blk.slot, r);
      *reinterpret_cast<float2*>(p.part_o + to * D + d) = make_float2(a0, a1);
      if (d == 0) p.part_ml[to] = make_float2(mm, ll);
    } else {
      const float rl = ll == 0.0f ? 0.0f : __frcp_rn(ll);
      const bool real = node < sq.n;
      *reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + b * p.o_st[0] + head * p.o_st[1] + node * p.o_st[2] + d) =
          pack2<T>(real ? a0 * rl : 0.0f, real ? a1 * rl : 0.0f);
    }
  }
  __syncthreads();  // the next block's keys go where the rows were joined
  }
}

template <typename T, int D, bool Q8, bool FEW>
int launch_rows(const Params& p, cudaStream_t s) {
  constexpr int bytes = Cfg<D, Q8, FEW>::kSmem;
  static OptIn opted;
  if (!opted.shared(tree_dec_kernel<T, D, Q8, FEW>, bytes)) return FPK_ERR_CUDA;
  return launch_dependent(tree_dec_kernel<T, D, Q8, FEW>, dim3(static_cast<unsigned>(p.ctas)), kThreads, bytes, s, p);
}
template <typename T, int D, bool Q8>
int launch(const Params& p, cudaStream_t s) {
  return p.group * p.nodes <= 8 ? launch_rows<T, D, Q8, true>(p, s) : launch_rows<T, D, Q8, false>(p, s);
}
template <typename T, bool Q8>
int launch_t(const Params& p, int D, cudaStream_t s) {
  switch (D) {
    case 16: return launch<T, 16, Q8>(p, s);
    case 32: return launch<T, 32, Q8>(p, s);
    case 64: return launch<T, 64, Q8>(p, s);
    default: return launch<T, 128, Q8>(p, s);
  }
}

}  // namespace

int launch_dec(const Params& p, int dtype, int D, cudaStream_t s) {
  if (dtype == FPK_F16) return p.ks ? launch_t<__half, true>(p, D, s) : launch_t<__half, false>(p, D, s);
  return p.ks ? launch_t<__nv_bfloat16, true>(p, D, s) : launch_t<__nv_bfloat16, false>(p, D, s);
}

}  // namespace tree
}  // namespace fpk
