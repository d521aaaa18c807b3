// Score attention for few query rows (f16 and bf16): the form for single tokens.
//
// The queries of all heads of a group read the same keys and values, so up to 16 rows
// (row r: head r / q_len of the group, query r % q_len) are one m16 operand of the
// mma.sync matrix instruction, and the cache is read once whatever the group.  The work
// is bound by reading the cache; 16 rows of tensor work are far below that.
//
// A CTA takes a part of one sequence's key tiles; its 4 warps take 16 keys at a time in
// turn, each with its own ring of cp.async stages (no barrier between warps), its own
// running maximum and sum and its own 16 x D result in registers, joined through shared
// memory at the end.  With several parts, unnormalised rows go to the workspace and
// score_combine_kernel joins them.
//
// Values behind a row's mask must not reach it: in chunks that some row sees in part, what
// is not finite in V is replaced by zeros before the product and added for the rows that
// see it.
#include <cuda_runtime.h>

#include <cmath>
#include <type_traits>

#include "internal.h"
#include "score_common.cuh"
#include "vec_types.cuh"

namespace fpk {
namespace score {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 16;
constexpr int kChunk = 16;  // keys a warp takes at a time
constexpr int kPer = kKeyTile / kChunk;

template <int D>
struct Cfg {
  static constexpr int kPitch = D * 2 + 16;  // bytes: an odd number of 16-byte units, no bank conflicts
  static constexpr int kHalf = kChunk * kPitch;
  static constexpr int kStage = 2 * kHalf;   // K, V
  static constexpr int kStages = D == 128 ? 3 : 4;
  static constexpr int kWarpBytes = kStages * kStage;
  static constexpr int kJoin = kWarps * kRows * (D + 2) * 4;
  static constexpr int kSmem = kWarps * kWarpBytes > kJoin ? kWarps * kWarpBytes : kJoin;
};

template <typename T>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t bad_bits(uint32_t u) {
  constexpr bool kHalfT = std::is_same<T, __half>::value;
  return ((u & (kHalfT ? 0x7c007c00u : 0x7f807f80u)) + (kHalfT ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}
__device__ __forceinline__ float quad_max(float v) {
  // a NaN among the four is kept
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, v, off);
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(v), "f"(o));
  }
  return v;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) score_dec_kernel(const __grid_constant__ Params p) {
  using C = Cfg<D>;
  constexpr int NS = C::kStages;
  extern __shared__ __align__(16) uint8_t dec_smem[];
  __shared__ int s_range[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q4 = lane & 3;
  int item = static_cast<int>(blockIdx.x);
  const int sp = item % p.splits;
  item /= p.splits;
  const int kvh = item % p.kv_heads, b = item / p.kv_heads;
  const int rows = p.group * p.q_len;
  grid_wait();
  const Seq sq = seq_of(p, b);
  const Tiles tl = tiles_of(p, sq, sq.base, sq.base + p.q_len - 1);

  // this thread's two rows: g and g + 8
  int pos[2], id[2];
  Span span[2];
  float slope2[2];
  bool real[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = min(g + 8 * h, rows - 1);
    real[h] = g + 8 * h < rows;
    pos[h] = sq.base + r % p.q_len;
    span[h] = span_of(p, sq, pos[h]);
    id[h] = p.ids ? id_at(p, b, pos[h], sq.len) : 0;
    slope2[h] = p.slopes ? __ldg(p.slopes + kvh * p.group + r / p.q_len) * 1.4426950408889634f : 0.0f;
  }
  int i0 = 0, i1 = tl.n;
  if (p.ids) {  // the ends of the tile list that hold none of the rows' ids
    int lo = min(id[0] < 0 ? 0x7fffffff : id[0], id[1] < 0 ? 0x7fffffff : id[1]), hi = max(id[0], id[1]);
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (warp == 0) {
      const IdRange* rg = p.ranges + static_cast<int64_t>(b) * p.k_tiles;
      int a = tl.n, z = 0;
      for (int i = lane; i < tl.n; i += 32) {
        const IdRange r = rg[tl.at(i)];
        if (r.hi >= lo && r.lo <= hi) {
          a = min(a, i);
          z = max(z, i + 1);
        }
      }
      a = __reduce_min_sync(0xffffffffu, a);
      z = __reduce_max_sync(0xffffffffu, z);
      if (lane == 0) {
        s_range[0] = a;
        s_range[1] = max(a, z);
      }
    }
    __syncthreads();
    i0 = s_range[0];
    i1 = s_range[1];
  }
  // this CTA's chunks, shared by its warps in turn
  const int nc = (i1 - i0) * kPer;
  const int c0 = i0 * kPer + static_cast<int>(static_cast<int64_t>(nc) * sp / p.splits);
  const int c1 = i0 * kPer + static_cast<int>(static_cast<int64_t>(nc) * (sp + 1) / p.splits);

  // Q as A fragments: k-step s, rows g / g + 8, columns 16 s + 2 q4 (+8)
  uint32_t qa[D / 16][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = min(g + 8 * h, rows - 1);
    const T* qr = static_cast<const T*>(p.q) + b * p.q_st[0] + (kvh * p.group + r / p.q_len) * p.q_st[1] +
                  (r % p.q_len) * p.q_st[2];
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      qa[s][h] = real[h] ? __ldg(reinterpret_cast<const uint32_t*>(qr + 16 * s + 2 * q4)) : 0u;
      qa[s][2 + h] = real[h] ? __ldg(reinterpret_cast<const uint32_t*>(qr + 16 * s + 8 + 2 * q4)) : 0u;
    }
  }
  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

  const uint32_t ring = smem_u32(dec_smem) + warp * C::kWarpBytes;
  const T* kb = static_cast<const T*>(p.k) + b * p.k_st[0] + kvh * p.k_st[1];
  const T* vb = static_cast<const T*>(p.v) + b * p.v_st[0] + kvh * p.v_st[1];
  auto key0 = [&](int c) { return tl.at(c / kPer) * kKeyTile + (c % kPer) * kChunk; };
  auto fetch = [&](int c, int stage) {
    if (c < c1) {
      const int j0 = key0(c);
      const uint32_t at = ring + stage * C::kStage;
      constexpr int kUnits = D / 8;  // 16-byte units a row
#pragma unroll
      for (int x = lane; x < kChunk * kUnits; x += 32) {
        const int r = x / kUnits, u = x % kUnits;
        const bool in = j0 + r < sq.len;  // beyond the length: zeros, nothing read
        const int64_t row = in ? j0 + r : 0;
        cp16(at + r * C::kPitch + u * 16, kb + row * p.k_st[2] + u * 8, in);
        cp16(at + C::kHalf + r * C::kPitch + u * 16, vb + row * p.v_st[2] + u * 8, in);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int first = c0 + warp;
#pragma unroll
  for (int s = 0; s < NS - 1; ++s) fetch(first + s * kWarps, s);

  int stage = 0;
  for (int c = first; c < c1; c += kWarps) {
    asm volatile("cp.async.wait_group %0;" ::"n"(NS - 2) : "memory");
    __syncwarp();
    const int j0 = key0(c);
    const uint32_t sk = ring + stage * C::kStage, sv = sk + C::kHalf;
    // S = Q K^T: two n-tiles of 8 keys
    float s[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
    const uint32_t krow = sk + ((lane & 7) + ((lane >> 4) << 3)) * C::kPitch + ((lane >> 3) & 1) * 16;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint32_t r[4];  // keys 0-7: k 0-7, k 8-15; keys 8-15: k 0-7, k 8-15
      ldsm4(r, krow + ks * 32);
      mma16816<T>(s[0], qa[ks], r[0], r[1]);
      mma16816<T>(s[1], qa[ks], r[2], r[3]);
    }
    // exponents of base 2
    bool part = false;
    const bool inside = j0 + kChunk <= sq.pre;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int h = e >> 1, j = j0 + n * 8 + q4 * 2 + (e & 1);
        float x = s[n][e];
        if (p.cap > 0.0f) x = p.cap * 1.4426950408889634f * tanh_ex2(x * (p.scale / p.cap));
        else x *= p.scale_log2;
        if (p.slopes) x = __fmaf_rn(-slope2[h], fabsf(static_cast<float>(pos[h] - j)), x);
        bool seen = inside || j < sq.pre || (j >= span[h].lo && j < span[h].hi);
        if (p.ids) seen = seen && id[h] >= 0 && id_at(p, b, j, sq.len) == id[h];
        part |= !seen;
        s[n][e] = seen ? x : -INFINITY;
      }
    float alpha[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx;
      asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(mx) : "f"(s[0][2 * h]), "f"(s[0][2 * h + 1]), "f"(s[1][2 * h]));
      asm("max.NaN.f32 %0, %1, %2;" : "=f"(mx) : "f"(mx), "f"(s[1][2 * h + 1]));
      mx = quad_max(mx);
      if (!(mx < INFINITY)) l[h] = __uint_as_float(0x7fc00000u);  // a NaN or an infinite score
      const float mn = fmaxf(m[h], mx);
      const float ref = mn == -INFINITY ? 0.0f : mn;
      alpha[h] = ex2_approx(m[h] - ref);
      m[h] = mn;
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[n][2 * h + e] = ex2_approx(s[n][2 * h + e] - ref);
          sum += s[n][2 * h + e];
        }
      l[h] = __fmaf_rn(l[h], alpha[h], sum);  // this thread's columns; joined over the quad at the end
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        o[n][0] *= alpha[0];
        o[n][1] *= alpha[0];
        o[n][2] *= alpha[1];
        o[n][3] *= alpha[1];
      }
    }
    if (__any_sync(0xffffffffu, part)) {
      bool bad = false;
      for (int x = lane; x < kChunk * (D / 8); x += 32) {
        uint4* at = reinterpret_cast<uint4*>(dec_smem + (sv - smem_u32(dec_smem)) + (x / (D / 8)) * C::kPitch +
                                             (x % (D / 8)) * 16);
        uint4 u = *at;
        uint32_t* e = reinterpret_cast<uint32_t*>(&u);
        bool hit = false;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t nf = bad_bits<T>(e[q]);
          if (nf & 0x8000u) e[q] &= 0xffff0000u;
          if (nf & 0x80000000u) e[q] &= 0x0000ffffu;
          hit |= nf != 0u;
        }
        if (hit) *at = u;
        bad |= hit;
      }
      __syncwarp();
      if (__any_sync(0xffffffffu, bad)) {
        for (int k = 0; k < kChunk && j0 + k < sq.len; ++k) {
          const int j = j0 + k;
          const T* vr = vb + j * p.v_st[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            bool seen = j < sq.pre || (j >= span[h].lo && j < span[h].hi);
            if (p.ids) seen = seen && id[h] >= 0 && id_at(p, b, j, sq.len) == id[h];
            if (!seen) continue;
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
    // O += P V
    const uint32_t pa[4] = {pack2<T>(s[0][0], s[0][1]), pack2<T>(s[0][2], s[0][3]), pack2<T>(s[1][0], s[1][1]),
                            pack2<T>(s[1][2], s[1][3])};
    const uint32_t vrow = sv + (lane & 15) * C::kPitch + (lane >> 4) * 16;
#pragma unroll
    for (int n = 0; n < D / 8; n += 2) {
      uint32_t r[4];  // columns 8 n: keys 0-7, 8-15; columns 8 n + 8: keys 0-7, 8-15
      ldsm4t(r, vrow + n * 16);
      mma16816<T>(o[n], pa, r[0], r[1]);
      mma16816<T>(o[n + 1], pa, r[2], r[3]);
    }
    __syncwarp();  // every lane has read the stage that is filled next
    const int ahead = stage + NS - 1 >= NS ? stage - 1 : stage + NS - 1;
    fetch(c + (NS - 1) * kWarps, ahead);
    stage = stage + 1 == NS ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], off);

  // join the warps
  __syncthreads();
  float* jo = reinterpret_cast<float*>(dec_smem);         // [warp][row][D]
  float* jm = jo + kWarps * kRows * D;                    // [warp][row]
  float* jl = jm + kWarps * kRows;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = g + 8 * h;
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
      *reinterpret_cast<float2*>(jo + (warp * kRows + r) * D + n * 8 + q4 * 2) =
          make_float2(o[n][2 * h], o[n][2 * h + 1]);
    if (q4 == 0) {
      jm[warp * kRows + r] = m[h];
      jl[warp * kRows + r] = l[h];
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < rows * (D / 2); x += kThreads) {
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
    const int head = kvh * p.group + r / p.q_len, qi = r % p.q_len;
    if (p.splits > 1) {
      const int64_t at = ((static_cast<int64_t>(b) * p.heads + head) * p.q_len + qi) * p.splits + sp;
      *reinterpret_cast<float2*>(p.part_o + at * D + d) = make_float2(a0, a1);
      if (d == 0) p.part_ml[at] = make_float2(mm, ll);
    } else {
      const float rl = ll == 0.0f ? 0.0f : __frcp_rn(ll);
      *reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + b * p.o_st[0] + head * p.o_st[1] + qi * p.o_st[2] + d) =
          pack2<T>(a0 * rl, a1 * rl);
    }
  }
}

template <typename T, int D>
int launch(const Params& p, cudaStream_t s) {
  const int64_t grid = static_cast<int64_t>(p.items) * p.splits;
  if (grid > 0x7fffffffLL) return FPK_ERR_UNSUPPORTED;
  constexpr int bytes = Cfg<D>::kSmem;
  static OptIn opted;
  if (!opted.shared(score_dec_kernel<T, D>, bytes)) return FPK_ERR_CUDA;
  return launch_dependent(score_dec_kernel<T, D>, dim3(static_cast<unsigned>(grid)), kThreads, bytes, s, p);
}
template <typename T>
int launch_t(const Params& p, int D, cudaStream_t s) {
  switch (D) {
    case 16: return launch<T, 16>(p, s);
    case 32: return launch<T, 32>(p, s);
    case 64: return launch<T, 64>(p, s);
    case 128: return launch<T, 128>(p, s);
    default: return FPK_ERR_UNSUPPORTED;
  }
}

}  // namespace

int launch_dec(const Params& p, int dtype, int D, cudaStream_t s) {
  return dtype == FPK_F16 ? launch_t<__half>(p, D, s) : launch_t<__nv_bfloat16>(p, D, s);
}

}  // namespace score
}  // namespace fpk
