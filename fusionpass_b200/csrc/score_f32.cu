// Score attention in f32 on the FMA pipe (score_common.cuh: which key a query sees).
//
// A CTA takes BM rows of one key/value head, where the rows are the queries of all heads
// of the group (row r: head r / q_len of the group, query r % q_len), so that a single
// token of grouped heads reads its cache once.  64-key tiles of K and V go through shared
// memory; a thread owns RPT rows x 4 keys of the scores and RPT rows x D / 16 columns of
// the result, 16 threads share a row.  BM = 64 for long queries, 16 for few rows.
// A key that a row does not see contributes nothing, whatever its values are: in tiles that
// some row sees in part a product with p = 0 is skipped.
#include <cuda_runtime.h>

#include <cmath>

#include "internal.h"
#include "score_common.cuh"

namespace fpk {
namespace score {
namespace {

constexpr int kBK = 64;       // keys a tile
constexpr int kThreads = 256; // 16 rows of threads x 16 threads

template <int D, int RPT>
struct Smem {
  static constexpr int kBM = 16 * RPT;
  static constexpr int kPitch = D + 4;  // floats: rows of one column fall on distinct banks by 16 bytes
  float q[kBM][kPitch], k[kBK][kPitch], v[kBK][D];
  float p[kBM][kBK + 4];
};

__device__ __forceinline__ float row_max(float v) {
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, v, off);
    v = (v != v || o != o) ? v + o : fmaxf(v, o);
  }
  return v;
}
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// a thread's part of a tile of kBK rows of D floats: from memory into registers (rows from n
// on are zeros), and from there into shared memory
template <int D>
struct Part {
  static constexpr int kN = kBK * (D / 4) / kThreads;
  float4 f[kN];
  __device__ __forceinline__ void load(const float* src, int64_t stride, int n) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int x = threadIdx.x + i * kThreads, r = x / (D / 4), c = (x % (D / 4)) * 4;
      f[i] = r < n ? __ldg(reinterpret_cast<const float4*>(src + r * stride + c)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
  }
  __device__ __forceinline__ void store(float* dst, int pitch) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int x = threadIdx.x + i * kThreads, r = x / (D / 4), c = (x % (D / 4)) * 4;
      *reinterpret_cast<float4*>(dst + r * pitch + c) = f[i];
    }
  }
};

// o += P V over the tile; PART: a key with p = 0 adds nothing, whatever its values
template <bool PART, int D, int RPT>
__device__ __forceinline__ void weigh(const Smem<D, RPT>& sm, int ty, int tx, float (&o)[RPT][D / 16]) {
#pragma unroll 2
  for (int j = 0; j < kBK; j += 4) {
    float4 e[RPT];
#pragma unroll
    for (int a = 0; a < RPT; ++a) e[a] = *reinterpret_cast<const float4*>(&sm.p[ty * RPT + a][j]);
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = sm.v[j + i][tx + 16 * c];
#pragma unroll
      for (int a = 0; a < RPT; ++a) {
        const float w[4] = {e[a].x, e[a].y, e[a].z, e[a].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) o[a][c] = __fmaf_rn(w[i], PART && w[i] == 0.0f ? 0.0f : v[i], o[a][c]);
      }
    }
  }
}

template <int D, int RPT>
__global__ void __launch_bounds__(kThreads) score_f32_kernel(const __grid_constant__ Params p) {
  using S = Smem<D, RPT>;
  constexpr int BM = S::kBM;
  constexpr int DC = D / 16;  // result columns a thread: tx + 16 c
  extern __shared__ float smem_raw[];
  S& sm = *reinterpret_cast<S*>(smem_raw);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int item = static_cast<int>(blockIdx.x);
  const int sp = item % p.splits;
  item /= p.splits;
  const int mb = p.mblocks - 1 - item % p.mblocks;
  const int kvh = (item / p.mblocks) % p.kv_heads;
  const int b = item / p.mblocks / p.kv_heads;
  const int rows = p.group * p.q_len;
  const int r0 = mb * BM;
  grid_wait();
  const Seq sq = seq_of(p, b);
  const int rl = min(r0 + BM, rows) - 1;  // last row
  int first = 0, last = p.q_len - 1;      // queries among the rows
  if (r0 / p.q_len == rl / p.q_len) {
    first = r0 % p.q_len;
    last = rl % p.q_len;
  }
  const Tiles tl = tiles_of(p, sq, sq.base + first, sq.base + last);
  const int n2 = tl.n * (kKeyTile / kBK);
  const int i0 = static_cast<int>(static_cast<int64_t>(n2) * sp / p.splits);
  const int i1 = static_cast<int>(static_cast<int64_t>(n2) * (sp + 1) / p.splits);

  // queries of the group's heads
  for (int x = threadIdx.x; x < BM * (D / 4); x += kThreads) {
    const int r = r0 + x / (D / 4), c = (x % (D / 4)) * 4;
    float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r < rows)
      f = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + b * p.q_st[0] +
                                                (kvh * p.group + r / p.q_len) * p.q_st[1] +
                                                (r % p.q_len) * p.q_st[2] + c));
    *reinterpret_cast<float4*>(&sm.q[x / (D / 4)][c]) = f;
  }
  int pos[RPT], id[RPT];
  Span span[RPT];
  float slope[RPT], m[RPT], l[RPT], o[RPT][DC];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = min(r0 + ty * RPT + i, rows - 1);
    pos[i] = sq.base + r % p.q_len;
    span[i] = span_of(p, sq, pos[i]);
    id[i] = p.ids ? id_at(p, b, pos[i], sq.len) : 0;
    slope[i] = p.slopes ? __ldg(p.slopes + kvh * p.group + r / p.q_len) : 0.0f;
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < DC; ++c) o[i][c] = 0.0f;
  }
  const float* kb = static_cast<const float*>(p.k) + b * p.k_st[0] + kvh * p.k_st[1];
  const float* vb = static_cast<const float*>(p.v) + b * p.v_st[0] + kvh * p.v_st[1];

  // the next tile's K and V are asked for before this one is worked on
  Part<D> pk, pv;
  const auto fetch = [&](int i) {
    const int j0 = tl.at(i / 2) * kKeyTile + (i & 1) * kBK;
    const int n = max(sq.len - j0, 0);  // the second half of the last tile may lie beyond the keys
    pk.load(kb + j0 * p.k_st[2], p.k_st[2], n);
    pv.load(vb + j0 * p.v_st[2], p.v_st[2], n);
  };
  if (i0 < i1) fetch(i0);
  for (int i = i0; i < i1; ++i) {
    const int j0 = tl.at(i / 2) * kKeyTile + (i & 1) * kBK;
    __syncthreads();
    pk.store(&sm.k[0][0], S::kPitch);
    pv.store(&sm.v[0][0], D);
    __syncthreads();
    if (i + 1 < i1) fetch(i + 1);
    if (j0 >= sq.len) continue;  // the same for the whole block
    float x[RPT][4];
#pragma unroll
    for (int a = 0; a < RPT; ++a)
#pragma unroll
      for (int c = 0; c < 4; ++c) x[a][c] = 0.0f;
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      float4 qv[RPT], kv[4];
#pragma unroll
      for (int a = 0; a < RPT; ++a) qv[a] = *reinterpret_cast<const float4*>(&sm.q[ty * RPT + a][d]);
#pragma unroll
      for (int c = 0; c < 4; ++c) kv[c] = *reinterpret_cast<const float4*>(&sm.k[tx + 16 * c][d]);
#pragma unroll
      for (int a = 0; a < RPT; ++a)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          x[a][c] = __fmaf_rn(qv[a].x, kv[c].x, x[a][c]);
          x[a][c] = __fmaf_rn(qv[a].y, kv[c].y, x[a][c]);
          x[a][c] = __fmaf_rn(qv[a].z, kv[c].z, x[a][c]);
          x[a][c] = __fmaf_rn(qv[a].w, kv[c].w, x[a][c]);
        }
    }
    bool part = false;  // some row does not see some key
#pragma unroll
    for (int a = 0; a < RPT; ++a) {
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = j0 + tx + 16 * c;
        bool seen = j < sq.pre || (j >= span[a].lo && j < span[a].hi);
        if (p.ids) seen = seen && id[a] >= 0 && id_at(p, b, j, sq.len) == id[a];
        float s = x[a][c] * p.scale;
        if (p.cap > 0.0f) s = p.cap * tanhf(s / p.cap);
        if (p.slopes) s = __fmaf_rn(-slope[a], fabsf(static_cast<float>(pos[a] - j)), s);
        x[a][c] = seen ? s : -INFINITY;
        part |= !seen;
        mx = (s != s && seen) ? s : (mx != mx ? mx : fmaxf(mx, x[a][c]));
      }
      mx = row_max(mx);
      if (!(mx < INFINITY)) l[a] = __uint_as_float(0x7fc00000u);  // a NaN or an infinite score
      const float mn = fmaxf(m[a], mx);
      const float ref = mn == -INFINITY ? 0.0f : mn;
      const float alpha = expf(m[a] - ref);
      m[a] = mn;
      float sum = 0.0f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float e = expf(x[a][c] - ref);
        sum += e;
        sm.p[ty * RPT + a][tx + 16 * c] = e;
      }
      l[a] = __fmaf_rn(l[a], alpha, row_sum(sum));
#pragma unroll
      for (int c = 0; c < DC; ++c) o[a][c] *= alpha;
    }
    __syncwarp();  // a row's 16 threads are of one warp
    if (__any_sync(0xffffffffu, part)) weigh<true>(sm, ty, tx, o);
    else weigh<false>(sm, ty, tx, o);
    __syncwarp();
  }
#pragma unroll
  for (int a = 0; a < RPT; ++a) {
    const int r = r0 + ty * RPT + a;
    if (r >= rows) continue;
    const int head = kvh * p.group + r / p.q_len, qi = r % p.q_len;
    if (p.splits > 1) {
      const int64_t g = ((static_cast<int64_t>(b) * p.heads + head) * p.q_len + qi) * p.splits + sp;
#pragma unroll
      for (int c = 0; c < DC; ++c) p.part_o[g * D + tx + 16 * c] = o[a][c];
      if (tx == 0) p.part_ml[g] = make_float2(m[a] * 1.4426950408889634f, l[a]);
    } else {
      float* out = static_cast<float*>(p.o) + b * p.o_st[0] + head * p.o_st[1] + qi * p.o_st[2];
      const float rl = l[a] == 0.0f ? 0.0f : __frcp_rn(l[a]);
#pragma unroll
      for (int c = 0; c < DC; ++c) out[tx + 16 * c] = o[a][c] * rl;
    }
  }
}

template <int D, int RPT>
int launch(const Params& p, cudaStream_t s) {
  const int64_t grid = static_cast<int64_t>(p.items) * p.splits;
  if (grid > 0x7fffffffLL) return FPK_ERR_UNSUPPORTED;
  constexpr int bytes = sizeof(Smem<D, RPT>);
  static OptIn opted;
  if (!opted.shared(score_f32_kernel<D, RPT>, bytes)) return FPK_ERR_CUDA;
  return launch_dependent(score_f32_kernel<D, RPT>, dim3(static_cast<unsigned>(grid)), kThreads, bytes, s, p);
}

}  // namespace

int launch_f32(const Params& p, int D, bool few, cudaStream_t s) {
  switch (D) {
    case 16: return few ? launch<16, 1>(p, s) : launch<16, 4>(p, s);
    case 32: return few ? launch<32, 1>(p, s) : launch<32, 4>(p, s);
    case 64: return few ? launch<64, 1>(p, s) : launch<64, 4>(p, s);
    case 128: return few ? launch<128, 1>(p, s) : launch<128, 4>(p, s);
    default: return FPK_ERR_UNSUPPORTED;
  }
}

}  // namespace score
}  // namespace fpk
