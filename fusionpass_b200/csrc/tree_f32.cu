// Tree attention in f32 on the FMA pipe (tree_common.cuh: which key a node sees), over a cache in
// f32 or in 8 bits.
//
// A CTA takes BM rows of one key/value head, the nodes of all heads of the group (row r: head
// r / nodes, node r % nodes).  64-key tiles of K and V go through shared memory, where 8-bit rows
// arrive as f32, q * scale; a thread owns RPT rows x 4 keys of the scores and RPT rows x D / 16
// columns of the result, 16 threads share a row.  BM = 64, or 16 where few rows leave SMs idle.
// The next tile is asked for before this one is worked on.  Bound by the FMA pipe for many rows, by
// the latency of a step for few.
#include <cuda_runtime.h>

#include <cmath>

#include "internal.h"
#include "tree_common.cuh"

namespace fpk {
namespace tree {
namespace {

constexpr int kBK = 64;       // keys a tile
constexpr int kThreads = 256; // 16 rows of threads x 16 threads
constexpr uint32_t kUnseen = 0x80000000u;

template <int D, int RPT>
struct Smem {
  static constexpr int kBM = 16 * RPT;
  static constexpr int kPitch = D + 4;  // floats: rows of one column fall on distinct banks by 16 bytes
  float q[kBM][kPitch], k[kBK][kPitch], v[kBK][D];
  float p[kBM][kBK + 4];
  uint32_t bits[kBM][kWords + 1];
  int parent[kMaxNodes];
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

// a thread's part of a tile of kBK rows of D elements: from memory into registers (rows from n on
// are zeros), and from there, as f32, into shared memory
template <int D, bool Q8>
struct Part {
  static constexpr int kN = kBK * (D / 4) / kThreads;
  float4 f[Q8 ? 1 : kN];
  uint32_t w[Q8 ? kN : 1];
  float one[Q8 ? kN : 1];
  __device__ __forceinline__ void load(const void* src, int64_t stride, const float* scale, int64_t scale_st, int64_t j0,
                                       int n) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int x = threadIdx.x + i * kThreads, r = x / (D / 4), c = (x % (D / 4)) * 4;
      if constexpr (Q8) {
        w[i] = 0u;
        one[i] = 0.0f;
        if (r < n) {
          w[i] = __ldg(reinterpret_cast<const uint32_t*>(static_cast<const int8_t*>(src) + (j0 + r) * stride + c));
          one[i] = __ldg(scale + (j0 + r) * scale_st);
        }
      } else {
        f[i] = r < n ? __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(src) + (j0 + r) * stride + c))
                     : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
    }
  }
  __device__ __forceinline__ void store(float* dst, int pitch) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int x = threadIdx.x + i * kThreads, r = x / (D / 4), c = (x % (D / 4)) * 4;
      float4 a;
      if constexpr (Q8) {
        const uint32_t u = w[i];
        a = make_float4(static_cast<float>(static_cast<int8_t>(u)) * one[i], static_cast<float>(static_cast<int8_t>(u >> 8)) * one[i],
                        static_cast<float>(static_cast<int8_t>(u >> 16)) * one[i],
                        static_cast<float>(static_cast<int8_t>(u >> 24)) * one[i]);
      } else {
        a = f[i];
      }
      *reinterpret_cast<float4*>(dst + r * pitch + c) = a;
    }
  }
};

// o += P V over the tile; PART: a key that is not seen, marked by p = -0, adds nothing, whatever its values
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
        for (int i = 0; i < 4; ++i) o[a][c] = __fmaf_rn(w[i], PART && __float_as_uint(w[i]) == kUnseen ? 0.0f : v[i], o[a][c]);
      }
    }
  }
}

template <int D, int RPT, bool Q8>
__global__ void __launch_bounds__(kThreads) tree_f32_kernel(const __grid_constant__ Params p) {
  using S = Smem<D, RPT>;
  constexpr int BM = S::kBM;
  constexpr int DC = D / 16;  // result columns a thread: tx + 16 c
  extern __shared__ float smem_raw[];
  S& sm = *reinterpret_cast<S*>(smem_raw);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int cta = static_cast<int>(blockIdx.x), rows = p.group * p.nodes;
  grid_wait();
  Walk walk(p, cta);
  while (walk.more()) {
  const Block blk = next_block(p, walk);
  const Seq sq = blk.sq;
  const int b = blk.b, kvh = blk.kvh, r0 = blk.mb * BM;
  const int i0 = blk.t0 * (kUnit / kBK), i1 = min(blk.t1 * (kUnit / kBK), (sq.len + kBK - 1) / kBK);

  const int64_t unit = Q8 ? 1 : 4;
  const char* kb = static_cast<const char*>(p.k) + (b * p.k_st[0] + kvh * p.k_st[1]) * unit;
  const char* vb = static_cast<const char*>(p.v) + (b * p.v_st[0] + kvh * p.v_st[1]) * unit;
  const float* ksb = Q8 ? p.ks + b * p.ks_st[0] + kvh * p.ks_st[1] : nullptr;
  const float* vsb = Q8 ? p.vs + b * p.vs_st[0] + kvh * p.vs_st[1] : nullptr;
  Part<D, Q8> pk, pv;
  const auto fetch = [&](int i) {
    const int j0 = i * kBK;
    pk.load(kb, p.k_st[2], ksb, p.ks_st[2], j0, sq.len - j0);
    pv.load(vb, p.v_st[2], vsb, p.vs_st[2], j0, sq.len - j0);
  };
  if (i0 < i1) fetch(i0);
  // the rows' queries, and what they see of the tree
  for (int x = threadIdx.x; x < BM * (D / 4); x += kThreads) {
    const int r = r0 + x / (D / 4), c = (x % (D / 4)) * 4;
    float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r < rows)
      f = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + b * p.q_st[0] +
                                                (kvh * p.group + r / p.nodes) * p.q_st[1] +
                                                (r % p.nodes) * p.q_st[2] + c));
    *reinterpret_cast<float4*>(&sm.q[x / (D / 4)][c]) = f;
  }
  if (i1 * kBK > sq.all) {
    load_parents(p, sq, b, sm.parent, kThreads);
    __syncthreads();
    if (threadIdx.x < BM)
      walk_up(sq, sm.parent, min(r0 + static_cast<int>(threadIdx.x), rows - 1) % p.nodes, sm.bits[threadIdx.x]);
  }
  float m[RPT], l[RPT], o[RPT][DC];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < DC; ++c) o[i][c] = 0.0f;
  }
  for (int i = i0; i < i1; ++i) {
    const int j0 = i * kBK;
    __syncthreads();
    pk.store(&sm.k[0][0], S::kPitch);
    pv.store(&sm.v[0][0], D);
    __syncthreads();
    if (i + 1 < i1) fetch(i + 1);
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
    const bool inside = j0 + kBK <= sq.all;
#pragma unroll
    for (int a = 0; a < RPT; ++a) {
      float mx = -INFINITY;
      bool seen[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        seen[c] = inside || sees(sq, sm.bits[ty * RPT + a], j0 + tx + 16 * c);
        const float s = x[a][c] * p.scale;
        x[a][c] = seen[c] ? s : -INFINITY;
        mx = (s != s && seen[c]) ? s : (mx != mx ? mx : fmaxf(mx, x[a][c]));
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
        sm.p[ty * RPT + a][tx + 16 * c] = seen[c] ? e : __uint_as_float(kUnseen);
      }
      l[a] = __fmaf_rn(l[a], alpha, row_sum(sum));
#pragma unroll
      for (int c = 0; c < DC; ++c) o[a][c] *= alpha;
    }
    __syncwarp();  // a row's 16 threads are of one warp
    if (inside) weigh<false>(sm, ty, tx, o);
    else weigh<true>(sm, ty, tx, o);
    __syncwarp();
  }
#pragma unroll
  for (int a = 0; a < RPT; ++a) {
    const int r = r0 + ty * RPT + a;
    if (r >= rows) continue;
    const int head = kvh * p.group + r / p.nodes, node = r % p.nodes;
    if (!blk.whole) {
      const int64_t to = part_row(p, cta, blk.slot, r - r0);
#pragma unroll
      for (int c = 0; c < DC; ++c) p.part_o[to * D + tx + 16 * c] = o[a][c];
      if (tx == 0) p.part_ml[to] = make_float2(m[a] * kLog2e, l[a]);
    } else {
      float* out = static_cast<float*>(p.o) + b * p.o_st[0] + head * p.o_st[1] + node * p.o_st[2];
      const float rl = l[a] == 0.0f ? 0.0f : __frcp_rn(l[a]);
#pragma unroll
      for (int c = 0; c < DC; ++c) out[tx + 16 * c] = node < sq.n ? o[a][c] * rl : 0.0f;
    }
  }
  __syncthreads();  // the next block's rows and parents go where this one's are read
  }
}

template <int D, int RPT, bool Q8>
int launch(const Params& p, cudaStream_t s) {
  constexpr int bytes = sizeof(Smem<D, RPT>);
  static OptIn opted;
  if (!opted.shared(tree_f32_kernel<D, RPT, Q8>, bytes)) return FPK_ERR_CUDA;
  return launch_dependent(tree_f32_kernel<D, RPT, Q8>, dim3(static_cast<unsigned>(p.ctas)), kThreads, bytes, s, p);
}
template <int D>
int launch_d(const Params& p, bool few, cudaStream_t s) {
  if (p.ks) return few ? launch<D, 1, true>(p, s) : launch<D, 4, true>(p, s);
  return few ? launch<D, 1, false>(p, s) : launch<D, 4, false>(p, s);
}

}  // namespace

int launch_f32(const Params& p, int D, bool few, cudaStream_t s) {
  switch (D) {
    case 16: return launch_d<16>(p, few, s);
    case 32: return launch_d<32>(p, few, s);
    case 64: return launch_d<64>(p, few, s);
    default: return launch_d<128>(p, few, s);
  }
}

}  // namespace tree
}  // namespace fpk
