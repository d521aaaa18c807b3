// Tree attention: the choice of kernel and of the parts that the keys are split into, the kernel
// that joins the parts, and the C entry points (include/fpkern.h).
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "internal.h"
#include "tree_common.cuh"
#include "vec_types.cuh"

namespace fpk {
namespace tree {
namespace {

// With many sequences each CTA, and each warp that joins rows, would add up all lengths anew: they are added up
// once, by one block.
constexpr int kManySequences = 256;
constexpr int kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads) tree_before_kernel(const __grid_constant__ Params p, int64_t* before) {
  __shared__ int64_t warp_sum[32];
  grid_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t run = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kSumThreads) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    const int64_t mine = b < p.batch ? units_of(seq_of(p, b)) : 0;
    int64_t upto = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += o;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int64_t ahead = run;
    for (int w = 0; w < warp; ++w) ahead += warp_sum[w];
    if (b < p.batch) before[b] = ahead + upto - mine;
    for (int w = 0; w < 32; ++w) run += warp_sum[w];
    __syncthreads();
  }
  if (threadIdx.x == 0) before[p.batch] = run;
}

// The rows of blocks that several CTAs share.  Bound by the latency of the chain lengths -> parts -> rows, so
// that a warp has several rows of a head, or several parts of one, on their way at once, and with
// many parts a row four warps have one row.  (us for 32768 rows of D 128 in two or three parts: a warp a row 30,
// so 14.)
// the CTAs that have a block's units
struct Parts {
  int first, n, head;  // CTA; how many; the first one's slot
  int row0;            // the block's first row (of its key/value head)
  __device__ __forceinline__ int64_t row(const Params& p, int s, int r) const {
    return part_row(p, first + s, s == 0 ? head : 0, r - row0);
  }
};
__device__ __forceinline__ Parts parts_of_row(const Params& p, int64_t total, int64_t before, int units, int kvh, int row) {
  const int mb = row / p.block_rows, ctas = ctas_of(p, total);
  const int64_t a0 = before + static_cast<int64_t>(kvh * p.mblocks + mb) * units;
  Parts x;
  x.first = cta_of(total, a0, ctas);
  x.n = cta_of(total, a0 + units - 1, ctas) - x.first + 1;
  // the first CTA's part is its last one, unless its part of the work begins with this block
  x.head = first_unit(total, x.first, ctas) < a0 ? 1 : 0;
  x.row0 = mb * p.block_rows;
  return x;
}
// all units, and those of the sequences before b; by a converged warp
__device__ __forceinline__ void units_around(const Params& p, int b, int64_t* total, int64_t* before) {
  if (p.before) {
    *total = p.before[p.batch] * p.per;
    *before = p.before[b] * p.per;
    return;
  }
  int64_t t = 0, f = 0;
  for (int i = threadIdx.x & 31; i < p.batch; i += 32) {
    const int64_t n = units_of(seq_of(p, i));
    t += n;
    if (i < b) f += n;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    t += __shfl_xor_sync(0xffffffffu, t, off);
    f += __shfl_xor_sync(0xffffffffu, f, off);
  }
  *total = t * p.per;
  *before = f * p.per;
}
template <typename T>
__device__ __forceinline__ void store4(const Params& p, int b, int h, int node, int n, int col, float4 a, float l) {
  const float rl = l == 0.0f ? 0.0f : __frcp_rn(l);
  a = node < n ? make_float4(a.x * rl, a.y * rl, a.z * rl, a.w * rl) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  T* out = static_cast<T*>(p.o) + b * p.o_st[0] + h * p.o_st[1] + node * p.o_st[2] + col;
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out) = a;
  else *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(a.x, a.y), pack2<T>(a.z, a.w));
}

// D / 4 lanes a row, 4 columns each, and with D < 128 more rows at once; RW such steps of rows a warp, S parts
// of each on their way
template <typename T, int D, int RW, int S>
__global__ void __launch_bounds__(128) tree_join_kernel(const __grid_constant__ Params p, int groups) {
  constexpr int kCols = D / 4, kAtOnce = 32 / kCols, kN = RW * kAtOnce;  // rows a warp
  grid_wait();
  const int lane = threadIdx.x & 31, col = lane % kCols * 4;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);  // (sequence, head, group of nodes)
  if (at >= static_cast<int64_t>(p.batch) * p.heads * groups) return;
  const int h = static_cast<int>(at / groups % p.heads), b = static_cast<int>(at / groups / p.heads);
  const int node0 = static_cast<int>(at % groups) * kN, row0 = h % p.group * p.nodes + node0;
  int64_t total, before;
  units_around(p, b, &total, &before);
  const Seq sq = seq_of(p, b);
  const int units = units_of(sq), rows = min(kN, p.nodes - node0);
  for (int r = 0; r < rows;) {  // the rows of one block, then those of the next
    const Parts x = parts_of_row(p, total, before, units, h / p.group, row0 + r);
    const int end = min(rows, x.row0 + p.block_rows - row0);
    if (x.n > 1) {  // else its CTA has written them
      float m[RW], l[RW];
      float4 a[RW];
#pragma unroll
      for (int i = 0; i < RW; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.0f;
        a[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      for (int s0 = 0; s0 < x.n; s0 += S) {
        float2 ml[S][RW];
        float4 o[S][RW];
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
          for (int i = 0; i < RW; ++i) {
            const int k = lane / kCols + i * kAtOnce;
            ml[s][i] = make_float2(-INFINITY, 0.0f);
            if (s0 + s < x.n && k >= r && k < end) {
              const int64_t from = x.row(p, s0 + s, row0 + k);
              ml[s][i] = p.part_ml[from];
              o[s][i] = *reinterpret_cast<const float4*>(p.part_o + from * D + col);
            }
          }
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
          for (int i = 0; i < RW; ++i) {
            const float2 v = ml[s][i];
            const bool none = v.x == -INFINITY && v.y == 0.0f;  // saw no key, whatever its row holds
            const float top = fmaxf(m[i], v.x), ref = top == -INFINITY ? 0.0f : top;
            const float f = ex2_approx(m[i] - ref), w = none ? 0.0f : ex2_approx(v.x - ref);
            m[i] = top;
            l[i] = __fmaf_rn(v.y, w, l[i] * f);  // a NaN stays, also where the weight is 0
            a[i] = make_float4(a[i].x * f, a[i].y * f, a[i].z * f, a[i].w * f);
            if (!none) {  // also where the weight is 0: what is not finite in a value that was seen stays so
              a[i].x = __fmaf_rn(o[s][i].x, w, a[i].x);
              a[i].y = __fmaf_rn(o[s][i].y, w, a[i].y);
              a[i].z = __fmaf_rn(o[s][i].z, w, a[i].z);
              a[i].w = __fmaf_rn(o[s][i].w, w, a[i].w);
            }
          }
      }
#pragma unroll
      for (int i = 0; i < RW; ++i) {
        const int k = lane / kCols + i * kAtOnce;
        if (k >= r && k < end) store4<T>(p, b, h, node0 + k, sq.n, col, a[i], l[i]);
      }
    }
    r = end;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(128) tree_combine_kernel(const __grid_constant__ Params p) {
  constexpr int kCols = D / 4, kSlots = 32 / kCols;  // lanes a part, parts at once
  __shared__ float4 s_o[4][32];
  grid_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int node = static_cast<int>(blockIdx.x % p.nodes), h = static_cast<int>(blockIdx.x / p.nodes % p.heads);
  const int b = static_cast<int>(blockIdx.x / p.nodes / p.heads);
  const int col = lane % kCols, slot = lane / kCols;
  int64_t total, before;
  units_around(p, b, &total, &before);
  const Seq sq = seq_of(p, b);
  const int row = h % p.group * p.nodes + node;
  const Parts x = parts_of_row(p, total, before, units_of(sq), h / p.group, row);
  const int parts = x.n;
  if (parts == 1) return;  // written by its CTA
  constexpr float2 kNone = {-INFINITY, 0.0f};
  const float2 own = lane < parts ? p.part_ml[x.row(p, lane, row)] : kNone;  // the first 32 parts', kept
  float m = own.x;
  for (int s = lane + 32; s < parts; s += 32) m = fmaxf(m, p.part_ml[x.row(p, s, row)].x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  const float ref = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int s0 = 0; s0 < parts; s0 += 32) {
    const float2 v = s0 == 0 ? own : (s0 + lane < parts ? p.part_ml[x.row(p, s0 + lane, row)] : kNone);
    // a part that saw no key is passed over (-1), whatever its row holds
    const float f = v.x == -INFINITY && v.y == 0.0f ? -1.0f : ex2_approx(v.x - ref);
    l = __fmaf_rn(v.y, f, l);  // a NaN stays, also where the weight is 0
    const int n = min(32, parts - s0);
#pragma unroll 4
    for (int s = warp * kSlots; s < n; s += 4 * kSlots) {  // the same for the warp
      const int mine = s + slot;
      const float w = __shfl_sync(0xffffffffu, f, mine & 31);
      if (mine < n && !(w < 0.0f)) {
        const float4 o = *reinterpret_cast<const float4*>(p.part_o + x.row(p, s0 + mine, row) * D + col * 4);
        a.x = __fmaf_rn(o.x, w, a.x);
        a.y = __fmaf_rn(o.y, w, a.y);
        a.z = __fmaf_rn(o.z, w, a.z);
        a.w = __fmaf_rn(o.w, w, a.w);
      }
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
#pragma unroll
  for (int off = kCols; off < 32; off <<= 1) {
    a.x += __shfl_xor_sync(0xffffffffu, a.x, off);
    a.y += __shfl_xor_sync(0xffffffffu, a.y, off);
    a.z += __shfl_xor_sync(0xffffffffu, a.z, off);
    a.w += __shfl_xor_sync(0xffffffffu, a.w, off);
  }
  s_o[warp][lane] = a;
  __syncthreads();
  if (warp != 0 || slot != 0) return;
#pragma unroll
  for (int k = 1; k < 4; ++k) {
    const float4 o = s_o[k][lane];
    a.x += o.x;
    a.y += o.y;
    a.z += o.z;
    a.w += o.w;
  }
  store4<T>(p, b, h, node, sq.n, col * 4, a, l);
}

template <typename T, int D, int RW, int S>
int join(const Params& p, cudaStream_t s) {
  constexpr int kN = RW * (128 / D);
  const int groups = (p.nodes + kN - 1) / kN;
  const int64_t warps = static_cast<int64_t>(p.batch) * p.heads * groups;
  return launch_dependent(tree_join_kernel<T, D, RW, S>, dim3(static_cast<unsigned>((warps + 3) / 4)), 128, 0, s, p, groups);
}
template <typename T, int D>
int combine(const Params& p, cudaStream_t s) {
  const int64_t parts = (p.ctas + static_cast<int64_t>(p.batch) * p.per - 1) / (static_cast<int64_t>(p.batch) * p.per);  // a row, about
  if (parts <= 3) return join<T, D, 4, 2>(p, s);
  if (parts <= 8) return join<T, D, 1, 8>(p, s);
  const int64_t rows = static_cast<int64_t>(p.batch) * p.heads * p.nodes;
  return launch_dependent(tree_combine_kernel<T, D>, dim3(static_cast<unsigned>(rows)), 128, 0, s, p);
}
template <typename T>
int combine_t(const Params& p, int D, cudaStream_t s) {
  switch (D) {
    case 16: return combine<T, 16>(p, s);
    case 32: return combine<T, 32>(p, s);
    case 64: return combine<T, 64>(p, s);
    default: return combine<T, 128>(p, s);
  }
}

int64_t up(int64_t x) { return (x + 255) / 256 * 256; }

// Rows that mma.sync's kernel takes, 16 a block.  us on tcgen05 / mma.sync, heads 32 over 8, 24 rows, 32, 48:
//   1 x 2048    D 128 8-bit f16 16/14 17/15 17/23, bf16 16/15 17/15 17/17, 16-bit 15.5/15.8 15.8/16.0 16/19
//               D 64 8-bit 14/12 14/12 14/13, 16-bit 14/12 14/12 14/14;  D 32 12/10 12/10 13/11;  D 16 12/9 12/9 12/10
//   1 x 16384   D 128 8-bit f16 34/32 34/33 35/52, bf16 36/35 36/37 36/45, 16-bit 30/34 31/36 31/42
//               D 64 8-bit 27/23 27/24 28/29, 16-bit 25/23 26/23 26/28;  D 32 24/18 24/19 25/23;  D 16 22/17 22/17 23/21
//   16 x 4096   D 128 8-bit f16 78/64 73/68 79/117, bf16 82/68 79/73 84/97, 16-bit 66/70 70/80 67/97
//               D 64 8-bit 57/45 56/44 58/62, 16-bit 49/39 53/40 50/53;  D 32 52/36 49/34 49/49;  D 16 44/31 46/31 48/45
int64_t dec_rows(const fpk_tree_desc* d) { return d->head_dim == 128 && !(d->flags & FPK_TREE_Q8) ? 16 : 32; }

struct Plan {
  enum Kind { kDec, kTc, kF32 } kind;
  bool few;
  Params p;
  int64_t ml_at, before_at, bytes;
};

int make_plan(const fpk_tree_desc* d, const DeviceInfo& dev, Plan* out) {
  Plan& pl = *out;
  Params& p = pl.p;
  p = Params{};
  const int sms = dev.num_sms > 0 ? dev.num_sms : 148;
  const int64_t group = d->heads / d->kv_heads, rows = group * d->nodes, bh = d->batch * d->kv_heads;
  if (d->batch * d->heads > 0x7fffffffLL / d->nodes) return FPK_ERR_UNSUPPORTED;
  if (rows > 0x7fff0000LL) return FPK_ERR_UNSUPPORTED;
  p.batch = static_cast<int32_t>(d->batch);
  p.heads = static_cast<int32_t>(d->heads);
  p.kv_heads = static_cast<int32_t>(d->kv_heads);
  p.group = static_cast<int32_t>(group);
  p.nodes = static_cast<int32_t>(d->nodes);
  p.room = static_cast<int32_t>(d->room);
  p.scale = d->scale;
  p.scale_log2 = d->scale * kLog2e;
  p.ks = d->flags & FPK_TREE_Q8 ? d->k_scale : nullptr;
  p.vs = d->flags & FPK_TREE_Q8 ? d->v_scale : nullptr;
  p.parents = d->parents;
  p.parents_st = d->parents_stride;
  p.past = d->past_lens;
  p.lens = d->tree_lens;
  for (int i = 0; i < 3; ++i) {
    p.q_st[i] = d->q_strides[i];
    p.k_st[i] = d->k_strides[i];
    p.v_st[i] = d->v_strides[i];
    p.o_st[i] = d->o_strides[i];
    p.ks_st[i] = d->k_scale_strides[i];
    p.vs_st[i] = d->v_scale_strides[i];
  }
  p.status = dev.status;
  int64_t slots;  // CTAs that run at once
  if (d->dtype == FPK_F32) {
    pl.kind = Plan::kF32;
    pl.few = bh * ((rows + 63) / 64) < sms;
    p.block_rows = pl.few ? 16 : 64;
    slots = 2 * sms;
  } else if (rows <= dec_rows(d)) {
    pl.kind = Plan::kDec;
    p.block_rows = 16;
    // What registers and shared memory leave room for; with one more an SM its CTAs wait for a place.  us with 2 / 3
    // an SM, heads 32 over 8, 24 ragged caches of 8192 and 1 of 32768:
    //   D 128  1 row a head (4 a block): 8-bit f16 68/88 24/33, bf16 76/99 25/35, 16-bit 108/110 35/42;
    //          4: 8-bit f16 84/109 30/44, bf16 107/94 35/38, 16-bit 119/131 38/51
    //   D 64   1: 8-bit 49/45 18/19, 16-bit 59/59 18/20;  4: 8-bit 71/60 23/25, 16-bit 64/71 22/25
    //   D 32   1: 8-bit 38/33 15/16, 16-bit 38/38 15/16;  4: 8-bit 59/48 20/20, 16-bit 49/41 18/19
    //   D 16   1: 8-bit 32/28 13/14, 16-bit 33/29 14/14;  4: 8-bit 53/43 18/17, 16-bit 40/33 16/16
    const bool bf16_rows = p.ks && d->dtype == FPK_BF16 && rows > 8;  // the one form of D 128 with 168 registers or less
    slots = sms * (d->head_dim == 128 && !bf16_rows ? 2 : 3);
  } else {
    pl.kind = Plan::kTc;
    p.by_rows = rows > 128;
    p.block_rows = p.by_rows ? 256 : 128;
    slots = sms;
  }
  p.mblocks = static_cast<int32_t>((rows + p.block_rows - 1) / p.block_rows);
  if (static_cast<int64_t>(d->kv_heads) * p.mblocks > 0x7fffffffLL) return FPK_ERR_UNSUPPORTED;
  p.per = static_cast<int32_t>(d->kv_heads * p.mblocks);
  // all CTAs that run at once, where each gets a unit at least (by the room: lengths are not known here)
  const int64_t units = std::max<int64_t>(1, (d->room + kUnit - 1) / kUnit);
  if (units > (1LL << 48) / p.per / d->batch) return FPK_ERR_UNSUPPORTED;
  p.ctas = static_cast<int32_t>(std::min(slots, bh * p.mblocks * units));
  const int64_t parts = static_cast<int64_t>(p.ctas) * 2 * p.block_rows;
  pl.ml_at = up(parts * d->head_dim * 4);
  pl.before_at = pl.ml_at + up(parts * 8);
  pl.bytes = pl.before_at + (p.batch > kManySequences ? up((p.batch + 1LL) * 8) : 0);
  return FPK_OK;
}

int check(const fpk_tree_desc* d) {
  if (!d || d->size != sizeof(fpk_tree_desc) || d->version != FPK_ABI_VERSION) return FPK_ERR_INVALID;
  if (d->dtype != FPK_F16 && d->dtype != FPK_BF16 && d->dtype != FPK_F32) return FPK_ERR_INVALID;
  if (d->flags & ~FPK_TREE_Q8) return FPK_ERR_INVALID;
  if (d->batch < 0 || d->heads < 0 || d->nodes < 0 || d->room < 0) return FPK_ERR_INVALID;
  if (d->heads > 0 && (d->kv_heads < 1 || d->heads % d->kv_heads)) return FPK_ERR_INVALID;
  if (!std::isfinite(d->scale)) return FPK_ERR_INVALID;
  if (!std::isfinite(d->scale * kLog2e)) return FPK_ERR_UNSUPPORTED;
  if (d->head_dim != 16 && d->head_dim != 32 && d->head_dim != 64 && d->head_dim != 128) return FPK_ERR_UNSUPPORTED;
  if (d->nodes > FPK_TREE_MAX_NODES || d->room > (1 << 30) || d->batch > 65535 || d->heads > (1 << 30))
    return FPK_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(d->parents) | reinterpret_cast<uintptr_t>(d->past_lens) |
       reinterpret_cast<uintptr_t>(d->tree_lens) | reinterpret_cast<uintptr_t>(d->k_scale) |
       reinterpret_cast<uintptr_t>(d->v_scale)) % 4)
    return FPK_ERR_ALIGN;
  return FPK_OK;
}
bool nothing(const fpk_tree_desc* d) { return d->batch == 0 || d->heads == 0 || d->nodes == 0; }

int run(const fpk_tree_desc* d, const void* q, const void* k, const void* v, void* o, void* ws, int64_t ws_bytes,
        cudaStream_t s, const DeviceInfo& dev) {
  Plan pl;
  int rc = make_plan(d, dev, &pl);
  if (rc != FPK_OK) return rc;
  if (ws_bytes < pl.bytes || (pl.bytes > 0 && (!ws || reinterpret_cast<uintptr_t>(ws) % 16))) return FPK_ERR_INVALID;
  Params& p = pl.p;
  p.q = q;
  p.k = k ? k : q;  // a cache without rows: never read
  p.v = v ? v : q;
  p.o = o;
  if (pl.bytes > 0) {
    p.part_o = static_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + pl.ml_at);
  }
  if (p.batch > kManySequences) {
    int64_t* before = reinterpret_cast<int64_t*>(static_cast<char*>(ws) + pl.before_at);
    rc = launch_dependent(tree_before_kernel, dim3(1), kSumThreads, 0, s, p, before);
    if (rc != FPK_OK) return rc;
    p.before = before;
  }
  if (pl.kind == Plan::kF32) rc = launch_f32(p, d->head_dim, pl.few, s);
  else if (pl.kind == Plan::kDec) rc = launch_dec(p, d->dtype, d->head_dim, s);
  else rc = d->dtype == FPK_F16 ? launch_tc_f16(p, d->head_dim, s) : launch_tc_bf16(p, d->head_dim, s);
  if (rc != FPK_OK || p.ctas == 1) return rc;
  if (d->dtype == FPK_F16) return combine_t<__half>(p, d->head_dim, s);
  if (d->dtype == FPK_BF16) return combine_t<__nv_bfloat16>(p, d->head_dim, s);
  return combine_t<float>(p, d->head_dim, s);
}

}  // namespace
}  // namespace tree
}  // namespace fpk

extern "C" {

int64_t fpk_tree_attention_workspace(const fpk_tree_desc* d) {
  int rc = fpk::tree::check(d);
  if (rc != FPK_OK) return rc;
  if (fpk::tree::nothing(d)) return 0;
  fpk::DeviceInfo dev;
  rc = fpk::current_device_info(&dev);
  if (rc != FPK_OK) return rc;
  fpk::tree::Plan pl;
  rc = fpk::tree::make_plan(d, dev, &pl);
  return rc == FPK_OK ? pl.bytes : rc;
}

int fpk_tree_attention_fwd(const fpk_tree_desc* d, const void* q, const void* k, const void* v, void* o,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = fpk::tree::check(d);
  if (rc != FPK_OK) return rc;
  if (fpk::tree::nothing(d)) return FPK_OK;
  const bool q8 = d->flags & FPK_TREE_Q8;
  if (!q || !o || !d->parents || !d->past_lens || (d->room > 0 && (!k || !v || (q8 && (!d->k_scale || !d->v_scale)))))
    return FPK_ERR_INVALID;
  const uintptr_t mis = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                        reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(o);
  if (mis % 16) return FPK_ERR_ALIGN;
  const int64_t unit = d->dtype == FPK_F32 ? 4 : 8, kv_unit = q8 ? 16 : unit;  // elements in 16 bytes
  for (int i = 0; i < 3; ++i) {
    if (d->q_strides[i] <= 0 || d->q_strides[i] % unit || d->o_strides[i] <= 0 || d->o_strides[i] % unit) return FPK_ERR_ALIGN;
    if (d->k_strides[i] <= 0 || d->k_strides[i] % kv_unit || d->v_strides[i] <= 0 || d->v_strides[i] % kv_unit) return FPK_ERR_ALIGN;
    if (q8 && (d->k_scale_strides[i] <= 0 || d->v_scale_strides[i] <= 0)) return FPK_ERR_INVALID;
  }
  fpk::DeviceInfo dev;
  rc = fpk::current_device_info(&dev);
  if (rc != FPK_OK) return rc;
  return fpk::tree::run(d, q, k, v, o, workspace, workspace_bytes, static_cast<cudaStream_t>(stream), dev);
}

}  // extern "C"
