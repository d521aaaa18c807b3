// Host side of score attention: argument checks, the choice of the kernel and of how many
// CTAs share the keys of one, the workspace, and the two small kernels around the others
// (ranges of document ids per key tile before, joining the parts after).
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "internal.h"
#include "score_common.cuh"
#include "vec_types.cuh"

namespace fpk {
namespace score {

int launch_tc_f16(const Params& p, int D, cudaStream_t s);
int launch_tc_bf16(const Params& p, int D, cudaStream_t s);
int launch_dec(const Params& p, int dtype, int D, cudaStream_t s);
int launch_f32(const Params& p, int D, bool few, cudaStream_t s);

namespace {

// smallest and largest document id of each 128 keys, and whether they are all one
__global__ void __launch_bounds__(128) id_range_kernel(const int32_t* ids, int64_t stride, int k_len, int k_tiles,
                                                       IdRange* out) {
  grid_wait();
  const int tile = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = tile * kKeyTile + threadIdx.x;
  const int id = j < k_len ? __ldg(ids + b * stride + j) : -1;
  __shared__ int s_lo[4], s_hi[4], s_none[4];
  const int lo = __reduce_min_sync(0xffffffffu, id >= 0 ? id : 0x7fffffff);
  const int hi = __reduce_max_sync(0xffffffffu, id >= 0 ? id : -1);
  const int none = __any_sync(0xffffffffu, j < k_len && id < 0);
  if (lane == 0) {
    s_lo[warp] = lo;
    s_hi[warp] = hi;
    s_none[warp] = none;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    IdRange r{0x7fffffff, -1, 1};
    for (int w = 0; w < 4; ++w) {
      r.lo = min(r.lo, s_lo[w]);
      r.hi = max(r.hi, s_hi[w]);
      if (s_none[w]) r.same = 0;
    }
    if (r.lo != r.hi) r.same = 0;
    out[static_cast<int64_t>(b) * k_tiles + tile] = r;
  }
}

// o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s over the parts of a row, a block a row.  A
// thread holds 4 columns of every (512 / D)-th part; the maximum and the sum of the weights
// are taken a part a lane.  Parts that saw no key (m = -inf, l = 0) are skipped; with no parts
// at all the row is zero.  (A thread for all parts of 4 columns took 20 us at 64 parts of one
// token's 32 heads, as long as the attention itself.)
template <typename T, int D>
__global__ void __launch_bounds__(128) score_combine_kernel(const __grid_constant__ Params p) {
  constexpr int kCols = D / 4, kSlots = 128 / kCols;
  __shared__ float4 s_o[128];
  grid_wait();
  const int64_t row = blockIdx.x;
  const int col = threadIdx.x % kCols, slot = threadIdx.x / kCols, lane = threadIdx.x & 31;
  const float2* ml = p.part_ml + row * p.splits;
  float m = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, ml[s].x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  const float ref = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  for (int s = lane; s < p.splits; s += 32) {
    const float2 v = ml[s];
    if (!(v.x == -INFINITY && v.y == 0.0f)) l = __fmaf_rn(v.y, ex2_approx(v.x - ref), l);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
  float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int s = slot; s < p.splits; s += kSlots) {
    const float2 v = ml[s];
    const float4 o = *reinterpret_cast<const float4*>(p.part_o + (row * p.splits + s) * D + col * 4);
    if (v.x == -INFINITY && v.y == 0.0f) continue;
    const float f = ex2_approx(v.x - ref);
    a.x = __fmaf_rn(o.x, f, a.x);
    a.y = __fmaf_rn(o.y, f, a.y);
    a.z = __fmaf_rn(o.z, f, a.z);
    a.w = __fmaf_rn(o.w, f, a.w);
  }
  s_o[threadIdx.x] = a;
  __syncthreads();
  if (slot != 0) return;
  for (int k = 1; k < kSlots; ++k) {
    const float4 o = s_o[k * kCols + col];
    a.x += o.x;
    a.y += o.y;
    a.z += o.z;
    a.w += o.w;
  }
  const float rl = l == 0.0f ? 0.0f : __frcp_rn(l);
  const int qi = static_cast<int>(row % p.q_len), h = static_cast<int>(row / p.q_len % p.heads);
  const int64_t b = row / p.q_len / p.heads;
  T* out = static_cast<T*>(p.o) + b * p.o_st[0] + h * p.o_st[1] + qi * p.o_st[2] + col * 4;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(out) = make_float4(a.x * rl, a.y * rl, a.z * rl, a.w * rl);
  } else {
    *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(a.x * rl, a.y * rl), pack2<T>(a.z * rl, a.w * rl));
  }
}

template <typename T, int D>
int combine(const Params& p, cudaStream_t s) {
  const int64_t blocks = static_cast<int64_t>(p.batch) * p.heads * p.q_len;
  if (blocks > 0x7fffffffLL) return FPK_ERR_UNSUPPORTED;
  return launch_dependent(score_combine_kernel<T, D>, dim3(static_cast<unsigned>(blocks)), 128, 0, s, p);
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

struct Plan {
  enum Kind { kTc, kDec, kF32, kZero } kind;
  bool few;
  Params p;
  int64_t ranges_at, part_at, ml_at, bytes;
};

// Key tiles that a query block of `queries` rows walks at most
int64_t most_tiles(const fpk_score_desc* d, int64_t queries) {
  int64_t n = d->k_len;
  if (d->window > 0 && !d->prefix_lens) {
    const int64_t wide = queries + (d->flags & FPK_SCORE_CAUSAL ? 1 : 2) * std::min(d->window, n) + 2 * kKeyTile;
    n = std::min(n, wide + std::min(d->prefix, n));
  }
  return (n + kKeyTile - 1) / kKeyTile;
}

int make_plan(const fpk_score_desc* d, const DeviceInfo& dev, Plan* out) {
  Plan& pl = *out;
  Params& p = pl.p;
  p = Params{};
  const int sms = dev.num_sms > 0 ? dev.num_sms : 148;
  const int64_t group = d->heads / d->kv_heads;
  p.batch = static_cast<int32_t>(d->batch);
  p.heads = static_cast<int32_t>(d->heads);
  p.kv_heads = static_cast<int32_t>(d->kv_heads);
  p.group = static_cast<int32_t>(group);
  p.q_len = static_cast<int32_t>(d->q_len);
  p.k_len = static_cast<int32_t>(d->k_len);
  p.k_tiles = static_cast<int32_t>((d->k_len + kKeyTile - 1) / kKeyTile);
  p.causal = d->flags & FPK_SCORE_CAUSAL ? 1 : 0;
  p.window = static_cast<int32_t>(std::min<int64_t>(d->window, 1 << 30));
  p.prefix = static_cast<int32_t>(std::min<int64_t>(d->prefix, 1 << 30));
  p.scale = d->scale;
  p.scale_log2 = d->scale * 1.4426950408889634f;
  p.cap = d->softcap;
  p.slopes = d->slopes;
  p.prefixes = d->prefix_lens;
  p.ids = d->doc_ids;
  p.ids_stride = d->ids_stride;
  p.lens = d->kv_lens;
  for (int i = 0; i < 3; ++i) {
    p.q_st[i] = d->q_strides[i];
    p.k_st[i] = d->k_strides[i];
    p.v_st[i] = d->v_strides[i];
    p.o_st[i] = d->o_strides[i];
  }
  p.status = dev.status;
  p.mblocks = 1;
  int64_t items, splits = 1;
  const int64_t rows = group * d->q_len;
  if (d->k_len == 0) {
    pl.kind = Plan::kZero;
    items = 0;
    splits = 0;
  } else if (d->dtype == FPK_F32) {
    pl.kind = Plan::kF32;
    if (rows > 0x7fff0000LL) return FPK_ERR_UNSUPPORTED;
    // blocks of 64 rows when they fill the SMs, of 16 when they do not: a quarter of the work in
    // each step of a chain that latency bounds (2 x 6 heads over 3, 77 queries, 130 keys, D 32: 29 us in
    // blocks of 64, 11 in blocks of 16, with the next tile fetched ahead in the latter)
    pl.few = d->batch * d->kv_heads * ((rows + 63) / 64) < sms;
    const int64_t bm = pl.few ? 16 : 64;
    p.mblocks = static_cast<int32_t>((rows + bm - 1) / bm);
    items = d->batch * d->kv_heads * p.mblocks;
    if (items < sms) splits = std::min<int64_t>(2 * sms / items, most_tiles(d, std::min(d->q_len, bm)) / 2);
  } else if (rows <= 16) {
    // two CTAs an SM are resident; the least number of parts with the least time, in key tiles:
    // rounds of CTAs times the tiles of a part and one for starting and joining it.  (f16, D 128, 32
    // heads over 8, us: 24 x 8192 keys in 4 / 3 parts 153.9 / 134.8; 1 x 8192 in 64 / 37 30.4 / 16.0.)
    pl.kind = Plan::kDec;
    items = d->batch * d->kv_heads;
    const int64_t slots = 2 * sms, tiles = most_tiles(d, d->q_len);
    int64_t least = INT64_MAX;
    for (int64_t n = 1; n <= std::min<int64_t>(tiles, 128); ++n) {
      const int64_t t = (items * n + slots - 1) / slots * ((tiles + n - 1) / n + 1);
      if (t < least) {
        least = t;
        splits = n;
      }
    }
  } else {
    pl.kind = Plan::kTc;
    const int64_t q_tiles = d->head_dim == 128 ? 2 : 1;  // of a CTA, and with one tile two CTAs an SM
    const int64_t bm = q_tiles * kKeyTile;
    p.pair_heads = q_tiles == 2 && d->q_len <= kKeyTile && group % 2 == 0 ? 1 : 0;
    p.mblocks = p.pair_heads ? 1 : static_cast<int32_t>((d->q_len + bm - 1) / bm);
    items = d->batch * (p.pair_heads ? d->heads / 2 : d->heads) * p.mblocks;
    // fewer blocks than run at once: several CTAs share a block's keys, four key tiles each at least
    const int64_t slots = q_tiles == 2 ? sms : 2 * sms;
    if (items < slots) splits = std::min<int64_t>(slots / items, most_tiles(d, std::min(d->q_len, bm)) / 4);
  }
  if (pl.kind != Plan::kZero) splits = std::max<int64_t>(splits, 1);
  if (items > 0x7fffffffLL / std::max<int64_t>(splits, 1)) return FPK_ERR_UNSUPPORTED;
  p.items = static_cast<int32_t>(items);
  p.splits = static_cast<int32_t>(splits);
  int64_t at = 0;
  pl.ranges_at = at;
  if (d->doc_ids && pl.kind != Plan::kF32) at += up(d->batch * p.k_tiles * static_cast<int64_t>(sizeof(IdRange)));
  const int64_t parts = splits > 1 ? d->batch * d->heads * d->q_len * splits : 0;
  pl.part_at = at;
  at += up(parts * d->head_dim * 4);
  pl.ml_at = at;
  at += up(parts * 8);
  pl.bytes = at;
  return FPK_OK;
}

int check(const fpk_score_desc* d) {
  if (!d || d->size != sizeof(fpk_score_desc) || d->version != FPK_ABI_VERSION) return FPK_ERR_INVALID;
  if (d->dtype != FPK_F16 && d->dtype != FPK_BF16 && d->dtype != FPK_F32) return FPK_ERR_INVALID;
  if ((d->flags & ~FPK_SCORE_CAUSAL) || d->reserved != 0) return FPK_ERR_INVALID;
  if (d->batch < 0 || d->heads < 0 || d->q_len < 0 || d->k_len < 0 || d->window < 0 || d->prefix < 0)
    return FPK_ERR_INVALID;
  if (d->heads > 0 && (d->kv_heads < 1 || d->heads % d->kv_heads)) return FPK_ERR_INVALID;
  if (!std::isfinite(d->scale) || !std::isfinite(d->softcap) || d->softcap < 0.0f) return FPK_ERR_INVALID;
  // the factors of a score must be finite in f32: infinity times a score of 0 is NaN
  if (!std::isfinite(d->scale * 1.4426950408889634f) ||
      (d->softcap > 0.0f && !std::isfinite(2.8853900817779268f * d->scale / d->softcap)))
    return FPK_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(d->slopes) | reinterpret_cast<uintptr_t>(d->prefix_lens) |
       reinterpret_cast<uintptr_t>(d->doc_ids) | reinterpret_cast<uintptr_t>(d->kv_lens)) % 4)
    return FPK_ERR_ALIGN;
  if (d->head_dim != 16 && d->head_dim != 32 && d->head_dim != 64 && d->head_dim != 128) return FPK_ERR_UNSUPPORTED;
  if (d->softcap > FPK_SCORE_MAX_CAP && d->dtype != FPK_F32) return FPK_ERR_UNSUPPORTED;
  if (d->q_len > (1 << 30) || d->k_len > (1 << 30) || d->batch > 65535 || d->heads > (1 << 30)) return FPK_ERR_UNSUPPORTED;
  return FPK_OK;
}

}  // namespace

int64_t workspace(const fpk_score_desc* d, const DeviceInfo& dev) {
  Plan pl;
  const int rc = make_plan(d, dev, &pl);
  return rc == FPK_OK ? pl.bytes : rc;
}

int run(const fpk_score_desc* d, const void* q, const void* k, const void* v, void* o, void* ws, int64_t ws_bytes,
        cudaStream_t s, const DeviceInfo& dev) {
  Plan pl;
  int rc = make_plan(d, dev, &pl);
  if (rc != FPK_OK) return rc;
  if (ws_bytes < pl.bytes || (pl.bytes > 0 && (!ws || reinterpret_cast<uintptr_t>(ws) % 16))) return FPK_ERR_INVALID;
  Params& p = pl.p;
  p.q = q;
  p.k = k;
  p.v = v;
  p.o = o;
  char* w = static_cast<char*>(ws);
  if (pl.bytes > 0) {
    p.part_o = reinterpret_cast<float*>(w + pl.part_at);
    p.part_ml = reinterpret_cast<float2*>(w + pl.ml_at);
  }
  if (p.ids && pl.kind != Plan::kF32 && pl.kind != Plan::kZero) {
    IdRange* r = reinterpret_cast<IdRange*>(w + pl.ranges_at);
    p.ranges = r;
    rc = launch_dependent(id_range_kernel, dim3(p.k_tiles, p.batch), 128, 0, s, p.ids, p.ids_stride, p.k_len, p.k_tiles, r);
    if (rc != FPK_OK) return rc;
  }
  if (pl.kind == Plan::kF32) rc = launch_f32(p, d->head_dim, pl.few, s);
  else if (pl.kind == Plan::kDec) rc = launch_dec(p, d->dtype, d->head_dim, s);
  else if (pl.kind == Plan::kTc)
    rc = d->dtype == FPK_F16 ? launch_tc_f16(p, d->head_dim, s) : launch_tc_bf16(p, d->head_dim, s);
  if (rc != FPK_OK || p.splits == 1) return rc;
  if (d->dtype == FPK_F16) return combine_t<__half>(p, d->head_dim, s);
  if (d->dtype == FPK_BF16) return combine_t<__nv_bfloat16>(p, d->head_dim, s);
  return combine_t<float>(p, d->head_dim, s);
}

}  // namespace score
}  // namespace fpk

extern "C" {

int64_t fpk_score_attention_workspace(const fpk_score_desc* d) {
  int rc = fpk::score::check(d);
  if (rc != FPK_OK) return rc;
  if (d->batch == 0 || d->heads == 0 || d->q_len == 0) return 0;
  fpk::DeviceInfo dev;
  rc = fpk::current_device_info(&dev);
  return rc == FPK_OK ? fpk::score::workspace(d, dev) : rc;
}

int fpk_score_attention_fwd(const fpk_score_desc* d, const void* q, const void* k, const void* v, void* o,
                            void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = fpk::score::check(d);
  if (rc != FPK_OK) return rc;
  if (d->batch == 0 || d->heads == 0 || d->q_len == 0) return FPK_OK;
  if (!q || !o || (d->k_len > 0 && (!k || !v))) return FPK_ERR_INVALID;
  const int64_t unit = d->dtype == FPK_F32 ? 4 : 8;  // elements in 16 bytes
  uintptr_t mis = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                  reinterpret_cast<uintptr_t>(o);
  if (mis % 16) return FPK_ERR_ALIGN;
  for (const int64_t* st : {d->q_strides, d->k_strides, d->v_strides, d->o_strides})
    for (int i = 0; i < 3; ++i)
      if (st[i] <= 0 || st[i] % unit) return FPK_ERR_ALIGN;
  fpk::DeviceInfo dev;
  rc = fpk::current_device_info(&dev);
  if (rc != FPK_OK) return rc;
  return fpk::score::run(d, q, k, v, o, workspace, workspace_bytes, static_cast<cudaStream_t>(stream), dev);
}

}  // extern "C"
