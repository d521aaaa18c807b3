// What the score attention kernels share: the call's parameters, which keys a query sees,
// and how a score becomes the exponent of the softmax.
//
// Query i of sequence b stands at position p = len_b - q_len + i, so the queries are the
// last ones of the len_b keys.  It sees key j when
//
//   j < len_b  and  (j < prefix_b  or  (causal: j <= p) and (window w: |p - j| < w))
//   and, with document ids, id_b[p] == id_b[j] >= 0 (a position below 0 has no document).
//
// Without the ids that is the union of two intervals, [0, pre) and [lo, hi), which is what
// the kernels carry for each row; keys outside of both are never read when they fill a
// tile.  Lengths and prefixes come from device memory and are clamped to the buffers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <atomic>
#include <cstring>

#include "common.cuh"

namespace fpk {
namespace score {

constexpr int kKeyTile = 128;  // keys a tile, and a document range

// smallest and largest id >= 0 of a tile's keys; same: all of them one id >= 0
struct alignas(16) IdRange {
  int lo, hi, same;
};

struct Params {
  int* status;
  const float* slopes;       // [heads] or null
  const int32_t* prefixes;   // [batch] or null
  const int32_t* ids;        // [batch, k_len], rows ids_stride apart, or null
  const int32_t* lens;       // [batch] or null
  const IdRange* ranges;     // [batch, k_tiles] of ids
  float* part_o;             // [rows][splits][D] unnormalised partial results
  float2* part_ml;           // [rows][splits] (running maximum, sum)
  int64_t ids_stride;
  int64_t q_st[3], k_st[3], v_st[3], o_st[3];
  const void *q, *k, *v;
  void* o;
  int32_t batch, heads, kv_heads, group, q_len, k_len, k_tiles;
  int32_t causal, window, prefix;  // window 0: none
  int32_t splits;
  int32_t items;
  int32_t mblocks;
  int32_t pair_heads;
  float scale;
  float scale_log2;          // scale * log2(e)
  float cap;                 // 0: none
};

struct Seq {
  int len;   // keys of this sequence
  int base;  // position of query 0
  int pre;   // keys that every query sees
};
__device__ __forceinline__ Seq seq_of(const Params& p, int b) {
  Seq s;
  s.len = p.lens ? min(max(__ldg(p.lens + b), 0), p.k_len) : p.k_len;
  s.base = s.len - p.q_len;
  s.pre = min(max(p.prefixes ? __ldg(p.prefixes + b) : p.prefix, 0), s.len);
  return s;
}

struct Span {
  int lo, hi;
};
__device__ __forceinline__ Span span_of(const Params& p, const Seq& s, int pos) {
  Span r{0, s.len};
  if (p.window) {
    r.lo = max(0, pos - p.window + 1);
    r.hi = min(r.hi, max(0, pos + p.window));
  }
  if (p.causal) r.hi = min(r.hi, max(0, pos + 1));
  r.hi = max(r.hi, 0);
  return r;
}

// id of the document at a position; -1: none
__device__ __forceinline__ int id_at(const Params& p, int b, int pos, int len) {
  return pos >= 0 && pos < len ? __ldg(p.ids + b * p.ids_stride + pos) : -1;
}

// stream order towards the kernel before (programmatic dependent launch): what stands ahead of
// this, barriers and TMEM, may run while that kernel finishes
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A kernel's opt-in to more than 48 KB of shared memory, made once a device.
struct OptIn {
  std::atomic<int> done[64];
  template <typename K>
  bool shared(K kern, int bytes) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (done[dev].load(std::memory_order_acquire)) return true;
    if (bytes > 48 * 1024 &&
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return false;
    done[dev].store(1, std::memory_order_release);
    return true;
  }
};

// launch as a programmatic dependent of the stream's previous kernel
template <typename K, typename... A>
inline int launch_dependent(K kern, dim3 grid, int threads, int smem, cudaStream_t s, const A&... args) {
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? FPK_OK : FPK_ERR_CUDA;
}

// bits of [lo, hi) that fall on the 32 keys from j0
__device__ __forceinline__ uint32_t span_bits(int lo, int hi, int j0) {
  const int a = max(lo - j0, 0), b = min(hi - j0, 32);
  if (a >= b) return 0u;
  return (b >= 32 ? 0xffffffffu : (1u << b) - 1u) & ~((1u << a) - 1u);
}

// The key tiles that rows with positions [first, last] need, as a list: 0 .. n - 1 maps to
// the prefix's tiles, then to those of [lo, hi).
struct Tiles {
  int pre, from, n;
  __device__ __forceinline__ int at(int i) const { return i < pre ? i : from + (i - pre); }
};
__device__ __forceinline__ Tiles tiles_of(const Params& p, const Seq& s, int first, int last) {
  const int lo = span_of(p, s, first).lo, hi = span_of(p, s, last).hi;
  Tiles t;
  t.pre = (s.pre + kKeyTile - 1) / kKeyTile;
  t.from = max(lo / kKeyTile, t.pre);
  const int to = hi > lo ? (hi + kKeyTile - 1) / kKeyTile : 0;
  t.n = t.pre + max(to - t.from, 0);
  return t;
}

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 - 2 / (1 + e^(2x)): e^(2x) to infinity gives 1, to zero -1, NaN stays NaN.  The error is
// absolute, also near zero, where the difference cancels: in steps of 2^-24, 6 by the sum and its
// reciprocal, 2 by the ex2, 1.8 by its argument and 1 at the end, 6.5e-7 at most.
__device__ __forceinline__ float tanh_ex2(float x) {
  return __fmaf_rn(-2.0f, rcp_approx(1.0f + ex2_approx(2.8853900817779268f * x)), 1.0f);
}

}  // namespace score
}  // namespace fpk
