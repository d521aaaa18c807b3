// Root-mean-square norm of a sum of addends over the last axis, its output in the
// input's type or in 8 bits with one scale a row; and that 8-bit form alone.
//
//   s = a_0 + a_1 + ...            f32, in the given order (a residual and a branch)
//   y = s * r * w,  r = 1 / sqrt(mean(s^2) + eps)
//   q = rint(y / scale),  scale = max|y| / 127          (8-bit output)
//
// Every row is read once and held in registers as f32, so the bound is the bytes of
// the addends, the kept sum and the output.  Since r is one factor for the whole row it
// drops out of q: q = rint(s w * 127 / max|s w|) and scale = r * max|s w| / 127.  The sum
// of squares and the maximum are therefore reduced together, with one block barrier
// instead of two in a row.  A row whose s w holds an infinity or a NaN gets the scale NaN
// and zeros, so that what is computed from it is NaN; a row whose largest |s w| is below
// 127 times the smallest normal number counts as zero (scale 0).
#include <cuda_runtime.h>

#include "../../include/fpkern.h"
#include "internal.h"
#include "vec_types.cuh"

namespace fpk {
namespace rms {

constexpr int kMaxThreads = 1024;

struct Args {
  const void* a[4];
  uint32_t col_mask;  // bit i: addend i is per column
  int n;
  const void* w;      // null: ones
  void* sum;          // null: not kept
  void* y;            // null: 8-bit output
  int8_t* q;
  float* scale;
  int64_t rows;
  int64_t q_stride;
  int cols;
  float eps;
  int norm;           // 0: r = 1 (quantise only)
};

// largest magnitude as the integer order of its bits: NaN > infinity > finite, so neither is lost
__device__ __forceinline__ uint32_t mag(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct Red {
  float ss;
  uint32_t top;
};

__device__ __forceinline__ Red warp_red(Red v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v.ss += __shfl_xor_sync(0xffffffffu, v.ss, off);
  v.top = __reduce_max_sync(0xffffffffu, v.top);
  return v;
}

// over the threads of one row: a warp (ONE_WARP) or the block
template <bool ONE_WARP>
__device__ __forceinline__ Red row_red(Red v) {
  v = warp_red(v);
  if constexpr (!ONE_WARP) {
    __shared__ float s_ss[32];
    __shared__ uint32_t s_top[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    if (lane == 0) {
      s_ss[warp] = v.ss;
      s_top[warp] = v.top;
    }
    __syncthreads();
    v.ss = lane < nw ? s_ss[lane] : 0.0f;
    v.top = lane < nw ? s_top[lane] : 0u;
    v = warp_red(v);  // every warp sums the same values in the same order
  }
  return v;
}

template <typename T, int VEC>
__device__ __forceinline__ void load_sum(const Args& a, int64_t row_off, int col, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // constant indices keep the pointers in registers
    if (i < a.n) {
      float t[VEC];
      const T* base = static_cast<const T*>(a.a[i]);
      load_vec<T, VEC>((a.col_mask >> i) & 1u ? base + col : base + row_off + col, t);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = i == 0 ? t[e] : __fadd_rn(v[e], t[e]);
    }
  }
}

// the row's factors: y = s w * r;  q = rint(s w * inv)
struct Factors {
  float r, scale, inv;
};
__device__ __forceinline__ Factors factors(const Args& a, Red t) {
  Factors f;
  f.r = a.norm ? __frsqrt_rn(__fadd_rn(__fdiv_rn(t.ss, static_cast<float>(a.cols)), a.eps)) : 1.0f;
  const float top = __uint_as_float(t.top);
  if (t.top >= 0x7f800000u) {
    f.scale = __uint_as_float(0x7fc00000u);
    f.inv = 0.0f;
  } else if (top < 127.0f * 1.17549435e-38f) {
    f.scale = 0.0f;
    f.inv = 0.0f;
  } else {
    f.scale = __fdiv_rn(__fmul_rn(f.r, top), 127.0f);
    f.inv = __fdiv_rn(127.0f, top);
  }
  return f;
}

template <int VEC>
__device__ __forceinline__ void store_q(int8_t* p, const float* sw, float inv) {
  int b[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    // |s w * inv| <= 127 (1 + 2^-23): rounds to 127 at most; inf * 0 and NaN * 0 convert to 0
    b[e] = __float2int_rn(__fmul_rn(sw[e], inv));
  }
  if constexpr (VEC == 1) {
    *p = static_cast<int8_t>(b[0]);
  } else {
    uint32_t u[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i)
      u[i] = (b[4 * i] & 0xff) | (b[4 * i + 1] & 0xff) << 8 | (b[4 * i + 2] & 0xff) << 16 | b[4 * i + 3] << 24;
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
    else *reinterpret_cast<uint32_t*>(p) = u[0];
  }
}

// One row a block (ONE_WARP: one row a warp), at most VPT vectors a thread.
template <typename T, int VEC, int VPT, bool ONE_WARP>
__global__ void __launch_bounds__(ONE_WARP ? 128 : kMaxThreads) rms_kernel(const Args a) {
  const int tid = ONE_WARP ? threadIdx.x & 31 : threadIdx.x;
  const int tpr = ONE_WARP ? 32 : blockDim.x;
  const int64_t row = ONE_WARP ? static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.rows) return;  // whole warps of one row leave together
  const int nv = a.cols / VEC;
  const int64_t off = row * a.cols;
  float v[VPT * VEC];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int c = k * tpr + tid;
    if (c < nv) {
      load_sum<T, VEC>(a, off, c * VEC, v + k * VEC);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[k * VEC + e] = 0.0f;
    }
  }
  Red t{0.0f, 0u};
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int c = k * tpr + tid;
    if (c >= nv) continue;
    if (a.sum) store_vec<T, VEC>(static_cast<T*>(a.sum) + off + c * VEC, v + k * VEC);
    float w[VEC];
    if (a.w) load_vec<T, VEC>(static_cast<const T*>(a.w) + c * VEC, w);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float& s = v[k * VEC + e];
      t.ss = __fmaf_rn(s, s, t.ss);
      if (a.w && a.q) s = __fmul_rn(s, w[e]);
      t.top = max(t.top, mag(s));
    }
  }
  t = row_red<ONE_WARP>(t);
  const Factors f = factors(a, t);
  if (a.q) {
    if (tid == 0) a.scale[row] = f.scale;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = k * tpr + tid;
      if (c < nv) store_q<VEC>(a.q + row * a.q_stride + c * VEC, v + k * VEC, f.inv);
    }
  } else {
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = k * tpr + tid;
      if (c >= nv) continue;
      float w[VEC], o[VEC];
      if (a.w) load_vec<T, VEC>(static_cast<const T*>(a.w) + c * VEC, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        o[e] = __fmul_rn(v[k * VEC + e], f.r);
        if (a.w) o[e] = __fmul_rn(o[e], w[e]);
      }
      store_vec<T, VEC>(static_cast<T*>(a.y) + off + c * VEC, o);
    }
  }
}

// Rows too long for the registers of one block: the addends are read again (from L2)
// for the output.
template <typename T, int VEC>
__global__ void __launch_bounds__(kMaxThreads) rms_long_kernel(const Args a) {
  const int64_t row = blockIdx.x;
  const int nv = a.cols / VEC;
  const int64_t off = row * a.cols;
  Red t{0.0f, 0u};
  for (int c = threadIdx.x; c < nv; c += blockDim.x) {
    float v[VEC], w[VEC];
    load_sum<T, VEC>(a, off, c * VEC, v);
    if (a.sum) store_vec<T, VEC>(static_cast<T*>(a.sum) + off + c * VEC, v);
    if (a.w && a.q) load_vec<T, VEC>(static_cast<const T*>(a.w) + c * VEC, w);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      t.ss = __fmaf_rn(v[e], v[e], t.ss);
      t.top = max(t.top, mag(a.w && a.q ? __fmul_rn(v[e], w[e]) : v[e]));
    }
  }
  t = row_red<false>(t);
  const Factors f = factors(a, t);
  if (a.q && threadIdx.x == 0) a.scale[row] = f.scale;
  for (int c = threadIdx.x; c < nv; c += blockDim.x) {
    float v[VEC], w[VEC];
    load_sum<T, VEC>(a, off, c * VEC, v);
    if (a.w) load_vec<T, VEC>(static_cast<const T*>(a.w) + c * VEC, w);
    if (a.q) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (a.w) v[e] = __fmul_rn(v[e], w[e]);
      store_q<VEC>(a.q + row * a.q_stride + c * VEC, v, f.inv);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[e] = __fmul_rn(v[e], f.r);
        if (a.w) v[e] = __fmul_rn(v[e], w[e]);
      }
      store_vec<T, VEC>(static_cast<T*>(a.y) + off + c * VEC, v);
    }
  }
}

template <typename T, int VEC>
static int launch_vec(const Args& a, cudaStream_t s) {
  const int nv = a.cols / VEC;
  if (nv <= 64) {
    const int64_t grid = (a.rows + 3) / 4;
    if (grid > 0x7fffffffLL) return FPK_ERR_UNSUPPORTED;
    if (nv <= 32) rms_kernel<T, VEC, 1, true><<<static_cast<unsigned>(grid), 128, 0, s>>>(a);
    else rms_kernel<T, VEC, 2, true><<<static_cast<unsigned>(grid), 128, 0, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? FPK_OK : FPK_ERR_CUDA;
  }
  if (a.rows > 0x7fffffffLL) return FPK_ERR_UNSUPPORTED;
  const unsigned grid = static_cast<unsigned>(a.rows);
  const auto threads = [&](int vpt) { return (((nv + vpt - 1) / vpt + 31) / 32) * 32; };
  if (threads(1) <= 256) rms_kernel<T, VEC, 1, false><<<grid, threads(1), 0, s>>>(a);
  else if (threads(2) <= 512) rms_kernel<T, VEC, 2, false><<<grid, threads(2), 0, s>>>(a);
  else if (threads(4) <= kMaxThreads) rms_kernel<T, VEC, 4, false><<<grid, threads(4), 0, s>>>(a);
  else rms_long_kernel<T, VEC><<<grid, kMaxThreads, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? FPK_OK : FPK_ERR_CUDA;
}

template <typename T>
static int launch_t(const Args& a, bool vec, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  return vec ? launch_vec<T, V>(a, s) : launch_vec<T, 1>(a, s);
}

}  // namespace rms

int launch_rms_norm(const fpk_rms_desc* d, const void* const* addends, const int32_t* bcast, int n_addends,
                    const void* w, void* sum, void* y, int8_t* q, float* scale, cudaStream_t stream) {
  using namespace rms;
  Args a{};
  const int esize = d->dtype == FPK_F32 ? 4 : 2;
  uintptr_t mis = reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(sum) | reinterpret_cast<uintptr_t>(y);
  for (int i = 0; i < n_addends; ++i) {
    a.a[i] = addends[i];
    if (bcast[i] == FPK_BCAST_COL) a.col_mask |= 1u << i;
    mis |= reinterpret_cast<uintptr_t>(addends[i]);
  }
  a.n = n_addends;
  a.w = w;
  a.sum = sum;
  a.y = y;
  a.q = q;
  a.scale = scale;
  a.rows = d->rows;
  a.cols = static_cast<int>(d->cols);
  a.q_stride = d->q_stride;
  a.eps = d->eps;
  a.norm = (d->flags & FPK_RMS_QUANT_ONLY) ? 0 : 1;
  // 16-byte vectors need every row of every buffer on a 16-byte boundary (8 for q)
  const bool vec = mis % 16 == 0 && (d->cols * esize) % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0 &&
                   (!q || d->q_stride % 8 == 0);
  if (d->dtype == FPK_F16) return launch_t<__half>(a, vec, stream);
  if (d->dtype == FPK_BF16) return launch_t<__nv_bfloat16>(a, vec, stream);
  return launch_t<float>(a, vec, stream);
}

}  // namespace fpk
