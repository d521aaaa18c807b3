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

#include <algorithm>
#include <atomic>
#include <cstring>

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

// stream order towards the kernel before (programmatic dependent launch)
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

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
  grid_wait();
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

// Many rows: a resident grid whose threads ask for their next row before they reduce and
// store the one in hand, so that the loads never stop.  TPR threads a row, VPT 16-byte
// vectors a thread, NA full addends held as raw vectors (in flight: 16 VPT NA bytes a
// thread).  bf16 [16384, 4096], two addends, sum and 8 bits: 98.7 us with a block a row
// (4.8 TB/s), 83.5 us so (5.6 TB/s).  Of the splits of a row, four vectors a thread with as
// few threads as hold it was best or within 2 % for rows of 256 to 8192 (on rows of zeros,
// 4096: 128 threads x 4 78.3 us, 256 x 2 81.4; 1024: 32 x 4 77.9, 64 x 2 81.2, 128 x 1 91.9).
//
// VEC = 1: rows that are not all on 16 bytes, an element at a time (a warp reads 32 neighbours).
// Vectors from the boundary before the row, with the ends and the weights by element, took twice
// the time: f32 1500 x 2049 8.5 us against 5.5, f16 8000 x 1001 20.1 against 13.4.  At most ten
// elements a thread, while they last: sixteen of two addends do not fit the 64 registers that a
// thread of 1024 has (13104 x 5121 f16, one addend 352 us with sixteen, 168 with ten; two 712 and
// 239; a block a row 346 and 428).
constexpr int kStreamThreads = 256;
// Blocks an SM that the registers are cut for: two where a block barrier holds a row's warps up
// (16384 x 4096 88.5 -> 83.5 us); warps of their own, and element rows, do better with what the
// compiler takes (65536 x 1024 83.6 against 91.4).
constexpr int stream_blocks(int tpr, int vec) { return vec > 1 && tpr >= 64 && tpr <= kStreamThreads ? 2 : 0; }

// VEC elements as they lie in memory: 16 bytes, or one
template <typename T, int VEC>
struct Raw {
  using type = uint4;
  static __device__ __forceinline__ void f32(const uint4& u, float* f) { raw_to_f32<T>(u, f); }
};
template <typename T>
struct Raw<T, 1> {
  using type = T;
  static __device__ __forceinline__ void f32(const T& u, float* f) { *f = to_f32(u); }
};

template <typename T, int VEC, int VPT, int NA, int TPR>
__global__ void __launch_bounds__(TPR > kStreamThreads ? TPR : kStreamThreads, stream_blocks(TPR, VEC))
    rms_stream_kernel(const Args a) {
  using R = Raw<T, VEC>;
  using U = typename R::type;
  constexpr int kThreads = TPR > kStreamThreads ? TPR : kStreamThreads;
  constexpr int kRows = kThreads / TPR;  // rows a block has in hand
  constexpr int kWarps = TPR / 32;       // a row
  __shared__ float s_ss[2][kThreads / 32];
  __shared__ uint32_t s_top[2][kThreads / 32];
  grid_wait();
  const int group = threadIdx.x / TPR, tid = threadIdx.x % TPR;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  U w[VPT], raw[NA][VPT];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int c = k * TPR + tid;
    w[k] = a.w && c * VEC < a.cols ? __ldg(static_cast<const U*>(a.w) + c) : U{};
  }
  const auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const T* p = static_cast<const T*>(a.a[i]) + row * a.cols;
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int e0 = (k * TPR + tid) * VEC;
        raw[i][k] = U{};
        if (e0 + VEC <= a.cols) raw[i][k] = __ldcs(reinterpret_cast<const U*>(p + e0));
      }
    }
  };
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + group;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  if (row < a.rows) fetch(row);
  for (uint32_t turn = 0; row < a.rows; row += step, turn ^= 1u) {
    float v[VPT * VEC];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      R::f32(raw[0][k], v + k * VEC);
#pragma unroll
      for (int i = 1; i < NA; ++i) {
        float t[VEC];
        R::f32(raw[i][k], t);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[k * VEC + e] = __fadd_rn(v[k * VEC + e], t[e]);
      }
    }
    if (row + step < a.rows) fetch(row + step);
    Red t{0.0f, 0u};
    const int64_t off = row * a.cols;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int e0 = (k * TPR + tid) * VEC;
      if (a.sum && e0 + VEC <= a.cols) store_vec<T, VEC>(static_cast<T*>(a.sum) + off + e0, v + k * VEC);
      float wf[VEC];
      if (a.w && a.q) R::f32(w[k], wf);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {  // beyond the row the vectors are zeros
        float& s = v[k * VEC + e];
        t.ss = __fmaf_rn(s, s, t.ss);
        if (a.w && a.q) s = __fmul_rn(s, wf[e]);
        t.top = max(t.top, mag(s));
      }
    }
    t = warp_red(t);
    if constexpr (kWarps > 1) {
      // by turns in two sets of slots: the next row's barrier lies between a read and the next write
      if (lane == 0) {
        s_ss[turn][warp] = t.ss;
        s_top[turn][warp] = t.top;
      }
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(TPR) : "memory");
      const int at = group * kWarps + (lane < kWarps ? lane : 0);
      t.ss = lane < kWarps ? s_ss[turn][at] : 0.0f;
      t.top = s_top[turn][at];
      t = warp_red(t);
    }
    const Factors f = factors(a, t);
    if (a.q && tid == 0) a.scale[row] = f.scale;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int e0 = (k * TPR + tid) * VEC;
      if (a.q) {
        int8_t* q = a.q + row * a.q_stride;
        if (e0 < a.cols) store_q<VEC>(q + e0, v + k * VEC, f.inv);
      } else {
        float wf[VEC], o[VEC];
        if (a.w) R::f32(w[k], wf);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          o[e] = __fmul_rn(v[k * VEC + e], f.r);
          if (a.w) o[e] = __fmul_rn(o[e], wf[e]);
        }
        if (e0 + VEC <= a.cols) store_vec<T, VEC>(static_cast<T*>(a.y) + off + e0, o);
      }
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
  grid_wait();
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

// programmatic dependent launch: every kernel here waits for the stream's previous kernel
// before its first access
template <typename K>
static int launch_k(K kern, int64_t grid, int threads, const Args& a, cudaStream_t s) {
  if (grid > 0x7fffffffLL) return FPK_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a) == cudaSuccess ? FPK_OK : FPK_ERR_CUDA;
}

template <typename T, int VEC, int VPT, int NA, int TPR>
static int launch_stream(const Args& a, int num_sms, cudaStream_t s) {
  constexpr int kThreads = TPR > kStreamThreads ? TPR : kStreamThreads;
  auto kern = rms_stream_kernel<T, VEC, VPT, NA, TPR>;
  static std::atomic<int> resident{0};  // blocks an SM
  int per = resident.load(std::memory_order_relaxed);
  if (per == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, kThreads, 0) != cudaSuccess || per < 1) return FPK_ERR_CUDA;
    resident.store(per, std::memory_order_relaxed);
  }
  const int64_t blocks = (a.rows + kThreads / TPR - 1) / (kThreads / TPR);
  return launch_k(kern, std::min<int64_t>(blocks, static_cast<int64_t>(num_sms) * per), kThreads, a, s);
}
template <typename T, int NA>
static int launch_rows(const Args& a, int num_sms, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int nv = a.cols / V;
  if (nv <= 32) return launch_stream<T, V, 1, NA, 32>(a, num_sms, s);
  if (nv <= 64) return launch_stream<T, V, 2, NA, 32>(a, num_sms, s);
  if (nv <= 96) return launch_stream<T, V, 3, NA, 32>(a, num_sms, s);
  if (nv <= 128) return launch_stream<T, V, 4, NA, 32>(a, num_sms, s);
  if (nv <= 192) return launch_stream<T, V, 3, NA, 64>(a, num_sms, s);
  if (nv <= 256) return launch_stream<T, V, 4, NA, 64>(a, num_sms, s);
  if (nv <= 384) return launch_stream<T, V, 3, NA, 128>(a, num_sms, s);
  if (nv <= 512) return launch_stream<T, V, 4, NA, 128>(a, num_sms, s);
  if (nv <= 768) return launch_stream<T, V, 3, NA, 256>(a, num_sms, s);
  if (nv <= 1024) return launch_stream<T, V, 4, NA, 256>(a, num_sms, s);
  return launch_stream<T, V, 4, NA, 512>(a, num_sms, s);
}
template <typename T, int NA>
static int launch_elements(const Args& a, int num_sms, cudaStream_t s) {
  const int n = a.cols;
  if (n <= 4 * 32) return launch_stream<T, 1, 4, NA, 32>(a, num_sms, s);
  if (n <= 10 * 32) return launch_stream<T, 1, 10, NA, 32>(a, num_sms, s);
  if (n <= 10 * 64) return launch_stream<T, 1, 10, NA, 64>(a, num_sms, s);
  if (n <= 10 * 128) return launch_stream<T, 1, 10, NA, 128>(a, num_sms, s);
  if (n <= 10 * 256) return launch_stream<T, 1, 10, NA, 256>(a, num_sms, s);
  if (n <= 10 * 512) return launch_stream<T, 1, 10, NA, 512>(a, num_sms, s);
  if (n <= 10 * 1024) return launch_stream<T, 1, 10, NA, 1024>(a, num_sms, s);
  return launch_stream<T, 1, 16, NA, 1024>(a, num_sms, s);
}

template <typename T, int VEC>
static int launch_vec(const Args& a, cudaStream_t s) {
  const int nv = a.cols / VEC;
  if (nv <= 32) return launch_k(rms_kernel<T, VEC, 1, true>, (a.rows + 3) / 4, 128, a, s);
  if (nv <= 64) return launch_k(rms_kernel<T, VEC, 2, true>, (a.rows + 3) / 4, 128, a, s);
  const auto threads = [&](int vpt) { return (((nv + vpt - 1) / vpt + 31) / 32) * 32; };
  if (threads(1) <= 512) return launch_k(rms_kernel<T, VEC, 1, false>, a.rows, threads(1), a, s);
  if (threads(2) <= kMaxThreads) return launch_k(rms_kernel<T, VEC, 2, false>, a.rows, threads(2), a, s);
  if (threads(4) <= kMaxThreads) return launch_k(rms_kernel<T, VEC, 4, false>, a.rows, threads(4), a, s);
  return launch_k(rms_long_kernel<T, VEC>, a.rows, kMaxThreads, a, s);
}

// Which form: the streaming one for 1 or 2 full addends whose rows fit it (2048 vectors, 16384
// elements; of two f32 addends 10240, since with sixteen elements a thread their registers spill:
// 2718 x 12345 178 us against 157 a block a row, in f16 312 against 384), when there are more rows than SMs (with fewer there is no next row to ask for, and
// a row spread over more threads is done sooner); else a block (or warp) a row with the row in
// registers; else, beyond 4096 vectors, rows read twice.
template <typename T>
static int launch_t(const Args& a, bool vec, int num_sms, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int most = vec ? 2048 * V : sizeof(T) == 4 && a.n == 2 ? 10240 : 16384;
  if (a.rows > num_sms && a.col_mask == 0 && a.n <= 2 && a.cols <= most) {
    if (vec) return a.n == 1 ? launch_rows<T, 1>(a, num_sms, s) : launch_rows<T, 2>(a, num_sms, s);
    return a.n == 1 ? launch_elements<T, 1>(a, num_sms, s) : launch_elements<T, 2>(a, num_sms, s);
  }
  return vec ? launch_vec<T, V>(a, s) : launch_vec<T, 1>(a, s);
}

}  // namespace rms

int launch_rms_norm(const fpk_rms_desc* d, const void* const* addends, const int32_t* bcast, int n_addends,
                    const void* w, void* sum, void* y, int8_t* q, float* scale, int num_sms, cudaStream_t stream) {
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
  if (d->dtype == FPK_F16) return launch_t<__half>(a, vec, num_sms, stream);
  if (d->dtype == FPK_BF16) return launch_t<__nv_bfloat16>(a, vec, num_sms, stream);
  return launch_t<float>(a, vec, num_sms, stream);
}

}  // namespace fpk
