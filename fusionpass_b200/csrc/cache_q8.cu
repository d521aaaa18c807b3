// The 8-bit cache: rows of keys and values quantised as they are written, read back in the
// model's type, and the rows of an accepted branch moved up behind those that were there.
//
// All three only move bytes; what bounds them is the memory, and for a few rows the launch.
// A warp takes a unit of rows of one head of one tensor, several vectors of 16 bytes a thread
// asked for before the first is used.
#include <cuda_runtime.h>

#include <algorithm>

#include "internal.h"
#include "score_common.cuh"
#include "vec_types.cuh"

namespace fpk {
namespace cache {
namespace {

using score::grid_wait;
using score::launch_dependent;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;

struct Side {
  void* x;         // rows in the model's type
  void* cache;     // 8-bit rows
  float* scale;
  int64_t x_st[3], c_st[3], s_st[3];
};
struct Params {
  Side side[2];    // keys, values
  const int32_t* past;
  const int32_t* lens;
  int32_t batch, heads, rows, room;
};

// the warp's unit: side, sequence, head and first row (a block is of one head: no division)
struct Unit {
  int side, b, h, row;
};
__device__ __forceinline__ bool unit_of(const Params& p, int rows_a_unit, Unit* u) {
  u->side = static_cast<int>(blockIdx.x & 1u);
  u->row = ((blockIdx.x >> 1) * (blockDim.x >> 5) + (threadIdx.x >> 5)) * rows_a_unit;
  u->h = static_cast<int>(blockIdx.y);
  u->b = static_cast<int>(blockIdx.z);
  return u->row < p.rows;
}

// The nearest whole number to 127 x / top, |x| <= top, exactly; ties to even.  t = x * inv with
// inv = 127 / top rounded is off by at most two roundings of a value up to 127, 127 * 2^-23 < 1.6e-5:
// only next to the middle of two whole numbers can it lie on the wrong side (near), and there (exactly)
// 254 x is compared with (2 n + 1) top for the whole number n below, both exact in 64 bits (24 + 8 bits
// each).  Adding 1.5 * 2^23 rounds to a whole number, which the low byte of the sum then holds: a
// conversion to integer, at a quarter of the rate, and a branch an element took 42 us of [2, 8, 8192, 128] f16 under
// ncu, so 31 (0.82 of the issue slots).
constexpr float kWhole = 12582912.0f;
__device__ __forceinline__ float near_of(float x, float inv, uint32_t* low, float near) {
  const float t = __fmul_rn(x, inv), r = __fadd_rn(t, kWhole);
  *low = __float_as_uint(r);
  return fmaxf(near, fabsf(__fsub_rn(t, __fsub_rn(r, kWhole))));
}
__device__ __forceinline__ uint32_t exactly(float x, float inv, float top) {
  const float t = __fmul_rn(x, inv);
  const int a = __float2int_rd(t - 0.25f);  // the middle that is near is a + 1/2, if one is
  int n = __float2int_rn(t);
  if (fabsf(t - (static_cast<float>(a) + 0.5f)) < 0.01f) {
    const double d = 254.0 * static_cast<double>(x) - static_cast<double>(2 * a + 1) * static_cast<double>(top);
    n = d > 0.0 ? a + 1 : (d < 0.0 ? a : a + (a & 1));
  }
  return static_cast<uint32_t>(n);
}
// four low bytes
__device__ __forceinline__ uint32_t bytes_of(const uint32_t* b) {
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

// 8 elements a thread: 16 bytes of a 16-bit type, 32 of f32
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) write_kernel(const __grid_constant__ Params p) {
  constexpr int LANES = D / 8;           // of a row
  constexpr int ROWS = 32 / LANES;       // rows a warp holds at once
  constexpr int N = 4;                   // of which it asks for so many
  constexpr int WORDS = sizeof(T) / 2;   // 16-byte vectors
  Unit u;
  grid_wait();
  if (!unit_of(p, ROWS * N, &u)) return;
  const Side& s = p.side[u.side];
  const int lane = threadIdx.x & 31, c = (lane % LANES) * 8;
  const int fresh = p.lens ? min(max(__ldg(p.lens + u.b), 0), p.rows) : p.rows;
  const int64_t past = __ldg(p.past + u.b);
  const T* x = static_cast<const T*>(s.x) + u.b * s.x_st[0] + u.h * s.x_st[1] + c;
  int8_t* cache = static_cast<int8_t*>(s.cache) + u.b * s.c_st[0] + u.h * s.c_st[1] + c;
  float* scale = s.scale + u.b * s.s_st[0] + u.h * s.s_st[1];
  uint4 w[N][WORDS];
  bool in[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int row = u.row + i * ROWS + lane / LANES;
    const int64_t to = past + row;
    in[i] = row < fresh && to >= 0 && to < p.room;
#pragma unroll
    for (int k = 0; k < WORDS; ++k)
      w[i][k] = in[i] ? __ldg(reinterpret_cast<const uint4*>(x + row * s.x_st[2]) + k) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float f[8];
#pragma unroll
    for (int k = 0; k < WORDS; ++k) raw_to_f32<T>(w[i][k], f + k * (8 / WORDS));
    uint32_t top = 0u;  // magnitudes as the integer order of their bits: NaN > infinity > finite
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float t = __uint_as_float(top);
    const bool odd = top >= 0x7f800000u, none = t < 127.0f * 1.17549435e-38f;
    const float one = odd ? __uint_as_float(0x7fc00000u) : (none ? 0.0f : __fdiv_rn(t, 127.0f));
    const float inv = odd || none ? 0.0f : __fdiv_rn(127.0f, t);
    uint32_t b[8];
    float near = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) near = near_of(f[e], inv, &b[e], near);
    // inf * 0 and NaN * 0 are NaN: such a row's bytes are made zero below
    if (near > 0.4999f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = exactly(f[e], inv, t);
    }
    if (!in[i]) continue;
    const int64_t to = past + u.row + i * ROWS + lane / LANES;
    const uint32_t keep = odd || none ? 0u : 0xffffffffu;
    *reinterpret_cast<uint2*>(cache + to * s.c_st[2]) = make_uint2(bytes_of(b) & keep, bytes_of(b + 4) & keep);
    if (c == 0) scale[to * s.s_st[2]] = one;
  }
}

// 16 bytes of the result a thread
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ Params p) {
  constexpr int E = 16 / sizeof(T);      // elements a thread
  constexpr int LANES = D / E;
  constexpr int ROWS = 32 / LANES;
  constexpr int N = 4;
  Unit u;
  grid_wait();
  if (!unit_of(p, ROWS * N, &u)) return;
  const Side& s = p.side[u.side];
  const int lane = threadIdx.x & 31, c = (lane % LANES) * E;
  const int held = p.lens ? min(max(__ldg(p.lens + u.b), 0), p.rows) : p.rows;
  T* x = static_cast<T*>(s.x) + u.b * s.x_st[0] + u.h * s.x_st[1] + c;
  const int8_t* cache = static_cast<const int8_t*>(s.cache) + u.b * s.c_st[0] + u.h * s.c_st[1] + c;
  const float* scale = s.scale + u.b * s.s_st[0] + u.h * s.s_st[1];
  uint2 w[N];
  float one[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t row = u.row + i * ROWS + lane / LANES;
    w[i] = make_uint2(0u, 0u);
    one[i] = 0.0f;
    if (row < held) {
      if constexpr (E == 8) w[i] = __ldg(reinterpret_cast<const uint2*>(cache + row * s.c_st[2]));
      else w[i].x = __ldg(reinterpret_cast<const uint32_t*>(cache + row * s.c_st[2]));
      one[i] = __ldg(scale + row * s.s_st[2]);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t row = u.row + i * ROWS + lane / LANES;
    if (row >= p.rows) continue;
    float f[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
      // the byte with its sign bit flipped below 2^23, less 2^23 + 128: exact, without a conversion
      f[e] = (__uint_as_float(__byte_perm((e < 4 ? w[i].x : w[i].y) ^ 0x80808080u, 0x4b000000u, 0x7440 | (e & 3))) - 8388736.0f) *
             one[i];
    store_vec<T, E>(x + row * s.x_st[2], f);
  }
}

// ------------------------------------------------------------------ keep ---
struct Keep {
  fpk_keep_cache c[FPK_KEEP_MAX_CACHES];
  const int32_t *path, *counts, *past;
  int64_t path_stride;
  int32_t batch, n_path;
};
constexpr int kSlice = 128;  // bytes of a row that are moved at a time

template <typename U>
__device__ __forceinline__ void move_rows(char* base, int64_t st, int bytes, int n, const int* from, const int* to,
                                          char* room) {
  const int units = bytes / static_cast<int>(sizeof(U));
  for (int x = threadIdx.x; x < n * units; x += kThreads) {
    const int r = x / units, c = x % units;
    if (from[r] >= 0) reinterpret_cast<U*>(room)[x] = *reinterpret_cast<const U*>(base + from[r] * st + c * sizeof(U));
  }
  __syncthreads();
  for (int x = threadIdx.x; x < n * units; x += kThreads) {
    const int r = x / units, c = x % units;
    if (from[r] >= 0) *reinterpret_cast<U*>(base + to[r] * st + c * sizeof(U)) = reinterpret_cast<const U*>(room)[x];
  }
  __syncthreads();
}

__global__ void __launch_bounds__(kThreads) keep_kernel(const __grid_constant__ Keep p) {
  __shared__ __align__(16) char room[FPK_TREE_MAX_NODES * kSlice];
  __shared__ int from[FPK_TREE_MAX_NODES], to[FPK_TREE_MAX_NODES];
  const fpk_keep_cache& c = p.c[blockIdx.y];
  const int b = static_cast<int>(blockIdx.x % p.batch), h = static_cast<int>(blockIdx.x / p.batch);
  if (h >= c.heads) return;
  grid_wait();
  const int n = min(max(__ldg(p.counts + b), 0), p.n_path);
  const int64_t past = __ldg(p.past + b);
  for (int i = threadIdx.x; i < p.n_path; i += kThreads) {  // all of them: not behind the load of the count
    const int64_t step = __ldg(p.path + b * p.path_stride + i), a = past + step, z = past + i;
    // a row that stays where it is is not moved
    const bool ok = step >= 0 && step != i && a >= 0 && a < c.room && z >= 0 && z < c.room;
    from[i] = ok ? static_cast<int>(a) : -1;
    to[i] = static_cast<int>(z);
  }
  __syncthreads();
  char* base = static_cast<char*>(c.data) + b * c.strides[0] + h * c.strides[1];
  const uint64_t mis = reinterpret_cast<uintptr_t>(c.data) | static_cast<uint64_t>(c.strides[0]) |
                       static_cast<uint64_t>(c.strides[1]) | static_cast<uint64_t>(c.strides[2]) |
                       static_cast<uint64_t>(c.row_bytes);
  for (int at = 0; at < c.row_bytes; at += kSlice) {
    const int bytes = min(kSlice, c.row_bytes - at);
    if (mis % 16 == 0) move_rows<uint4>(base + at, c.strides[2], bytes, n, from, to, room);
    else if (mis % 4 == 0) move_rows<uint32_t>(base + at, c.strides[2], bytes, n, from, to, room);
    else if (mis % 2 == 0) move_rows<uint16_t>(base + at, c.strides[2], bytes, n, from, to, room);
    else move_rows<uint8_t>(base + at, c.strides[2], bytes, n, from, to, room);
  }
}

// ------------------------------------------------------------- host side ---
template <typename T, int D>
int launch(const Params& p, bool write, cudaStream_t s) {
  const int lanes = write ? D / 8 : D * static_cast<int>(sizeof(T)) / 16;
  const int rows = 32 / lanes * 4, units = (p.rows + rows - 1) / rows, warps = std::min(kWarps, units);
  const dim3 grid(2u * static_cast<unsigned>((units + warps - 1) / warps), static_cast<unsigned>(p.heads),
                  static_cast<unsigned>(p.batch));
  return write ? launch_dependent(write_kernel<T, D>, grid, 32 * warps, 0, s, p)
               : launch_dependent(read_kernel<T, D>, grid, 32 * warps, 0, s, p);
}
template <typename T>
int launch_t(const Params& p, int D, bool write, cudaStream_t s) {
  switch (D) {
    case 16: return launch<T, 16>(p, write, s);
    case 32: return launch<T, 32>(p, write, s);
    case 64: return launch<T, 64>(p, write, s);
    default: return launch<T, 128>(p, write, s);
  }
}

int check(const fpk_cache_desc* d) {
  if (!d || d->size != sizeof(fpk_cache_desc) || d->version != FPK_ABI_VERSION) return FPK_ERR_INVALID;
  if (d->dtype != FPK_F16 && d->dtype != FPK_BF16 && d->dtype != FPK_F32) return FPK_ERR_INVALID;
  if (d->batch < 0 || d->heads < 0 || d->rows < 0 || d->room < 0) return FPK_ERR_INVALID;
  if (d->head_dim != 16 && d->head_dim != 32 && d->head_dim != 64 && d->head_dim != 128) return FPK_ERR_UNSUPPORTED;
  if (d->batch > 65535 || d->heads > 65535 || d->rows > (1 << 30) || d->room > (1 << 30)) return FPK_ERR_UNSUPPORTED;
  return FPK_OK;
}

int run(const fpk_cache_desc* d, bool write, const void* k, const void* v, const void* kc, const void* vc,
        const float* ks, const float* vs, void* stream) {
  int rc = check(d);
  if (rc != FPK_OK) return rc;
  if (d->batch == 0 || d->heads == 0 || d->rows == 0 || (write && d->room == 0)) return FPK_OK;
  if (!k || !v || !kc || !vc || !ks || !vs || (write && !d->past_lens)) return FPK_ERR_INVALID;
  if (!write && d->rows != d->room) return FPK_ERR_INVALID;
  const uintptr_t at16 = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                         reinterpret_cast<uintptr_t>(kc) | reinterpret_cast<uintptr_t>(vc);
  const uintptr_t at4 = reinterpret_cast<uintptr_t>(ks) | reinterpret_cast<uintptr_t>(vs) |
                        reinterpret_cast<uintptr_t>(d->past_lens) | reinterpret_cast<uintptr_t>(d->lens);
  if (at16 % 16 || at4 % 4) return FPK_ERR_ALIGN;
  const int64_t unit = d->dtype == FPK_F32 ? 4 : 8;
  for (int i = 0; i < 3; ++i) {
    if (d->k_strides[i] % unit || d->v_strides[i] % unit) return FPK_ERR_ALIGN;
    if (d->k_cache_strides[i] % 16 || d->v_cache_strides[i] % 16) return FPK_ERR_ALIGN;
  }
  DeviceInfo dev;
  rc = current_device_info(&dev);
  if (rc != FPK_OK) return rc;
  Params p{};
  for (int i = 0; i < 2; ++i) {
    Side& s = p.side[i];
    s.x = const_cast<void*>(i ? v : k);
    s.cache = const_cast<void*>(i ? vc : kc);
    s.scale = const_cast<float*>(i ? vs : ks);
    for (int j = 0; j < 3; ++j) {
      s.x_st[j] = (i ? d->v_strides : d->k_strides)[j];
      s.c_st[j] = (i ? d->v_cache_strides : d->k_cache_strides)[j];
      s.s_st[j] = (i ? d->v_scale_strides : d->k_scale_strides)[j];
    }
  }
  p.past = d->past_lens;
  p.lens = d->lens;
  p.batch = static_cast<int32_t>(d->batch);
  p.heads = static_cast<int32_t>(d->heads);
  p.rows = static_cast<int32_t>(d->rows);
  p.room = static_cast<int32_t>(d->room);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->dtype == FPK_F16) return launch_t<__half>(p, d->head_dim, write, s);
  if (d->dtype == FPK_BF16) return launch_t<__nv_bfloat16>(p, d->head_dim, write, s);
  return launch_t<float>(p, d->head_dim, write, s);
}

int keep(const fpk_keep_desc* d, const fpk_keep_cache* caches, void* stream) {
  if (!d || d->size != sizeof(fpk_keep_desc) || d->version != FPK_ABI_VERSION) return FPK_ERR_INVALID;
  if (d->batch < 0 || d->n_caches < 0 || d->n_path < 0) return FPK_ERR_INVALID;
  if (d->n_caches > FPK_KEEP_MAX_CACHES || d->n_path > FPK_TREE_MAX_NODES) return FPK_ERR_UNSUPPORTED;
  if (d->batch == 0 || d->n_caches == 0 || d->n_path == 0) return FPK_OK;
  if (!caches || !d->path || !d->counts || !d->past_lens) return FPK_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(d->path) | reinterpret_cast<uintptr_t>(d->counts) |
       reinterpret_cast<uintptr_t>(d->past_lens)) % 4)
    return FPK_ERR_ALIGN;
  Keep p{};
  int64_t heads = 0;
  for (int i = 0; i < d->n_caches; ++i) {
    const fpk_keep_cache& c = caches[i];
    if (c.heads < 0 || c.room < 0 || c.row_bytes < 1) return FPK_ERR_INVALID;
    if (c.room > (1 << 30)) return FPK_ERR_UNSUPPORTED;
    if (c.heads > 0 && c.room > 0 && !c.data) return FPK_ERR_INVALID;
    p.c[i] = c;
    if (c.room == 0) p.c[i].heads = 0;
    heads = std::max<int64_t>(heads, p.c[i].heads);
  }
  if (heads == 0) return FPK_OK;
  if (heads > 0x7fffffffLL / d->batch) return FPK_ERR_UNSUPPORTED;
  p.path = d->path;
  p.counts = d->counts;
  p.past = d->past_lens;
  p.path_stride = d->path_stride;
  p.batch = static_cast<int32_t>(d->batch);
  p.n_path = d->n_path;
  DeviceInfo dev;
  const int rc = current_device_info(&dev);
  if (rc != FPK_OK) return rc;
  return launch_dependent(keep_kernel, dim3(static_cast<unsigned>(heads * d->batch), static_cast<unsigned>(d->n_caches)),
                          kThreads, 0, static_cast<cudaStream_t>(stream), p);
}

}  // namespace
}  // namespace cache
}  // namespace fpk

extern "C" {

int fpk_cache_write(const fpk_cache_desc* d, const void* k, const void* v, void* k_cache, void* v_cache,
                    float* k_scale, float* v_scale, void* stream) {
  return fpk::cache::run(d, true, k, v, k_cache, v_cache, k_scale, v_scale, stream);
}

int fpk_cache_read(const fpk_cache_desc* d, const void* k_cache, const void* v_cache, const float* k_scale,
                   const float* v_scale, void* k, void* v, void* stream) {
  return fpk::cache::run(d, false, k, v, k_cache, v_cache, k_scale, v_scale, stream);
}

int fpk_cache_keep(const fpk_keep_desc* d, const fpk_keep_cache* caches, void* stream) {
  return fpk::cache::keep(d, caches, stream);
}

}  // extern "C"
