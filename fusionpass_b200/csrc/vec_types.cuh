// f16 / bf16 / f32 element access for the row kernels: 16-byte vectors and single
// elements, converted to and from f32 (one rounding to nearest even at a store).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace fpk {

__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(float x) { return x; }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }

// two f32 packed into one 32-bit word of T (lower address first)
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// 16 bytes of T as f32
template <typename T>
__device__ __forceinline__ void raw_to_f32(const uint4& u, float* a) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      a[i] = __uint_as_float(w[i]);
    } else {
      const float2 f = unpack2<T>(w[i]);
      a[2 * i] = f.x;
      a[2 * i + 1] = f.y;
    }
  }
}

// VEC elements at p (VEC = 1, or 16 bytes' worth with p 16-byte aligned) as f32
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* a) {
  if constexpr (VEC == 1) {
    a[0] = to_f32(__ldg(p));
  } else if constexpr (sizeof(T) == 4) {
    static_assert(VEC == 4, "16-byte vectors");
    const float4 x = __ldg(reinterpret_cast<const float4*>(p));
    a[0] = x.x; a[1] = x.y; a[2] = x.z; a[3] = x.w;
  } else {
    static_assert(VEC == 8, "16-byte vectors");
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(w[i]);
      a[2 * i] = f.x;
      a[2 * i + 1] = f.y;
    }
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* a) {
  if constexpr (VEC == 1) {
    *p = from_f32<T>(a[0]);
  } else if constexpr (sizeof(T) == 4) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(a[0], a[1], a[2], a[3]));
  } else {
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(pack2<T>(a[0], a[1]), pack2<T>(a[2], a[3]), pack2<T>(a[4], a[5]),
                                                   pack2<T>(a[6], a[7])));
  }
}

}  // namespace fpk
