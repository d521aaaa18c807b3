// The matrix instruction of a warp and what feeds it from shared memory, for the kernels that
// have too few rows for the 5th-generation tensor cores.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

namespace fpk {

// c += a b: 16 x 16 by 16 x 8, f32 sums
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
// 16 bytes, zeros where !in (nothing is read then)
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
// sign bits of the 16-bit halves of u that are not finite
template <typename T>
__device__ __forceinline__ uint32_t bad_bits(uint32_t u) {
  constexpr bool kHalfT = std::is_same<T, __half>::value;
  return ((u & (kHalfT ? 0x7c007c00u : 0x7f807f80u)) + (kHalfT ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}
// the largest among the four threads of a quad; a NaN among them is kept
__device__ __forceinline__ float quad_max(float v) {
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, v, off);
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(v), "f"(o));
  }
  return v;
}

}  // namespace fpk
