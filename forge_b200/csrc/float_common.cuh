// Pieces shared by the kernels that take fp16 or bf16 activations (int4*.cu, gated_*.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <type_traits>

#include "common.cuh"

namespace fb200 {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two values as the 32-bit word they make in memory, lo first
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) { return pack_half2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// (v & mask) | bits in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(bits));
    return r;
}

// D = A B + C, A 16 rows x 16 inputs, B 16 inputs x 8 tokens; C is D, or zero (`first`, a constant where it is inlined)
#define FB200_MMA(TYPE)                                                                                                 \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE                                                 \
                 ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"                                       \
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                                       \
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(first ? 0.f : d[0]), "f"(first ? 0.f : d[1]), \
                   "f"(first ? 0.f : d[2]), "f"(first ? 0.f : d[3]))
template <typename T>
__device__ __forceinline__ void mma16816(bool first, float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value) {
        FB200_MMA("f16");
    } else {
        FB200_MMA("bf16");
    }
}
#undef FB200_MMA

}  // namespace fb200
