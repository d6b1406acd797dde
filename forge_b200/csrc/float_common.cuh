// Pieces shared by the kernels that take fp16 or bf16 activations (wstream.cu, int4.cu, gated_linear.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

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

// Word of 8 four-bit weights (weight 2i in nibble i, weight 2i + 1 in nibble i + 4, stored as the integer + 8) ->
// four pairs of 16-bit floats. A nibble placed in the low mantissa bits of 1024 (fp16) or 128 (bf16) is that number
// plus the nibble, exactly; subtracting the offset + 8 leaves the integer, exactly.
template <typename T>
struct Int4Pairs;
template <>
struct Int4Pairs<__half> {
    static __device__ __forceinline__ void unpack(uint32_t w, uint32_t (&f)[4]) {
        const __half2 off = __half2half2(__ushort_as_half(0x6408));   // 1032
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t b = ((w >> (4 * i)) & 0x000F000Fu) | 0x64006400u;
            const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
            f[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
};
template <>
struct Int4Pairs<__nv_bfloat16> {
    static __device__ __forceinline__ void unpack(uint32_t w, uint32_t (&f)[4]) {
        const __nv_bfloat162 off = __bfloat162bfloat162(__ushort_as_bfloat16(0x4308));   // 136
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t b = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
            const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&b), off);
            f[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
};

}  // namespace fb200
