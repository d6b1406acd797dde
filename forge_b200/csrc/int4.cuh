// Internal declarations of the 4-bit weight launchers (int4.cu, int4_stream.cu, int4_gemm.cu).
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace fb200 {

// w (N, K), dtype 0 fp32 / 1 fp16 / 2 bf16 -> packed (N, ceil(K / 128) * 64) and scale (ceil(K / group), N).
int prepare_weight_int4(const void* w, int dtype, uint8_t* packed, __half* scale, int N, int K, int group,
                        cudaStream_t stream);

// Few tokens (int4_stream.cu), and many (int4_gemm.cu). w1 == nullptr: out = x w0^T + b0, else out = SiLU(x w0^T + b0) * (x w1^T + b1).
int int4_stream(const void* x, const uint8_t* w0, const uint8_t* w1, const __half* s0, const __half* s1, const void* b0,
                const void* b1, void* out, int M, int K, int N, int group, bool bf16, cudaStream_t st);
int int4_gemm(const void* x, const uint8_t* w0, const uint8_t* w1, const __half* s0, const __half* s1, const void* b0,
              const void* b1, void* out, int M, int K, int N, int group, bool bf16, cudaStream_t st);

}  // namespace fb200
