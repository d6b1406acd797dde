// Internal declarations of the 4-bit weight launchers (int4.cu).
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace fb200 {

// w (N, K), dtype 0 fp32 / 1 fp16 / 2 bf16 -> packed (N, ceil(K / 128) * 64) and scale (ceil(K / group), N).
int prepare_weight_int4(const void* w, int dtype, uint8_t* packed, __half* scale, int N, int K, int group,
                        cudaStream_t stream);

}  // namespace fb200
