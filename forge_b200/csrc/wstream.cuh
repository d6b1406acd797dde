// Internal declaration of the weight-streaming launcher for few tokens (wstream.cu).
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace fb200 {

// w1 == nullptr: out = x w0^T + b0. Else out = SiLU(x w0^T + b0) * (x w1^T + b1). group 32 / 64 / 128: 4-bit weights
// with scales s0, s1 (ceil(K / group), N); 0: 16-bit weights (N, K). K % 8 == 0, x and weights 16-byte aligned.
int wstream(const void* x, const void* w0, const void* w1, const __half* s0, const __half* s1, const void* b0,
            const void* b1, void* out, int M, int K, int N, int group, bool bf16, cudaStream_t st);

}  // namespace fb200
