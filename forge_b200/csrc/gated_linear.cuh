// Internal declarations of the gated linear layer on 16-bit weights (gated_linear.cu, gated_stream.cu).
// Arguments are checked in capi.cu.
#pragma once
#include <cuda_runtime.h>
#include <cstddef>

namespace fb200 {

// h = SiLU(x wg^T + bg) * (x wu^T + bu); g, u (M, N) fp32: the two products, kept for the backward pass (both or neither).
int gated_linear(const void* x, const void* wg, const void* wu, const void* bg, const void* bu, void* h, float* g,
                 float* u, int M, int K, int N, bool bf16, cudaStream_t stream);

// The same without g and u for M <= 16: one pass over the weights (gated_stream.cu).
int gated_stream(const void* x, const void* wg, const void* wu, const void* bg, const void* bu, void* h, int M, int K,
                 int N, bool bf16, cudaStream_t stream);

size_t gated_linear_backward_workspace(int M, int N);

// dx, the weight gradients (both or neither), dbg and dbu may be null.
int gated_linear_backward(const void* dh, const void* x, const void* wg, const void* wu, const float* g, const float* u,
                          void* dx, void* dwg, void* dwu, void* dbg, void* dbu, int M, int K, int N, bool bf16,
                          void* workspace, cudaStream_t stream);

}  // namespace fb200
