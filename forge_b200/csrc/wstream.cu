// Few-token linear layers on 4-bit or 16-bit weights: a weight-streaming kernel on mma.sync.
//
//   plain:  out[m][n] = sum_k x[m][k] w[n][k] + b[n]
//   gated:  out[m][n] = SiLU(g) u, g = x Wg^T + bg, u = x Wu^T + bu
//
// With a handful of tokens the call is one pass over the weight, so the kernel is built around bytes in
// flight: a warp owns 16 output channels of each matrix and every W-th block of 128 inputs, loads its
// weights straight into mma fragments with 16-byte loads, kDepth blocks ahead, and never touches shared
// memory before the final sum. Tensor-core fragments rather than FMAs because their cost does not grow with
// the tokens up to 8 per instruction.
//
// 4-bit weights are multiplied as the integers they are (exact in fp16 and in bf16) and each group's fp32 sum
// is scaled once, so nothing is rounded before the result. The weight layout (forge_prepare_weight_int4) makes
// this possible for every group size: a lane's 16-byte load of a 128-input block holds 8 inputs of each of the
// block's four 32-input runs, so one instruction multiplies inputs of one run only.
//
// The order of the sums is fixed (blocks of a warp, warps of a CTA, CTAs of a cluster): results do not change
// from run to run. Rows past N and tokens past M are computed on clamped addresses and not stored.
#include "common.cuh"
#include "float_common.cuh"
#include "gemv_common.cuh"
#include "ptx.cuh"
#include "wstream.cuh"

namespace fb200 {

using gemv::ldg_stream16;

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTokStride = 20;   // floats per token of a partial sum: 16 rows + 4, conflict-free fragment writes

// C += A B, A 16 rows x 16 inputs, B 16 inputs x 8 tokens
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                 uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                                        uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t u32(uint4 v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// G: group size, 0 = 16-bit weights. GATED: two matrices. NT: blocks of 8 tokens.
template <typename T, int G, bool GATED, int NT>
__global__ void __launch_bounds__(kThreads, 2)
wstream_kernel(const T* __restrict__ x, const void* __restrict__ w0, const void* __restrict__ w1,
               const __half* __restrict__ s0, const __half* __restrict__ s1, const T* __restrict__ b0,
               const T* __restrict__ b1, T* __restrict__ out, int M, int K, int N, int cluster) {
    constexpr bool INT4 = G != 0;
    constexpr int MATS = GATED ? 2 : 1;
    constexpr int CHUNK_K = INT4 ? 128 : 32;            // inputs of a chunk: one 16-byte load per row
    constexpr int STEPS = INT4 ? 4 : 1;                 // runs of 32 inputs in it
    constexpr int FLUSH = INT4 ? G / 32 : 1;            // runs per group
    constexpr int DEPTH = GATED ? 4 : (INT4 ? 4 : 8);   // chunks loaded ahead
    __shared__ float red[kWarps][MATS][NT * 8 * kTokStride];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % cluster;
    const int n0 = (blockIdx.x / cluster) * 16;
    const int m0 = blockIdx.y * (NT * 8);
    const int chunks = (K + CHUNK_K - 1) / CHUNK_K;
    const size_t row_bytes = INT4 ? (size_t)chunks * 64 : (size_t)K * 2;
    const int first = rank * kWarps + warp, stride = cluster * kWarps;
    const int mine = first < chunks ? (chunks - first + stride - 1) / stride : 0;

    const uint8_t* wp[MATS][2];
#pragma unroll
    for (int a = 0; a < MATS; a++)
#pragma unroll
        for (int r = 0; r < 2; r++)
            wp[a][r] = static_cast<const uint8_t*>(a == 0 ? w0 : w1) + (size_t)min(n0 + g + 8 * r, N - 1) * row_bytes + t * 16;
    const T* xp[NT];
#pragma unroll
    for (int i = 0; i < NT; i++) xp[i] = x + (size_t)min(m0 + i * 8 + g, M - 1) * K + t * 8;

    uint4 wbuf[DEPTH][MATS][2];
    uint32_t sbuf[DEPTH][MATS];   // lane l: scales of rows 2 (l % 8) and 2 (l % 8) + 1 in the chunk's group l / 8
    auto load = [&](int i, int d) {
        const int c = first + i * stride;
        const bool in = INT4 || c * CHUNK_K + t * 8 < K;   // 16-bit rows end at K, packed rows at a whole block
#pragma unroll
        for (int a = 0; a < MATS; a++) {
#pragma unroll
            for (int r = 0; r < 2; r++)
                wbuf[d][a][r] = in ? ldg_stream16(wp[a][r] + (size_t)c * 64) : make_uint4(0, 0, 0, 0);
            if constexpr (INT4) {
                constexpr int PER = 128 / G;
                const int groups = (K + G - 1) / G;
                const int j = min(c * PER + min(lane >> 3, PER - 1), groups - 1);
                const unsigned short* s = reinterpret_cast<const unsigned short*>(a == 0 ? s0 : s1) + (size_t)j * N;
                const int r = n0 + (lane & 7) * 2;
                sbuf[d][a] = __ldg(s + min(r, N - 1)) | (uint32_t)__ldg(s + min(r + 1, N - 1)) << 16;
            }
        }
    };

    float acc[MATS][NT][4];
#pragma unroll
    for (int a = 0; a < MATS; a++)
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[a][i][e] = 0.f;

    auto compute = [&](int i, int d) {
        const int k0 = (first + i * stride) * CHUNK_K;
        float part[MATS][NT][4];
#pragma unroll
        for (int j = 0; j < STEPS; j++) {
            uint4 xv[NT];
#pragma unroll
            for (int n = 0; n < NT; n++)
                xv[n] = k0 + j * 32 + t * 8 < K ? __ldg(reinterpret_cast<const uint4*>(xp[n] + k0 + j * 32))
                                                : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int a = 0; a < MATS; a++) {
                uint32_t f[2][4];   // the 8 inputs of each of the lane's two rows, in order
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    if constexpr (INT4) {
                        Int4Pairs<T>::unpack(u32(wbuf[d][a][r], j), f[r]);
                    } else {
                        f[r][0] = wbuf[d][a][r].x;
                        f[r][1] = wbuf[d][a][r].y;
                        f[r][2] = wbuf[d][a][r].z;
                        f[r][3] = wbuf[d][a][r].w;
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float (&c)[4] = INT4 ? part[a][n] : acc[a][n];
                    if (INT4 && j % FLUSH == 0) c[0] = c[1] = c[2] = c[3] = 0.f;
                    mma16816<T>(c, f[0][0], f[1][0], f[0][1], f[1][1], xv[n].x, xv[n].y);
                    mma16816<T>(c, f[0][2], f[1][2], f[0][3], f[1][3], xv[n].z, xv[n].w);
                }
            }
            if constexpr (INT4) {
                if (j % FLUSH == FLUSH - 1) {
#pragma unroll
                    for (int a = 0; a < MATS; a++) {
                        const int src = (j / FLUSH) * 8 + (g >> 1);
                        const uint32_t lo = __shfl_sync(0xffffffffu, sbuf[d][a], src);
                        const uint32_t hi = __shfl_sync(0xffffffffu, sbuf[d][a], src + 4);
                        const float sl = __half2float(__ushort_as_half((unsigned short)(g & 1 ? lo >> 16 : lo)));
                        const float sh = __half2float(__ushort_as_half((unsigned short)(g & 1 ? hi >> 16 : hi)));
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            acc[a][n][0] = fmaf(part[a][n][0], sl, acc[a][n][0]);
                            acc[a][n][1] = fmaf(part[a][n][1], sl, acc[a][n][1]);
                            acc[a][n][2] = fmaf(part[a][n][2], sh, acc[a][n][2]);
                            acc[a][n][3] = fmaf(part[a][n][3], sh, acc[a][n][3]);
                        }
                    }
                }
            }
        }
    };

#pragma unroll
    for (int d = 0; d < DEPTH; d++)
        if (d < mine) load(d, d);
    for (int i = 0; i < mine; i += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            if (i + d < mine) {
                compute(i + d, d);
                if (i + d + DEPTH < mine) load(i + d + DEPTH, d);
            }
        }
    }

#pragma unroll
    for (int a = 0; a < MATS; a++)
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float* p = &red[warp][a][(n * 8 + 2 * t) * kTokStride + g];
            p[0] = acc[a][n][0];
            p[kTokStride] = acc[a][n][1];
            p[8] = acc[a][n][2];
            p[kTokStride + 8] = acc[a][n][3];
        }
    __syncthreads();
    // sum over the CTA's warps; with a cluster, rank 0 then adds the other CTAs' sums
    if (cluster > 1) {
        for (int i = threadIdx.x; i < MATS * NT * 128; i += kThreads) {
            const int a = i / (NT * 128), tok = (i / 16) % (NT * 8), row = i % 16;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) v += red[w][a][tok * kTokStride + row];
            red[0][a][tok * kTokStride + row] = v;
        }
        ptx::cluster_sync_all();
    }
    if (rank == 0) {
        for (int i = threadIdx.x; i < NT * 128; i += kThreads) {
            const int tok = i / 16, row = i % 16;
            float v[MATS];
#pragma unroll
            for (int a = 0; a < MATS; a++) {
                float* p = &red[0][a][tok * kTokStride + row];
                v[a] = 0.f;
                if (cluster > 1) {
                    for (int c = 0; c < cluster; c++) {
                        float r;
                        asm volatile("ld.shared::cluster.f32 %0, [%1];"
                                     : "=f"(r)
                                     : "r"(ptx::mapa_shared(ptx::smem_u32(p), c))
                                     : "memory");
                        v[a] += r;
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < kWarps; w++) v[a] += red[w][a][tok * kTokStride + row];
                }
            }
            const int m = m0 + tok, n = n0 + row;
            if (m < M && n < N) {
                float r = v[0] + (b0 != nullptr ? to_float(b0[n]) : 0.f);
                if constexpr (GATED) r = silu_mul(r, v[MATS - 1] + (b1 != nullptr ? to_float(b1[n]) : 0.f));
                out[(size_t)m * N + n] = from_float<T>(r);
            }
        }
    }
    if (cluster > 1) ptx::cluster_sync_all();   // rank 0 has read the others' shared memory
}

template <typename T, int G, bool GATED, int NT>
int launch(const void* x, const void* w0, const void* w1, const __half* s0, const __half* s1, const void* b0,
           const void* b1, void* out, int M, int K, int N, cudaStream_t stream) {
    const int chunks = (K + (G ? 128 : 32) - 1) / (G ? 128 : 32);
    const long long tiles = ((long long)N + 15) / 16;
    const int token_blocks = (M + NT * 8 - 1) / (NT * 8);
    // K is split over a cluster while that leaves the GPU short of CTAs and every warp a chunk
    int cluster = 1;
    while (cluster < 8 && tiles * cluster * token_blocks < 2 * sm_count() && chunks >= 2 * cluster * kWarps) cluster *= 2;
    if (tiles * cluster > 0x7fffffffll || token_blocks > 65535) return kTooLarge;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(tiles * cluster), (unsigned)token_blocks, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, wstream_kernel<T, G, GATED, NT>, static_cast<const T*>(x), w0, w1, s0, s1,
                              static_cast<const T*>(b0), static_cast<const T*>(b1), static_cast<T*>(out), M, K, N,
                              cluster) == cudaSuccess
               ? kOk
               : kLaunchFailed;
}

template <typename T, int G, bool GATED>
int by_tokens(const void* x, const void* w0, const void* w1, const __half* s0, const __half* s1, const void* b0,
              const void* b1, void* out, int M, int K, int N, cudaStream_t st) {
    if (M <= 8) return launch<T, G, GATED, 1>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    if (M <= 16) return launch<T, G, GATED, 2>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    return launch<T, G, GATED, 4>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
}

template <typename T, bool GATED>
int by_group(const void* x, const void* w0, const void* w1, const __half* s0, const __half* s1, const void* b0,
             const void* b1, void* out, int M, int K, int N, int group, cudaStream_t st) {
    switch (group) {
    case 0: return by_tokens<T, 0, GATED>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    case 32: return by_tokens<T, 32, GATED>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    case 64: return by_tokens<T, 64, GATED>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    case 128: return by_tokens<T, 128, GATED>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    default: return kBadShape;
    }
}

}  // namespace

int wstream(const void* x, const void* w0, const void* w1, const __half* s0, const __half* s1, const void* b0,
            const void* b1, void* out, int M, int K, int N, int group, bool bf16, cudaStream_t st) {
    if (w1 != nullptr)
        return bf16 ? by_group<__nv_bfloat16, true>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, group, st)
                    : by_group<__half, true>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, group, st);
    return bf16 ? by_group<__nv_bfloat16, false>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, group, st)
                : by_group<__half, false>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, group, st);
}

}  // namespace fb200
