// Few-token linear layers on 4-bit weights: a weight-streaming kernel on mma.sync.
//
//   plain:  out[m][n] = sum_k x[m][k] w[n][k] + b[n]
//   gated:  out[m][n] = SiLU(g) u, g = x Wg^T + bg, u = x Wu^T + bu
//
// With a handful of tokens the call is one pass over the weight. What bounds it, once enough bytes are under way, is the
// instructions that make 16-bit numbers of the weights, so there are few of them:
//   - The stored n = q + 8 is cut out where it lies and multiplied as it is, sum_k x[k] n[k] per group, and 8 sum_k x[k],
//     which all rows share, is taken off before the group's scale is applied (Nibbles below). n and its products are exact
//     and the sums are fp32: nothing is rounded before the result, but a token with an infinite activation comes out as
//     NaN.
//   - The products are tensor-core fragments, whose cost does not grow with the tokens up to 8 per instruction.
//   - A CTA owns up to 32 output channels of the call (gated: 16 of each matrix) and its warps divide the blocks of 128
//     inputs. A lane copies exactly the bytes that it later reads as its fragment (cp.async, a ring of its own), so warps
//     run without barriers, 24 on an SM, up to the sum over a CTA's warps at the end. Activations are read through L1:
//     copied into the ring as well they cost a third of the weights' stages, and calls with 8 and 16 tokens 5 to 20 %.
// The weight layout (forge_prepare_weight_int4) makes this possible for every group size: a lane's 16-byte load of a
// 128-input block holds 8 inputs of each of the block's four 32-input runs, so one instruction multiplies inputs of one run
// only.
//
// Cold weights: 11008 x 4096 fp16, groups of 128, 9.7 us at 1 token and 10.6 at 8 (22.9 MB: 2.4 TB/s; 3.5 us at the copy
// rate, an empty launch 2); 4096 x 14336 bf16, groups of 64, 14 and 15 us; 8192 x 8192 12 and 12.6; 28672 x 8192 32 us (3.7
// TB/s); gated 14336 x 4096 twice 22 and 24 us (60.6 MB: 2.8 TB/s). 4096 x 14336: half of the issue slots are used and a
// fifth of the memory's rate; what is left is latency, of the activations from L2 and of few blocks for each warp, and
// registers: with two row blocks and groups of 32 or 64 every instance spills, 60 to 96 bytes of stores a thread with 80
// registers (up to 8 tokens), 40 to 268 with 128; groups of 128 at most 36. 16
// tokens need two products a fragment and the registers of 16 warps an SM: 17 us for the first.
//
// The order of the sums is fixed (blocks of a warp, warps of a CTA): results do not change from run to run. Rows past N
// and tokens past M are computed on the last one's addresses and not stored.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "float_common.cuh"
#include "int4.cuh"

namespace fb200 {

namespace {

constexpr int kRing = 6;              // KB of a warp's weights under way: 6 * 24 warps, and room for activations in L1 (8: 5 % slower)
constexpr int kTokStride = 20;        // floats per token of a partial sum: 16 rows + 4, conflict-free fragment writes

// Word of 8 four-bit weights (weight 2i in nibble i, weight 2i + 1 in nibble i + 4, stored as the integer + 8) -> four
// pairs of 16-bit floats, the first two for one accumulator (A), the others for another (B); their sum is A + B * kB.
//   fp16: a nibble alone in a half is the subnormal number n 2^-24, or 16 n 2^-24 where it lies four bits up; tensor
//         cores take subnormals as they are. The factor 2^24 comes in behind the last sum.
//   bf16: its subnormals would make subnormal fp32 products, so the nibble becomes the upper mantissa bits of (16 + n) 2^-12:
//         the most that a sum over a group can be is 128 * 31 * 2^-12 < 1 times the largest activation, so none overflows,
//         whatever the activations are.
template <typename T>
struct Nibbles;
template <>
struct Nibbles<__half> {
    static constexpr float kB = 0.0625f, kFactor = 16777216.f;
    static constexpr uint32_t kMinusOffsetA = 0x80088008u, kMinusOffsetB = 0x80808080u;   // -8 as A and as B holds it
    static __device__ __forceinline__ void unpack(uint32_t w, uint32_t (&f)[4]) {
        const uint32_t v = w >> 4;
        f[0] = w & 0x000F000Fu;
        f[1] = v & 0x000F000Fu;
        f[2] = v & 0x00F000F0u;
        f[3] = (w >> 8) & 0x00F000F0u;
    }
};
template <>
struct Nibbles<__nv_bfloat16> {
    static constexpr float kB = 1.f, kFactor = 4096.f;
    static constexpr uint32_t kMinusOffsetA = 0xBBC0BBC0u, kMinusOffsetB = 0xBBC0BBC0u;   // -24 2^-12
    static __device__ __forceinline__ void unpack(uint32_t w, uint32_t (&f)[4]) {
        f[0] = and_or(w * 8u, 0x00780078u, 0x3B803B80u);
        f[1] = and_or(w >> 1, 0x00780078u, 0x3B803B80u);
        f[2] = and_or(w >> 5, 0x00780078u, 0x3B803B80u);
        f[3] = and_or(w >> 9, 0x00780078u, 0x3B803B80u);
    }
};

__device__ __forceinline__ uint32_t u32(uint4 v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                 "l"(src)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// UNITS: blocks of 16 rows of a CTA. NT: blocks of 8 tokens.
template <typename T, int G, bool GATED, int UNITS, int WARPS, int NT>
__global__ void __launch_bounds__(WARPS * 32, (NT == 1 ? 24 : 16) / WARPS)
int4_stream_kernel(const T* __restrict__ x, const uint8_t* __restrict__ w0, const uint8_t* __restrict__ w1,
                   const __half* __restrict__ s0, const __half* __restrict__ s1, const T* __restrict__ b0,
                   const T* __restrict__ b1, T* __restrict__ out, int M, int K, int N, int rows) {
    using F = Nibbles<T>;
    constexpr int PER = 128 / G, FLUSH = G / 32;   // groups of a block; runs of a group
    constexpr int kDepth = kRing / UNITS;          // blocks under way
    constexpr int RED_UNIT = NT * 8 * kTokStride;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * rows;
    const int m0 = blockIdx.y * (NT * 8);
    const int blocks = (K + 127) / 128;
    const int mine = warp < blocks ? (blocks - warp + WARPS - 1) / WARPS : 0;
    const bool ragged = K % 128 != 0 && mine > 0 && warp + (mine - 1) * WARPS == blocks - 1;

    const uint8_t* wp[UNITS][2];
#pragma unroll
    for (int u = 0; u < UNITS; u++)
#pragma unroll
        for (int r = 0; r < 2; r++)
            wp[u][r] = (GATED && u == 1 ? w1 : w0) +
                       (size_t)min(n0 + g + 8 * r + (GATED ? 0 : 16 * u), N - 1) * ((size_t)blocks * 64) + warp * 64 + t * 16;
    // lane l: its bytes of the ring are [stage][unit][row half][lane], 16 each
    uint8_t* const ring = smem + warp * (kDepth * UNITS * 1024) + lane * 16;
    int in_stage = 0;
    auto load = [&]() {
#pragma unroll
        for (int u = 0; u < UNITS; u++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                cp_async16(ring + in_stage * (UNITS * 1024) + u * 1024 + r * 512, wp[u][r]);
                wp[u][r] += WARPS * 64;
            }
        in_stage = in_stage + 1 == kDepth ? 0 : in_stage + 1;
    };
#pragma unroll 1
    for (int i = 0; i < kDepth; i++) {
        if (i < mine) load();
        cp_commit();
    }

    // Scales, a block ahead: lane l holds that of row l % 16 of unit l / 16, from where the lanes that need it take it.
    const int groups = (K + G - 1) / G;
    const unsigned short* sp =
        reinterpret_cast<const unsigned short*>(GATED && lane >= 16 ? s1 : s0) + min(n0 + (GATED ? lane % 16 : lane), N - 1);
    unsigned short sv[PER], sn[PER];   // of this block and the next
    auto load_scales = [&](int block, unsigned short (&v)[PER]) {
#pragma unroll
        for (int k = 0; k < PER; k++) v[k] = __ldg(sp + (size_t)min(block * PER + k, groups - 1) * N);
    };
    load_scales(min(warp, blocks - 1), sn);

    const T* xp[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) xp[n] = x + (size_t)min(m0 + n * 8 + g, M - 1) * K + warp * 128 + t * 8;

    float acc[UNITS][NT][4];
#pragma unroll
    for (int i = 0; i < UNITS * NT * 4; i++) (&acc[0][0][0])[i] = 0.f;

    int block = warp, stage = 0;
    // The next block's products. WHOLE: all of its inputs exist.
    auto compute = [&](auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        uint4 xv[4][NT];   // under way while the weights are waited for
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int n = 0; n < NT; n++) {
                xv[j][n] = make_uint4(0, 0, 0, 0);
                if (WHOLE || block * 128 + j * 32 + t * 8 < K) xv[j][n] = __ldg(reinterpret_cast<const uint4*>(xp[n] + j * 32));
            }
#pragma unroll
        for (int n = 0; n < NT; n++) xp[n] += WARPS * 128;
#pragma unroll
        for (int k = 0; k < PER; k++) sv[k] = sn[k];
        load_scales(min(block + WARPS, blocks - 1), sn);
        cp_wait<kDepth - 1>();
        float off[PER][NT][2];   // minus the offset's share of the lane's two tokens, per group
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float ca[4], cb[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                constexpr uint32_t A = F::kMinusOffsetA, B = F::kMinusOffsetB;
                const uint4 v = xv[j][n];
                mma16816<T>(j % FLUSH == 0, ca, A, A, A, A, v.x, v.y);
                mma16816<T>(j % FLUSH == 0, cb, B, B, B, B, v.z, v.w);
                if (j % FLUSH == FLUSH - 1) {
                    off[j / FLUSH][n][0] = fmaf(cb[0], F::kB, ca[0]);
                    off[j / FLUSH][n][1] = fmaf(cb[1], F::kB, ca[1]);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            const uint4* at = reinterpret_cast<const uint4*>(ring + stage * (UNITS * 1024) + u * 1024);
            const uint4 w[2] = {at[0], at[32]};   // rows g and g + 8
            float pa[NT][4], pb[NT][4];           // sums of the current group
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t f0[4], f1[4];
                F::unpack(u32(w[0], j), f0);
                F::unpack(u32(w[1], j), f1);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const uint4 v = xv[j][n];
                    mma16816<T>(j % FLUSH == 0, pa[n], f0[0], f1[0], f0[1], f1[1], v.x, v.y);
                    mma16816<T>(j % FLUSH == 0, pb[n], f0[2], f1[2], f0[3], f1[3], v.z, v.w);
                }
                if (j % FLUSH == FLUSH - 1) {
                    const int v = sv[j / FLUSH];
                    const float sl = __half2float(__ushort_as_half((unsigned short)__shfl_sync(0xffffffffu, v, u * 16 + g)));
                    const float sh = __half2float(__ushort_as_half((unsigned short)__shfl_sync(0xffffffffu, v, u * 16 + 8 + g)));
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            acc[u][n][e] = fmaf(fmaf(pb[n][e], F::kB, pa[n][e] + off[j / FLUSH][n][e & 1]), e < 2 ? sl : sh,
                                                acc[u][n][e]);
                }
            }
        }
        block += WARPS;
        stage = stage + 1 == kDepth ? 0 : stage + 1;
    };
    const int whole = mine - ragged;
#pragma unroll 1
    for (int i = 0; i < whole; i++) {
        compute(std::true_type());
        if (i + kDepth < mine) load();
        cp_commit();
    }
    if (ragged) compute(std::false_type());

    // ---- sum over the warps
    __syncthreads();   // every warp is done with the ring
    float* red = reinterpret_cast<float*>(smem);   // [warp][unit][token * kTokStride + row]
#pragma unroll
    for (int u = 0; u < UNITS; u++)
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float* p = red + (warp * UNITS + u) * RED_UNIT + (n * 8 + 2 * t) * kTokStride + g;
            p[0] = acc[u][n][0];
            p[kTokStride] = acc[u][n][1];
            p[8] = acc[u][n][2];
            p[kTokStride + 8] = acc[u][n][3];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < (GATED ? 1 : UNITS) * NT * 128; i += WARPS * 32) {
        const int row = i % 16, u = GATED ? 0 : i / 16 % UNITS, tok = i / 16 / (GATED ? 1 : UNITS);
        const int m = m0 + tok, n = n0 + u * 16 + row;
        if (m >= M || n >= N || u * 16 + row >= rows) continue;
        auto sum = [&](int unit) {
            const float* p = red + unit * RED_UNIT + tok * kTokStride + row;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) v += p[w * (UNITS * RED_UNIT)];
            return v * F::kFactor;
        };
        float v = sum(u) + (b0 != nullptr ? to_float(b0[n]) : 0.f);
        if constexpr (GATED) v = silu_mul(v, sum(UNITS - 1) + (b1 != nullptr ? to_float(b1[n]) : 0.f));
        out[(size_t)m * N + n] = from_float<T>(v);
    }
}

template <typename T, int G, bool GATED, int UNITS, int WARPS, int NT>
int launch(const void* x, const uint8_t* w0, const uint8_t* w1, const __half* s0, const __half* s1, const void* b0,
           const void* b1, void* out, int M, int K, int N, int rows, cudaStream_t stream) {
    static bool ready[64] = {};
    auto kern = int4_stream_kernel<T, G, GATED, UNITS, WARPS, NT>;
    constexpr int kSmem = std::max(WARPS * kRing * 1024, WARPS * UNITS * NT * 8 * kTokStride * 4);
    int dev = 0;
    cudaGetDevice(&dev);
    if (!ready[dev & 63]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
            return kLaunchFailed;
        ready[dev & 63] = true;
    }
    const dim3 grid((unsigned)(((long long)N + rows - 1) / rows), (M + NT * 8 - 1) / (NT * 8), 1);
    if (grid.y > 65535) return kTooLarge;
    kern<<<grid, WARPS * 32, kSmem, stream>>>(static_cast<const T*>(x), w0, w1, s0, s1, static_cast<const T*>(b0),
                                              static_cast<const T*>(b1), static_cast<T*>(out), M, K, N, rows);
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
}

template <typename T, int G, bool GATED>
int dispatch(const void* x, const uint8_t* w0, const uint8_t* w1, const __half* s0, const __half* s1, const void* b0,
             const void* b1, void* out, int M, int K, int N, cudaStream_t st) {
    // Output channels of a CTA: as many as a warp can hold, or, where that makes up to three CTAs for each SM, so many that
    // all SMs have the same number. The warps that an SM runs at a time (24; 16 with more than 8 tokens) are divided over
    // them: 4096 x 14336 14 us with 24 warps on 28 channels, 17 with 8 on 14 twice; 8192 x 8192 12 us with 12 warps on 28
    // channels twice, 17 with 8 on 14 four times.
    const int most = GATED ? 16 : 32, sms = sm_count();
    const long long per_sm = ((long long)N + (long long)most * sms - 1) / ((long long)most * sms);
    const int rows = per_sm <= 3 ? (int)((N + per_sm * sms - 1) / (per_sm * sms)) : most;
    if (!GATED && rows <= 16)   // 2048 x 2048: 3.3 us, 4.2 with fragments for 32
        return M <= 8 ? launch<T, G, false, 1, 24, 1>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, rows, st)
                      : launch<T, G, false, 1, 16, 2>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, rows, st);
    if (M <= 8) {
        if (per_sm == 1) return launch<T, G, GATED, 2, 24, 1>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, rows, st);
        if (per_sm == 2) return launch<T, G, GATED, 2, 12, 1>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, rows, st);
        return launch<T, G, GATED, 2, 8, 1>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, rows, st);
    }
    if (per_sm == 1) return launch<T, G, GATED, 2, 16, 2>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, rows, st);
    return launch<T, G, GATED, 2, 8, 2>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, rows, st);
}

template <typename T, int G>
int dispatch(const void* x, const uint8_t* w0, const uint8_t* w1, const __half* s0, const __half* s1, const void* b0,
             const void* b1, void* out, int M, int K, int N, cudaStream_t st) {
    return w1 != nullptr ? dispatch<T, G, true>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st)
                         : dispatch<T, G, false>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
}

}  // namespace

int int4_stream(const void* x, const uint8_t* w0, const uint8_t* w1, const __half* s0, const __half* s1, const void* b0,
                const void* b1, void* out, int M, int K, int N, int group, bool bf16, cudaStream_t st) {
    switch (group * 2 + (bf16 ? 1 : 0)) {
    case 64: return dispatch<__half, 32>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    case 65: return dispatch<__nv_bfloat16, 32>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    case 128: return dispatch<__half, 64>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    case 129: return dispatch<__nv_bfloat16, 64>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    case 256: return dispatch<__half, 128>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    case 257: return dispatch<__nv_bfloat16, 128>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    default: return kBadShape;
    }
}

}  // namespace fb200
