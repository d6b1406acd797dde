// 4-bit weights with group scales: quantization of a float weight into the layout that the linear kernels read.
//
// Per row and group of G inputs: s = fp16(absmax / 7), q = clamp(round_half_even(w / s), -7, 7), both quotients taken
// exactly (a float quotient that lands on a rounding border is resolved by its remainder), so the integers do not
// depend on how a division rounds. A group that holds an infinity or a NaN, or whose scale is beyond fp16, gets the
// scale NaN and zeros: its outputs are NaN, not plausible numbers.
//
// Layout: row n is ceil(K / 128) blocks of 64 bytes. Eight neighbouring weights make one 32-bit word: weight 2i in
// nibble i, weight 2i + 1 in nibble i + 4, each stored as q + 8 (pairs of neighbours come out of one mask). Of the 16
// words of a block word 4t + j holds the block's run 4j + t, so that 16 bytes hold 8 weights of each run of 32.
// Weights past K are 0. Scales are (ceil(K / G), N): what a tile of rows needs of a group is contiguous.
//
// Bound by HBM: 2 or 4 bytes read and half a byte written per weight. A CTA takes 16 rows so that the two-byte scale
// stores of neighbouring rows meet in a 32-byte sector. 28672 x 8192, groups of 128: fp32 200 us (82 % of the copy rate),
// fp16 206 us, there bound by the arithmetic of the exact quotients.
#include "common.cuh"
#include "float_common.cuh"
#include "int4.cuh"

namespace fb200 {

namespace {

constexpr int kRows = 16;

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
    const T* h = reinterpret_cast<const T*>(&a);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = to_float(h[i]);
}

// absmax / 7 rounded once to fp16: the quotient is first cut to fp32, with its last bit set when it is inexact. The product
// with 1 / 7 is less than a step off the quotient, and the remainders are exact. Infinities and NaNs become NaN on the way,
// a scale beyond fp16 at the end.
__device__ __forceinline__ __half group_scale(float amax) {
    float q = amax * (1.f / 7.f);
    if (fmaf(-7.f, q, amax) < 0.f) q = __uint_as_float(__float_as_uint(q) - 1u);
    if (fmaf(-7.f, q, amax) != 0.f) q = __uint_as_float(__float_as_uint(q) | 1u);
    const __half s = __float2half_rn(q);
    return __hisinf(s) || __hisnan(s) ? __ushort_as_half(0x7FFF) : s;
}

// Four integers -8 .. 7 -> n = q + 8 in the nibbles of the low half, q0 lowest
__device__ __forceinline__ uint32_t nibbles4(float q0, float q1, float q2, float q3) {
    const float sum = fmaf(fmaf(fmaf(q3, 16.f, q2), 16.f, q1), 16.f, q0);
    return __float_as_uint(sum + (8388608.f + 34952.f));   // 34952 = 8 (1 + 16 + 256 + 4096)
}

// Eight weights against the scale s > 0, packed as the layout says. Adding 1.5 * 2^23 rounds to an integer, half to even.
// w (1 / s) is not the quotient, but near it: the remainder w - q s, which is exact, tells whether q is the nearest integer,
// and where w lies on a border.
__device__ __forceinline__ uint32_t quantize8(const float (&w)[8], float s) {
    constexpr float kRound = 12582912.f;
    const float inv = __fdividef(1.f, s), half = 0.5f * s;
    float q[8], worst = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        q[i] = (w[i] * inv + kRound) - kRound;
        worst = fmaxf(worst, fabsf(fmaf(-q[i], s, w[i])));
    }
    // some weight is on a border or beside the integer that 1 / s gave; a subnormal scale may be far from absmax / 7
    if (!(worst < half) || s < 6.1035156e-5f) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float n = (fminf(fmaxf(w[i] * inv, -7.f), 7.f) + kRound) - kRound, r = fmaf(-n, s, w[i]);
            const bool away = fabsf(r) > half || (fabsf(r) == half && ((int)n & 1) != 0);   // from n, on the side of r
            q[i] = fminf(fmaxf(n + (away ? copysignf(1.f, r) : 0.f), -7.f), 7.f);
        }
    }
    return __byte_perm(nibbles4(q[0], q[2], q[4], q[6]), nibbles4(q[1], q[3], q[5], q[7]), 0x5410);
}

// A lane holds 8 weights; half a warp a block of 128. A warp takes two rows at a time, whose loads are under way together.
// Grid: x over pairs of blocks, y over 16 rows.
template <typename T, int G>
__global__ void __launch_bounds__(256)
prepare_int4_kernel(const T* __restrict__ w, uint32_t* __restrict__ packed, __half* __restrict__ scale, int N, int K) {
    constexpr int LANES = G / 8, EACH = kRows / 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, run = lane & 15;
    const int blocks = (K + 127) / 128;
    const int blk = blockIdx.x * 2 + (lane >> 4);
    const int k = blk * 128 + run * 8;
    for (long long row0 = (long long)blockIdx.y * kRows + warp * EACH; row0 < N; row0 += (long long)gridDim.y * kRows) {
        float v[EACH][8];
#pragma unroll
        for (int r = 0; r < EACH; r++) {
            if (row0 + r < N && k < K) {
                load8(w + (size_t)(row0 + r) * K + k, v[r]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) v[r][i] = 0.f;
            }
        }
#pragma unroll
        for (int r = 0; r < EACH; r++) {
            // the bits of |w| order as numbers do, infinities and NaNs above all
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(v[r][i]) & 0x7FFFFFFFu);
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const __half s = group_scale(__uint_as_float(m));
            const float sf = __half2float(s);
            const uint32_t word = sf > 0.f ? quantize8(v[r], sf) : 0x88888888u;
            const long long row = row0 + r;
            if (row < N && blk < blocks) {
                packed[((size_t)row * blocks + blk) * 16 + (run & 3) * 4 + (run >> 2)] = word;
                if (run % LANES == 0 && k < K) scale[(size_t)(k / G) * N + row] = s;
            }
        }
    }
}

template <typename T>
int prepare(const void* w, uint8_t* packed, __half* scale, int N, int K, int group, cudaStream_t stream) {
    const int blocks = (K + 127) / 128;
    const dim3 grid((blocks + 1) / 2, (unsigned)std::min<long long>(((long long)N + kRows - 1) / kRows, 65535), 1);
    const T* src = static_cast<const T*>(w);
    uint32_t* dst = reinterpret_cast<uint32_t*>(packed);
    switch (group) {
    case 32: prepare_int4_kernel<T, 32><<<grid, 256, 0, stream>>>(src, dst, scale, N, K); break;
    case 64: prepare_int4_kernel<T, 64><<<grid, 256, 0, stream>>>(src, dst, scale, N, K); break;
    case 128: prepare_int4_kernel<T, 128><<<grid, 256, 0, stream>>>(src, dst, scale, N, K); break;
    default: return kBadShape;
    }
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
}

}  // namespace

int prepare_weight_int4(const void* w, int dtype, uint8_t* packed, __half* scale, int N, int K, int group,
                        cudaStream_t stream) {
    switch (dtype) {
    case 0: return prepare<float>(w, packed, scale, N, K, group, stream);
    case 1: return prepare<__half>(w, packed, scale, N, K, group, stream);
    case 2: return prepare<__nv_bfloat16>(w, packed, scale, N, K, group, stream);
    default: return kBadShape;
    }
}

}  // namespace fb200
