// The gate of a gated feed-forward block on 16-bit weights for a few tokens: a weight-streaming kernel on mma.sync.
//
//   h[m][n] = SiLU(g) u, g = x Wg^T + bg, u = x Wu^T + bu
//
// With a handful of tokens the call is one pass over the weights, so the kernel is built around an even share of their
// bytes for every SM and enough of them under way:
//   - one CTA per SM, each with the same number of rows of both matrices (up to 32 of each a pass);
//   - columns of 128 bytes (64 inputs) of those rows come with one TMA copy a matrix, and the activations that belong to
//     them, into a ring as deep as shared memory allows; the warp that has read a stage fetches the column that comes into
//     it next, so no warp is kept for that;
//   - the warps divide the columns and sum over each other once, at the end of a pass.
// The products are tensor-core fragments rather than FMAs because their cost does not grow with the tokens up to 8 per
// instruction. The columns lie in shared memory with the 128-byte swizzle; fragment row g is row (g / 2 | g % 2 * 4) of
// its block, which spreads eight lanes' 16-byte reads over all banks.
//
// The order of the sums is fixed (columns of a warp, warps of the CTA): results do not change from run to run. What lies past
// the last row, token or input arrives as zeros or is stale in rows of its own; it is not stored.
//
// 14336 x 4096 bf16, cold weights: 38.6 us at 1 token and 39 us at 8 (235 MB: 6.1 TB/s; 36 us at the copy rate). Columns of
// 64 bytes, a ring for each warp: 48 us.
#include <algorithm>

#include "common.cuh"
#include "float_common.cuh"
#include "gated_linear.cuh"
#include "gemm_dense.cuh"
#include "ptx.cuh"

namespace fb200 {

namespace {

constexpr int kTokStride = 20;                    // floats per token of a partial sum: 16 rows + 4, conflict-free writes
constexpr int kSmemMax = 226 * 1024;              // dynamic; the barriers are static
constexpr int kColK = 64;                         // inputs of a column
constexpr int kMaxBlocks = 2;                     // blocks of 16 rows of a matrix in a pass
constexpr int kMaxDepth = 32;
template <int NT>
struct Warps {
    static constexpr int kMax = NT == 1 ? 16 : 12;
    static constexpr int kBlock = NT * 8 * kTokStride;              // floats of a block's partial sums
    static constexpr int kRed = 2 * kMaxBlocks * kBlock * 4;        // bytes of a warp's partial sums
};

// How a call is cut.
struct Cut {
    int rows;            // of each matrix, in a pass
    int passes;          // of a CTA
    int blocks;          // of 16 rows, in a pass
    int warps;
    int depth;           // ring stages
    int stage;           // bytes of one
    int tokens;          // of which a stage holds the activations: those of the call, if they are fewer than 8 NT
    int red;             // where the sums over warps lie: behind the ring, or, with one pass, where it was
};

// Bounded wait for a word of shared memory to become `value`.
__device__ __forceinline__ bool wait_equal(const volatile int* word, int value, volatile int* abort_flag) {
    if (*word == value) return true;
    const uint64_t t0 = ptx::globaltimer_ns();
    for (uint32_t spins = 1;; spins++) {
        if (*word == value) return true;
        if ((spins & 0x3f) == 0) {
            if (*abort_flag != 0) return false;
            if (ptx::globaltimer_ns() - t0 > 2000000000ull) {
                *abort_flag = 1;
                return false;
            }
        }
    }
}

// NT: blocks of 8 tokens
template <typename T, int NT>
__global__ void __launch_bounds__(Warps<NT>::kMax * 32, 1)
gated_stream_kernel(const __grid_constant__ CUtensorMap tm_g, const __grid_constant__ CUtensorMap tm_u,
                    const __grid_constant__ CUtensorMap tm_x, const T* __restrict__ bg, const T* __restrict__ bu,
                    T* __restrict__ out, int M, int K, int N, Cut cut, int* __restrict__ status) {
    constexpr int BLOCK = Warps<NT>::kBlock, RED = Warps<NT>::kRed / 4;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ uint64_t full[kMaxDepth];
    __shared__ volatile int lap_of[kMaxDepth];   // how often a stage has been filled anew
    __shared__ volatile int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3, row_g = (g >> 1) | (g & 1) << 2;
    const int columns = (K + kColK - 1) / kColK;
    const int mat_bytes = cut.blocks * 2048;
    const long long row_first = (long long)blockIdx.x * cut.passes * cut.rows;
    const int passes = (int)min((long long)cut.passes, (N - row_first + cut.rows - 1) / cut.rows);
    const int turns = passes * columns;   // columns that this CTA goes through

    if ((ptx::smem_u32(smem) & 1023u) != 0) {
        if (threadIdx.x == 0) atomicExch(status, 800);
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < cut.depth; i++) {
            ptx::mbar_init(&full[i], 1);
            lap_of[i] = 0;
        }
        abort_flag = 0;
        ptx::fence_mbar_init();
    }
    __syncthreads();

    auto load = [&](int turn, int stage) {
        const int p = turn / columns, c = turn - p * columns, row0 = (int)row_first + p * cut.rows;
        uint8_t* d = smem + stage * cut.stage;
        ptx::mbar_expect_tx(&full[stage], 2 * cut.rows * 128 + cut.tokens * 128);
        ptx::tma_load_2d(d, &tm_g, &full[stage], c * kColK, row0);
        ptx::tma_load_2d(d + mat_bytes, &tm_u, &full[stage], c * kColK, row0);
        ptx::tma_load_2d(d + 2 * mat_bytes, &tm_x, &full[stage], c * kColK, 0);
    };
    if (lane == 0)
        for (int i = warp; i < min(cut.depth, turns); i += cut.warps) load(i, i);

    float* red = reinterpret_cast<float*>(smem + cut.red);   // [warp][matrix][block]
    bool ok = true;
    for (int p = 0; p < passes; p++) {
        const int row0 = (int)row_first + p * cut.rows;
        float acc[2][kMaxBlocks][NT][4];
#pragma unroll
        for (int i = 0; i < 2 * kMaxBlocks * NT * 4; i++) (&acc[0][0][0][0])[i] = 0.f;
        for (int c = warp; c < columns; c += cut.warps) {
            const int turn = p * columns + c, lap = turn / cut.depth, stage = turn - lap * cut.depth;
            // A barrier's parity tells a lap from its neighbours only, and this warp may be a lap ahead of those that read
            // the stage before it: it first waits for the stage to be in its lap.
            ok = __all_sync(0xffffffffu, wait_equal(&lap_of[stage], lap, &abort_flag) &&
                                             ptx::mbar_wait(&full[stage], lap & 1, &abort_flag));
            if (!ok) break;
            const int src = stage * cut.stage;
            const uint8_t* xs = smem + src + 2 * mat_bytes + t * 16;
            const int at = src + row_g * 128 + ((t ^ row_g) << 4);
#pragma unroll
            for (int j = 0; j < 2; j++) {   // runs of 32 inputs
                uint4 xv[NT];
#pragma unroll
                for (int n = 0; n < NT; n++)
                    xv[n] = *reinterpret_cast<const uint4*>(xs + min(n * 8 + g, cut.tokens - 1) * 128 + j * 64);
#pragma unroll
                for (int b = 0; b < kMaxBlocks; b++)
                    if (b < cut.blocks) {
#pragma unroll
                        for (int a = 0; a < 2; a++) {
                            const uint8_t* w = smem + ((at + a * mat_bytes + b * 2048) ^ (j * 64));
                            const uint4 lo = *reinterpret_cast<const uint4*>(w);             // fragment row g
                            const uint4 hi = *reinterpret_cast<const uint4*>(w + 1024);      // and g + 8
#pragma unroll
                            for (int n = 0; n < NT; n++) {
                                mma16816<T>(false, acc[a][b][n], lo.x, hi.x, lo.y, hi.y, xv[n].x, xv[n].y);
                                mma16816<T>(false, acc[a][b][n], lo.z, hi.z, lo.w, hi.w, xv[n].z, xv[n].w);
                            }
                        }
                    }
            }
            __syncwarp();   // the stage has been read
            if (lane == 0 && turn + cut.depth < turns) {
                lap_of[stage] = lap + 1;
                load(turn + cut.depth, stage);
            }
        }
        if (!ok && lane == 0) atomicExch(status, 801);

        // ---- sum over the warps
        if (cut.red == 0) __syncthreads();   // every warp is done with the ring
#pragma unroll
        for (int a = 0; a < 2; a++)
#pragma unroll
            for (int b = 0; b < kMaxBlocks; b++)
                if (b < cut.blocks) {
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        float* d = red + warp * RED + (a * kMaxBlocks + b) * BLOCK + (n * 8 + 2 * t) * kTokStride + row_g;
                        d[0] = acc[a][b][n][0];
                        d[kTokStride] = acc[a][b][n][1];
                        d[8] = acc[a][b][n][2];
                        d[kTokStride + 8] = acc[a][b][n][3];
                    }
                }
        __syncthreads();
        if (abort_flag != 0) break;
        for (int i = threadIdx.x; i < cut.blocks * NT * 128; i += cut.warps * 32) {
            const int row = i % 16, b = i / 16 % cut.blocks, m = i / 16 / cut.blocks;
            const float* q = red + b * BLOCK + m * kTokStride + row;
            float gate = 0.f, up = 0.f;
            for (int w = 0; w < cut.warps; w++) {
                gate += q[w * RED];
                up += q[w * RED + kMaxBlocks * BLOCK];
            }
            const int r = b * 16 + row, n = row0 + r;
            if (m < M && r < cut.rows && n < N) {
                if (bg != nullptr) gate += to_float(bg[n]);
                if (bu != nullptr) up += to_float(bu[n]);
                out[(size_t)m * N + n] = from_float<T>(silu_mul(gate, up));
            }
        }
        if (p + 1 < passes) __syncthreads();   // before the sums are written over
    }
    if (abort_flag != 0) {   // copies may still be under way into this CTA's memory
        const uint64_t t0 = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - t0 < 200000ull) { }
    }
}

// ---------------------------------------------------------------------- host

template <typename T>
bool encode(CUtensorMap* m, const void* base, long long dim0, long long dim1, int rows, CUtensorMapSwizzle swizzle) {
    PFN_encodeTiled fn = get_encode_fn();
    if (fn == nullptr) return false;
    const CUtensorMapDataType type =
        std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const cuuint64_t dims[2] = {(cuuint64_t)dim0, (cuuint64_t)dim1}, strides[1] = {(cuuint64_t)dim0 * 2};
    const cuuint32_t box[2] = {kColK, (cuuint32_t)rows}, es[2] = {1, 1};
    return fn(m, type, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NT>
Cut make_cut(int M, int K, int N) {
    Cut best = {};
    const int sms = sm_count(), columns = (K + kColK - 1) / kColK;
    // fewest blocks of 16 rows per SM, then fewest passes
    const int least = (int)(((long long)N + (long long)sms * kMaxBlocks * 16 - 1) / ((long long)sms * kMaxBlocks * 16));
    for (int p = least; p < least + 4; p++) {
        const int rows = (int)(((long long)N + (long long)sms * p - 1) / ((long long)sms * p));
        const int blocks = (rows + 15) / 16;
        if (best.passes == 0 || p * blocks < best.passes * best.blocks) {
            best.rows = rows;
            best.passes = p;
            best.blocks = blocks;
        }
    }
    best.tokens = std::min(M, NT * 8);
    best.stage = 2 * best.blocks * 2048 + ((best.tokens * 128 + 1023) & ~1023);
    // the fewest warps that need no more turns than all of them would
    const int turns = (columns + Warps<NT>::kMax - 1) / Warps<NT>::kMax;
    best.warps = (columns + turns - 1) / turns;
    const int red = best.warps * Warps<NT>::kRed;
    best.depth = std::min((kSmemMax - (best.passes > 1 ? red : 0)) / best.stage, kMaxDepth);
    best.red = best.passes > 1 ? best.depth * best.stage : 0;
    return best;
}

template <typename T, int NT>
int launch(const void* x, const void* wg, const void* wu, const void* bg, const void* bu, void* out, int M, int K, int N,
           cudaStream_t stream) {
    static_assert(Warps<NT>::kMax * Warps<NT>::kRed + 3 * (4 * 2048 + NT * 1024) <= kSmemMax, "a ring of three at least");
    static bool ready[64] = {};
    auto kern = gated_stream_kernel<T, NT>;
    int dev = 0;
    cudaGetDevice(&dev);
    if (!ready[dev & 63]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax) != cudaSuccess)
            return kLaunchFailed;
        ready[dev & 63] = true;
    }
    const Cut cut = make_cut<NT>(M, K, N);
    CUtensorMap tm_g, tm_u, tm_x;
    if (!encode<T>(&tm_g, wg, K, N, cut.rows, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode<T>(&tm_u, wu, K, N, cut.rows, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode<T>(&tm_x, x, K, M, cut.tokens, CU_TENSOR_MAP_SWIZZLE_NONE))
        return kLaunchFailed;
    int* status = status_word();
    if (status == nullptr) return kLaunchFailed;
    const int smem = std::max(cut.depth * cut.stage, cut.red + cut.warps * Warps<NT>::kRed);
    const long long per_cta = (long long)cut.rows * cut.passes;
    kern<<<(unsigned)(((long long)N + per_cta - 1) / per_cta), cut.warps * 32, smem, stream>>>(
        tm_g, tm_u, tm_x, static_cast<const T*>(bg), static_cast<const T*>(bu), static_cast<T*>(out), M, K, N, cut, status);
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
}

}  // namespace

int gated_stream(const void* x, const void* wg, const void* wu, const void* bg, const void* bu, void* h, int M, int K,
                 int N, bool bf16, cudaStream_t stream) {
    if (M <= 8)
        return bf16 ? launch<__nv_bfloat16, 1>(x, wg, wu, bg, bu, h, M, K, N, stream)
                    : launch<__half, 1>(x, wg, wu, bg, bu, h, M, K, N, stream);
    return bf16 ? launch<__nv_bfloat16, 2>(x, wg, wu, bg, bu, h, M, K, N, stream)
                : launch<__half, 2>(x, wg, wu, bg, bu, h, M, K, N, stream);
}

}  // namespace fb200
