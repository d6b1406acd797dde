// Pieces shared by the CTA-pair (tcgen05 cta_group::2) kernels on 16-bit operands: gated_linear.cu and int4_gemm.cu.
#pragma once

#include "common.cuh"
#include "ptx.cuh"

namespace fb200 {
namespace pair16 {

using namespace ptx;

constexpr int kEpiWarps = 4;
constexpr int kEpiThreads = 128;
constexpr int kBand = 16;       // 256-row blocks of A per raster band

struct Cfg {
    static constexpr int kStages = 6;
    static constexpr int kOperandBytes = 128 * 128;          // 128 rows (or channels) x 64 inputs of a CTA's half
    static constexpr int kStageBytes = 2 * kOperandBytes;
    static constexpr int kEpiBufs = 2;
    static constexpr int kEpiBufBytes = 32 * 128;
    static constexpr int kEpiBytes = kEpiWarps * kEpiBufs * kEpiBufBytes;
    static constexpr int kBiasBytes = 2 * 256 * (int)sizeof(float);
    static constexpr int kBarBytes = 256;
    static constexpr int kSmemBytes = kStages * kStageBytes + kEpiBytes + kBiasBytes + kBarBytes;
    static constexpr int kTmemCols = 512;
    static_assert(kSmemBytes <= 232448, "exceeds the 227 KB shared memory limit");
};

struct Bars {
    uint64_t *full, *empty, *tmem_full, *tmem_empty;
    uint32_t* tmem_slot;
    volatile int* abort_flag;
};
__device__ __forceinline__ Bars carve(uint8_t* p) {
    Bars b;
    b.full = reinterpret_cast<uint64_t*>(p);      // in the leader: bytes of both CTAs' loads
    b.empty = b.full + Cfg::kStages;              // one per CTA, committed by the leader's MMA thread
    b.tmem_full = b.empty + Cfg::kStages;         // one per CTA
    b.tmem_empty = b.tmem_full + 2;               // in the leader: both CTAs' epilogue warps
    b.tmem_slot = reinterpret_cast<uint32_t*>(b.tmem_empty + 2);
    b.abort_flag = reinterpret_cast<volatile int*>(b.tmem_slot + 1);
    return b;
}

// Instruction descriptor of kind::f16: fp32 accumulator, both operands fp16 or both bf16, each K-major or MN-major.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool bf16, bool a_mn, bool b_mn) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void umma_f16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// MN-major slab: chunks of 64 channels, each 64 rows (inputs) of 128 bytes with the 128-byte swizzle, 8 KB apart
// (leading offset); groups of 8 inputs are 1024 bytes apart (stride offset).
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t addr) {
    return static_cast<uint64_t>((addr & 0x3FFFF) >> 4) | static_cast<uint64_t>(8192 >> 4) << 16 |
           static_cast<uint64_t>(1024 >> 4) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}

struct Tile {
    int a_blk, b_blk;
};
__device__ __forceinline__ Tile tile_of(int t, int a_blocks, int b_blocks) {
    const int band_tiles = kBand * b_blocks;
    const int band = t / band_tiles;
    const int rows = min(kBand, a_blocks - band * kBand);
    const int r = t - band * band_tiles;
    return {band * kBand + r % rows, r / rows};
}

// (dim1, dim0) row-major elements, 128-byte wide swizzled boxes of `box_rows` rows; encoded anew in every call
inline bool encode_sw128(CUtensorMap* m, CUtensorMapDataType type, int elem, const void* base, long long dim0, long long dim1,
                         int box_rows) {
    PFN_encodeTiled fn = get_encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)dim0, (cuuint64_t)dim1};
    const cuuint64_t strides[1] = {(cuuint64_t)dim0 * elem};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / elem), (cuuint32_t)box_rows};
    const cuuint32_t es[2] = {1, 1};
    return fn(m, type, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

inline CUtensorMapDataType type16(bool bf16) {
    return bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// kern<<<2 * min(tiles, pairs that run at a time)>>> in clusters of two; `max_pairs` keeps the latter per device.
template <typename Kern, typename... Args>
int launch_pairs16(Kern kern, int threads, long long tiles, cudaStream_t stream, int* max_pairs, Args... args) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = Cfg::kSmemBytes;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int& cap = max_pairs[dev & 63];
    if (cap == 0) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes) != cudaSuccess)
            return kLaunchFailed;
        cfg.gridDim = dim3(2 * sm_count(), 1, 1);
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            return kLaunchFailed;
        }
        cap = n;
    }
    if (tiles > 0x7fffffffll / 2) return kTooLarge;
    cfg.gridDim = dim3(2 * (unsigned)(tiles < cap ? tiles : cap), 1, 1);
    return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? kOk : kLaunchFailed;
}

}  // namespace pair16
}  // namespace fb200
