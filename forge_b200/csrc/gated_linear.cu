// The gate of a gated feed-forward block on fp16 / bf16 weights, forward and backward, on CTA pairs
// (tcgen05 cta_group::2, kind::f16, fp32 accumulators in tensor memory).
//
//   g = x Wg^T + bg     u = x Wu^T + bu     h = SiLU(g) u                      x (M, K), W (N, K)
//   du = dh SiLU(g)     dg = dh u s (1 + g (1 - s)),  s = 1 / (1 + exp(-g))
//   dx = dg Wg + du Wu  dWg = dg^T x        dWu = du^T x   dbg, dbu = column sums of dg, du
//
// All of it is matrix products with tokens and channels in the thousands, bound by the tensor pipe, so the three
// products share one kernel skeleton (that of the INT8 pair GEMM): 256 x 256 accumulator tiles per pair of SMs, six
// stages of 64-deep operand slabs, two TMA-issuing threads per CTA, one MMA-issuing thread per pair, a
// double-buffered accumulator whose epilogue overlaps the next tile.
//   forward  the pair's B tile is 128 rows of Wg (staged by CTA 0) and the same rows of Wu (CTA 1), so each accumulator
//            row holds gate and up of 128 channels and the gate is applied where the products are read.
//   dx       one product over 2 N inputs: first dg with Wg, then du with Wu, into the same accumulator.
//   dW       both weight gradients in one launch, over the tokens.
// dx reads Wg, Wu and dW reads dg, du, x against their memory order; tensor cores take such 16-bit operands as they
// lie ("MN-major": 64 channels x 8 inputs per swizzle atom), so nothing is ever transposed in memory.
//
// 8192 tokens, 4096 -> 14336, bf16: forward 1.20 ms (1600 TFLOP/s, the burst rate of the tensor pipe), with g and u saved
// 1.31 ms; backward 2.7-3.0 ms, of which the elementwise part takes 265 us and the products the rest (1500 TFLOP/s), and
// in fp16 0.15-0.19 ms more (see Precision). 1001 tokens, 1032 -> 2744: forward 25 us, backward 64 us (fp16 69), with tens
// of tiles for 74 pairs; a step through autograd takes 155-160 us of host time.
//
// Precision: the forward keeps g and u in fp32 for the backward - 8 bytes per element, where rounding them to 16 bits
// would put another two roundings into every gradient. dg and du are rounded to 16 bits, which the tensor cores
// need; the bias gradients are summed from them before that rounding, in fp32, in a fixed order. Gradients are often so
// small (or, with a scaled loss, so large) that fp16 would flush or overflow them although their products are in its
// range: fp16 calls go through them once more beforehand for their largest value, store them times the power of two that
// puts it into [2^14, 2^15), and take that off the fp32 sums. What lies 2^29 below the largest is still rounded to 11 bits.
#include <algorithm>

#include "common.cuh"
#include "float_common.cuh"
#include "gated_linear.cuh"
#include "gemm_dense.cuh"
#include "pair16.cuh"
#include "ptx.cuh"

namespace fb200 {

using namespace pair16;

namespace {

constexpr int kThreads = 224;   // TMA warp (A), MMA warp, 4 epilogue warps, TMA warp (B)

enum Mode { kForward = 0, kForwardSave = 1, kDx = 2, kDw = 3 };

struct Maps {
    CUtensorMap a[2], b[2];   // operands of the first and second half of the work (see Mode)
    CUtensorMap out[2];       // h | dx | dWg, dWu
    CUtensorMap save[2];      // g, u (kForwardSave)
};

// Rows (256 per tile) are tokens, or channels for kDw; columns are channels (kForward*: 128 per tile) or inputs.
// rows, cols: extent of one output matrix; kb1: K blocks of the first operand pair, kbs: of both. unscale (kDx and kDw, fp16):
// what the products are multiplied by.
template <int MODE, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
gated_pair_kernel(const __grid_constant__ Maps maps, const void* __restrict__ bias_g, const void* __restrict__ bias_u,
                  int rows, int cols, int kb1, int kbs, const float* __restrict__ unscale, int* __restrict__ status) {
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    constexpr bool FWD = MODE == kForward || MODE == kForwardSave;
    constexpr bool A_MN = MODE == kDw, B_MN = !FWD;
    constexpr int TILE_N = FWD ? 128 : 256;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* smem_epi = smem + Cfg::kStages * Cfg::kStageBytes;
    float* smem_bias = reinterpret_cast<float*>(smem_epi + Cfg::kEpiBytes);
    const Bars bars = carve(smem_epi + Cfg::kEpiBytes + Cfg::kBiasBytes);

    const int warp_id = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    if ((smem_u32(smem) & 1023u) != 0) {   // the same in both CTAs
        if (threadIdx.x == 0) atomicExch(status, 700);
        return;
    }

    const int row_blocks = (rows + 255) / 256;
    const int a_blocks = MODE == kDw ? 2 * row_blocks : row_blocks;   // kDw: dWg's blocks, then dWu's
    const int b_blocks = (cols + TILE_N - 1) / TILE_N;
    const int num_tiles = a_blocks * b_blocks;
    const int pair_id = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::kStages; s++) {
            mbar_init(&bars.full[s], 1);
            mbar_init(&bars.empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&bars.tmem_full[i], 1);
            mbar_init(&bars.tmem_empty[i], 2 * kEpiWarps);
        }
        *bars.abort_flag = 0;
        fence_mbar_init();
    }
    if (warp_id == 1) {
        tmem_alloc_pair(bars.tmem_slot, Cfg::kTmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();   // the peer's barriers are initialised before anything signals them
    tc_fence_after();
    const uint32_t tmem_base = *bars.tmem_slot;

    const bool second = warp_id == kThreads / 32 - 1;
    if (warp_id == 0 || second) {
        // ------------------------------------------------------------------ TMA producers: A, and B
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = pair_id; t < num_tiles && ok; t += num_pairs) {
                const Tile tc = tile_of(t, a_blocks, b_blocks);
                const int half = MODE == kDw && tc.a_blk >= row_blocks;   // kDw: the tile is dWu's
                for (int kb = 0; kb < kbs; kb++) {
                    if (!mbar_wait(&bars.empty[stage], phase ^ 1, bars.abort_flag)) {
                        atomicExch(status, 701);
                        ok = false;
                        break;
                    }
                    uint8_t* dst = smem + stage * Cfg::kStageBytes + (second ? Cfg::kOperandBytes : 0);
                    const uint32_t full = mapa_shared(smem_u32(&bars.full[stage]), 0);
                    const int seg = MODE == kDx && kb >= kb1;             // kDx: the inputs are du's
                    const int k = (seg ? kb - kb1 : kb) * 64;
                    if (!second) {
                        if (leader) mbar_expect_tx(&bars.full[stage], 2 * Cfg::kStageBytes);
                        const CUtensorMap* m = &maps.a[MODE == kDw ? half : seg];
                        const int r = (tc.a_blk - half * row_blocks) * 256 + (int)rank * 128;
                        if (A_MN) {
                            tma_load_2d_pair(dst, m, full, r, k);
                            tma_load_2d_pair(dst + 8192, m, full, r + 64, k);
                        } else {
                            tma_load_2d_pair(dst, m, full, k, r);
                        }
                    } else {
                        const CUtensorMap* m = &maps.b[FWD ? (int)rank : seg];
                        const int c = tc.b_blk * TILE_N + (FWD ? 0 : (int)rank * 128);
                        if (B_MN) {
                            tma_load_2d_pair(dst, m, full, c, k);
                            tma_load_2d_pair(dst + 8192, m, full, c + 64, k);
                        } else {
                            tma_load_2d_pair(dst, m, full, k, c);
                        }
                    }
                    if (++stage == Cfg::kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        }
    } else if (warp_id == 1) {
        // ------------------------------------------------------------------ MMA issuer (leader only)
        if (leader && lane == 0) {
            constexpr uint32_t idesc = idesc_f16(256, 256, BF16, A_MN, B_MN);
            constexpr int STEP_A = A_MN ? 2048 >> 4 : 32 >> 4, STEP_B = B_MN ? 2048 >> 4 : 32 >> 4;   // 16 inputs on
            int stage = 0;
            uint32_t phase = 0;
            int local = 0;
            bool ok = true;
            for (int t = pair_id; t < num_tiles && ok; t += num_pairs, local++) {
                const int buf = local & 1;
                if (!mbar_wait(&bars.tmem_empty[buf], ((local >> 1) & 1) ^ 1, bars.abort_flag)) {
                    atomicExch(status, 702);
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t acc = tmem_base + buf * 256;
                for (int kb = 0; kb < kbs; kb++) {
                    if (!mbar_wait(&bars.full[stage], phase, bars.abort_flag)) {
                        atomicExch(status, 703);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sa = smem_u32(smem + stage * Cfg::kStageBytes);
                    const uint64_t da = A_MN ? desc_mn_sw128(sa) : make_desc_sw128(sa);
                    const uint64_t db =
                        B_MN ? desc_mn_sw128(sa + Cfg::kOperandBytes) : make_desc_sw128(sa + Cfg::kOperandBytes);
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        umma_f16_pair(acc, da + k * STEP_A, db + k * STEP_B, idesc, (kb | k) != 0 ? 1u : 0u);
                    tc_commit_pair_mask(smem_u32(&bars.empty[stage]), 3);
                    if (++stage == Cfg::kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (ok) tc_commit_pair_mask(smem_u32(&bars.tmem_full[buf]), 3);
            }
        }
    } else {
        // ------------------------------------------------------------------ epilogue (both CTAs)
        const int q = warp_id & 3;
        const int epi_tid = (warp_id - 2) * 32 + lane;
        uint8_t* my_stage = smem_epi + (warp_id - 2) * Cfg::kEpiBufs * Cfg::kEpiBufBytes;
        const uint64_t policy = l2_policy_evict_first();   // outputs must not push operands out of L2
        constexpr bool SCALED = !FWD && !BF16;
        const float factor = SCALED ? *unscale : 1.f;
        int sbuf = 0, local = 0;
        bool ok = true;
        // 32 rows x 128 bytes from this lane's 32 words, through a staging buffer, to column x, row y of `m`
        auto store = [&](const CUtensorMap* m, const uint32_t (&v)[32], int x, int y) {
            uint8_t* stg = my_stage + sbuf * Cfg::kEpiBufBytes;
            if (lane == 0) tma_store_wait_read<Cfg::kEpiBufs - 1>();
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 8; j++)
                *reinterpret_cast<uint4*>(stg + lane * 128 + (j ^ (lane & 7)) * 16) =
                    make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                tma_store_2d_hint(m, stg, x, y, policy);
                tma_store_commit();
            }
            sbuf = (sbuf + 1) % Cfg::kEpiBufs;
        };
        for (int t = pair_id; t < num_tiles; t += num_pairs, local++) {
            const Tile tc = tile_of(t, a_blocks, b_blocks);
            const int half = MODE == kDw && tc.a_blk >= row_blocks;
            const int buf = local & 1;
            const int row0 = (tc.a_blk - half * row_blocks) * 256 + (int)rank * 128 + q * 32;
            const int n0 = tc.b_blk * TILE_N;
            float* s_bg = smem_bias + buf * 256;
            float* s_bu = s_bg + 128;
            if (FWD) {
                const int n = n0 + epi_tid;
                const T* bg = static_cast<const T*>(bias_g);
                const T* bu = static_cast<const T*>(bias_u);
                s_bg[epi_tid] = bg != nullptr && n < cols ? to_float(bg[n]) : 0.f;
                s_bu[epi_tid] = bu != nullptr && n < cols ? to_float(bu[n]) : 0.f;
                named_barrier_sync(1, kEpiThreads);
            }
            if (ok) {
                ok = __all_sync(0xffffffffu, mbar_wait(&bars.tmem_full[buf], (local >> 1) & 1, bars.abort_flag));
                if (!ok) atomicExch(status, 704);
            }
            if (!ok) continue;
            tc_fence_after();
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * 256;
            // a store past the output's last row or column must not be issued: its box would start outside
#pragma unroll 1
            for (int c = 0; c < TILE_N / 64; c++) {
                uint32_t packed[32];
#pragma unroll
                for (int hh = 0; hh < 2; hh++) {
                    const int col = c * 64 + hh * 32;
                    uint32_t va[32], vb[32];
                    tmem_ld_32x32b_x32(taddr + col, va);
                    if (FWD) tmem_ld_32x32b_x32(taddr + 128 + col, vb);
                    tmem_ld_wait();
                    if (FWD) {
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            va[i] = __float_as_uint(__uint_as_float(va[i]) + s_bg[col + i]);
                            vb[i] = __float_as_uint(__uint_as_float(vb[i]) + s_bu[col + i]);
                        }
                        if (MODE == kForwardSave && row0 < rows && n0 + col < cols) {
                            store(&maps.save[0], va, n0 + col, row0);
                            store(&maps.save[1], vb, n0 + col, row0);
                        }
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            packed[hh * 16 + i] =
                                pack2<T>(silu_mul(__uint_as_float(va[2 * i]), __uint_as_float(vb[2 * i])),
                                         silu_mul(__uint_as_float(va[2 * i + 1]), __uint_as_float(vb[2 * i + 1])));
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            packed[hh * 16 + i] =
                                SCALED ? pack2<T>(__uint_as_float(va[2 * i]) * factor, __uint_as_float(va[2 * i + 1]) * factor)
                                       : pack2<T>(__uint_as_float(va[2 * i]), __uint_as_float(va[2 * i + 1]));
                    }
                }
                if (row0 < rows && n0 + c * 64 < cols) store(&maps.out[half], packed, n0 + c * 64, row0);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote_cta_scope(mapa_shared(smem_u32(&bars.tmem_empty[buf]), 0));
        }
        if (lane == 0) tma_store_wait_all<0>();
    }

    // ---------------------------------------------------------------------- teardown
    if (*bars.abort_flag != 0) {
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) { }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();   // neither CTA frees TMEM or exits while the peer can still touch it
    if (warp_id == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, Cfg::kTmemCols);
    }
}

// ---------------------------------------------------------------------- elementwise part of the backward pass

constexpr int kGateRows = 64;   // tokens per CTA
constexpr int kMaxima = 1000;   // CTAs that look for the largest gradient, at most

// dg and du of an element
__device__ __forceinline__ float2 gate_gradients(float dh, float g, float u) {
    const float s = __fdividef(1.f, 1.f + __expf(-g));
    return make_float2(dh * u * s * (1.f + g * (1.f - s)), dh * g * s);
}

template <typename T>
struct Loaded {   // 8 neighbouring elements
    uint4 d;
    float4 g[2], u[2];
    __device__ __forceinline__ float2 gradients(int i) const {
        const float4 a = g[i / 4], b = u[i / 4];
        const int e = i % 4;
        return gate_gradients(to_float(reinterpret_cast<const T*>(&d)[i]), e == 0 ? a.x : e == 1 ? a.y : e == 2 ? a.z : a.w,
                              e == 0 ? b.x : e == 1 ? b.y : e == 2 ? b.z : b.w);
    }
};

__device__ __forceinline__ float block_max(float v) {   // of 256 threads, for all of them
    __shared__ float warp_max[8];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = v;
    __syncthreads();
    v = warp_max[0];
#pragma unroll
    for (int i = 1; i < 8; i++) v = fmaxf(v, warp_max[i]);
    return v;
}

// maxima[CTA] = the largest finite |dg| or |du| of the CTA's share of `pieces` of 8 elements. Bound by HBM (10 bytes an
// element). From the end to the beginning, where gate_backward_kernel starts: what is read last it finds in L2.
template <typename T>
__global__ void __launch_bounds__(256)
gate_maxima_kernel(const T* __restrict__ dh, const float* __restrict__ gate, const float* __restrict__ up,
                   float* __restrict__ maxima, long long pieces) {
    float most = 0.f;
    const long long step = (long long)gridDim.x * 256;
    for (long long p = (long long)blockIdx.x * 256 + threadIdx.x; p < pieces; p += 2 * step) {
        const bool two = p + step < pieces;   // two at a time, so that 160 bytes a thread are under way
        Loaded<T> v[2];
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (k == 0 || two) {
                const long long at = pieces - 1 - (p + k * step);
                v[k].d = __ldg(reinterpret_cast<const uint4*>(dh) + at);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    v[k].g[h] = __ldg(reinterpret_cast<const float4*>(gate) + 2 * at + h);
                    v[k].u[h] = __ldg(reinterpret_cast<const float4*>(up) + 2 * at + h);
                }
            }
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (k == 0 || two) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float2 d = v[k].gradients(i);
                    const float a = fabsf(d.x), b = fabsf(d.y);
                    if (a < __int_as_float(0x7f800000)) most = fmaxf(most, a);   // infinities and NaNs stay what they are
                    if (b < __int_as_float(0x7f800000)) most = fmaxf(most, b);
                }
            }
    }
    most = block_max(most);
    if (threadIdx.x == 0) maxima[blockIdx.x] = most;
}

// A CTA takes 256 channels x kGateRows tokens: 32 threads across (8 channels each), 8 down. Bound by HBM (14 bytes an
// element). BIAS: per-CTA column sums into part (2, row chunks, N), reduced by sum_parts_kernel. fp16: dg and du are stored
// times the power of two that the maxima ask for, whose inverse goes to `unscale`.
template <typename T, bool BIAS>
__global__ void __launch_bounds__(256)
gate_backward_kernel(const T* __restrict__ dh, const float* __restrict__ gate, const float* __restrict__ up,
                     T* __restrict__ dg, T* __restrict__ du, float* __restrict__ part, const float* __restrict__ maxima,
                     int num_maxima, float* __restrict__ unscale, int M, int N) {
    constexpr bool SCALED = std::is_same<T, __half>::value;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int n = (blockIdx.x * 32 + tx) * 8;
    const long long m0 = (long long)blockIdx.y * kGateRows;
    float scale = 1.f;
    if constexpr (SCALED) {
        float most = 0.f;
        for (int i = threadIdx.x; i < num_maxima; i += 256) most = fmaxf(most, maxima[i]);
        most = block_max(most);
        // both powers stay normal numbers
        const int e = most > 0.f ? min(14 - ((int)(__float_as_uint(most) >> 23) - 127), 126) : 0;
        scale = __uint_as_float((uint32_t)(127 + e) << 23);
        if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *unscale = __uint_as_float((uint32_t)(127 - e) << 23);
    }
    float sg[8] = {}, su[8] = {};
    if (n < N) {
        // two rows at a time, so that 160 bytes a thread are under way
        for (int r0 = ty; r0 < kGateRows && m0 + r0 < M; r0 += 16) {
            const bool two = r0 + 8 < kGateRows && m0 + r0 + 8 < M;
            Loaded<T> v[2];
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (k == 0 || two) {
                    const size_t at = (size_t)(m0 + r0 + 8 * k) * N + n;
                    v[k].d = __ldcs(reinterpret_cast<const uint4*>(dh + at));
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        v[k].g[h] = __ldcs(reinterpret_cast<const float4*>(gate + at) + h);
                        v[k].u[h] = __ldcs(reinterpret_cast<const float4*>(up + at) + h);
                    }
                }
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (k == 0 || two) {
                    const size_t at = (size_t)(m0 + r0 + 8 * k) * N + n;
                    float a[8], b[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float2 d = v[k].gradients(i);
                        if (BIAS) {
                            sg[i] += d.x;
                            su[i] += d.y;
                        }
                        a[i] = SCALED ? d.x * scale : d.x;
                        b[i] = SCALED ? d.y * scale : d.y;
                    }
                    *reinterpret_cast<uint4*>(dg + at) = make_uint4(pack2<T>(a[0], a[1]), pack2<T>(a[2], a[3]),
                                                                    pack2<T>(a[4], a[5]), pack2<T>(a[6], a[7]));
                    *reinterpret_cast<uint4*>(du + at) = make_uint4(pack2<T>(b[0], b[1]), pack2<T>(b[2], b[3]),
                                                                    pack2<T>(b[4], b[5]), pack2<T>(b[6], b[7]));
                }
        }
    }
    if constexpr (BIAS) {
        __shared__ float sum[2][8][32 * 9];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            sum[0][ty][tx * 9 + i] = sg[i];
            sum[1][ty][tx * 9 + i] = su[i];
        }
        __syncthreads();
        const int c = threadIdx.x;   // one of the 256 channels
        const int at = (c >> 3) * 9 + (c & 7);
        const int col = blockIdx.x * 256 + c;
        if (col < N) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                float v = 0.f;
#pragma unroll
                for (int r = 0; r < 8; r++) v += sum[k][r][at];
                part[((size_t)k * gridDim.y + blockIdx.y) * N + col] = v;
            }
        }
    }
}

// out[k][n] = sum over `chunks` rows of part[k][.][n], k = blockIdx.y; 32 channels x 8 interleaved partial sums a CTA
template <typename T>
__global__ void __launch_bounds__(256)
sum_parts_kernel(const float* __restrict__ part, T* __restrict__ dbg, T* __restrict__ dbu, int chunks, int N) {
    __shared__ float s[8][32];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, n = blockIdx.x * 32 + tx;
    float v = 0.f;
    if (n < N)
        for (int c = ty; c < chunks; c += 8) v += part[((size_t)blockIdx.y * chunks + c) * N + n];
    s[ty][tx] = v;
    __syncthreads();
    T* out = blockIdx.y == 0 ? dbg : dbu;
    if (ty == 0 && n < N && out != nullptr) {
        float r = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) r += s[i][tx];
        out[n] = from_float<T>(r);
    }
}

// ---------------------------------------------------------------------- host

template <int MODE, bool BF16>
int launch_pair(const Maps& maps, const void* bg, const void* bu, int rows, int cols, int kb1, int kbs,
                const float* unscale, cudaStream_t stream) {
    static int max_pairs[64] = {};
    constexpr int TILE_N = MODE <= kForwardSave ? 128 : 256;
    const long long tiles = ((long long)rows + 255) / 256 * (MODE == kDw ? 2 : 1) * (((long long)cols + TILE_N - 1) / TILE_N);
    int* status = status_word();
    if (status == nullptr) return kLaunchFailed;
    return launch_pairs16(gated_pair_kernel<MODE, BF16>, kThreads, tiles, stream, max_pairs, maps, bg, bu, rows, cols, kb1,
                          kbs, unscale, status);
}

inline size_t pad256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }
inline int row_chunks(int M) { return (M + kGateRows - 1) / kGateRows; }

template <typename T>
int gate_backward(const void* dh, const float* g, const float* u, void* dg, void* du, float* part, float* maxima,
                  float* unscale, void* dbg, void* dbu, int M, int N, cudaStream_t stream) {
    const dim3 grid((N + 255) / 256, row_chunks(M), 1);
    if (grid.y > 65535) return kTooLarge;
    const T* d = static_cast<const T*>(dh);
    T *a = static_cast<T*>(dg), *b = static_cast<T*>(du);
    int num_maxima = 0;
    if constexpr (std::is_same<T, __half>::value) {
        const long long pieces = (long long)M * N / 8;
        num_maxima = (int)std::min<long long>((pieces + 511) / 512, std::min(4 * sm_count(), kMaxima));
        gate_maxima_kernel<T><<<num_maxima, 256, 0, stream>>>(d, g, u, maxima, pieces);
        if (cudaGetLastError() != cudaSuccess) return kLaunchFailed;
    }
    if (dbg != nullptr || dbu != nullptr) {
        gate_backward_kernel<T, true><<<grid, 256, 0, stream>>>(d, g, u, a, b, part, maxima, num_maxima, unscale, M, N);
        if (cudaGetLastError() != cudaSuccess) return kLaunchFailed;
        sum_parts_kernel<T><<<dim3((N + 31) / 32, 2, 1), 256, 0, stream>>>(part, static_cast<T*>(dbg), static_cast<T*>(dbu),
                                                                          (int)grid.y, N);
    } else {
        gate_backward_kernel<T, false><<<grid, 256, 0, stream>>>(d, g, u, a, b, part, maxima, num_maxima, unscale, M, N);
    }
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
}

}  // namespace

int gated_linear(const void* x, const void* wg, const void* wu, const void* bg, const void* bu, void* h, float* g,
                 float* u, int M, int K, int N, bool bf16, cudaStream_t stream) {
    // a few tokens: one pass over the weights without tensor-memory tiles that would be mostly empty (14336 x 4096: 39
    // against 51 us at 1 token, 48 against 51 at 16)
    if (g == nullptr && M <= 16) return gated_stream(x, wg, wu, bg, bu, h, M, K, N, bf16, stream);
    Maps m = {};
    const CUtensorMapDataType t = type16(bf16), f = CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    if (!encode_sw128(&m.a[0], t, 2, x, K, M, 128) || !encode_sw128(&m.b[0], t, 2, wg, K, N, 128) ||
        !encode_sw128(&m.b[1], t, 2, wu, K, N, 128) || !encode_sw128(&m.out[0], t, 2, h, N, M, 32))
        return kLaunchFailed;
    if (g != nullptr && (!encode_sw128(&m.save[0], f, 4, g, N, M, 32) || !encode_sw128(&m.save[1], f, 4, u, N, M, 32)))
        return kLaunchFailed;
    const int kbs = (K + 63) / 64;
    if (g != nullptr)
        return bf16 ? launch_pair<kForwardSave, true>(m, bg, bu, M, N, kbs, kbs, nullptr, stream)
                    : launch_pair<kForwardSave, false>(m, bg, bu, M, N, kbs, kbs, nullptr, stream);
    return bf16 ? launch_pair<kForward, true>(m, bg, bu, M, N, kbs, kbs, nullptr, stream)
                : launch_pair<kForward, false>(m, bg, bu, M, N, kbs, kbs, nullptr, stream);
}

size_t gated_linear_backward_workspace(int M, int N) {
    return 2 * pad256((size_t)M * N * 2) + pad256((size_t)2 * row_chunks(M) * N * sizeof(float)) +
           pad256((kMaxima + 1) * sizeof(float));
}

int gated_linear_backward(const void* dh, const void* x, const void* wg, const void* wu, const float* g, const float* u,
                          void* dx, void* dwg, void* dwu, void* dbg, void* dbu, int M, int K, int N, bool bf16,
                          void* workspace, cudaStream_t stream) {
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    void* dg = ws;
    void* du = ws + pad256((size_t)M * N * 2);
    float* part = reinterpret_cast<float*>(ws + 2 * pad256((size_t)M * N * 2));
    float* unscale = part + pad256((size_t)2 * row_chunks(M) * N * sizeof(float)) / sizeof(float);
    float* maxima = unscale + 1;
    int r = bf16 ? gate_backward<__nv_bfloat16>(dh, g, u, dg, du, part, maxima, unscale, dbg, dbu, M, N, stream)
                 : gate_backward<__half>(dh, g, u, dg, du, part, maxima, unscale, dbg, dbu, M, N, stream);
    if (r != kOk) return r;
    const CUtensorMapDataType t = type16(bf16);
    if (dx != nullptr) {
        Maps m = {};
        if (!encode_sw128(&m.a[0], t, 2, dg, N, M, 128) || !encode_sw128(&m.a[1], t, 2, du, N, M, 128) ||
            !encode_sw128(&m.b[0], t, 2, wg, K, N, 64) || !encode_sw128(&m.b[1], t, 2, wu, K, N, 64) ||
            !encode_sw128(&m.out[0], t, 2, dx, K, M, 32))
            return kLaunchFailed;
        const int kb = (N + 63) / 64;
        r = bf16 ? launch_pair<kDx, true>(m, nullptr, nullptr, M, K, kb, 2 * kb, unscale, stream)
                 : launch_pair<kDx, false>(m, nullptr, nullptr, M, K, kb, 2 * kb, unscale, stream);
        if (r != kOk) return r;
    }
    if (dwg != nullptr) {
        Maps m = {};
        if (!encode_sw128(&m.a[0], t, 2, dg, N, M, 64) || !encode_sw128(&m.a[1], t, 2, du, N, M, 64) ||
            !encode_sw128(&m.b[0], t, 2, x, K, M, 64) || !encode_sw128(&m.out[0], t, 2, dwg, K, N, 32) ||
            !encode_sw128(&m.out[1], t, 2, dwu, K, N, 32))
            return kLaunchFailed;
        const int kb = (M + 63) / 64;
        r = bf16 ? launch_pair<kDw, true>(m, nullptr, nullptr, N, K, kb, kb, unscale, stream)
                 : launch_pair<kDw, false>(m, nullptr, nullptr, N, K, kb, kb, unscale, stream);
    }
    return r;
}

}  // namespace fb200
