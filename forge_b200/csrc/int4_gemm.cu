// Linear layers on 4-bit weights for many tokens: CTA-pair tcgen05 GEMM (cta_group::2, kind::f16) whose weight operand
// is made in the kernel.
//
//   plain:  out[m][n] = sum_k x[m][k] w[n][k] + b[n]            w[n][k] = s[k / G][n] q[n][k]
//   gated:  out[m][n] = SiLU(g) u, g = x Wg^T + bg, u = x Wu^T + bu
//
// The skeleton of the other pair kernels (256 tokens x BN weight rows per pair), with the weight's TMA producer replaced by
// twelve warps per CTA that read packed weights from L2, multiply the integers by their scales and write 16-bit numbers
// in the swizzled layout that the tensor cores read; nothing of the unpacked weight ever reaches memory. A stage is a
// whole block of 128 inputs (three of 64 KB). Making one takes longer than the tensor cores need for it, so each stage has
// four warps of its own, three blocks being made at a time; the warps signal a barrier of their own CTA only, and one
// thread passes CTA 1's on to the leader (with eight warps on each 64-deep slab in turn and arrivals across the cluster,
// 2048 x 4096 x 11008 took 308 us; 142 us like this).
//
// s q has more bits than a 16-bit number. Plain calls round it once, which with the rounding of the output makes 1.4 times
// (fp16: 1.25 times) the error of the latter. Behind the gate two such products would meet and make it 1.7 times, so
// gated calls take both parts: CTA 0 makes the rounded weights and CTA 1 what the rounding left, which is exact, for the
// same 64 rows of both matrices; their products lie in neighbouring accumulator columns and are added in the epilogue.
// That is twice the tensor work (333 tokens, 4096 x 14336 twice: 190 us instead of 114) and no error beyond fp32 sums.
//
// Beyond 128 tokens: 2048 x 4096 x 11008 142 us (1300 TFLOP/s, tensor pipe 71 % busy), 4096 x 4096 x 11008 285 us; gated,
// 4096 -> 14336, 2048 tokens 705 us (74 %) and 8192 tokens 2.8-3.0 ms (1300 TFLOP/s, half of them the rest's). A block takes
// 0.88 us where its tensor instructions take 0.55: a stage is refilled once they are done with it, and 192 KB are three.
// Weights made in registers ahead of the stage do not help (156 us: the registers spill; of what is here, 96 registers a
// thread, the gated kernel spills 68 to 72 bytes, the plain one 8 to 32, the kernel for 17 to 128 tokens 102 to 136 with
// 128 columns and up to 46 with fewer).
// The kernel for 17 to 128 tokens is described below. It pays up to 128, apart from its sums: at 65 to 96 tokens 31 us
// against 34 here with 11008 x 4096 and groups of 128 (with groups of 32 50), 45 against 95 with 4096 x 14336, gated 67
// against 115; at 128 tokens 34 on both sides, 48 against 95 and 78 against 117.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "float_common.cuh"
#include "gemm_dense.cuh"
#include "int4.cuh"
#include "pair16.cuh"
#include "ptx.cuh"

namespace fb200 {

using namespace pair16;

namespace {

constexpr int kRing = 3;          // stages: two 64-deep slabs of both operands each
constexpr int kGroupWarps = 4;    // that make a stage's weights
constexpr int kWeightWarps = kRing * kGroupWarps;
constexpr int kSlab = Cfg::kOperandBytes;
constexpr int kTokensMax = 128;   // tokens up to which weight rows are the tensor cores' lanes

struct RingBars {
    uint64_t *full, *empty, *made, *tmem_full, *tmem_empty;
    uint32_t* tmem_slot;
    volatile int* abort_flag;
};
__device__ __forceinline__ RingBars carve_ring(uint8_t* p) {
    RingBars b;
    b.full = reinterpret_cast<uint64_t*>(p);   // in the leader: both CTAs' activations, its weight warps, CTA 1's relay
    b.empty = b.full + kRing;                  // one per CTA, committed by the leader's MMA thread
    b.made = b.empty + kRing;                  // in CTA 1: its weight warps
    b.tmem_full = b.made + kRing;              // one per CTA
    b.tmem_empty = b.tmem_full + 2;            // in the leader: both CTAs' epilogue warps
    b.tmem_slot = reinterpret_cast<uint32_t*>(b.tmem_empty + 2);
    b.abort_flag = reinterpret_cast<volatile int*>(b.tmem_slot + 1);
    return b;
}
constexpr int kThreads = 32 * (2 + kEpiWarps + kWeightWarps);   // TMA warp, MMA warp, epilogue, weights

// Word of 8 four-bit weights -> the integers q as 8 numbers of type T in order. A nibble in the low mantissa bits of 1024
// (fp16) or 128 (bf16) is that number plus the nibble, exactly; subtracting the offset + 8 leaves q, exactly.
__device__ __forceinline__ void unpack_q(uint32_t w, __half2 (&q)[4]) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t v = w >> (8 * i);
        const uint32_t lo = and_or(v, 0x000F000Fu, 0x64006400u), hi = and_or(v, 0x00F000F0u, 0x64006400u);
        q[2 * i] = __hsub2(reinterpret_cast<const __half2&>(lo), __half2half2(__ushort_as_half(0x6408)));
        q[2 * i + 1] = __hfma2(reinterpret_cast<const __half2&>(hi), __half2half2(__ushort_as_half(0x2C00)),
                               __half2half2(__ushort_as_half(0xD480)));   // / 16 - 72
    }
}
// SHIFT: q 2^-SHIFT
template <int SHIFT = 0>
__device__ __forceinline__ void unpack_q(uint32_t w, __nv_bfloat162 (&q)[4]) {
    constexpr uint32_t kOffset = 0x4300 - (SHIFT << 7), kOffset8 = kOffset + 8;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t b = and_or(w >> (4 * i), 0x000F000Fu, kOffset * 0x10001u);
        q[i] = __hsub2(reinterpret_cast<const __nv_bfloat162&>(b), __bfloat162bfloat162(__ushort_as_bfloat16(kOffset8)));
    }
}
template <typename V>
__device__ __forceinline__ uint4 bits4(const V (&v)[4]) {
    return make_uint4(reinterpret_cast<const uint32_t&>(v[0]), reinterpret_cast<const uint32_t&>(v[1]),
                      reinterpret_cast<const uint32_t&>(v[2]), reinterpret_cast<const uint32_t&>(v[3]));
}

// A word's weights s q rounded to T, or (`rest`) what that rounding left, exactly.
template <typename T>
struct Scaled;
template <>
struct Scaled<__half> {
    __half2 s;
    __device__ __forceinline__ explicit Scaled(unsigned short bits) : s(__half2half2(__ushort_as_half(bits))) {}
    __device__ __forceinline__ uint4 operator()(uint32_t w, bool rest) const {
        __half2 q[4];
        unpack_q(w, q);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __half2 v = __hmul2(q[i], s);
            q[i] = rest ? __hfma2(q[i], s, __hneg2(v)) : v;   // a multiple of 2^-24 as s is, so never out of range below
        }
        return bits4(q);
    }
};
template <>
struct Scaled<__nv_bfloat16> {
    __nv_bfloat162 hi, lo;   // s = hi + lo; their products with q are exact
    __device__ __forceinline__ explicit Scaled(unsigned short bits) {
        const float s = __half2float(__ushort_as_half(bits));
        const __nv_bfloat16 h = __float2bfloat16_rn(s);
        hi = __bfloat162bfloat162(h);
        lo = __bfloat162bfloat162(__float2bfloat16_rn(s - __bfloat162float(h)));
    }
    __device__ __forceinline__ uint4 operator()(uint32_t w, bool rest) const {
        __nv_bfloat162 q[4];
        unpack_q(w, q);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 small = __hmul2(q[i], lo), v = __hfma2(q[i], hi, small);
            q[i] = rest ? __hadd2(__hfma2(q[i], hi, __hneg2(v)), small) : v;
        }
        return bits4(q);
    }
};

// One thread of CTA 1: tells the leader, stage after stage, that CTA 1's half of the weights is there.
__device__ __forceinline__ void relay(const RingBars& bars, long long turns, int* status) {
    int stage = 0;
    uint32_t phase = 0;
    for (long long i = 0; i < turns; i++) {
        if (!mbar_wait(&bars.made[stage], phase, bars.abort_flag)) {
            atomicExch(status, 856);
            return;
        }
        mbar_arrive_cluster(mapa_shared(smem_u32(&bars.full[stage]), 0));
        if (++stage == kRing) {
            stage = 0;
            phase ^= 1;
        }
    }
}

// BN: rows of the pair's weight operand (256 or 128); GATED 256: 64 rows of each matrix, rounded and rest.
template <typename T, int G, bool GATED, int BN>
__global__ void __launch_bounds__(kThreads, 1)
int4_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_out,
                 const uint8_t* __restrict__ w0, const uint8_t* __restrict__ w1, const __half* __restrict__ s0,
                 const __half* __restrict__ s1, const T* __restrict__ b0, const T* __restrict__ b1, T* __restrict__ out,
                 int M, int N, int K, int tma_out, int* __restrict__ status) {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    static_assert(!GATED || BN == 256, "the gated tile");
    constexpr int TILE_N = GATED ? BN / 4 : BN;   // output columns
    constexpr int HALF = BN / 2;                  // weight rows that a CTA makes
    constexpr int PER = 128 / G;
    extern __shared__ __align__(1024) uint8_t smem[];
    static_assert(kRing * 4 * kSlab == Cfg::kStages * Cfg::kStageBytes, "the shared-memory plan of Cfg");
    uint8_t* smem_epi = smem + kRing * 4 * kSlab;   // a stage: activations of both slabs, weights of both
    float* smem_bias = reinterpret_cast<float*>(smem_epi + Cfg::kEpiBytes);
    const RingBars bars = carve_ring(smem_epi + Cfg::kEpiBytes + Cfg::kBiasBytes);

    const int warp_id = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    if ((smem_u32(smem) & 1023u) != 0) {   // the same in both CTAs
        if (threadIdx.x == 0) atomicExch(status, 850);
        return;
    }
    const int a_blocks = (M + 255) / 256, b_blocks = (N + TILE_N - 1) / TILE_N;
    const int num_tiles = a_blocks * b_blocks;
    const int blocks = (K + 127) / 128;
    const int pair_id = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kRing; s++) {
            mbar_init(&bars.full[s], 1 + kGroupWarps + 1);
            mbar_init(&bars.empty[s], 1);
            mbar_init(&bars.made[s], kGroupWarps);
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

    if (warp_id == 0) {
        // ------------------------------------------------------------------ activations (TMA)
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = pair_id; t < num_tiles && ok; t += num_pairs) {
                const Tile tc = tile_of(t, a_blocks, b_blocks);
                for (int blk = 0; blk < blocks; blk++) {
                    if (!mbar_wait(&bars.empty[stage], phase ^ 1, bars.abort_flag)) {
                        atomicExch(status, 851);
                        ok = false;
                        break;
                    }
                    if (leader) mbar_expect_tx(&bars.full[stage], 4 * kSlab);
                    const uint32_t full = mapa_shared(smem_u32(&bars.full[stage]), 0);
                    uint8_t* dst = smem + stage * 4 * kSlab;
                    tma_load_2d_pair(dst, &tm_x, full, blk * 128, tc.a_blk * 256 + (int)rank * 128);
                    tma_load_2d_pair(dst + kSlab, &tm_x, full, blk * 128 + 64, tc.a_blk * 256 + (int)rank * 128);
                    if (++stage == kRing) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        }
    } else if (warp_id == 1) {
        // ------------------------------------------------------------------ MMA issuer (leader only)
        if (leader && lane == 0) {
            constexpr uint32_t idesc = idesc_f16(256, BN, BF16, false, false);
            int stage = 0;
            uint32_t phase = 0;
            int local = 0;
            bool ok = true;
            for (int t = pair_id; t < num_tiles && ok; t += num_pairs, local++) {
                const int buf = local & 1;
                if (!mbar_wait(&bars.tmem_empty[buf], ((local >> 1) & 1) ^ 1, bars.abort_flag)) {
                    atomicExch(status, 852);
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t acc = tmem_base + buf * 256;
                for (int blk = 0; blk < blocks; blk++) {
                    // cluster scope: the other CTA's relay signals this barrier with a plain arrival
                    if (!mbar_wait_cluster(&bars.full[stage], phase, bars.abort_flag)) {
                        atomicExch(status, 853);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sa = smem_u32(smem + stage * 4 * kSlab);
                    const uint64_t da = make_desc_sw128(sa), db = make_desc_sw128(sa + 2 * kSlab);
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const int step = (k / 4) * (kSlab >> 4) + 2 * (k % 4);
                        umma_f16_pair(acc, da + step, db + step, idesc, (blk | k) != 0 ? 1u : 0u);
                    }
                    tc_commit_pair_mask(smem_u32(&bars.empty[stage]), 3);
                    if (++stage == kRing) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (ok) tc_commit_pair_mask(smem_u32(&bars.tmem_full[buf]), 3);
            }
        } else if (!leader && lane == 0) {
            relay(bars, (long long)((num_tiles - pair_id + num_pairs - 1) / num_pairs) * blocks, status);
        }
    } else if (warp_id >= 2 + kEpiWarps) {
        // ------------------------------------------------------------------ weights (both CTAs)
        // A lane makes a quarter (16 packed bytes: runs t, 4 + t, 8 + t, 12 + t) of a block of two or four rows. Rows go to
        // lanes so that eight lanes write all banks.
        constexpr int ROWS = HALF / (8 * kGroupWarps);
        const int t4 = lane & 3;
        const int row8 = (lane >> 3) | ((lane >> 2) & 1) << 2;
        const int group = (warp_id - 2 - kEpiWarps) / kGroupWarps;
        const int local_row = (warp_id - 2 - kEpiWarps) % kGroupWarps * 8 + row8;
        const int groups = (K + G - 1) / G;
        // Every third block of those that the CTA goes through, always into the same stage: a barrier's parity tells a lap
        // from its neighbours only, so whoever waits on it has to see every lap.
        const int stage = group;
        uint32_t phase = 0;
        bool ok = true;
        int blk = group;     // in its tile
        for (int t = pair_id; t < num_tiles && ok; t += num_pairs) {
            const Tile tc = tile_of(t, a_blocks, b_blocks);
            const uint8_t* wp[ROWS];
            const unsigned short* sp[ROWS];
#pragma unroll
            for (int i = 0; i < ROWS; i++) {
                const bool second = GATED && i >= ROWS / 2;   // gated: 64 rows of Wg, then the same of Wu
                const int r = local_row + 8 * kGroupWarps * (GATED ? i % (ROWS / 2) : i);
                const int row = min(tc.b_blk * TILE_N + (GATED ? 0 : (int)rank * HALF) + r, N - 1);
                wp[i] = (second ? w1 : w0) + (size_t)row * ((size_t)blocks * 64) + t4 * 16;
                sp[i] = reinterpret_cast<const unsigned short*>(second ? s1 : s0) + row;
            }
            uint4 next[ROWS];
            unsigned short next_s[ROWS][PER];
            auto load = [&](int b) {
#pragma unroll
                for (int i = 0; i < ROWS; i++) {
                    next[i] = __ldg(reinterpret_cast<const uint4*>(wp[i] + (size_t)b * 64));
#pragma unroll
                    for (int k = 0; k < PER; k++) next_s[i][k] = __ldg(sp[i] + (size_t)min(b * PER + k, groups - 1) * N);
                }
            };
            if (blk < blocks) load(blk);
            for (; blk < blocks; blk += kRing) {
                uint4 cur[ROWS];
                unsigned short cur_s[ROWS][PER];
#pragma unroll
                for (int i = 0; i < ROWS; i++) {
                    cur[i] = next[i];
#pragma unroll
                    for (int k = 0; k < PER; k++) cur_s[i][k] = next_s[i][k];
                }
                load(min(blk + kRing, blocks - 1));
                ok = __all_sync(0xffffffffu, mbar_wait(&bars.empty[stage], phase ^ 1, bars.abort_flag));
                if (!ok) {
                    if (lane == 0) atomicExch(status, 854);
                    break;
                }
                phase ^= 1;
                uint8_t* dst = smem + stage * 4 * kSlab + 2 * kSlab + local_row * 128;
#pragma unroll
                for (int i = 0; i < ROWS; i++) {
                    const uint32_t word[4] = {cur[i].x, cur[i].y, cur[i].z, cur[i].w};
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        *reinterpret_cast<uint4*>(dst + (j / 2) * kSlab + i * (8 * kGroupWarps * 128) +
                                                  (((4 * (j % 2) + t4) ^ row8) << 4)) =
                            Scaled<T>(cur_s[i][j * 32 / G])(word[j], GATED && rank == 1);
                }
                fence_proxy_async_smem();   // the tensor cores read through the async proxy
                __syncwarp();
                if (lane == 0) mbar_arrive(leader ? &bars.full[stage] : &bars.made[stage]);
            }
            blk -= blocks;
        }
    } else {
        // ------------------------------------------------------------------ epilogue (both CTAs)
        const int q = warp_id & 3;
        const int epi_tid = (warp_id - 2) * 32 + lane;
        uint8_t* my_stage = smem_epi + (warp_id - 2) * Cfg::kEpiBufs * Cfg::kEpiBufBytes;
        const uint64_t policy = l2_policy_evict_first();   // outputs must not push operands out of L2
        int sbuf = 0, local = 0;
        bool ok = true;
        for (int t = pair_id; t < num_tiles; t += num_pairs, local++) {
            const Tile tc = tile_of(t, a_blocks, b_blocks);
            const int buf = local & 1;
            const int row0 = tc.a_blk * 256 + (int)rank * 128 + q * 32;
            const int n0 = tc.b_blk * TILE_N;
            float* bias = smem_bias + buf * 256;   // TILE_N of b0; gated: then TILE_N of b1
            for (int i = epi_tid; i < (GATED ? 2 : 1) * TILE_N; i += kEpiThreads) {
                const int n = n0 + i % TILE_N;
                const T* b = i < TILE_N ? b0 : b1;
                bias[i] = b != nullptr && n < N ? to_float(b[n]) : 0.f;
            }
            named_barrier_sync(1, kEpiThreads);
            if (ok) {
                ok = __all_sync(0xffffffffu, mbar_wait(&bars.tmem_full[buf], (local >> 1) & 1, bars.abort_flag));
                if (!ok) atomicExch(status, 855);
            }
            if (!ok) continue;
            tc_fence_after();
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * 256;
#pragma unroll 1
            for (int c = 0; c < TILE_N / 64; c++) {
                uint32_t packed[32];
#pragma unroll
                for (int hh = 0; hh < 4; hh++) {
                    const int col = c * 64 + hh * 16;
                    uint32_t va[16], vb[16];
                    tmem_ld_32x32b_x16(taddr + col, va);
                    if (GATED) {   // gate, up, and the products of what the rounding left
                        uint32_t ra[16], rb[16];
                        tmem_ld_32x32b_x16(taddr + TILE_N + col, vb);
                        tmem_ld_32x32b_x16(taddr + 2 * TILE_N + col, ra);
                        tmem_ld_32x32b_x16(taddr + 3 * TILE_N + col, rb);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            va[i] = __float_as_uint(__uint_as_float(va[i]) + __uint_as_float(ra[i]));
                            vb[i] = __float_as_uint(__uint_as_float(vb[i]) + __uint_as_float(rb[i]));
                        }
                    } else {
                        tmem_ld_wait();
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        float o[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            o[e] = __uint_as_float(va[2 * i + e]) + bias[col + 2 * i + e];
                            if (GATED) o[e] = silu_mul(o[e], __uint_as_float(vb[2 * i + e]) + bias[TILE_N + col + 2 * i + e]);
                        }
                        packed[hh * 8 + i] = pack2<T>(o[0], o[1]);
                    }
                }
                if (row0 >= M || n0 + c * 64 >= N) continue;   // nothing to store; a box must not start outside
                uint8_t* stg = my_stage + sbuf * Cfg::kEpiBufBytes;
                if (lane == 0) tma_store_wait_read<Cfg::kEpiBufs - 1>();
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; j++)
                    *reinterpret_cast<uint4*>(stg + lane * 128 + (j ^ (lane & 7)) * 16) =
                        make_uint4(packed[4 * j], packed[4 * j + 1], packed[4 * j + 2], packed[4 * j + 3]);
                if (tma_out) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d_hint(&tm_out, stg, n0 + c * 64, row0, policy);
                        tma_store_commit();
                    }
                } else {   // rows that are no multiple of 16 bytes: two neighbouring columns a lane, row after row
                    __syncwarp();
                    const int n = n0 + c * 64 + 2 * lane;
                    for (int r = 0; r < 32 && row0 + r < M; r++) {
                        const T* v = reinterpret_cast<const T*>(stg + r * 128 + ((lane >> 2) ^ (r & 7)) * 16 + (lane & 3) * 4);
                        T* o = out + (size_t)(row0 + r) * N + n;
                        if (n < N) o[0] = v[0];
                        if (n + 1 < N) o[1] = v[1];
                    }
                }
                sbuf = (sbuf + 1) % Cfg::kEpiBufs;
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

// Up to 128 tokens: the operands change places. Weight rows are the lanes, tokens the columns, as many as there are (`cols`,
// a multiple of 32), so the tensor instructions shrink with the batch, and what bounds the call is how fast weights become
// operands. One CTA per tile of `rows` rows (gated: of each matrix, Wg in lanes 0-63 and Wu in lanes 64-127), chosen so
// that all SMs have the same number; rows beyond it are stale shared memory in accumulator lanes of their own, not stored.
// A tensor instruction of so few columns takes 75 clocks however few there are, so a tile costs 600 clocks a block of 128
// inputs; where 128-row tiles leave SMs free, a cluster of CTAs divides a tile's inputs, and sums its parts through
// distributed shared memory, in rank order (64 tokens, 4096 x 14336: 61 us without, 25 with; 4096 x 4096: 21 and 13).
//
// With so few columns there is time to keep the sums exact: the operand holds the integers, every group of inputs has
// accumulator columns of its own (a ring of four or eight), and eight warps multiply them by the scale of their lane's
// row and add them up in registers, in fp32. Nothing is rounded before the result. A block's groups are waited for and
// released together; what sums cost otherwise is registers: 32 columns where there are no more tokens, and as few scales ahead
// as hide a load (11008 x 4096, groups of 32, 64 tokens: 51 us without these, 28 with; 32 tokens: 51 and 22).
//
// 64 tokens, cold weights: 11008 x 4096 22 us, 4096 x 14336 25 us, gated 14336 x 4096 twice 45 us (floors 4, 5 and 9): the
// conversion of the weights and the per-block work of the issuers and sums take the time, not the memory.
//
// Waiting for three barriers and issuing eight tensor instructions, one after the other, takes a thread twice the time of
// the instructions, so two threads issue, one every other block (64 tokens, 11008 x 4096: 31 us with one, 22 with two).
// Rings have even numbers of stages: a barrier's parity tells a lap from its neighbours only, so whoever waits on one has
// to see every lap of it.
struct TokenBars {
    uint64_t *full_w, *empty_w;   // [kTokenRing]: the stage's weight warps; committed by the MMA thread
    uint64_t *full_x, *empty_x;   // [kMaxRingX]
    uint64_t *tmem_full, *tmem_empty;   // [kMaxAccs], one for each set of accumulators
    uint32_t* tmem_slot;
    volatile int* abort_flag;
};
constexpr int kMaxRingX = 8;
constexpr int kMaxAccs = 8;               // accumulators: 8 of 64 columns, or 4 of 128
constexpr int kTokenRing = 4;             // weight stages
constexpr int kTokenGroupWarps = 2;       // that make a stage's weights
constexpr int kSumWarps = 8;              // two for each quarter of the lanes, half of the columns each
constexpr int kFirstSum = 3;              // warps: TMA, two MMA issuers, sums, weights
constexpr int kFirstWeight = kFirstSum + kSumWarps;
constexpr int kTokenThreads = 32 * (kFirstWeight + kTokenRing * kTokenGroupWarps);
constexpr int kSwapBytes = 32 * 64 * 4;   // gated: the up products of 32 tokens x 64 rows
// bf16: the integers are multiplied as q 2^-11, so that a group's sum, 128 * 8 of the largest activation at most, stays
// below it: no sum overflows before the scale is applied, whatever the activations are.
constexpr int kShift = 11;
__device__ __forceinline__ TokenBars carve_tokens(uint8_t* p) {
    TokenBars b;
    b.full_w = reinterpret_cast<uint64_t*>(p);
    b.empty_w = b.full_w + kTokenRing;
    b.full_x = b.empty_w + kTokenRing;
    b.empty_x = b.full_x + kMaxRingX;
    b.tmem_full = b.empty_x + kMaxRingX;
    b.tmem_empty = b.tmem_full + kMaxAccs;
    b.tmem_slot = reinterpret_cast<uint32_t*>(b.tmem_empty + kMaxAccs);
    b.abort_flag = reinterpret_cast<volatile int*>(b.tmem_slot + 1);
    return b;
}

__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// MAX_COLS: 32, 64 or 128
template <typename T, int G, bool GATED, int MAX_COLS>
__global__ void __launch_bounds__(kTokenThreads, 1)
int4_tokens_kernel(const __grid_constant__ CUtensorMap tm_x, const uint8_t* __restrict__ w0, const uint8_t* __restrict__ w1,
                   const __half* __restrict__ s0, const __half* __restrict__ s1, const T* __restrict__ b0,
                   const T* __restrict__ b1, T* __restrict__ out, int M, int N, int K, int rows, int cols, int ring_x,
                   int split, int* __restrict__ status) {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    constexpr int PER = 128 / G;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int slab_x = cols * 128;
    uint8_t* smem_x = smem + kTokenRing * 2 * kSlab;
    uint8_t* smem_swap = smem_x + ring_x * 2 * slab_x;
    const TokenBars bars = carve_tokens(smem_swap + kSwapBytes);

    const int warp_id = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if ((smem_u32(smem) & 1023u) != 0) {
        if (threadIdx.x == 0) atomicExch(status, 850);
        return;
    }
    const int num_tiles = (N + rows - 1) / rows;
    // a cluster has one tile, a CTA without one takes every gridDim.x-th
    const int rank = split > 1 ? (int)(blockIdx.x % split) : 0;
    const int first_tile = blockIdx.x / split, tile_step = gridDim.x / split;
    const int all_blocks = (K + 127) / 128;
    const int blk0 = (int)((long long)all_blocks * rank / split);                    // of this CTA
    const int blocks = (int)((long long)all_blocks * (rank + 1) / split) - blk0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kTokenRing; s++) {
            mbar_init(&bars.full_w[s], kTokenGroupWarps);
            mbar_init(&bars.empty_w[s], 1);
        }
        for (int s = 0; s < ring_x; s++) {
            mbar_init(&bars.full_x[s], 1);
            mbar_init(&bars.empty_x[s], 1);
        }
        for (int i = 0; i < kMaxAccs; i++) {
            mbar_init(&bars.tmem_full[i], 1);
            mbar_init(&bars.tmem_empty[i], kSumWarps);
        }
        *bars.abort_flag = 0;
        fence_mbar_init();
    }
    if (warp_id == 1) {
        tmem_alloc(bars.tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *bars.tmem_slot;
    // Accumulators change hands in sets: a block's groups, or as many of them as leave another set to work on
    constexpr int accs = MAX_COLS > 64 ? 4 : 8, acc_cols = MAX_COLS;
    constexpr int SET = PER <= accs / 2 ? PER : accs / 2, SETS = accs / SET, BLOCK_SETS = PER / SET;

    if (warp_id == 0) {
        // ------------------------------------------------------------------ activations (TMA)
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = first_tile; t < num_tiles && ok; t += tile_step) {
                for (int blk = 0; blk < blocks; blk++) {
                    if (!mbar_wait(&bars.empty_x[stage], phase ^ 1, bars.abort_flag)) {
                        atomicExch(status, 851);
                        ok = false;
                        break;
                    }
                    uint8_t* dst = smem_x + stage * 2 * slab_x;
                    mbar_expect_tx(&bars.full_x[stage], 2 * slab_x);
                    tma_load_2d(dst, &tm_x, &bars.full_x[stage], (blk0 + blk) * 128, 0);
                    tma_load_2d(dst + slab_x, &tm_x, &bars.full_x[stage], (blk0 + blk) * 128 + 64, 0);
                    if (++stage == ring_x) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        }
    } else if (warp_id == 1 || warp_id == 2) {
        // ------------------------------------------------------------------ MMA issuers: of every other block, or one of all
        // where a block's groups take all accumulators
        constexpr int issuers = accs >= 2 * PER ? 2 : 1;
        if (lane == 0 && warp_id <= issuers) {
            const uint32_t idesc = idesc_f16(128, cols, BF16, false, false);
            const int total = (num_tiles - first_tile + tile_step - 1) / tile_step * blocks;   // blocks of all tiles
            bool ok = true;
            for (int i = warp_id - 1; i < total && ok; i += issuers) {
                const int stage = i % kTokenRing, stage_x = i & (ring_x - 1);
                if (!mbar_wait(&bars.full_x[stage_x], (i / ring_x) & 1, bars.abort_flag) ||
                    !mbar_wait(&bars.full_w[stage], (i / kTokenRing) & 1, bars.abort_flag)) {
                    atomicExch(status, 853);
                    break;
                }
                tc_fence_after();
                const uint64_t da = make_desc_sw128(smem_u32(smem + stage * 2 * kSlab));
                const uint64_t db = make_desc_sw128(smem_u32(smem_x + stage_x * 2 * slab_x));
#pragma unroll
                for (int h = 0; h < BLOCK_SETS; h++) {
                    const int a = i * BLOCK_SETS + h, set = a & (SETS - 1);
                    if (!mbar_wait(&bars.tmem_empty[set], ((a / SETS) & 1) ^ 1, bars.abort_flag)) {
                        atomicExch(status, 852);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
#pragma unroll
                    for (int e = 0; e < SET * (G / 16); e++) {
                        const int step = h * SET * (G / 16) + e;   // of the block's eight
                        umma_f16(tmem_base + (set * SET + e / (G / 16)) * acc_cols,
                                 da + (step / 4) * (kSlab >> 4) + 2 * (step % 4),
                                 db + (step / 4) * (slab_x >> 4) + 2 * (step % 4), idesc, e % (G / 16) != 0 ? 1u : 0u);
                    }
                    tc_commit(&bars.tmem_full[set]);
                }
                tc_commit(&bars.empty_w[stage]);
                tc_commit(&bars.empty_x[stage_x]);
            }
        }
    } else if (warp_id >= kFirstWeight) {
        // ------------------------------------------------------------------ weights, as in int4_pair_kernel, unscaled
        constexpr int ROWS = 128 / (8 * kTokenGroupWarps);   // of a lane; the last ones only where a CTA has so many
        constexpr int STEP = 8 * kTokenGroupWarps;
        const int t4 = lane & 3;
        const int row8 = (lane >> 3) | ((lane >> 2) & 1) << 2;
        const int stage = (warp_id - kFirstWeight) / kTokenGroupWarps;
        const int local_row = (warp_id - kFirstWeight) % kTokenGroupWarps * 8 + row8;
        uint32_t phase = 0;
        bool ok = true;
        int blk = stage;   // of its tile
        // i-th row of a lane: i * STEP + local_row (gated: 64 rows of Wg, then of Wu)
        auto used = [&](int i) { return (GATED ? i % (ROWS / 2) : i) * STEP < rows; };
        for (int t = first_tile; t < num_tiles && ok; t += tile_step) {
            auto row_of = [&](int i) {
                const int row = min(t * rows + (GATED ? i % (ROWS / 2) : i) * STEP + local_row, N - 1);
                return (GATED && i >= ROWS / 2 ? w1 : w0) + (size_t)row * ((size_t)all_blocks * 64) + (size_t)blk0 * 64 + t4 * 16;
            };
            const uint8_t* wp[ROWS];
#pragma unroll
            for (int i = 0; i < ROWS; i++) wp[i] = row_of(i);
            uint4 next[ROWS];
            auto load = [&](int b) {
#pragma unroll
                for (int i = 0; i < ROWS; i++)
                    if (used(i)) next[i] = __ldg(reinterpret_cast<const uint4*>(wp[i] + (size_t)b * 64));
            };
            load(min(blk, blocks - 1));
            for (; blk < blocks; blk += kTokenRing) {
                // All of the next block's loads behind all uses of this one's: a load between two uses makes the second
                // wait for it (870 clocks a row).
                uint4 cur[ROWS];
#pragma unroll
                for (int i = 0; i < ROWS; i++)
                    if (used(i)) cur[i] = next[i];
                load(min(blk + kTokenRing, blocks - 1));
                ok = __all_sync(0xffffffffu, mbar_wait(&bars.empty_w[stage], phase ^ 1, bars.abort_flag));
                if (!ok) {
                    if (lane == 0) atomicExch(status, 854);
                    break;
                }
                phase ^= 1;
                uint8_t* dst = smem + stage * 2 * kSlab + local_row * 128;
#pragma unroll
                for (int i = 0; i < ROWS; i++)
                    if (used(i)) {
                        const uint32_t word[4] = {cur[i].x, cur[i].y, cur[i].z, cur[i].w};
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            typename std::conditional<BF16, __nv_bfloat162, __half2>::type q[4];
                            if constexpr (BF16) unpack_q<kShift>(word[j], q);
                            else unpack_q(word[j], q);
                            *reinterpret_cast<uint4*>(dst + (j / 2) * kSlab + i * (STEP * 128) +
                                                      (((4 * (j % 2) + t4) ^ row8) << 4)) = bits4(q);
                        }
                    }
                fence_proxy_async_smem();   // the tensor cores read through the async proxy
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.full_w[stage]);
            }
            blk -= blocks;
        }
    } else {
        // ------------------------------------------------------------------ sums: a lane has a row's products with half of the tokens
        const int q = warp_id & 3, half = (warp_id - kFirstSum) / 4;
        const int width = cols / 2, col0 = half * width;   // a multiple of 16, at most 64
        float* swap = reinterpret_cast<float*>(smem_swap);
        int set = 0;
        uint32_t phase_set = 0;
        bool ok = true;
        for (int t = first_tile; t < num_tiles; t += tile_step) {
            const int r = GATED ? (q % 2) * 32 + lane : q * 32 + lane;
            const int n = t * rows + r;
            const bool live = r < rows && n < N;
            const T* b = GATED && q >= 2 ? b1 : b0;
            const float bias = live && b != nullptr ? to_float(b[n]) : 0.f;
            const unsigned short* sp = reinterpret_cast<const unsigned short*>(GATED && q >= 2 ? s1 : s0) + min(n, N - 1);
            const int groups = (K + G - 1) / G;
            // Scales of AHEAD blocks, and of the AHEAD behind them under way: a block takes less time than a load, and loads
            // between the uses of earlier ones would make those wait for them.
            constexpr int AHEAD = (MAX_COLS > 32 ? 4 : 8) / PER;   // as the registers allow
            unsigned short now[AHEAD][PER], next[AHEAD][PER];
            auto load = [&](int blk) {
#pragma unroll
                for (int u = 0; u < AHEAD; u++)
#pragma unroll
                    for (int k = 0; k < PER; k++) next[u][k] = __ldg(sp + (size_t)min((blk0 + blk + u) * PER + k, groups - 1) * N);
            };
            load(0);
            constexpr int SUMS = MAX_COLS / 2;
            float sum[SUMS];
#pragma unroll
            for (int i = 0; i < SUMS; i++) sum[i] = 0.f;
            auto add = [&](unsigned short (&scales)[PER]) {   // the products of the next block
#pragma unroll
                for (int h = 0; h < BLOCK_SETS; h++) {
                    ok = ok && __all_sync(0xffffffffu, mbar_wait(&bars.tmem_full[set], phase_set, bars.abort_flag));
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + set * SET * acc_cols + col0;
                    constexpr int CHUNK = SUMS == 32 ? 32 : 16;   // columns at a time, as the registers allow
#pragma unroll
                    for (int k = 0; k < SET; k++) {
                        const float s = __half2float(__ushort_as_half(scales[h * SET + k])) * (BF16 ? 1 << kShift : 1);
#pragma unroll
                        for (int c = 0; c < SUMS / CHUNK; c++) {
                            // columns past `width` may hold anything: theirs are sums that nobody takes
                            uint32_t v[CHUNK];
                            if (c * CHUNK < width) {
                                if constexpr (CHUNK == 16) tmem_ld_32x32b_x16(taddr + k * acc_cols + c * CHUNK, v);
                                else tmem_ld_32x32b_x32(taddr + k * acc_cols + c * CHUNK, v);
                                tmem_ld_wait();
                            }
                            if (k == SET - 1 && c == SUMS / CHUNK - 1) {   // all of the set is in registers
                                tc_fence_before();
                                __syncwarp();
                                if (lane == 0) mbar_arrive(&bars.tmem_empty[set]);
                            }
                            if (c * CHUNK < width) {
#pragma unroll
                                for (int e = 0; e < CHUNK; e++)
                                    sum[c * CHUNK + e] = fmaf(__uint_as_float(v[e]), s, sum[c * CHUNK + e]);
                            }
                        }
                    }
                    if (++set == SETS) {
                        set = 0;
                        phase_set ^= 1;
                    }
                }
            };
            for (int blk = 0; blk < blocks && ok; blk += AHEAD) {
#pragma unroll
                for (int i = 0; i < AHEAD * PER; i++) now[i / PER][i % PER] = next[i / PER][i % PER];
                load(blk + AHEAD);
#pragma unroll
                for (int u = 0; u < AHEAD; u++)
                    if (blk + u < blocks && ok) add(now[u]);
            }
            if (!ok && lane == 0) atomicExch(status, 855);
            if (split > 1) {   // this CTA's part, where the weights were
                float* part = reinterpret_cast<float*>(smem) + q * 32 + lane;
#pragma unroll
                for (int i = 0; i < SUMS; i++)
                    if (i < width) part[(col0 + i) * 128] = sum[i];
                continue;
            }
            if constexpr (GATED) {
#pragma unroll
                for (int c = 0; c < SUMS / 16; c++) {   // 16 tokens of each half at a time
                    if (c * 16 < width) {
                        if (q >= 2) {
#pragma unroll
                            for (int i = 0; i < 16; i++) swap[(half * 16 + i) * 64 + r] = sum[c * 16 + i] + bias;
                        }
                        named_barrier_sync(1, 32 * kSumWarps);
                        if (q < 2) {
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                const int m = col0 + c * 16 + i;
                                if (live && m < M && ok)
                                    out[(size_t)m * N + n] = from_float<T>(silu_mul(sum[c * 16 + i] + bias, swap[(half * 16 + i) * 64 + r]));
                            }
                        }
                        named_barrier_sync(1, 32 * kSumWarps);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < SUMS; i++)
                    if (i < width && live && col0 + i < M && ok)
                        out[(size_t)(col0 + i) * N + n] = from_float<T>(sum[i] + bias);
            }
        }
    }

    // ---------------------------------------------------------------------- teardown
    if (*bars.abort_flag != 0) {
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) { }
    }
    tc_fence_before();
    __syncthreads();
    if (warp_id == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
    if (split > 1) {
        cluster_sync_all();   // all parts are there
        if (*bars.abort_flag == 0) {
            const uint32_t part = smem_u32(smem);
            auto sum = [&](int m, int r) {
                float v = 0.f;
                for (int c = 0; c < split; c++) {
                    float p;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];"
                                 : "=f"(p)
                                 : "r"(mapa_shared(part + (m * 128 + r) * 4, c))
                                 : "memory");
                    v += p;
                }
                return v;
            };
            // every split-th token is this CTA's
            constexpr int LANES = GATED ? 64 : 128;
            for (int i = threadIdx.x; i < (M - rank + split - 1) / split * LANES; i += kTokenThreads) {
                const int m = rank + i / LANES * split, r = i % LANES, n = first_tile * rows + r;
                if (r < rows && n < N) {
                    float v = sum(m, r) + (b0 != nullptr ? to_float(b0[n]) : 0.f);
                    if constexpr (GATED) v = silu_mul(v, sum(m, 64 + r) + (b1 != nullptr ? to_float(b1[n]) : 0.f));
                    out[(size_t)m * N + n] = from_float<T>(v);
                }
            }
        }
        cluster_sync_all();   // nobody reads this CTA's memory any more
    }
}

// How a call is cut: rows of a tile, tiles, and CTAs that divide a tile's inputs.
struct TokenCut {
    int rows, tiles, split = 1;
    TokenCut(bool gated, int K, int N) {
        const int most = gated ? 64 : 128, sms = sm_count(), blocks = (K + 127) / 128;
        const long long full = ((long long)N + most - 1) / most;   // tiles of as many rows as the lanes hold
        while (split < 8 && full * split * 2 <= sms && blocks >= 4 * split) split *= 2;
        // without a split, so many rows that every SM has the same number
        const long long waves = (full + sms - 1) / sms;
        rows = split > 1 ? most : (int)((N + waves * sms - 1) / (waves * sms));
        tiles = (int)(((long long)N + rows - 1) / rows);
    }
    int blocks(int K) const { return split > 1 ? (K + 127) / 128 / split : (tiles + sm_count() - 1) / sm_count() * ((K + 127) / 128); }
};

template <typename T, int G, bool GATED, int MAX_COLS>
int launch_tokens(const void* x, const uint8_t* w0, const uint8_t* w1, const __half* s0, const __half* s1, const void* b0,
                  const void* b1, void* out, int M, int K, int N, cudaStream_t stream) {
    static bool ready[64] = {};
    auto kern = int4_tokens_kernel<T, G, GATED, MAX_COLS>;
    constexpr int kMaxSmem = 227 * 1024, kFixed = kTokenRing * 2 * kSlab + kSwapBytes + 512;
    int dev = 0;
    cudaGetDevice(&dev);
    if (!ready[dev & 63]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem) != cudaSuccess)
            return kLaunchFailed;
        ready[dev & 63] = true;
    }
    const int cols = (M + 31) / 32 * 32;
    int ring_x = kMaxRingX;   // a power of two
    while (ring_x * 2 * cols * 128 > kMaxSmem - kFixed) ring_x /= 2;
    const TokenCut cut(GATED, K, N);
    const int rows = cut.rows, tiles = cut.tiles, split = cut.split, sms = sm_count();
    CUtensorMap tm_x;
    if (!encode_sw128(&tm_x, type16(std::is_same<T, __nv_bfloat16>::value), 2, x, K, M, cols)) return kLaunchFailed;
    int* status = status_word();
    if (status == nullptr) return kLaunchFailed;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(split > 1 ? tiles * split : std::min(tiles, sms), 1, 1);
    cfg.blockDim = dim3(kTokenThreads, 1, 1);
    cfg.dynamicSmemBytes = kFixed + ring_x * 2 * cols * 128;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, tm_x, w0, w1, s0, s1, static_cast<const T*>(b0), static_cast<const T*>(b1),
                              static_cast<T*>(out), M, N, K, rows, cols, ring_x, split, status) == cudaSuccess
               ? kOk
               : kLaunchFailed;
}

template <typename T, int G, bool GATED, int BN>
int launch(const void* x, const uint8_t* w0, const uint8_t* w1, const __half* s0, const __half* s1, const void* b0,
           const void* b1, void* out, int M, int K, int N, cudaStream_t stream) {
    static int max_pairs[64] = {};
    constexpr int TILE_N = GATED ? BN / 4 : BN;
    const CUtensorMapDataType type = type16(std::is_same<T, __nv_bfloat16>::value);
    const int tma_out = N % 8 == 0 && aligned16(out);
    CUtensorMap tm_x, tm_out;
    if (!encode_sw128(&tm_x, type, 2, x, K, M, 128)) return kLaunchFailed;
    tm_out = tm_x;
    if (tma_out && !encode_sw128(&tm_out, type, 2, out, N, M, 32)) return kLaunchFailed;
    int* status = status_word();
    if (status == nullptr) return kLaunchFailed;
    const long long tiles = ((long long)M + 255) / 256 * (((long long)N + TILE_N - 1) / TILE_N);
    return launch_pairs16(int4_pair_kernel<T, G, GATED, BN>, kThreads, tiles, stream, max_pairs, tm_x, tm_out, w0, w1, s0, s1,
                          static_cast<const T*>(b0), static_cast<const T*>(b1), static_cast<T*>(out), M, N, K, tma_out,
                          status);
}

template <typename T, int G>
int dispatch(const void* x, const uint8_t* w0, const uint8_t* w1, const __half* s0, const __half* s1, const void* b0,
             const void* b1, void* out, int M, int K, int N, cudaStream_t st) {
    const bool gated = w1 != nullptr;
    if (M <= 32)
        return gated ? launch_tokens<T, G, true, 32>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st)
                     : launch_tokens<T, G, false, 32>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    if (M <= 64)
        return gated ? launch_tokens<T, G, true, 64>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st)
                     : launch_tokens<T, G, false, 64>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    // Sums of 128 tokens fill the registers of eight warps, and several groups a block make them what bounds the call: then
    // 64 tokens at a time, where a CTA has enough blocks (128 tokens, groups of 32: 11008 x 4096 55 against 79 us, 4096 x
    // 14336 56 against 76; groups of 64: 45 against 51, 47 against 51, gated 92 against 110; 8 blocks a CTA: 26 on both sides)
    if (G < 128 && M <= kTokensMax && TokenCut(gated, K, N).blocks(K) >= 16) {
        const int r = dispatch<T, G>(x, w0, w1, s0, s1, b0, b1, out, 64, K, N, st);
        return r != kOk ? r
                        : dispatch<T, G>(static_cast<const T*>(x) + (size_t)64 * K, w0, w1, s0, s1, b0, b1,
                                         static_cast<T*>(out) + (size_t)64 * N, M - 64, K, N, st);
    }
    if (M <= kTokensMax)
        return gated ? launch_tokens<T, G, true, 128>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st)
                     : launch_tokens<T, G, false, 128>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    if (gated) return launch<T, G, true, 256>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
    // A round of tiles of 128 weight rows takes 0.9 of the time of 256: worth it where even those fit into one round
    // (512 x 14336 x 4096: 88 against 94 us), not for shorter but more rounds (512 x 4096 x 11008: 81 against 59).
    const long long wide = ((long long)M + 255) / 256 * (((long long)N + 255) / 256);
    return 2 * wide <= sm_count() / 2 ? launch<T, G, false, 128>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st)
                                      : launch<T, G, false, 256>(x, w0, w1, s0, s1, b0, b1, out, M, K, N, st);
}

}  // namespace

int int4_gemm(const void* x, const uint8_t* w0, const uint8_t* w1, const __half* s0, const __half* s1, const void* b0,
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
