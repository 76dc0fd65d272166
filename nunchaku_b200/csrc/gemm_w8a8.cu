// 8-bit integer GEMM with a scale per token and per output channel on the tcgen05 tensor cores, sm_100a.
//
//   out[m][n] = ascales[m] * wscales[n] * sum_k act[m][k] * wgt[n][k] (+ bias[n])
//
// act int8 [M, K] and wgt int8 [N, K] row-major (both K-major operands as they lie in memory), the sum exact in int32
// (K <= 131071: 2^14 * K stays below 2^31), scales and bias applied in fp32 with one rounding to the 16-bit output.
// Reference: gemm_w8a8 / quantize_w8a8_act (src/kernels/zgemm/gemm_w8a8.cu), there on mma.sync with 16-bit scales.
//
// Two kernels.
//
// w8a8_pair_kernel (many tokens): the two SMs of a CTA pair walk 256 x BN output tiles (tcgen05.mma cta_group::2 kind::i8,
// M 256, K 32), each CTA holding its 128 token rows and half of the weight rows of a 128-deep K stage (128B-swizzled TMA
// boxes) in a ring; two accumulators of up to 256 columns alternate in TMEM, so that the epilogue of a tile runs under the
// next tile's products.  Warps: 0-3 producers, 4 MMA issuer (leader CTA), 8-15 epilogue (two per lane quadrant, alternating 32-column
// chunks).  Bound by the tensor pipe: 8192 x 4096 x 4096 87 us = 3153 TOPS (0.97 of what this instruction reaches without loads or epilogue,
// 3262); 15361 x 11200 x 2240 306 us = 2520 TOPS, where the last of 18 K stages is half zeros, tiles of 18 stages leave more to the
// hand-over, and the chip draws its power limit (sustained 386); 2147 x 4480 x 2240 22 us = 1960 TOPS: 9 x 24 tiles of 256 x 192 are 2.9 rounds
// of 74 pairs, a sixth of the rows and rounds padding, and 5 us are the first loads and the last epilogue.
//
// w8a8_skinny_kernel (few tokens, the serving form): there every weight is used for a handful of rows and the kernel streams
// weights.  The operands change places: 128 weight rows are the M side of the product, up to 16 tokens its N side, and K is split
// over a cluster of up to 8 CTAs to fill the SMs.  The int32 partial sums are exchanged through distributed shared memory (integers: the order
// does not matter).  Bound by the weights' bytes and, at these sizes, by launch and latency: 8 x 13440 x 2240 8 to 9 us = 3.6 TB/s (floor 4.6).
//
// Every wait is bounded; a role whose wait runs out records SVDQ_ERR_TIMEOUT and leaves its loop.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "host_common.h"
#include "ptx.cuh"

namespace svdq {

constexpr int W8_BK = 128;                        // K bytes per stage (one 128-byte swizzle row)
constexpr int W8_BM = 128;                        // token rows per CTA of a pair
constexpr int W8_BN_MAX = 256;
constexpr int W8_A_BYTES = W8_BM * W8_BK;         // 16384
constexpr int W8_B_BYTES = (W8_BN_MAX / 2) * W8_BK;
constexpr int W8_STAGE_BYTES = W8_A_BYTES + W8_B_BYTES;
constexpr int W8_STAGES = 6;
constexpr int W8_EPI_WARPS = 8;
constexpr int W8_MMA_WARP = 4, W8_EPI_WARP0 = 8;   // 0-3 producers, 5-7 nothing
constexpr int W8_THREADS = (W8_EPI_WARP0 + W8_EPI_WARPS) * 32;
constexpr int W8_COL_BYTES = 2 * W8_BN_MAX * 4;   // column scales and bias of one tile
constexpr int W8_SMEM = 1024 + W8_STAGES * W8_STAGE_BYTES + W8_COL_BYTES + 256;
constexpr int W8_MAX_K = 131071;
constexpr long long W8_WAIT_CYCLES = 4000000000ll;   // ~2 s

struct W8Params {
    const float* ascales;
    const float* wscales;
    const void* bias;
    void* out;
    long long out_stride;
    int M, N, K;
    int bn, tiles_m, tiles_n;
    int* status;
};

struct W8Shared {
    uint64_t full[W8_STAGES];     // leader: the stage's operands of both CTAs have landed
    uint64_t empty[W8_STAGES];    // each CTA: the MMAs of the stage are done
    uint64_t tfull[2];            // each CTA: accumulator complete
    uint64_t tempty[2];           // leader: accumulator drained by the epilogue warps of both CTAs
    uint64_t drain;
    uint32_t tmem_base;
    volatile int abort_flag;
};

__device__ __forceinline__ bool w8_wait(uint64_t* bar, uint32_t parity, W8Shared* sh, int* status, int where) {
#pragma unroll 1
    for (int i = 0; i < 512; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 64; ++i) {
            if (mbar_try_wait(bar, parity)) return true;
            __nanosleep(32);
        }
        if (sh->abort_flag) return false;
        if (clock64() - t0 > W8_WAIT_CYCLES) {
            sh->abort_flag = 1;
            st_shared_cluster_u32(mapa_shared(smem_u32(const_cast<int*>(&sh->abort_flag)), cluster_ctarank() ^ 1u), 1u);
            atomicExch(&status[0], SVDQ_ERR_TIMEOUT);
            atomicExch(&status[1], where);
            return false;
        }
    }
}

template <bool F16>
__device__ __forceinline__ uint32_t w8_pack(float lo, float hi) {
    uint32_t r;
    if constexpr (F16) asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));   // saturates as the W4A4 GEMM's output does
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <bool F16>
__device__ __forceinline__ float w8_load16(const void* p, int i) {
    if constexpr (F16) return __half2float(static_cast<const __half*>(p)[i]);
    else return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

template <bool F16>
__global__ void __launch_bounds__(W8_THREADS, 1)
w8a8_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const W8Params p) {
    extern __shared__ __align__(1024) uint8_t w8_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(w8_smem_raw) + 1023) & ~uintptr_t(1023));
    float* colv = reinterpret_cast<float*>(smem + W8_STAGES * W8_STAGE_BYTES);     // [0, 256) scales, [256, 512) bias
    W8Shared* sh = reinterpret_cast<W8Shared*>(reinterpret_cast<uint8_t*>(colv) + W8_COL_BYTES);
    static_assert(sizeof(W8Shared) <= 256, "barrier block");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int kstages = (p.K + W8_BK - 1) / W8_BK;
    const int ntiles = p.tiles_m * p.tiles_n;
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const int bnh = p.bn >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < W8_STAGES; ++s) {
            mbar_init(&sh->full[s], 4);       // two copies in each CTA
            mbar_init(&sh->empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh->tfull[i], 1);
            mbar_init(&sh->tempty[i], 2 * W8_EPI_WARPS);
        }
        mbar_init(&sh->drain, 1);
        sh->abort_flag = 0;
        fence_mbar_init();
        prefetch_tmap(&tm_a);
        prefetch_tmap(&tm_b);
    }
    if (warp == W8_MMA_WARP) {
        tmem_alloc_pair(&sh->tmem_base, 512);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    cluster_sync_all();   // barriers of both CTAs are initialised before anything remote touches them
    tc_fence_after_sync();
    pdl_launch_dependents();
    pdl_wait();           // nothing above touches global memory
    const uint32_t tmem = sh->tmem_base;

    if (warp < 4) {
        // ------------------------------------------------------------------ producers: warps 0, 2 tokens, 1, 3 weights, of every other stage each (the
        // copies of one issuing warp are worked off one after the other, in about the time a stage's products take)
        const bool wgt = warp & 1;
        const uint32_t turn = warp >> 1, bytes = wgt ? bnh * W8_BK : W8_A_BYTES;
        uint32_t it = 0;      // stages so far
        bool ok = true;
        for (int tile = pair; tile < ntiles && ok; tile += npairs) {
            const int row = wgt ? (tile / p.tiles_m) * p.bn + rank * bnh : (tile % p.tiles_m) * (2 * W8_BM) + rank * W8_BM;
            for (int ks = 0; ks < kstages; ++ks, ++it) {
                if ((it & 1) != turn) continue;
                const uint32_t slot = it % W8_STAGES;
                ok = __all_sync(0xffffffffu, w8_wait(&sh->empty[slot], ((it / W8_STAGES) & 1) ^ 1, sh, p.status, 810 + warp));
                if (!ok) break;
                uint8_t* dst = smem + slot * W8_STAGE_BYTES + (wgt ? W8_A_BYTES : 0);
                const uint32_t lfull = mapa_shared(smem_u32(&sh->full[slot]), 0);
                if (elect_one()) {
                    mbar_arrive_expect_tx_cluster(lfull, bytes);
                    tma_load_2d_pair(dst, wgt ? &tm_b : &tm_a, lfull, ks * W8_BK, row);
                }
                __syncwarp();
            }
        }
        if (!ok)   // The copies still in flight land on the leader's barriers, whose phases may never complete: wait many times a copy's time.
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    } else if (warp == W8_MMA_WARP && rank == 0) {
        // ------------------------------------------------------------------ MMA issuer
        const uint32_t idesc = idesc_i8(2 * W8_BM, p.bn, true);
        const uint64_t desc0 = smem_desc_sw128(smem_u32(smem));
        const uint32_t hi = static_cast<uint32_t>(desc0 >> 32), lo0 = static_cast<uint32_t>(desc0);
        const uint32_t full0 = smem_u32(&sh->full[0]), empty0 = smem_u32(&sh->empty[0]);
        uint32_t slot = 0, phase = 0, off = 0;
        bool ok = true;
        int ti = 0;
        for (int tile = pair; tile < ntiles && ok; tile += npairs, ++ti) {
            const uint32_t as = ti & 1;
            ok = __all_sync(0xffffffffu, w8_wait(&sh->tempty[as], ((ti >> 1) & 1) ^ 1, sh, p.status, 820));
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t d_tmem = tmem + as * W8_BN_MAX;
            for (int ks = 0; ks < kstages; ++ks) {
                if (!mbar_try_wait_addr(full0 + 8 * slot, phase)) ok = w8_wait(&sh->full[slot], phase, sh, p.status, 821);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after_sync();
                if (elect_one()) {
                    const uint32_t a_lo = lo0 + off, b_lo = a_lo + (W8_A_BYTES >> 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j)   // four K = 32 steps; the columns past K are zeros
                        tc_mma_pair_i8(d_tmem, a_lo + 2 * j, b_lo + 2 * j, hi, idesc, (ks | j) ? 1u : 0u);
                    tc_commit_pair_addr(empty0 + 8 * slot, 3);
                }
                __syncwarp();
                if (++slot == W8_STAGES) {
                    slot = 0;
                    phase ^= 1;
                    off = 0;
                } else {
                    off += W8_STAGE_BYTES >> 4;
                }
            }
            if (ok) {
                if (elect_one()) tc_commit_pair(&sh->tfull[as], 3);
                __syncwarp();
            }
        }
        if (sh->abort_flag) {   // let whatever was issued finish before TMEM is released
            if (lane == 0) {
                tc_commit_pair(&sh->drain, 1);
                mbar_wait(&sh->drain, 0, 400000000ll);
            }
            __syncwarp();
        }
    } else if (warp >= W8_EPI_WARP0) {
        // ------------------------------------------------------------------ epilogue
        const int quad = warp & 3, set = (warp - W8_EPI_WARP0) >> 2;
        const int et = threadIdx.x - W8_EPI_WARP0 * 32;
        int ti = 0;
        for (int tile = pair; tile < ntiles; tile += npairs, ++ti) {
            const uint32_t as = ti & 1;
            const int m = (tile % p.tiles_m) * (2 * W8_BM) + rank * W8_BM + quad * 32 + lane;
            const int n0 = (tile / p.tiles_m) * p.bn;
            // this tile's column scales and bias (every epilogue warp has left the previous tile at the first barrier)
            named_barrier_sync(1, W8_EPI_WARPS * 32);
            if (et < p.bn) {
                const int n = n0 + et;
                colv[et] = n < p.N ? p.wscales[n] : 0.f;
                colv[W8_BN_MAX + et] = (p.bias && n < p.N) ? w8_load16<F16>(p.bias, n) : 0.f;
            }
            const float sa = m < p.M ? p.ascales[m] : 0.f;
            named_barrier_sync(1, W8_EPI_WARPS * 32);
            const bool ok = __all_sync(0xffffffffu, w8_wait(&sh->tfull[as], (ti >> 1) & 1, sh, p.status, 830));
            if (ok) {
                tc_fence_after_sync();
                uint8_t* orow = static_cast<uint8_t*>(p.out) + 2 * (static_cast<long long>(m) * p.out_stride + n0);
                for (int c = set * 32; c < p.bn; c += 64) {
                    uint32_t r[32];
                    tc_ld_32x32b_x32(tmem + (static_cast<uint32_t>(quad * 32) << 16) + as * W8_BN_MAX + c, r);
                    tc_wait_ld();
                    if (m < p.M) {
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            if (n0 + c + u * 8 < p.N) {   // N is a multiple of 8
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int i = u * 8 + 2 * e;
                                    const float2 sc = *reinterpret_cast<const float2*>(colv + c + i);
                                    const float2 bi = *reinterpret_cast<const float2*>(colv + W8_BN_MAX + c + i);
                                    w[e] = w8_pack<F16>(fmaf(static_cast<float>(static_cast<int>(r[i])) * sa, sc.x, bi.x),
                                                        fmaf(static_cast<float>(static_cast<int>(r[i + 1])) * sa, sc.y, bi.y));
                                }
                                *reinterpret_cast<uint4*>(orow + 2 * (c + u * 8)) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    }
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&sh->tempty[as]), 0));
            }
            // a warp that gave up still takes part in the block's named barriers, tile by tile
        }
    }
    // Neither CTA may leave (or give up its TMEM) while the other can still signal its barriers or the leader's MMAs can
    // still read its shared memory: both have passed all their tiles here.
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();
    if (warp == W8_MMA_WARP) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem, 512);
    }
}

// ---------------------------------------------------------------------------------------------------------------- few tokens
constexpr int W8S_BW = 128;                       // weight rows per CTA (the M side)
constexpr int W8S_W_BYTES = W8S_BW * W8_BK;
constexpr int W8S_THREADS = 6 * 32;
constexpr int W8S_STAGES = 4;
constexpr int W8S_TOKENS = 16;                    // the N side; more tokens are the other kernel's
constexpr int W8S_MAX_SPLIT = 8;
constexpr int W8S_STAGE_BYTES = W8S_W_BYTES + W8S_TOKENS * W8_BK;
constexpr int W8S_TMEM_COLS = 32;
constexpr int W8S_SMEM = 1024 + W8S_STAGES * W8S_STAGE_BYTES + 256;   // 73 KB: three CTAs per SM

struct W8SShared {
    uint64_t full[W8S_STAGES], empty[W8S_STAGES], done;
    uint32_t tmem_base;
};
static_assert(W8S_STAGES * W8S_STAGE_BYTES >= W8S_TOKENS * W8S_BW * 4 && sizeof(W8SShared) <= 256, "the exchange buffer lies over the ring");

// grid (weight tiles * split), cluster (split, 1, 1)
template <bool F16>
__global__ void __launch_bounds__(W8S_THREADS)
w8a8_skinny_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_t, const W8Params p, const int split) {
    extern __shared__ __align__(1024) uint8_t w8_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(w8_smem_raw) + 1023) & ~uintptr_t(1023));
    W8SShared* sh = reinterpret_cast<W8SShared*>(smem + W8S_STAGES * W8S_STAGE_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int n0 = (blockIdx.x / split) * W8S_BW;
    const int kstages = (p.K + W8_BK - 1) / W8_BK;
    const int ks0 = kstages * rank / split, ks1 = kstages * (rank + 1) / split;

    if (threadIdx.x == 0) {
        for (int s = 0; s < W8S_STAGES; ++s) {
            mbar_init(&sh->full[s], 1);
            mbar_init(&sh->empty[s], 1);
        }
        mbar_init(&sh->done, 1);
        fence_mbar_init();
        prefetch_tmap(&tm_w);
        prefetch_tmap(&tm_t);
    }
    if (warp == 1) {
        tmem_alloc(&sh->tmem_base, W8S_TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    pdl_launch_dependents();
    pdl_wait();           // nothing above touches global memory
    const uint32_t tmem = sh->tmem_base;

    if (warp == 0) {
        if (lane == 0) {
            int i = 0;
            for (; i < ks1 - ks0; ++i) {
                const int s = i % W8S_STAGES;
                if (!mbar_wait(&sh->empty[s], ((i / W8S_STAGES) & 1) ^ 1, W8_WAIT_CYCLES)) {
                    atomicExch(&p.status[0], SVDQ_ERR_TIMEOUT);
                    atomicExch(&p.status[1], 840);
                    break;
                }
                uint8_t* st = smem + s * W8S_STAGE_BYTES;
                mbar_arrive_expect_tx(&sh->full[s], W8S_STAGE_BYTES);
                tma_load_2d(st, &tm_w, &sh->full[s], (ks0 + i) * W8_BK, n0);
                tma_load_2d(st + W8S_W_BYTES, &tm_t, &sh->full[s], (ks0 + i) * W8_BK, 0);
            }
            for (int k = i > W8S_STAGES ? i - W8S_STAGES : 0; k < i; ++k)   // leave with none of the copies in flight, whatever the others met
                mbar_wait(&sh->full[k % W8S_STAGES], (k / W8S_STAGES) & 1, W8_WAIT_CYCLES);
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc_i8(W8S_BW, W8S_TOKENS, true);
        bool ok = true;
        for (int i = 0; i < ks1 - ks0; ++i) {
            const int s = i % W8S_STAGES;
            ok = __all_sync(0xffffffffu, mbar_wait(&sh->full[s], (i / W8S_STAGES) & 1, W8_WAIT_CYCLES));
            if (!ok) {
                if (lane == 0) {
                    atomicExch(&p.status[0], SVDQ_ERR_TIMEOUT);
                    atomicExch(&p.status[1], 841);
                }
                break;
            }
            tc_fence_after_sync();
            if (elect_one()) {
                const uint64_t wd = smem_desc_sw128(smem_u32(smem + s * W8S_STAGE_BYTES));
                const uint64_t td = smem_desc_sw128(smem_u32(smem + s * W8S_STAGE_BYTES + W8S_W_BYTES));
#pragma unroll
                for (int j = 0; j < 4; ++j) tc_mma_i8(tmem, wd + 2 * j, td + 2 * j, idesc, (i | j) ? 1u : 0u);
                tc_commit(&sh->empty[s]);
            }
            __syncwarp();
        }
        if (elect_one()) tc_commit(&sh->done);
        __syncwarp();
    }
    // ---- partial sums [token][weight row] into shared memory over the ring (all copies and products are done)
    int* red = reinterpret_cast<int*>(smem);
    const bool done = mbar_wait(&sh->done, 0, 2 * W8_WAIT_CYCLES);
    if (!done && lane == 0) {
        atomicExch(&p.status[0], SVDQ_ERR_TIMEOUT);
        atomicExch(&p.status[1], 842);
    }
    if (done && warp >= 2) {
        tc_fence_after_sync();
        const int quad = warp & 3;
        uint32_t r[16];
        tc_ld_32x32b_x16(tmem + (static_cast<uint32_t>(quad * 32) << 16), r);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < W8S_TOKENS; ++i) red[i * W8S_BW + quad * 32 + lane] = static_cast<int>(r[i]);
    }
    tc_fence_before_sync();
    if (split > 1) cluster_sync_all();
    else __syncthreads();
    if (warp >= 2) {
        const int row = (warp & 3) * 32 + lane, n = n0 + row;
        const float sw = n < p.N ? p.wscales[n] : 0.f;
        const float bias = p.bias && n < p.N ? w8_load16<F16>(p.bias, n) : 0.f;
        uint32_t peer[W8S_MAX_SPLIT];
#pragma unroll
        for (int q = 0; q < W8S_MAX_SPLIT; ++q) peer[q] = q < split ? mapa_shared(smem_u32(red + row), q) : 0;
        const int tokens = min(W8S_TOKENS, p.M);
        // this CTA's tokens, four at a time with every peer's value asked for before the first is used
        for (int t = rank; t < tokens; t += 4 * split) {
            int sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int q = 0; q < W8S_MAX_SPLIT; ++q)
                if (q < split) {
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (t + u * split < tokens) sum[u] += ld_shared_cluster_s32(peer[q] + (t + u * split) * (W8S_BW * 4));
                }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int m = t + u * split;
                if (m < tokens && n < p.N) {
                    const uint32_t w = w8_pack<F16>(fmaf(static_cast<float>(sum[u]) * p.ascales[m], sw, bias), 0.f);
                    static_cast<uint16_t*>(p.out)[static_cast<long long>(m) * p.out_stride + n] = static_cast<uint16_t>(w);
                }
            }
        }
    }
    if (split > 1) cluster_sync_all();   // peers may still read this CTA's partial sums
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, W8S_TMEM_COLS);
    }
}

// ---------------------------------------------------------------------------------------------------------------- host
static int w8_tmap(CUtensorMap* map, const void* base, int rows, int K, int box_rows) {
    return make_tmap_2d(map, base, CU_TENSOR_MAP_DATA_TYPE_UINT8, static_cast<uint64_t>(K), static_cast<uint64_t>(rows),
                        static_cast<uint64_t>(K), W8_BK, static_cast<uint32_t>(box_rows), true);
}

// `cluster` CTAs of a cluster along x; launched so that the prologue may run under the predecessor's tail (both kernels wait for it
// before they touch global memory)
template <typename Kernel, typename... Args>
static int launch_w8(Kernel kernel, int grid, int threads, int smem, int cluster, std::atomic<uint64_t>& attr_done, cudaStream_t stream, Args... args) {
    if (int rc = ensure_dynamic_smem(kernel, smem, attr_done)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    SVDQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    return SVDQ_OK;
}
template <bool F16>
static int launch_w8_pair(const CUtensorMap& ta, const CUtensorMap& tb, const W8Params& p, int pairs, cudaStream_t stream) {
    static std::atomic<uint64_t> attr_done{0};
    return launch_w8(w8a8_pair_kernel<F16>, 2 * pairs, W8_THREADS, W8_SMEM, 2, attr_done, stream, ta, tb, p);
}
template <bool F16>
static int launch_w8_skinny(const CUtensorMap& tw, const CUtensorMap& tt, const W8Params& p, int split, cudaStream_t stream) {
    static std::atomic<uint64_t> attr_done{0};
    return launch_w8(w8a8_skinny_kernel<F16>, (p.N + W8S_BW - 1) / W8S_BW * split, W8S_THREADS, W8S_SMEM, split, attr_done, stream, tw, tt, p, split);
}

}  // namespace svdq

extern "C" int svdq_gemm_w8a8(const svdq_gemm_w8a8_args* a, void* stream) {
    using namespace svdq;
    SVDQ_CHECK_ARG(a && a->act && a->wgt && a->ascales && a->wscales && a->out, "gemm_w8a8: null pointer");
    SVDQ_CHECK_ARG(a->M > 0 && a->N > 0 && a->N % 8 == 0, "gemm_w8a8: M (%d) must be positive and N (%d) a positive multiple of 8", a->M, a->N);
    SVDQ_CHECK_ARG(a->M <= (1 << 30) && a->N <= (1 << 30), "gemm_w8a8: at most 2^30 rows and columns");
    SVDQ_CHECK_ARG(a->K > 0 && a->K % 16 == 0 && a->K <= W8_MAX_K, "gemm_w8a8: K (%d) must be a positive multiple of 16, at most %d", a->K, W8_MAX_K);
    SVDQ_CHECK_ARG(a->dtype == SVDQ_DTYPE_BF16 || a->dtype == SVDQ_DTYPE_FP16, "gemm_w8a8: bad dtype %d", a->dtype);
    SVDQ_CHECK_ARG(a->out_stride >= a->N && a->out_stride % 8 == 0, "gemm_w8a8: the output's row stride must be a multiple of 8, at least N");
    SVDQ_CHECK_ARG(aligned(a->act, 16) && aligned(a->wgt, 16) && aligned(a->out, 16) && aligned(a->ascales, 4) && aligned(a->wscales, 4) &&
                       aligned(a->bias, 2),
                   "gemm_w8a8: act, wgt and out must be 16-byte aligned");
    if (int rc = check_arch()) return rc;
    W8Params p = {};
    p.ascales = a->ascales;
    p.wscales = a->wscales;
    p.bias = a->bias;
    p.out = a->out;
    p.out_stride = a->out_stride;
    p.M = a->M;
    p.N = a->N;
    p.K = a->K;
    if (int rc = status_words(&p.status)) return rc;
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool f16 = a->dtype == SVDQ_DTYPE_FP16;
    const int kstages = (a->K + W8_BK - 1) / W8_BK;
    CUtensorMap ta, tb;
    if (a->M <= W8S_TOKENS) {
        // Few tokens: against the other kernel 9.0 to 12.0 us on 8 x 13440 x 2240 and 7.7 to 15.6 on 16 x 4096 x 4096; with 64 tokens in steps
        // of 16 it took 26 us on 64 x 4480 x 2240, the other 7.4.
        // K over as many CTAs as give every SM one (16 x 4096 x 4096: 11.4 us unsplit, 7.7 so); more cost more in joining than they bring
        // (8 x 13440 x 2240: 19.5 us with up to four per SM, 9.0 so)
        const int tiles = (a->N + W8S_BW - 1) / W8S_BW;
        int split = 1;
        while (split < W8S_MAX_SPLIT && tiles * split < sms && 2 * split <= kstages) split *= 2;
        if (int rc = w8_tmap(&ta, a->wgt, a->N, a->K, W8S_BW)) return rc;
        if (int rc = w8_tmap(&tb, a->act, a->M, a->K, W8S_TOKENS)) return rc;
        return f16 ? launch_w8_skinny<true>(ta, tb, p, split, st) : launch_w8_skinny<false>(ta, tb, p, split, st);
    }
    const int max_pairs = sms / 2;
    p.tiles_m = (a->M + 2 * W8_BM - 1) / (2 * W8_BM);
    // tile width: the one whose rounds over the pairs take the least, a round costing its width plus a fixed part
    // (always 256 / always 64 / this, us: 32 x 4096 x 4096 13.4 / 9.8 / 9.8; 2147 x 4480 x 2240 25.9 / 36.4 / 21.7; 8192 x 4096 x 4096 88 / 183 / 88)
    long long best = -1;
    for (int bn = W8_BN_MAX; bn >= 64; bn -= 32) {
        const long long tiles = static_cast<long long>(p.tiles_m) * ((a->N + bn - 1) / bn);
        const long long cost = (tiles + max_pairs - 1) / max_pairs * (bn + 16);
        if (best < 0 || cost < best) {
            best = cost;
            p.bn = bn;
        }
    }
    p.tiles_n = (a->N + p.bn - 1) / p.bn;
    const int ntiles = p.tiles_m * p.tiles_n;
    if (int rc = w8_tmap(&ta, a->act, a->M, a->K, W8_BM)) return rc;
    if (int rc = w8_tmap(&tb, a->wgt, a->N, a->K, p.bn / 2)) return rc;
    const int pairs = ntiles < max_pairs ? ntiles : max_pairs;
    return f16 ? launch_w8_pair<true>(ta, tb, p, pairs, st) : launch_w8_pair<false>(ta, tb, p, pairs, st);
}
