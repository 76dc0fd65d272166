// Softmax attention of queries over an encoder's states of another length, sm_100a: out = softmax(scale * q k^T) v per (batch, head)
// over the states that exist for the sample.
//
// Heads of 8 to 128 channels (multiples of 8), kv_heads dividing heads (query head h reads stored head h / (heads / kv_heads)),
// states given as [batch, kv_len] rows (all of them, the first kv_lens[b], or those a byte mask keeps) or packed one sample after
// the other (kv_offsets).  A sample without states gets zeros.  States that do not take part may hold anything, infinities and
// NaN included: their scores are replaced, not added to, and their rows of V are zeroed before the second product.
// Scores, running maximum, sums and the output accumulator are fp32; the probabilities are rounded to the 16-bit type before the
// second product (the tensor cores take 16-bit operands; the row sum is taken before that rounding), the output once.
// Reference: MultiHeadCrossAttention, src/SanaModel.cpp:138-190, which calls a varlen library kernel on packed captions.
//
// Two kernels.
//
// cross_tile_kernel (many queries): an item is 128 query rows of one (batch, head), or two times 128 over the same states (two tiles of
// a head, or two heads that share a stored one); the states are walked in blocks of 64 with Q K^T and P V as tcgen05.mma kind::f16, S,
// P and O in tensor memory and a running maximum per row (O is rescaled only when a maximum has grown by more than 2^8, as in
// attention.cu).  State lists are short here (a caption has up to 300 states, five blocks), so filling and draining count as much as
// the loop: CTAs are resident (one of two tiles, or two of one tile, to an SM), each works through a run of items, and warps are
// specialised so that an item's output, the next one's queries and the products of both lie behind one another.  Per tile: four softmax
// warps (one query row per thread), four output warps (O / l, through shared memory and on by TMA), an issuer for Q K^T and one for P V (an
// MMA of these sizes takes longer to issue than to run); per CTA a producer of Q and K and one of V.
// Two S buffers of 64 columns: a block's Q K^T runs under the previous block's exponentials.  K and V have two slots each, and with two
// tiles Q has two buffers: the next item's queries are on their way while this one is worked on.  The last block's products, loads and
// exponentials are cut to the states that exist (in sixteens, sixteens and 32s).
// Items lie in the order batch, tile, head: the heads' channels are neighbours in token-major rows, and a row of 224 bytes shares
// its DRAM bursts with them (one block of states, 32 x 20 x 1024 x 64 x 112: 94 us with tiles innermost, 65 so).  A CTA's run of items
// is cut from the samples' lengths on the device, so that all runs cost alike.
// What bounds it: 32 x 20 x 1024 x <=300 x 112, packed, moves 342 MB (52 us at the copy rate) and takes 96 us; 69 us with one block of 64 for
// every item, about 17 for each further one (full lists of 300: 133 us).  Two waits set the pace.  The queries of an item come 2.5 us after
// they are asked for, and the copy unit takes four cycles for a row of up to 128 bytes, whether query, state or output (with one tile at a
// time and one Q buffer the same takes 105 us, full lists of 300 160).  And in a block the chain S -> maximum -> P -> P V is served by two
// softmax warps per scheduler, which leave half of the issue slots empty.  The code of all roles has to stay small: at 80 KB it ran 30 % slower than at 47,
// and with the output's loop unrolled (70 KB) it took twice as long.  Tried and no faster: a quarter of the exponentials on the FMA pipe,
// as in attention.cu, two threads per row (105 -> 117), the output out of Q's buffer (which then comes free late), in boxes of 128-byte rows
// (99 -> 125, by code and registers) or by the warps' own stores (1 to 2 %), waits without suspension, queries and output first to leave
// L2 (300 states 5 % faster, 64 states as much slower).
//
// cross_rows_kernel (few query rows per stored head: the serving form for single tokens): bound by streaming K and V once.
// Up to 16 rows (queries x heads that share a stored head) are the M side of mma.sync m16n8k16; four warps take 16 of every 64
// states each, with their own running maximum; a producer warp brings K and V by TMA through a ring of two or three 64-state stages; the states are
// split over a cluster of up to 16 CTAs, which push their sums to one another through distributed shared memory and join them in the
// same launch.  16 x 24 (8 stored) x 1 x <=4096 x 128, lengths as they come: 31 us = 5.3 TB/s (floor 25; the longest sample's CTAs finish
// last); one token of 20 heads over 300 states: 5.3 us, of which an empty launch takes more than two and the joining one and a half.
//
// Every wait is bounded; a role whose wait runs out records SVDQ_ERR_TIMEOUT and leaves its loop.
#include "attention_common.cuh"
#include "host_common.h"

namespace svdq {

struct CrossStates {
    const int* kv_lens;       // or NULL
    const int* kv_offsets;    // or NULL: packed, k / v have no batch dimension
    const uint8_t* mask;      // or NULL: [batch, kv_len], row stride mask_stride bytes
    long long mask_stride;
    int kv_len;               // padded length, or the number of packed rows
};

// first row and number of rows of sample b; whatever the device arrays hold, inside [0, kv_len]
__device__ __forceinline__ void cross_range(const CrossStates& s, int b, int& start, int& len) {
    start = 0;
    len = s.kv_len;
    if (s.kv_offsets) {
        const int a = min(max(s.kv_offsets[b], 0), s.kv_len), e = min(max(s.kv_offsets[b + 1], 0), s.kv_len);
        start = a;
        len = max(e - a, 0);
    } else if (s.kv_lens) {
        len = min(max(s.kv_lens[b], 0), s.kv_len);
    }
}

// ---------------------------------------------------------------------------------------------------------------- many queries
constexpr int CT_BM = 128, CT_BN = 64;
constexpr int CT_Q_HALF = CT_BM * 128;              // 128 rows x 64 channels
constexpr int CT_KV_HALF = CT_BN * 128;
constexpr int CT_Q_BYTES = 2 * CT_Q_HALF, CT_KV_BYTES = 2 * CT_KV_HALF;
constexpr int CT_SLOTS = 2;                         // of K and of V each
constexpr int CT_STAGE_BYTES = 4 * 32 * 64;         // output: 32 rows x 32 channels per output warp on their way to memory
constexpr int CT_BAR_BYTES = 512;
constexpr int CT_MASK_STATES = 32768;               // longest state list a mask may cover (its bits are kept in shared memory)
constexpr int CT_TABLE_BYTES = 6 * 1024;            // the samples' ranges or mask bits
constexpr int CT_TMEM_COLS = 256;                   // of a query tile.  S: 2 x 64, O: 128
constexpr int CT_WAIT_LOOKS = 1 << 20;              // each of up to a microsecond
constexpr int CT_MAX_STATES = 1 << 22;              // about 70 ms an item: its output warps wait that long, and are not to give up on it
constexpr float CT_RESCALE_STEP = 8.f;
static_assert(CT_TABLE_BYTES >= CT_MASK_STATES / 8 + 8, "the bits of one sample's mask");

// TILES: query tiles that a CTA works on at a time, over the same states
template <int TILES>
struct CrossTileSizes {
    static constexpr int Q_BUFFERS = TILES;             // two tiles leave room for the next item's queries as well
    static constexpr int WARPS = TILES == 1 ? 12 : 24;
    static constexpr int THREADS = 32 * WARPS;
    // softmax, 4 per tile; output, 4 per tile; then
    static constexpr int OUT_WARP = 4 * TILES, S_WARP = 8 * TILES, PV_WARP = S_WARP + TILES, QK_WARP = PV_WARP + TILES, V_WARP = QK_WARP + 1;
    static_assert(V_WARP < WARPS, "warps");
    // registers move inside the pool the CTA was launched with (80 a thread fill the file)
    static constexpr int REGS_SOFTMAX = 112, REGS_OUTPUT = 64, REGS_OTHER = 64;
    static constexpr int REGS_LAUNCH = 80;
    static_assert(4 * TILES * (REGS_SOFTMAX + REGS_OUTPUT) + (WARPS - 8 * TILES) * REGS_OTHER <= WARPS * REGS_LAUNCH, "register budget");
    static constexpr int SUM_BYTES = 3 * TILES * CT_BM * 4;   // row sums of three items
    static constexpr int SMEM = 1024 + Q_BUFFERS * TILES * CT_Q_BYTES + 2 * CT_SLOTS * CT_KV_BYTES + TILES * CT_STAGE_BYTES + SUM_BYTES + CT_BAR_BYTES;
    static constexpr int PER_SM = TILES == 1 ? 2 : 1;
    // what it takes to change queries and hand the output over, in tenths of a block of 64 states' time (32 x 20 x 1024 x <=300 x 112, packed: one
    // tile 134 us at 8, 112 at 12, 109 at 16, 110 at 20; two 97.5 at 10, 96.3 at 13, 99.5 at 16, 101.5 at 20)
    static constexpr int ITEM_COST = TILES == 1 ? 16 : 13;
    static_assert(PER_SM * (SMEM + CT_TABLE_BYTES + 1024) <= 228 * 1024, "CTAs per SM");
};

template <int TILES>
struct CrossTileShared {
    // A slot of K is free when every tile's Q K^T is done (s_full), one of V when every tile's P V is (pv_done): the producers wait for
    // those.  A block of V whose rows are all to be seen lands on v_full; one with rows to be zeroed lands on vh_full, and who zeroes them
    // arrives on vz_full.  Every barrier has one sequence of phases that its waiters follow without gaps.
    uint64_t q_full[TILES], q_free[TILES], k_full[CT_SLOTS], v_full[CT_SLOTS], vh_full[CT_SLOTS], vz_full[CT_SLOTS];
    struct {
        uint64_t s_full[2], p_full[2], pv_done[2], l_full[3], o_free;
    } tile[TILES];
    uint32_t tmem_base;
    int failed;            // the code of a wait that ran out
};
static_assert(sizeof(CrossTileShared<2>) <= CT_BAR_BYTES, "barrier block");

struct CrossTileParams {
    CrossStates st;
    int q_len, dim, group, q_tiles, batch;
    int units_h, units_t, items;                          // item = (batch * units_t + tile unit) * units_h + head unit
    bool pair_heads;                                      // two tiles at a time: of two query heads that share a stored head, else of one head
    int mask_words;                                       // 32-bit words of mask bits per sample
    int q_bmul, q_hmul, k_bmul, k_hmul, v_bmul, v_hmul, o_bmul, o_hmul;   // 0 where that dimension is broadcast (stride 0): its coordinate is then 0
    float scale_log2;
    int* status;
};

// Bounded wait of a whole warp that lets the hardware suspend it between looks (polling takes issue slots from the softmax warps).
// False, on every lane, when it runs out; the code is reported at the kernel's end.
__device__ __forceinline__ bool ct_wait(uint64_t* bar, uint32_t parity, int* failed, int code) {
    uint32_t ok = 0;
#pragma unroll 1
    for (int i = 0; i < CT_WAIT_LOOKS && !ok; ++i)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(1000u)
            : "memory");
    if (__all_sync(0xffffffffu, ok != 0)) return true;
    *failed = code;
    return false;
}

// The items that a CTA works through, as each of its roles sees them: states [start, start + count) of the item's sample (with a mask:
// up to the last one that is to be seen) in blocks of 64.  Starts in front of the first.
template <bool MASK, int TILES>
struct CrossItems {
    const CrossTileParams& p;
    const int2* ranges;
    const uint32_t* words;
    int item, end, batch, head_unit, tile_unit, start, count, blocks;   // end: behind this CTA's last item

    __device__ __forceinline__ CrossItems(const CrossTileParams& p_, const int2* r, const uint32_t* w, int first, int end_, int batch_, int head_, int tile_)
        : p(p_), ranges(r), words(w), item(first - 1), end(end_), batch(batch_), head_unit(head_ - 1), tile_unit(tile_), start(0), count(0), blocks(0) {}
    // to the next item (EMPTY: even if it has no states); false behind the last
    template <bool EMPTY = false>
    __device__ __forceinline__ bool advance() {
#pragma unroll 1
        do {
            if (++item >= end) return false;
            if (++head_unit == p.units_h) {   // heads first: their channels lie next to each other in token-major rows
                head_unit = 0;
                if (++tile_unit == p.units_t) {
                    tile_unit = 0;
                    ++batch;
                }
            }
            const int2 r = ranges[batch];
            start = r.x;
            count = r.y;
            blocks = (count + CT_BN - 1) / CT_BN;
        } while (!EMPTY && blocks == 0);
        return true;
    }
    // query head and tile of the CTA's tile t
    __device__ __forceinline__ int head(int t) const { return TILES == 2 && p.pair_heads ? 2 * head_unit + t : head_unit; }
    __device__ __forceinline__ int tile(int t) const { return TILES == 2 && !p.pair_heads ? 2 * tile_unit + t : tile_unit; }
    __device__ __forceinline__ int valid(int j) const { return min(count - j * CT_BN, CT_BN); }
    __device__ __forceinline__ const uint32_t* bits(int j) const { return words + batch * p.mask_words + 2 * j; }
    // some of the rows of V that P V reads (valid rounded up to 16) must not be seen and are not zeros already
    __device__ __forceinline__ bool holes(int j) const {
        if constexpr (MASK) {
            const int up = (valid(j) + 15) & ~15;
            const uint32_t wa = up >= 32 ? 0xffffffffu : (1u << up) - 1u, wb = up >= 64 ? 0xffffffffu : up > 32 ? (1u << (up - 32)) - 1u : 0u;
            return (bits(j)[0] & wa) != wa || (bits(j)[1] & wb) != wb;
        }
        return (count & 15) != 0 && j + 1 == blocks && (p.st.kv_lens || p.st.kv_offsets);   // without them the rows past the end are filled with zeros by the copy
    }
};

// What an item costs, in tenths of a block's time.
template <int TILES>
__device__ __forceinline__ float cross_item_cost(int count) {
    return static_cast<float>(10 * ((count + CT_BN - 1) / CT_BN) + CrossTileSizes<TILES>::ITEM_COST);
}

// largest of three; a NaN stays one (fmaxf drops it)
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Rows of a block of V whose states must not be seen -> zeros, up to the last that P V reads: eight lanes per row (and half), this lane's
// rows from `r` on in steps of `step`.  By the softmax warps where a mask makes holes anywhere (by one warp a masked 6 x 16 x 1000 x 77 x 64
// takes 18.4 us, so 15.6), by a P V issuer where at most 15 rows behind the last state are concerned (32 x 20 x 1024 x <=300 x 112: 99 against
// 103).
template <bool MASK, int TILES>
__device__ __forceinline__ void zero_rows(const CrossItems<MASK, TILES>& it, uint8_t* v, int j, int halves, int r, int step, int lane) {
    const int valid = it.valid(j), up = (valid + 15) & ~15;
#pragma unroll 1
    for (; r < up; r += step) {
        bool zero = r >= valid;
        if constexpr (MASK) zero = !((it.bits(j)[r >> 5] >> (r & 31)) & 1u);
        if (zero)
            for (int h = 0; h < halves; ++h) *reinterpret_cast<uint4*>(v + h * CT_KV_HALF + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
    __syncwarp();
}

template <bool F16, bool MASK, int TILES>
__global__ void __launch_bounds__(CrossTileSizes<TILES>::THREADS, CrossTileSizes<TILES>::PER_SM)
cross_tile_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const __grid_constant__ CUtensorMap tm_o, const __grid_constant__ CrossTileParams p) {
    using Sz = CrossTileSizes<TILES>;
    extern __shared__ __align__(1024) uint8_t ct_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ct_smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* q_s = smem;                                                    // [buffer][tile]
    uint8_t* k_s = q_s + Sz::Q_BUFFERS * TILES * CT_Q_BYTES;
    uint8_t* v_s = k_s + CT_SLOTS * CT_KV_BYTES;
    uint8_t* stage = v_s + CT_SLOTS * CT_KV_BYTES;                          // [output warp]
    float* sums = reinterpret_cast<float*>(stage + TILES * CT_STAGE_BYTES);   // [3][tile][row]
    auto* sh = reinterpret_cast<CrossTileShared<TILES>*>(reinterpret_cast<uint8_t*>(sums) + Sz::SUM_BYTES);
    uint8_t* table = reinterpret_cast<uint8_t*>(sh) + CT_BAR_BYTES;
    int2* ranges = reinterpret_cast<int2*>(table);
    uint32_t* words = reinterpret_cast<uint32_t*>(table + p.batch * 8);   // MASK: behind the ranges

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int halves = p.dim > 64 ? 2 : 1;

    if (tid == 0) {
        for (int i = 0; i < TILES; ++i) {
            mbar_init(&sh->q_full[i], 1);
            mbar_init(&sh->q_free[i], TILES);
            for (int s = 0; s < 2; ++s) {
                mbar_init(&sh->tile[i].s_full[s], 1);
                mbar_init(&sh->tile[i].p_full[s], 4);
                mbar_init(&sh->tile[i].pv_done[s], 1);
            }
            for (int s = 0; s < 3; ++s) mbar_init(&sh->tile[i].l_full[s], 4);
            mbar_init(&sh->tile[i].o_free, 4);
        }
        for (int i = 0; i < CT_SLOTS; ++i) {
            mbar_init(&sh->k_full[i], 1);
            mbar_init(&sh->v_full[i], 1);
            mbar_init(&sh->vh_full[i], 1);
            mbar_init(&sh->vz_full[i], MASK ? 4 * TILES : 1);
        }
        sh->failed = 0;
        fence_mbar_init();
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
        prefetch_tmap(&tm_o);
    }
    if (warp == Sz::S_WARP) {
        tmem_alloc(&sh->tmem_base, TILES * CT_TMEM_COLS);
        tmem_relinquish();
    }
    pdl_launch_dependents();
    pdl_wait();   // nothing above touches global memory
    // the samples' ranges and mask bits
    if constexpr (MASK) {
        for (int b = tid; b < p.batch; b += Sz::THREADS) ranges[b] = make_int2(0, 0);
        __syncthreads();
#pragma unroll 1
        for (int w = warp; w < p.batch * p.mask_words; w += Sz::WARPS) {
            const int b = w / p.mask_words, at = (w - b * p.mask_words) * 32, i = at + lane;
            const uint32_t bits = __ballot_sync(0xffffffffu, i < p.st.kv_len && p.st.mask[b * p.st.mask_stride + i] != 0);
            if (lane == 0) {
                words[w] = bits;
                if (bits) atomicMax(&ranges[b].y, at + 32 - __clz(bits));
            }
        }
    } else {
        for (int b = tid; b < p.batch; b += Sz::THREADS) {
            int2 r;
            cross_range(p.st, b, r.x, r.y);
            ranges[b] = r;
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sh->tmem_base;
    // This CTA's share: a run of items, cut so that the CTAs' costs are alike.  An item belongs to the CTA in whose span of the whole
    // cost its own begins.  (Every warp for itself, 32 samples a turn; a CTA's end and the next one's start are the same computation.)
    const int per_batch = p.units_h * p.units_t;
    int edge[2] = {static_cast<int>(blockIdx.x), static_cast<int>(blockIdx.x) + 1};
    if (gridDim.x < p.items) {
        float total = 0.f;
        for (int b = lane; b < p.batch; b += 32) total += cross_item_cost<TILES>(ranges[b].y);
#pragma unroll
        for (int m = 16; m >= 1; m >>= 1) total += __shfl_xor_sync(0xffffffffu, total, m);
#pragma unroll
        for (int e = 0; e < 2; ++e) edge[e] = p.items;
#pragma unroll 1
        for (int e = 0; e < 2; ++e) {
            const float at = total * (static_cast<float>(blockIdx.x + e) / static_cast<float>(gridDim.x));   // in costs of one item per sample
            float before = 0.f;
            int found = p.items;
#pragma unroll 1
            for (int b0 = 0; b0 < p.batch && blockIdx.x + e < gridDim.x; b0 += 32) {
                const int b = b0 + lane;
                const float c = b < p.batch ? cross_item_cost<TILES>(ranges[b].y) : 0.f;
                float to = c;   // cost up to and including sample b
#pragma unroll 1
                for (int m = 1; m < 32; m <<= 1) {
                    const float v = __shfl_up_sync(0xffffffffu, to, m);
                    if (lane >= m) to += v;
                }
                to += before;
                const uint32_t inside = __ballot_sync(0xffffffffu, b < p.batch && at < to);
                if (inside) {
                    const float share = fminf(fmaxf((at - (to - c)) / fmaxf(c, 1.f), 0.f), 1.f);
                    found = __shfl_sync(0xffffffffu, b * per_batch + static_cast<int>(ceilf(share * static_cast<float>(per_batch))), __ffs(inside) - 1);
                    break;
                }
                before = __shfl_sync(0xffffffffu, to, 31);
            }
            if (e == 0) edge[0] = found;
            else edge[1] = found;
        }
    }
    const int b_first = edge[0] / per_batch, t_first = (edge[0] - b_first * per_batch) / p.units_h,
              h_first = edge[0] - (b_first * p.units_t + t_first) * p.units_h;
    using Items = CrossItems<MASK, TILES>;
    int* const failed = &sh->failed;
#define CT_ITEMS(name) Items name(p, ranges, words, edge[0], edge[1], b_first, h_first, t_first)

    if (warp >= Sz::S_WARP) {
        reg_dealloc<Sz::REGS_OTHER>();
        const int ksteps = (p.dim + 15) >> 4;                    // of 16 channels; channels past the head read as zeros
        if (warp < Sz::PV_WARP) {
            // -------------------------------------------------------------- issuer of a tile's Q K^T (the whole warp walks the loop, one elected lane
            // issues).  The two products have a warp each: an MMA of these sizes takes longer to issue than to run.
            const int tile = TILES == 1 ? 0 : warp - Sz::S_WARP;
            auto& bar = sh->tile[tile];
            const uint32_t s_tmem = tmem + tile * CT_TMEM_COLS;
            const uint64_t qd = smem_desc_sw128(smem_u32(q_s + tile * CT_Q_BYTES)), kd = smem_desc_sw128(smem_u32(k_s));
            const uint32_t hi = static_cast<uint32_t>(qd >> 32), q_lo = static_cast<uint32_t>(qd), k_lo = static_cast<uint32_t>(kd);
            CT_ITEMS(it);
            uint32_t n = 0, items = 0;
            bool ok = true;
            while (ok && it.advance()) {
                const uint32_t q_buf = items % Sz::Q_BUFFERS, q0 = q_lo + q_buf * (TILES * CT_Q_BYTES >> 4);
                if (!ct_wait(&sh->q_full[q_buf], (items / Sz::Q_BUFFERS) & 1, failed, 910)) break;
                ++items;
#pragma unroll 1
                for (int j = 0; j < it.blocks; ++j, ++n) {
                    const uint32_t slot = n & 1;
                    // S = Q K_j^T over the block's states, rounded up to 16, where P of two blocks ago was
                    if (!(ok = ct_wait(&sh->k_full[slot], (n >> 1) & 1, failed, 911) && (n < 2 || ct_wait(&bar.pv_done[slot], ((n - 2) >> 1) & 1, failed, 912))))
                        break;
                    tc_fence_after_sync();
                    const uint32_t idesc = idesc_h16(CT_BM, 0, F16, false) | (static_cast<uint32_t>((it.valid(j) + 15) >> 4) << 18);
                    const uint32_t d = s_tmem + slot * CT_BN, k0 = k_lo + slot * (CT_KV_BYTES >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk)
                            if (kk < ksteps)
                                tc_mma_f16_lo(d, q0 + (kk >> 2) * (CT_Q_HALF >> 4) + (kk & 3) * 2, k0 + (kk >> 2) * (CT_KV_HALF >> 4) + (kk & 3) * 2, hi,
                                              idesc, kk > 0);
                        tc_commit(&bar.s_full[slot]);
                        if (j + 1 == it.blocks) tc_commit(&sh->q_free[q_buf]);
                    }
                    __syncwarp();
                }
            }
        } else if (warp < Sz::QK_WARP) {
            // -------------------------------------------------------------- issuer of a tile's P V
            const int tile = TILES == 1 ? 0 : warp - Sz::PV_WARP;
            auto& bar = sh->tile[tile];
            const uint32_t t_tmem = tmem + tile * CT_TMEM_COLS;
            const uint32_t idesc = idesc_h16(CT_BM, 0, F16, true) | (static_cast<uint32_t>(ksteps * 2) << 17);
            const uint64_t vd = smem_desc_sw128_mn(smem_u32(v_s), CT_KV_HALF, 1024);
            const uint32_t hi = static_cast<uint32_t>(vd >> 32), v_lo = static_cast<uint32_t>(vd);
            CT_ITEMS(it);
            uint32_t n = 0, items = 0, phase = 0;   // phase: bits of v_full and vz_full per slot
            bool ok = true;
            while (ok && it.advance()) {
                ++items;
#pragma unroll 1
                for (int j = 0; j < it.blocks; ++j, ++n) {
                    const uint32_t slot = n & 1;
                    const int up = (it.valid(j) + 15) & ~15;
                    const uint32_t kind = 2 * slot + it.holes(j);   // bit of `phase`
                    if constexpr (!MASK)   // rows of V behind the last state -> zeros
                        if (tile == 0 && (kind & 1)) {
                            if (!(ok = ct_wait(&sh->vh_full[slot], (phase >> kind) & 1, failed, 950))) break;
                            zero_rows(it, v_s + slot * CT_KV_BYTES, j, halves, it.valid(j) + (lane >> 3), 4, lane);
                            if (lane == 0) mbar_arrive(&sh->vz_full[slot]);
                            __syncwarp();
                        }
                    uint64_t* v_there = (kind & 1 ? sh->vz_full : sh->v_full) + slot;
                    if (!(ok = (j > 0 || items == 1 || ct_wait(&bar.o_free, items & 1, failed, 915)) &&   // the previous item's O has been read
                               ct_wait(v_there, (phase >> kind) & 1, failed, 920) && ct_wait(&bar.p_full[slot], (n >> 1) & 1, failed, 930)))
                        break;
                    phase ^= 1u << kind;
                    tc_fence_after_sync();
                    const uint32_t a = t_tmem + slot * CT_BN, v0 = v_lo + slot * (CT_KV_BYTES >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int k4 = 0; k4 < 4; ++k4)
                            if (k4 * 16 < up) tc_mma_f16_ts_lo(t_tmem + 2 * CT_BN, a + k4 * 8, v0 + k4 * 128, hi, idesc, (j | k4) ? 1u : 0u);
                        tc_commit(&bar.pv_done[slot]);
                    }
                    __syncwarp();
                }
            }
        } else if (warp == Sz::QK_WARP) {
            // -------------------------------------------------------------- producer of Q and K (the copies of one issuing warp are worked off one
            // after the other, so that V has its own)
            CT_ITEMS(qi);
            CT_ITEMS(it);
            uint32_t n = 0, items = 0;   // blocks of K, items of Q asked for
            // the next item's queries, if there is one, as soon as the buffer's last user is through with it
            auto load_q = [&]() {
                if (!qi.advance()) return true;
                const uint32_t buf = items % Sz::Q_BUFFERS;
                if (items >= Sz::Q_BUFFERS && !ct_wait(&sh->q_free[buf], (items / Sz::Q_BUFFERS - 1) & 1, failed, 900)) return false;
                ++items;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&sh->q_full[buf], TILES * halves * CT_Q_HALF);
#pragma unroll 1
                    for (int t = 0; t < TILES; ++t)
#pragma unroll 1
                        for (int h = 0; h < halves; ++h)
                            tma_load_4d(q_s + (buf * TILES + t) * CT_Q_BYTES + h * CT_Q_HALF, &tm_q, &sh->q_full[buf], h * 64, qi.tile(t) * CT_BM,
                                        qi.head(t) * p.q_hmul, qi.batch * p.q_bmul);
                }
                __syncwarp();
                return true;
            };
            bool ok = TILES == 1 || load_q();
            while (ok && it.advance()) {
                if (TILES == 1 && !(ok = load_q())) break;
                const int z = it.head(0) / p.group * p.k_hmul, w = p.st.kv_offsets ? 0 : it.batch * p.k_bmul;
                for (int j = 0; j < it.blocks; ++j, ++n) {
                    const int slot = n & 1;
                    for (int t = 0; t < TILES && ok; ++t) ok = n < 2 || ct_wait(&sh->tile[t].s_full[slot], ((n - 2) >> 1) & 1, failed, 901);
                    if (!ok) break;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&sh->k_full[slot], halves * CT_KV_HALF);
#pragma unroll 1
                        for (int h = 0; h < halves; ++h)
                            tma_load_4d(k_s + slot * CT_KV_BYTES + h * CT_KV_HALF, &tm_k, &sh->k_full[slot], h * 64, it.start + j * CT_BN, z, w);
                    }
                    __syncwarp();
                    // behind the second block, whose slot says that the previous item's Q K^T are done
                    if (TILES == 2 && j == min(1, it.blocks - 1) && !(ok = load_q())) {
                        ++n;
                        break;
                    }
                }
            }
            // leave with none of this warp's copies in flight (where all went well they have all been waited for)
            for (uint32_t i = items > Sz::Q_BUFFERS ? items - Sz::Q_BUFFERS : 0; i < items; ++i)
                ct_wait(&sh->q_full[i % Sz::Q_BUFFERS], (i / Sz::Q_BUFFERS) & 1, failed, 903);
            for (uint32_t i = n > 2 ? n - 2 : 0; i < n; ++i) ct_wait(&sh->k_full[i & 1], (i >> 1) & 1, failed, 904);
        } else if (warp == Sz::V_WARP) {
            // -------------------------------------------------------------- producer of V
            CT_ITEMS(it);
            uint32_t n = 0, used = 0, phase = 0;   // blocks; per slot and kind (bit 2 * slot + holes): any copy yet, and the next one's phase bit
            bool ok = true;
            while (ok && it.advance()) {
                const int z = it.head(0) / p.group * p.v_hmul, w = p.st.kv_offsets ? 0 : it.batch * p.v_bmul;
                for (int j = 0; j < it.blocks; ++j, ++n) {
                    const int slot = n & 1;
                    for (int t = 0; t < TILES && ok; ++t) ok = n < 2 || ct_wait(&sh->tile[t].pv_done[slot], ((n - 2) >> 1) & 1, failed, 902);
                    if (!ok) break;
                    const bool holes = it.holes(j);
                    used |= 1u << (2 * slot + holes);
                    phase ^= 1u << (2 * slot + holes);
                    if (lane == 0) {
                        uint64_t* full = (holes ? sh->vh_full : sh->v_full) + slot;
                        mbar_arrive_expect_tx(full, halves * CT_KV_HALF);
#pragma unroll 1
                        for (int h = 0; h < halves; ++h) tma_load_4d(v_s + slot * CT_KV_BYTES + h * CT_KV_HALF, &tm_v, full, h * 64, it.start + j * CT_BN, z, w);
                    }
                    __syncwarp();
                }
            }
#pragma unroll 1
            for (int i = 0; i < 4; ++i)   // as above
                if ((used >> i) & 1u) ct_wait((i & 1 ? sh->vh_full : sh->v_full) + (i >> 1), ((phase >> i) & 1u) ^ 1u, failed, 905);
        }
    } else if (warp >= Sz::OUT_WARP) {
        reg_dealloc<Sz::REGS_OUTPUT>();
        // ------------------------------------------------------------------ output: O / l -> global memory, while the softmax warps are at the
        // next item already
        const int quad = warp & 3, tile = TILES == 1 ? 0 : (warp - Sz::OUT_WARP) >> 2;
        auto& bar = sh->tile[tile];
        const uint32_t o_tmem = tmem + tile * CT_TMEM_COLS + (static_cast<uint32_t>(quad * 32) << 16) + 2 * CT_BN;
        uint8_t* box = stage + (warp - Sz::OUT_WARP) * (CT_STAGE_BYTES / 4);   // [32 rows][64 bytes], 16-byte pieces swizzled by row / 2
        CT_ITEMS(it);
        uint32_t n = 0, at = 0, phase = 0;   // blocks so far; the item's buffer of sums, phase bit of its barrier
        while (it.template advance<true>()) {
            n += it.blocks;
            const int row0 = it.tile(tile) * CT_BM + quad * 32;
            float inv = 0.f;
            if (it.blocks) {
                const uint32_t last = n - 1;
                if (!ct_wait(&bar.l_full[at], phase, failed, 980) || !ct_wait(&bar.pv_done[last & 1], (last >> 1) & 1, failed, 981)) break;
                inv = 1.f / sums[(at * TILES + tile) * CT_BM + quad * 32 + lane];
                if (++at == 3) {
                    at = 0;
                    phase ^= 1;
                }
                tc_fence_after_sync();
            }
#pragma unroll 1
            for (int c = 0; c < p.dim; c += 32) {
                uint32_t o[32];
                if (it.blocks) {
                    tc_ld_32x32b_x32(o_tmem + c, o);   // columns past the head hold anything and are not stored
                    tc_wait_ld();
                    if (c + 32 >= p.dim) {   // all of O has been read: the next item's P V may overwrite it
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar.o_free);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0u;   // no states: zeros
                }
                // into a box of 32 rows x 32 channels (64-byte swizzle) and on by TMA (with stores of the warps' own 1 to 2 % slower)
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 v = __fmul2_rn(make_float2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), make_float2(inv, inv));
                    w[i] = pack_h16<F16>(v.x, v.y);
                }
                if (lane == 0) bulk_wait_group_read<0>();   // the previous copy has read the box
                __syncwarp();
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    *reinterpret_cast<uint4*>(box + lane * 64 + ((u ^ ((lane >> 1) & 3)) << 4)) = make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {   // rows behind the last and channels past the head are cut off by the copy
                    if (row0 < p.q_len) tma_store_4d(&tm_o, box, c, row0, it.head(tile) * p.o_hmul, it.batch * p.o_bmul);
                    bulk_commit_group();
                }
                __syncwarp();
            }
        }
        if (lane == 0) bulk_wait_group<0>();
        __syncwarp();
    } else {
        reg_alloc<Sz::REGS_SOFTMAX>();
        // ------------------------------------------------------------------ softmax: thread = one query row
        const int quad = warp & 3, tile = TILES == 1 ? 0 : warp >> 2;
        auto& bar = sh->tile[tile];
        const uint32_t s_tmem = tmem + tile * CT_TMEM_COLS + (static_cast<uint32_t>(quad * 32) << 16), o_tmem = s_tmem + 2 * CT_BN;
        const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
        // 32 states -> 16 columns of packed 16-bit pairs, and their sum
        auto exp32 = [&](const uint32_t (&a)[32], float m, uint32_t (&w)[16]) {
            const float2 nm2 = make_float2(-m, -m);
            float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 x = __ffma2_rn(make_float2(__uint_as_float(a[2 * i]), __uint_as_float(a[2 * i + 1])), sc2, nm2);
                float2 r;
                r.x = ex2(x.x);
                r.y = ex2(x.y);
                sum2[i & 1] = __fadd2_rn(sum2[i & 1], r);
                w[i] = pack_h16<F16>(r.x, r.y);
            }
            return (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
        };
        auto max32 = [&](const uint32_t (&a)[32], float least) {   // and of `least`
            float m[4] = {least, __uint_as_float(a[0]), __uint_as_float(a[1]), __uint_as_float(a[2])};
#pragma unroll
            for (int i = 3; i < 27; i += 8)
#pragma unroll
                for (int c = 0; c < 4; ++c) m[c] = max3_nan(m[c], __uint_as_float(a[i + 2 * c]), __uint_as_float(a[i + 2 * c + 1]));
            m[0] = max3_nan(m[0], __uint_as_float(a[27]), __uint_as_float(a[28]));
            m[1] = max3_nan(m[1], __uint_as_float(a[29]), __uint_as_float(a[30]));
            return max3_nan(m[0], max3_nan(m[1], m[2], m[3]), __uint_as_float(a[31]));
        };
        auto hide = [&](uint32_t (&a)[32], uint32_t bits) {
            if (bits != 0xffffffffu) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (!((bits >> i) & 1u)) a[i] = 0xff800000u;
            }
        };
        CT_ITEMS(it);
        uint32_t n = 0, at = 0, hole_phase = 0;   // blocks; the item's buffer of sums; phase bits of vh_full per slot
        bool ok = true;
        while (ok && it.advance()) {
            float m_used = 0.f, l = 0.f;
#pragma unroll 1
            for (int j = 0; j < it.blocks; ++j, ++n) {
                const uint32_t slot = n & 1, st = s_tmem + slot * CT_BN;
                const int valid = it.valid(j);
                if (!(ok = ct_wait(&bar.s_full[slot], (n >> 1) & 1, failed, 960))) break;
                tc_fence_after_sync();
                // Scores that do not count are replaced by -inf (selected, not added: they may be anything).
                uint32_t a0[32], a1[32], w[16];
                const bool two = valid > 32;
                tc_ld_32x32b_x32(st, a0);
                if (two) tc_ld_32x32b_x32(st + 32, a1);
                tc_wait_ld();
                hide(a0, MASK ? it.bits(j)[0] : valid >= 32 ? 0xffffffffu : (1u << valid) - 1u);
                // (Not below a finite bound: a block of which nothing is to be seen, ahead of others, has only -inf, whose exponentials are 0
                // whatever the finite maximum.  A score that is NaN makes the maximum and with it the whole row NaN.)
                float mx = max32(a0, -INFINITY);
                if (two) {
                    hide(a1, MASK ? it.bits(j)[1] : valid >= 64 ? 0xffffffffu : (1u << (valid - 32)) - 1u);
                    mx = max32(a1, mx);
                }
                const float ms = max3_nan(mx * p.scale_log2, -3e38f, -3e38f);
                if (j == 0) {
                    m_used = ms;
                } else if (const bool grow = !(ms <= m_used + CT_RESCALE_STEP); __any_sync(0xffffffffu, grow)) {
                    // O is written by the previous P V product until it has completed
                    if (!(ok = ct_wait(&bar.pv_done[(n - 1) & 1], ((n - 1) >> 1) & 1, failed, 970))) break;
                    tc_fence_after_sync();
                    const float alpha = grow ? ex2(m_used - ms) : 1.f;
                    l *= alpha;
#pragma unroll 1
                    for (int c = 0; c < p.dim; c += 16) {
                        uint32_t o[16];
                        tc_ld_32x32b_x16(o_tmem + c, o);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tc_st_32x32b_x16(o_tmem + c, o);
                    }
                    if (grow) m_used = ms;
                }
                // P over scores of this thread that are in registers by now
                l += exp32(a0, m_used, w);
                tc_st_32x32b_x16(st, w);
                if (two) {
                    l += exp32(a1, m_used, w);
                    tc_st_32x32b_x16(st + 16, w);
                }
                if constexpr (MASK)
                    if (it.holes(j)) {
                        if (!(ok = ct_wait(&sh->vh_full[slot], (hole_phase >> slot) & 1, failed, 950))) break;
                        hole_phase ^= 1u << slot;
                        zero_rows(it, v_s + slot * CT_KV_BYTES, j, halves, warp * 4 + (lane >> 3), 16 * TILES, lane);
                        if (lane == 0) mbar_arrive(&sh->vz_full[slot]);
                    }
                tc_wait_st();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.p_full[slot]);
            }
            if (!ok) break;
            // Three buffers (and barriers) in turn.  The scores of this item's last block were only asked for when all but the last of the P V
            // ahead of them were done; with one block per item that is the P V of the item two ahead, which waited until the output warps had
            // read O and sums of the item three ahead: whose buffer and barrier these are.
            sums[(at * TILES + tile) * CT_BM + quad * 32 + lane] = l;
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.l_full[at]);
            at = at == 2 ? 0 : at + 1;
        }
    }
#undef CT_ITEMS
    tc_fence_before_sync();
    __syncthreads();
    if (tid == 0 && sh->failed) {
        atomicExch(&p.status[0], SVDQ_ERR_TIMEOUT);
        atomicExch(&p.status[1], sh->failed);
    }
    if (warp == Sz::S_WARP) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, TILES * CT_TMEM_COLS);
    }
}

// ---------------------------------------------------------------------------------------------------------------- few query rows
constexpr int CR_WARPS = 4, CR_THREADS = 32 * (CR_WARPS + 1), CR_KEYS = 16, CR_ROWS = 16, CR_MAX_SPLIT = 16;
constexpr int CR_TILE = CR_WARPS * CR_KEYS;          // states of a tile: 16 per warp
constexpr long long CR_WAIT_CYCLES = 600000000ll;   // ~0.3 s
constexpr int CR_HALF_BYTES = CR_TILE * 128;         // 64 states x 64 channels

struct CrossRowsParams {
    CrossStates st;
    const uint8_t* q;
    uint8_t* out;
    long long qs[3], os[3];                 // batch, head, token strides in bytes
    int kv_heads, group, q_rows, dim;       // q_rows = q_len * group: row r is query r / group, head kv_head * group + r % group
    int k_bmul, k_hmul, v_bmul, v_hmul;     // 0 where that dimension is broadcast: its coordinate is then 0
    float scale_log2;
    int* status;
};

// CTAs per SM, by the registers that the queries and the output take (a third CTA at 128 channels spills and is slower: 34 -> 38 us on
// [16, 24 over 8, 1 over <= 4096, 128])
__host__ __device__ constexpr int cross_rows_per_sm(int nk) { return nk > 7 ? 2 : nk > 4 ? 3 : nk > 2 ? 4 : 6; }

// stages of the ring: as many as the shared memory of that many CTAs takes (a third at 128 channels: 33 -> 31 us on the case above; full lists of
// 4096 go from 42 to 44)
__host__ __device__ constexpr int cross_rows_stages(int nk) { return nk > 7 ? 3 : nk > 4 ? 2 : nk > 2 ? 3 : 2; }

template <int NK>
struct CrossRowsSizes {
    static constexpr int STAGES = cross_rows_stages(NK);
    static constexpr int HALVES = NK > 4 ? 2 : 1;
    static constexpr int STAGE = 2 * HALVES * CR_HALF_BYTES;    // K and V
    static constexpr int RING = STAGES * STAGE;
    static constexpr int COLS = NK * 16;
    // afterwards over the ring: the warps' partial sums [4][16][COLS], maxima and sums [4][16] each
    static_assert(RING >= CR_WARPS * CR_ROWS * (COLS + 2) * 4, "the partial sums lie over the ring");
    // behind the ring, written by the CTAs of the cluster: each one's sums of the elements that this CTA finishes, and their maxima and sums
    static constexpr int mail_floats(int rows, int split) { return split * ((rows * COLS / 2 + split - 1) / split) * 2; }
    static constexpr int smem(int rows, int split) { return 1024 + RING + 64 + (mail_floats(rows, split) + 2 * split * rows) * 4; }
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t src) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(src) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t src) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(src) : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma_16816_t(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void st_shared_cluster_f32x2(uint32_t cluster_addr, float2 v) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(cluster_addr), "f"(v.x), "f"(v.y) : "memory");
}

// grid (batch * kv_heads * split, row tiles), cluster (split, 1, 1)
template <bool F16, int NK>
__global__ void __launch_bounds__(CR_THREADS, cross_rows_per_sm(NK))
cross_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CrossRowsParams p,
                  const int log_split) {
    using S = CrossRowsSizes<NK>;
    extern __shared__ __align__(1024) uint8_t cr_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(cr_smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::RING);
    uint64_t* empty = full + S::STAGES;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int split = 1 << log_split, rank = split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int pairix = blockIdx.x >> log_split, batch = pairix / p.kv_heads, kv_head = pairix % p.kv_heads;
    const int r0 = blockIdx.y * CR_ROWS, rows = min(CR_ROWS, p.q_rows - r0);
    if (tid == 0) {
#pragma unroll
        for (int i = 0; i < S::STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], CR_WARPS);
        }
        fence_mbar_init();
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
    }
    pdl_launch_dependents();
    pdl_wait();   // nothing above touches global memory
    int start, count;
    cross_range(p.st, batch, start, count);
    const int tiles = (count + CR_TILE - 1) / CR_TILE;
    const int t0 = static_cast<int>(static_cast<long long>(tiles) * rank / split), t1 = static_cast<int>(static_cast<long long>(tiles) * (rank + 1) / split);
    __syncthreads();

    float o[2 * NK][4];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    bool ok = true;
    if (warp == CR_WARPS) {
        // ------------------------------------------------------------------ producer
        if (lane == 0) {
            int i = 0;
#pragma unroll 1
            for (int tile = t0; tile < t1; ++tile, ++i) {
                const int s = i % S::STAGES;
                if (!mbar_wait(&empty[s], ((i / S::STAGES) & 1) ^ 1, CR_WAIT_CYCLES)) {
                    ok = false;
                    break;
                }
                mbar_arrive_expect_tx(&full[s], S::STAGE);
                uint8_t* st = smem + s * S::STAGE;
#pragma unroll
                for (int h = 0; h < S::HALVES; ++h) {
                    tma_load_4d(st + h * CR_HALF_BYTES, &tm_k, &full[s], h * 64, start + tile * CR_TILE, kv_head * p.k_hmul, p.st.kv_offsets ? 0 : batch * p.k_bmul);
                    tma_load_4d(st + (S::HALVES + h) * CR_HALF_BYTES, &tm_v, &full[s], h * 64, start + tile * CR_TILE, kv_head * p.v_hmul,
                                p.st.kv_offsets ? 0 : batch * p.v_bmul);
                }
            }
            if (!ok)   // leave with none of the copies in flight
                for (int k = i > S::STAGES ? i - S::STAGES : 0; k < i; ++k) mbar_wait(&full[k % S::STAGES], (k / S::STAGES) & 1, CR_WAIT_CYCLES);
        }
    } else {
        // ------------------------------------------------------------------ consumers
        const uint8_t* mask = p.st.mask ? p.st.mask + batch * p.st.mask_stride : nullptr;
        const bool cut = p.st.kv_lens || p.st.kv_offsets;   // rows behind the sample's last are somebody's: elsewhere the copy fills in zeros
        // query fragments: rows g and g + 8
        uint32_t qf[NK][4];
        {
            const uint8_t* qrow[2];
            bool there[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = g + 8 * i;
                there[i] = r < rows;
                const int row = r0 + (there[i] ? r : 0);
                qrow[i] = p.q + batch * p.qs[0] + (kv_head * p.group + row % p.group) * p.qs[1] + (row / p.group) * p.qs[2] + 4 * t;
            }
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    qf[kk][i] = there[i & 1] && kk * 16 + (i >> 1) * 8 < p.dim ? *reinterpret_cast<const uint32_t*>(qrow[i & 1] + kk * 32 + (i >> 1) * 16) : 0u;
        }
#pragma unroll
        for (int i = 0; i < 2 * NK; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
        // this lane's rows of the ldmatrix groups, and the 16-byte piece that stands for piece 0 / 1 of its row (128-byte swizzle)
        const uint32_t base = smem_u32(smem) + warp * CR_KEYS * 128;
        const uint32_t k_row = ((lane >> 4) * 8 + (lane & 7)) * 128, k_x = (((lane >> 3) & 1) ^ (lane & 7)) << 4;
        const uint32_t v_row = (((lane >> 3) & 1) * 8 + (lane & 7)) * 128, v_x = ((lane >> 4) ^ (lane & 7)) << 4;
        // which of this warp's 16 states of a tile are to be seen
        auto visible = [&](int tile) {
            const int left = count - tile * CR_TILE - warp * CR_KEYS;
            uint32_t bits = left >= CR_KEYS ? 0xffffu : left > 0 ? (1u << left) - 1u : 0u;
            if (mask) bits &= __ballot_sync(0xffffffffu, lane < CR_KEYS && lane < left && mask[tile * CR_TILE + warp * CR_KEYS + lane] != 0);
            return bits;
        };
        uint32_t next_bits = t0 < t1 ? visible(t0) : 0u;
#pragma unroll 1
        for (int tile = t0; tile < t1; ++tile) {
            const int i = tile - t0, slot = i % S::STAGES;
            const uint32_t bits = next_bits;
            if (tile + 1 < t1) next_bits = visible(tile + 1);
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&full[slot], (i / S::STAGES) & 1, CR_WAIT_CYCLES)))) break;
            if (bits) {
                const uint32_t ks = base + slot * S::STAGE, vs = ks + S::HALVES * CR_HALF_BYTES;
                float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int kk = 0; kk < NK; ++kk) {
                    uint32_t b[4];
                    ldmatrix_x4(b, ks + (kk >> 2) * CR_HALF_BYTES + k_row + (k_x ^ ((kk & 3) << 5)));
                    mma_16816_t<F16>(s[0], qf[kk], b[0], b[1]);
                    mma_16816_t<F16>(s[1], qf[kk], b[2], b[3]);
                }
                if (bits != 0xffffu && (mask || cut)) {   // rows of V that must not be seen -> zeros: two lanes per row
                    if (!((bits >> (lane >> 1)) & 1u))
#pragma unroll
                        for (int c = 0; c < 4 * S::HALVES; ++c)
                            *reinterpret_cast<uint4*>(smem + slot * S::STAGE + (S::HALVES + (c >> 2)) * CR_HALF_BYTES + (warp * CR_KEYS + (lane >> 1)) * 128 +
                                                      ((lane & 1) * 4 + (c & 3)) * 16) = make_uint4(0, 0, 0, 0);
                    __syncwarp();
                }
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[h][e] = (bits >> (h * 8 + 2 * t + (e & 1))) & 1u ? s[h][e] * p.scale_log2 : -INFINITY;
                        top[e >> 1] = fmaxf(top[e >> 1], s[h][e]);
                    }
                float alpha[2], ref[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                    const float mn = fmaxf(m[r], top[r]);
                    ref[r] = mn == -INFINITY ? 0.f : mn;         // nothing seen yet: every exponential below is 2^-inf = 0
                    alpha[r] = ex2(m[r] - ref[r]);
                    m[r] = mn;
                    l[r] *= alpha[r];
                }
                uint32_t pf[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float e[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) e[q] = ex2(s[h][q] - ref[q >> 1]);
                    l[0] += e[0] + e[1];
                    l[1] += e[2] + e[3];
                    pf[2 * h] = pack_h16<F16>(e[0], e[1]);
                    pf[2 * h + 1] = pack_h16<F16>(e[2], e[3]);
                }
                if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                    for (int c = 0; c < 2 * NK; ++c) {
                        o[c][0] *= alpha[0];
                        o[c][1] *= alpha[0];
                        o[c][2] *= alpha[1];
                        o[c][3] *= alpha[1];
                    }
                }
#pragma unroll
                for (int kk = 0; kk < NK; ++kk) {
                    uint32_t b[4];
                    ldmatrix_x4_trans(b, vs + (kk >> 2) * CR_HALF_BYTES + v_row + (v_x ^ ((kk & 3) << 5)));
                    mma_16816_t<F16>(o[2 * kk], pf, b[0], b[1]);
                    mma_16816_t<F16>(o[2 * kk + 1], pf, b[2], b[3]);
                }
                if (bits != 0xffffu && (mask || cut)) fence_proxy_async_smem();   // zeros written here, ahead of the next copy into the slot
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[slot]);
        }
    }
    if (!ok && lane == 0) {
        atomicExch(&p.status[0], SVDQ_ERR_TIMEOUT);
        atomicExch(&p.status[1], 880 + warp);
    }
    __syncwarp();   // the producer's lanes among them
    // Every CTA of the cluster has started (its shared memory may be written from here on); the wait is at the joining below.
    if (split > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    __syncthreads();
    // ---- the warps' sums into shared memory (over the ring: every copy has been waited for), rows that exist only
    float* part = reinterpret_cast<float*>(smem);                  // [4][16][COLS]
    float* pm = part + CR_WARPS * CR_ROWS * S::COLS;               // [4][16] maxima, then the warps' factors
    float* pl = pm + CR_WARPS * CR_ROWS;                           // [4][16] sums
    if (warp < CR_WARPS) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = g + 8 * i;
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if (r < rows) {
                if (t == 0) {
                    pm[warp * CR_ROWS + r] = m[i];
                    pl[warp * CR_ROWS + r] = l[i];
                }
                float* dst = part + (warp * CR_ROWS + r) * S::COLS + 2 * t;
#pragma unroll
                for (int c = 0; c < 2 * NK; ++c) *reinterpret_cast<float2*>(dst + c * 8) = make_float2(o[c][2 * i], o[c][2 * i + 1]);
            }
        }
    }
    __syncthreads();
    // ---- joined over the warps and sent to the CTA of the cluster that finishes the element: pair of channels e (row e / (COLS / 2))
    // belongs to CTA e % split, which keeps [source CTA][e / split] pairs, and every CTA every source's maximum and sum per row
    constexpr int HALF = S::COLS / 2;
    const int elems = rows * HALF, per = (elems + split - 1) >> log_split;
    float2* mail = reinterpret_cast<float2*>(smem + S::RING + 64);   // [split][per]
    float2* stat = mail + split * per;                               // [split][rows]: maximum, sum
    if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid < rows) {
        float mw[CR_WARPS], mm = -INFINITY, ls = 0.f;
#pragma unroll
        for (int w = 0; w < CR_WARPS; ++w) mm = fmaxf(mm, mw[w] = pm[w * CR_ROWS + tid]);
        const float b = mm == -INFINITY ? 0.f : mm;
#pragma unroll
        for (int w = 0; w < CR_WARPS; ++w) {
            const float f = ex2(mw[w] - b);
            pm[w * CR_ROWS + tid] = f;
            ls = fmaf(f, pl[w * CR_ROWS + tid], ls);
        }
#pragma unroll 1
        for (int q = 0; q < split; ++q) {
            float2* dst = stat + rank * rows + tid;
            if (split > 1) st_shared_cluster_f32x2(mapa_shared(smem_u32(dst), q), make_float2(mm, ls));
            else *dst = make_float2(mm, ls);
        }
    }
    __syncthreads();
#pragma unroll 2
    for (int e = tid; e < elems; e += CR_THREADS) {
        const int r = e / HALF, c = (e % HALF) * 2;
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < CR_WARPS; ++w) {
            const float f = pm[w * CR_ROWS + r];
            const float2 v = *reinterpret_cast<const float2*>(part + (w * CR_ROWS + r) * S::COLS + c);
            sum.x = fmaf(f, v.x, sum.x);
            sum.y = fmaf(f, v.y, sum.y);
        }
        float2* dst = mail + rank * per + (e >> log_split);
        if (split > 1) st_shared_cluster_f32x2(mapa_shared(smem_u32(dst), e & (split - 1)), sum);
        else *dst = sum;
    }
    if (split > 1) cluster_sync_all();   // nothing is read from or written to another CTA behind this
    else __syncthreads();
    // ---- joined over the CTAs: factors of the sources first (over the warps' sums, which have been read)
    float* factor = part;                // [split][rows], the quotient by the whole sum included
    if (tid < rows) {
        float mm = -INFINITY, ls = 0.f;
#pragma unroll 1
        for (int q = 0; q < split; ++q) mm = fmaxf(mm, stat[q * rows + tid].x);
        const float b = mm == -INFINITY ? 0.f : mm;
#pragma unroll 1
        for (int q = 0; q < split; ++q) {
            const float2 ml = stat[q * rows + tid];
            const float f = ex2(ml.x - b);
            factor[q * rows + tid] = f;
            ls = fmaf(f, ml.y, ls);
        }
        const float inv = ls == 0.f ? 0.f : 1.f / ls;   // nothing seen: zeros (a sum over anything is at least 1)
#pragma unroll 1
        for (int q = 0; q < split; ++q) factor[q * rows + tid] *= inv;
    }
    __syncthreads();
#pragma unroll 1
    for (int e = rank + split * tid; e < elems; e += split * CR_THREADS) {
        const int r = e / HALF, c = (e % HALF) * 2, row = r0 + r;
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll 2
        for (int q = 0; q < split; ++q) {
            const float f = factor[q * rows + r];
            const float2 v = mail[q * per + (e >> log_split)];
            sum.x = fmaf(f, v.x, sum.x);
            sum.y = fmaf(f, v.y, sum.y);
        }
        if (c < p.dim)
            *reinterpret_cast<uint32_t*>(p.out + batch * p.os[0] + (kv_head * p.group + row % p.group) * p.os[1] + (row / p.group) * p.os[2] + 2 * c) =
                pack_h16<F16>(sum.x, sum.y);
    }
}

// ---------------------------------------------------------------------------------------------------------------- host
struct CrossTensor {
    const void* base;
    int64_t stride[3];   // batch, head, token
    int batch, heads, tokens;
};

// 4-D tiled map (channel, token, head, batch).  A dimension of one, or broadcast with stride 0, is encoded with one entry and some
// valid stride; *bmul / *hmul say whether its coordinate counts.
static int cross_tmap(CUtensorMap* map, const CrossTensor& t, int dim, int dtype, int box_rows, int* bmul, int* hmul, int box_channels = 64) {
    const int64_t any = dim;   // a multiple of 8
    *bmul = t.batch > 1 && t.stride[0] != 0;
    *hmul = t.heads > 1 && t.stride[1] != 0;
    const uint64_t dims[4] = {static_cast<uint64_t>(dim), static_cast<uint64_t>(t.tokens), static_cast<uint64_t>(*hmul ? t.heads : 1),
                              static_cast<uint64_t>(*bmul ? t.batch : 1)};
    const uint64_t strides[3] = {2 * static_cast<uint64_t>(t.tokens > 1 ? t.stride[2] : any), 2 * static_cast<uint64_t>(*hmul ? t.stride[1] : any),
                                 2 * static_cast<uint64_t>(*bmul ? t.stride[0] : any)};
    const uint32_t box[4] = {static_cast<uint32_t>(box_channels), static_cast<uint32_t>(box_rows), 1, 1};
    return make_tmap_nd(map, t.base, dtype == SVDQ_DTYPE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, dims, strides,
                        box, box_channels == 64 ? 128 : 64);
}

template <bool F16, bool MASK, int TILES>
static int launch_cross_tile(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to, const CrossTileParams& p, int sms, cudaStream_t stream) {
    using Sz = CrossTileSizes<TILES>;
    auto kern = cross_tile_kernel<F16, MASK, TILES>;
    // the budget above is of the registers that the compiler gave the kernel: with fewer an increase would wait for good
    static const int regs = [&] {
        cudaFuncAttributes fa = {};
        return cudaFuncGetAttributes(&fa, kern) == cudaSuccess ? fa.numRegs : 0;
    }();
    if (regs < Sz::REGS_LAUNCH) return fail(SVDQ_ERR_CUDA, "cross_attention: built with %d registers a thread, %d needed", regs, Sz::REGS_LAUNCH);
    static std::atomic<uint64_t> attr_done{0};
    if (int rc = ensure_dynamic_smem(kern, Sz::SMEM + CT_TABLE_BYTES, attr_done)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.items < Sz::PER_SM * sms ? p.items : Sz::PER_SM * sms, 1, 1);   // all resident; each works through its share of the items
    cfg.blockDim = dim3(Sz::THREADS, 1, 1);
    cfg.dynamicSmemBytes = Sz::SMEM + p.batch * (8 + 4 * p.mask_words);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // the prologue may run under the predecessor's tail
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    SVDQ_CUDA(cudaLaunchKernelEx(&cfg, kern, tq, tk, tv, to, p));
    return SVDQ_OK;
}
template <bool F16, bool MASK>
static int launch_cross_tile(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to, const CrossTileParams& p, int tiles, int sms,
                             cudaStream_t stream) {
    return tiles == 2 ? launch_cross_tile<F16, MASK, 2>(tq, tk, tv, to, p, sms, stream) : launch_cross_tile<F16, MASK, 1>(tq, tk, tv, to, p, sms, stream);
}

template <bool F16, int NK>
static int launch_cross_rows(const CUtensorMap& tk, const CUtensorMap& tv, const CrossRowsParams& p, int pairs, int split, cudaStream_t stream) {
    auto kern = cross_rows_kernel<F16, NK>;
    static std::atomic<uint64_t> attr_done{0};
    if (int rc = ensure_dynamic_smem(kern, CrossRowsSizes<NK>::smem(CR_ROWS, CR_MAX_SPLIT), attr_done, true)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(pairs * split, (p.q_rows + CR_ROWS - 1) / CR_ROWS, 1);
    cfg.blockDim = dim3(CR_THREADS, 1, 1);
    cfg.dynamicSmemBytes = CrossRowsSizes<NK>::smem(p.q_rows < CR_ROWS ? p.q_rows : CR_ROWS, split);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // the prologue may run under the predecessor's tail
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    SVDQ_CUDA(cudaLaunchKernelEx(&cfg, kern, tk, tv, p, __builtin_ctz(split)));   // a power of two
    return SVDQ_OK;
}

template <bool F16>
static int launch_cross_rows_dim(const CUtensorMap& tk, const CUtensorMap& tv, const CrossRowsParams& p, int pairs, int split, cudaStream_t stream) {
    switch ((p.dim + 15) / 16) {
        case 1: return launch_cross_rows<F16, 1>(tk, tv, p, pairs, split, stream);
        case 2: return launch_cross_rows<F16, 2>(tk, tv, p, pairs, split, stream);
        case 3: return launch_cross_rows<F16, 3>(tk, tv, p, pairs, split, stream);
        case 4: return launch_cross_rows<F16, 4>(tk, tv, p, pairs, split, stream);
        case 5: return launch_cross_rows<F16, 5>(tk, tv, p, pairs, split, stream);
        case 6: return launch_cross_rows<F16, 6>(tk, tv, p, pairs, split, stream);
        case 7: return launch_cross_rows<F16, 7>(tk, tv, p, pairs, split, stream);
        default: return launch_cross_rows<F16, 8>(tk, tv, p, pairs, split, stream);
    }
}

}  // namespace svdq

extern "C" int svdq_cross_attention(const svdq_cross_attention_args* a, void* stream) {
    using namespace svdq;
    SVDQ_CHECK_ARG(a && a->q && a->k && a->v && a->out, "cross_attention: null tensor pointer");
    SVDQ_CHECK_ARG(a->batch > 0 && a->heads > 0 && a->kv_heads > 0 && a->q_len > 0 && a->kv_len > 0 && a->batch <= 65535 && a->heads <= 65535 &&
                       a->q_len <= (1 << 30) && a->kv_len <= (1 << 30),
                   "cross_attention: bad sizes");
    SVDQ_CHECK_ARG(a->heads % a->kv_heads == 0, "cross_attention: kv_heads (%d) must divide heads (%d)", a->kv_heads, a->heads);
    SVDQ_CHECK_ARG(a->head_dim > 0 && a->head_dim <= 128 && a->head_dim % 8 == 0, "cross_attention: head_dim %d (multiples of 8 up to 128)", a->head_dim);
    SVDQ_CHECK_ARG(a->dtype == SVDQ_DTYPE_BF16 || a->dtype == SVDQ_DTYPE_FP16, "cross_attention: bad dtype %d", a->dtype);
    SVDQ_CHECK_ARG(a->scale > 0.f && a->scale < 3e38f, "cross_attention: scale must be positive");
    SVDQ_CHECK_ARG((a->kv_lens != nullptr) + (a->kv_offsets != nullptr) + (a->mask != nullptr) <= 1,
                   "cross_attention: at most one of kv_lens, kv_offsets and mask");
    SVDQ_CHECK_ARG(!a->mask || a->mask_stride >= 0, "cross_attention: the mask's row stride must not be negative");
    SVDQ_CHECK_ARG(aligned(a->q, 16) && aligned(a->k, 16) && aligned(a->v, 16) && aligned(a->out, 16) && aligned(a->kv_lens, 4) && aligned(a->kv_offsets, 4),
                   "cross_attention: tensors must be 16-byte aligned");
    const int kv_batch = a->kv_offsets ? 1 : a->batch;
    const CrossTensor tq = {a->q, {a->q_stride[0], a->q_stride[1], a->q_stride[2]}, a->batch, a->heads, a->q_len};
    const CrossTensor tk = {a->k, {a->k_stride[0], a->k_stride[1], a->k_stride[2]}, kv_batch, a->kv_heads, a->kv_len};
    const CrossTensor tv = {a->v, {a->v_stride[0], a->v_stride[1], a->v_stride[2]}, kv_batch, a->kv_heads, a->kv_len};
    const CrossTensor to = {a->out, {a->o_stride[0], a->o_stride[1], a->o_stride[2]}, a->batch, a->heads, a->q_len};
    for (const CrossTensor* t : {&tq, &tk, &tv, &to}) {
        const int size[3] = {t->batch, t->heads, t->tokens};
        for (int i = 0; i < 3; ++i) {
            const int64_t s = t->stride[i];
            SVDQ_CHECK_ARG(size[i] == 1 || (s % 8 == 0 && s >= 0 && s < (1ll << 38)), "cross_attention: strides must be multiples of 8 elements");
            SVDQ_CHECK_ARG(size[i] == 1 || s >= a->head_dim || (s == 0 && i < 2 && t != &to),
                           "cross_attention: strides must be at least head_dim (batch and head strides of q, k and v may be 0)");
        }
    }
    const int group = a->heads / a->kv_heads;
    const long long q_rows = static_cast<long long>(a->q_len) * group;
    if (a->mask && a->kv_len > CT_MASK_STATES)
        return fail(SVDQ_ERR_UNSUPPORTED, "cross_attention: a mask covers at most %d states (got %d)", CT_MASK_STATES, a->kv_len);
    if (int rc = check_arch()) return rc;
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool f16 = a->dtype == SVDQ_DTYPE_FP16;
    const CrossStates states = {a->kv_lens, a->kv_offsets, static_cast<const uint8_t*>(a->mask), a->mask_stride, a->kv_len};
    const float scale_log2 = a->scale * 1.4426950408889634f;
    const long long kv_pairs = static_cast<long long>(a->batch) * a->kv_heads;
    // Which kernel: up to 16 rows per stored head the row kernel; beyond, the one that both kernels' times, fitted in microseconds to
    // 17 to 512 rows, 77 to 4096 states and 8 to 256 pairs of sample and stored head, say is faster.  The row kernel reads K and V again for every
    // 16 rows but splits the states; the tile kernel takes 128 rows of one query head at a time, a CTA per 128 x head, and walks all states.
    // (1 sample, 20 heads of 112, 32 queries over 4096 states: 16 us against 57; 16 x 16 x 64, 128 queries: 233 against 70.)
    const long long len = a->kv_offsets ? (a->kv_len + a->batch - 1) / a->batch : a->kv_len;   // states per sample as far as the host knows
    const long long tiles = (len + CR_TILE - 1) / CR_TILE, ctas = kv_pairs * ((q_rows + CR_ROWS - 1) / CR_ROWS);
    // Split while the CTAs are all resident at once: a further wave costs more than it balances (16 samples x 8 heads x 4096 x 128:
    // 43 us with 256 CTAs, 47 with 512, 57 with 1024).
    const long long resident = static_cast<long long>(sms) * cross_rows_per_sm((a->head_dim + 15) / 16);
    int split = 1;
    while (split < 8 && ctas * split * 2 <= resident && 2 * split <= tiles) split *= 2;
    // 16 where every CTA still has four tiles (1 x 24 heads (8 stored) x 30000 x 128: 38.5 -> 29 us, 1 x 20 x 4096 x 112: 13 -> 11.5; with one
    // tile each 1 x 24 x 1200 x 64 goes from 6.6 to 8.7).  Such clusters fit a GPC's SMs less well: three quarters of the places are counted on.
    if (split == 8 && ctas * 16 <= resident * 3 / 4 && tiles >= 4 * 16) split = 16;
    const long long q_items = static_cast<long long>(a->batch) * a->heads * ((a->q_len + CT_BM - 1) / CT_BM);
    const double rows_alone = 0.65 * static_cast<double>((tiles + split - 1) / split),
                 rows_shared = (a->head_dim > 64 ? 0.53 : 0.26) * static_cast<double>(ctas) * static_cast<double>(tiles) / sms;
    const double rows_us = 6.5 + (rows_alone > rows_shared ? rows_alone : rows_shared);
    const double tile_us = 5.0 + (q_items <= sms ? 0.8 : 1.0 * static_cast<double>((q_items + 2 * sms - 1) / (2 * sms))) * static_cast<double>(tiles);
    // (no wait of the row kernel lasts longer than a few tiles, however many states there are)
    if ((q_rows <= CR_ROWS || rows_us < tile_us || a->kv_len > CT_MAX_STATES) && kv_pairs * CR_MAX_SPLIT < (1ll << 31) && q_rows <= CR_ROWS * 65535ll) {
        CrossRowsParams p = {};
        p.st = states;
        p.q = static_cast<const uint8_t*>(a->q);
        p.out = static_cast<uint8_t*>(a->out);
        for (int i = 0; i < 3; ++i) {
            p.qs[i] = 2 * a->q_stride[i];
            p.os[i] = 2 * a->o_stride[i];
        }
        p.kv_heads = a->kv_heads;
        p.group = group;
        p.q_rows = static_cast<int>(q_rows);
        p.dim = a->head_dim;
        p.scale_log2 = scale_log2;
        if (int rc = status_words(&p.status)) return rc;
        CUtensorMap mk, mv;
        if (int rc = cross_tmap(&mk, tk, a->head_dim, a->dtype, CR_TILE, &p.k_bmul, &p.k_hmul)) return rc;
        if (int rc = cross_tmap(&mv, tv, a->head_dim, a->dtype, CR_TILE, &p.v_bmul, &p.v_hmul)) return rc;
        return f16 ? launch_cross_rows_dim<true>(mk, mv, p, static_cast<int>(kv_pairs), split, st)
                   : launch_cross_rows_dim<false>(mk, mv, p, static_cast<int>(kv_pairs), split, st);
    }
    if (a->kv_len > CT_MAX_STATES)
        return fail(SVDQ_ERR_UNSUPPORTED, "cross_attention: more than %d states (got %d) for so many queries", CT_MAX_STATES, a->kv_len);
    // The kernel keeps its samples' ranges and mask bits in shared memory: launches of as many samples as fit (hundreds, without a mask).
    const int q_tiles = (a->q_len + CT_BM - 1) / CT_BM;
    const int mask_words = a->mask ? (a->kv_len + CT_BN - 1) / CT_BN * (CT_BN / 32) : 0;
    const int most = CT_TABLE_BYTES / (8 + 4 * mask_words);
    SVDQ_CHECK_ARG(static_cast<long long>(a->heads) * q_tiles * (a->batch < most ? a->batch : most) < (1ll << 30), "cross_attention: too many query tiles");
    // Two tiles over the same states where there are more tiles than places for one-tile CTAs and they go into pairs, of one head or of two that
    // share a stored head (one tile / two, us: 32 x 20 x 1024 x 192 x 112 104 / 93, x 320 171 / 136, x 64 65 / 69; 3 x 20 x 1024 x 300 x 112 23 / 21;
    // with fewer tiles, 1 x 20 x 1000 x 77 x 64 6.7 / 7.2; with a tile twice to make nine a pair, 32 x 20 x 1152 x 200 x 112 115 / 122).
    const int tiles_at_once = q_items > 2 * sms && (group % 2 == 0 || q_tiles % 2 == 0) ? 2 : 1;
    for (int b0 = 0; b0 < a->batch; b0 += most) {
        const int nb = a->batch - b0 < most ? a->batch - b0 : most;
        auto from = [&](CrossTensor t, int count) {
            if (count) {
                t.base = static_cast<const uint8_t*>(t.base) + 2 * b0 * t.stride[0];
                t.batch = nb;
            }
            return t;
        };
        CrossTileParams p = {};
        p.st = states;
        if (p.st.kv_lens) p.st.kv_lens += b0;
        if (p.st.kv_offsets) p.st.kv_offsets += b0;
        if (p.st.mask) p.st.mask += b0 * p.st.mask_stride;
        p.q_len = a->q_len;
        p.dim = a->head_dim;
        p.group = group;
        p.scale_log2 = scale_log2;
        if (int rc = status_words(&p.status)) return rc;
        p.q_tiles = q_tiles;
        p.batch = nb;
        p.pair_heads = group % 2 == 0;
        p.units_h = tiles_at_once == 2 && p.pair_heads ? a->heads / 2 : a->heads;
        p.units_t = tiles_at_once == 2 && !p.pair_heads ? q_tiles / 2 : q_tiles;
        p.items = nb * p.units_h * p.units_t;
        p.mask_words = mask_words;
        CUtensorMap mq, mk, mv, mo;
        if (int rc = cross_tmap(&mq, from(tq, 1), a->head_dim, a->dtype, CT_BM, &p.q_bmul, &p.q_hmul)) return rc;
        if (int rc = cross_tmap(&mk, from(tk, !a->kv_offsets), a->head_dim, a->dtype, CT_BN, &p.k_bmul, &p.k_hmul)) return rc;
        if (int rc = cross_tmap(&mv, from(tv, !a->kv_offsets), a->head_dim, a->dtype, CT_BN, &p.v_bmul, &p.v_hmul)) return rc;
        if (int rc = cross_tmap(&mo, from(to, 1), a->head_dim, a->dtype, 32, &p.o_bmul, &p.o_hmul, 32)) return rc;
        const int rc = a->mask ? (f16 ? launch_cross_tile<true, true>(mq, mk, mv, mo, p, tiles_at_once, sms, st) : launch_cross_tile<false, true>(mq, mk, mv, mo, p, tiles_at_once, sms, st))
                               : (f16 ? launch_cross_tile<true, false>(mq, mk, mv, mo, p, tiles_at_once, sms, st) : launch_cross_tile<false, false>(mq, mk, mv, mo, p, tiles_at_once, sms, st));
        if (rc) return rc;
    }
    return SVDQ_OK;
}
