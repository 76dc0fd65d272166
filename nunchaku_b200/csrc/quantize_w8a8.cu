// Rows of a 16-bit matrix -> signed 8-bit codes with one fp32 scale per row, sm_100a; optionally behind a residual addition and
// an RMSNorm.
//
//   h = x (+ residual)                      fp32, and rounded once to the 16-bit type for the residual stream (`hidden`)
//   z = h * w  (z = h without the norm)
//   rstd = 1 / sqrt(sum h^2 / cols + eps)   (1 without the norm)
//   scale = rstd * max|z| / 127,  code = rint(z * (127 / max|z|))
//
// The normalised value is z * rstd, and rstd cancels in code = value / scale: so the sum of squares and the maximum are
// reduced together, in one pass over registers, and the row is read once and never kept in memory.  fp32 throughout; the
// one rounding to fewer bits besides the codes is `hidden`, the residual stream in the model's own type (the norm works on
// the sum before that rounding).
// A row of zeros has scale 0 and codes 0.  A row whose sum of squares or maximum is not finite (a NaN, an infinity, squares
// beyond fp32) has scale NaN and codes 0, so that a product with it is NaN as well and not quietly wrong.
//
// HBM bound: 3 bytes per element for the codes alone, 7 with the residual.  32768 x 2240 with residual and norm: 81 us = 6.3 TB/s (0.97 of the
// copy rate); codes alone, 18433 x 5600: 50 us = 6.2 TB/s; 2147 x 2304 with the norm 4.8 us and one row 1.5 us, which are latency.
// One row per block of W warps, V 16-byte vectors per thread and tensor (W * 32 * V >= cols / 8), weights in registers over
// all rows of a block.
// Compiled once per 16-bit type: bf16 here, fp16 from quantize_w8a8_f16.cu.
#include "dtype.cuh"
#include "host_common.h"
#include "ptx.cuh"

#include <type_traits>

namespace svdq {
namespace SVDQ_DT {

constexpr int Q8_MAX_WARPS = 16, Q8_MAX_V = 4;
constexpr int Q8_MAX_COLS = Q8_MAX_WARPS * 32 * Q8_MAX_V * 8;

struct Quant8Params {
    const h16* x;
    const h16* residual;
    const h16* weight;
    int8_t* codes;
    float* scales;
    h16* hidden;
    long long rows, x_stride, residual_stride;   // strides in elements
    int cols;
    float eps;
};

// largest magnitude of three; a NaN stays one (fmaxf drops it)
__device__ __forceinline__ float absmax3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float warp_max_nan(float v) {   // of magnitudes
    float d;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
    return d;
}

// rint of four values with |v| <= 127.5 as packed bytes: adding 1.5 * 2^23 leaves the integer (ties to even) in the low byte
__device__ __forceinline__ uint32_t pack_codes4(float a, float b, float c, float d) {
    constexpr float MAGIC = 12582912.f;
    const uint32_t ia = __float_as_uint(a + MAGIC), ib = __float_as_uint(b + MAGIC), ic = __float_as_uint(c + MAGIC),
                   id = __float_as_uint(d + MAGIC);
    return __byte_perm(__byte_perm(ia, ib, 0x0040), __byte_perm(ic, id, 0x0040), 0x5410);
}

template <bool NORM, bool RES, int V>
__global__ void __launch_bounds__(Q8_MAX_WARPS * 32, V == 4 ? 1 : 2)
quantize_w8a8_kernel(const Quant8Params p) {
    const int lane = threadIdx.x, W = blockDim.y;
    __shared__ float2 part[2][Q8_MAX_WARPS];
    const int nvec = p.cols >> 3;
    const int tid = threadIdx.y * 32 + lane, threads = W * 32;
    pdl_launch_dependents();
    pdl_wait();   // nothing above touches global memory
    uint4 wv[V];
    if constexpr (NORM) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            wv[j] = tid + j * threads < nvec ? reinterpret_cast<const uint4*>(p.weight)[tid + j * threads] : make_uint4(0, 0, 0, 0);
    }
    // the next row's loads go out while this row is reduced, where the registers for that are there (with a residual: at V = 2 only)
    constexpr bool AHEAD = !RES || V == 2;
    uint4 xv[V], rv[V];
    auto fetch = [&](long long row) {
        const uint4* xp = reinterpret_cast<const uint4*>(p.x + row * p.x_stride);
#pragma unroll
        for (int j = 0; j < V; ++j) xv[j] = tid + j * threads < nvec ? xp[tid + j * threads] : make_uint4(0, 0, 0, 0);
        if constexpr (RES) {
            const uint4* rp = reinterpret_cast<const uint4*>(p.residual + row * p.residual_stride);
#pragma unroll
            for (int j = 0; j < V; ++j) rv[j] = tid + j * threads < nvec ? rp[tid + j * threads] : make_uint4(0, 0, 0, 0);
        }
    };
    long long row = blockIdx.x;
    if (AHEAD && row < p.rows) fetch(row);
    int buf = 0;
    for (; row < p.rows; row += gridDim.x, buf ^= 1) {
        if (!AHEAD) fetch(row);
        float z[V][8];
        float ss = 0.f, top = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t xw[4] = {xv[j].x, xv[j].y, xv[j].z, xv[j].w};
            uint32_t hw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2 h = unpack2(xw[i]);
                if constexpr (RES) {
                    const uint32_t rw[4] = {rv[j].x, rv[j].y, rv[j].z, rv[j].w};
                    const float2 r = unpack2(rw[i]);
                    h.x += r.x;
                    h.y += r.y;
                    hw[i] = pack2(h);
                }
                if constexpr (NORM) {
                    const uint32_t ww[4] = {wv[j].x, wv[j].y, wv[j].z, wv[j].w};
                    const float2 w = unpack2(ww[i]);
                    ss = fmaf(h.x, h.x, fmaf(h.y, h.y, ss));
                    h.x *= w.x;
                    h.y *= w.y;
                }
                z[j][2 * i] = h.x;
                z[j][2 * i + 1] = h.y;
                top = absmax3_nan(top, h.x, h.y);
            }
            if constexpr (RES) {
                if (tid + j * threads < nvec)
                    reinterpret_cast<uint4*>(p.hidden + row * p.cols)[tid + j * threads] = make_uint4(hw[0], hw[1], hw[2], hw[3]);
            }
        }
        if (AHEAD && row + gridDim.x < p.rows) fetch(row + gridDim.x);   // while this row is reduced and written
        if constexpr (NORM) {
#pragma unroll
            for (int m = 16; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        }
        top = warp_max_nan(top);
        if (W > 1) {
            // two buffers in turn: a warp that writes row r + 2 has passed row r + 1's barrier, which every reader of row r's
            // values reaches behind its reads
            if (lane == 0) part[buf][threadIdx.y] = make_float2(ss, top);
            __syncthreads();
            const float2 o = lane < W ? part[buf][lane] : make_float2(0.f, 0.f);
            ss = o.x;
            if constexpr (NORM) {
#pragma unroll
                for (int m = 8; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);   // at most 16 warps
                ss = __shfl_sync(0xffffffffu, ss, 0);
            }
            top = warp_max_nan(o.y);
        }
        // Per-row scalars, which every thread computes: kept to a few instructions (with four full divisions and a root the kernel was
        // bound by them).
        const bool finite = top < __int_as_float(0x7f800000) && ss < __int_as_float(0x7f800000);   // false for NaN
        // 2^100 or 2^-100 (exact) for a row whose 127 / top would leave fp32, or its reciprocal lose bits
        const float up = top < 1e-30f ? 1.2676506002282294e30f : top > 1e30f ? 7.888609052210118e-31f : 1.0f;
        const float inv = top > 0.f ? 127.0f * __frcp_rn(top * up) : 0.f;
        // 127 / top to twice the precision: a value of half the row's largest, common among 16-bit inputs, stands exactly on the tie 63.5,
        // and is to be told from its neighbours by the quotient, not by the rounding of the reciprocal
        const float inv_lo = NORM ? 0.f : fmaf(-(top * up), inv, 127.0f) * (inv * (1.0f / 127.0f));
        if (up != 1.0f) {
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) z[j][i] *= up;
        }
        auto code = [&](float v) { return NORM ? v * inv : fmaf(v, inv, v * inv_lo); };
        uint2* cp = reinterpret_cast<uint2*>(p.codes + row * p.cols);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (tid + j * threads >= nvec) continue;
            const uint2 c = make_uint2(pack_codes4(code(z[j][0]), code(z[j][1]), code(z[j][2]), code(z[j][3])),
                                       pack_codes4(code(z[j][4]), code(z[j][5]), code(z[j][6]), code(z[j][7])));
            cp[tid + j * threads] = finite ? c : make_uint2(0u, 0u);
        }
        if (tid == 0) {
            const float rstd = NORM ? 1.0f / sqrtf(ss / static_cast<float>(p.cols) + p.eps) : 1.0f;
            p.scales[row] = finite ? top * rstd / 127.0f : __int_as_float(0x7fc00000);
        }
    }
}

// launched so that the start may lie under the predecessor's tail (both kernels wait for it before they touch global memory): behind
// one another on 2147 x 2304 9.2 -> 8.8 us for the two, on one row 3.4 -> 2.8
template <typename Kernel, typename... Args>
static int launch_q8(Kernel kernel, int grid, dim3 block, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = block;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    SVDQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    return SVDQ_OK;
}

template <bool NORM, bool RES, int V>
static int launch_quant8(const Quant8Params& p, int warps, int sms, cudaStream_t stream) {
    const long long per_sm = 2048 / (warps * 32) < 32 ? 2048 / (warps * 32) : 32;
    const long long cap = sms * (per_sm > 0 ? per_sm : 1);
    const int grid = static_cast<int>(p.rows < cap ? p.rows : cap);
    return launch_q8(quantize_w8a8_kernel<NORM, RES, V>, grid, dim3(32, warps), stream, p);
}

int quantize_w8a8_impl(const svdq_quantize_w8a8_args* a, void* stream) {
    SVDQ_CHECK_ARG(a && a->x && a->codes && a->scales, "quantize_w8a8: null pointer");
    SVDQ_CHECK_ARG(a->rows > 0 && a->cols > 0 && a->cols % 16 == 0, "quantize_w8a8: cols (%d) must be a positive multiple of 16", a->cols);
    if (a->cols > Q8_MAX_COLS) return fail(SVDQ_ERR_UNSUPPORTED, "quantize_w8a8: at most %d columns (got %d)", Q8_MAX_COLS, a->cols);
    SVDQ_CHECK_ARG(!a->residual == !a->hidden, "quantize_w8a8: residual and hidden go together");
    SVDQ_CHECK_ARG(!a->residual || a->weight, "quantize_w8a8: the residual form needs a norm weight");
    SVDQ_CHECK_ARG(a->x_stride >= a->cols && a->x_stride % 8 == 0 && (!a->residual || (a->residual_stride >= a->cols && a->residual_stride % 8 == 0)),
                   "quantize_w8a8: row strides must be multiples of 8 elements, at least cols");
    // (with less, a row whose squares vanish in fp32 would be divided by zero)
    SVDQ_CHECK_ARG(!a->weight || a->eps >= 1e-30f, "quantize_w8a8: eps must be at least 1e-30");
    SVDQ_CHECK_ARG(aligned(a->x, 16) && aligned(a->residual, 16) && aligned(a->weight, 16) && aligned(a->hidden, 16) && aligned(a->codes, 16) &&
                       aligned(a->scales, 4),
                   "quantize_w8a8: tensors must be 16-byte aligned");
    if (int rc = check_arch()) return rc;
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    Quant8Params p = {static_cast<const h16*>(a->x), static_cast<const h16*>(a->residual), static_cast<const h16*>(a->weight),
                      static_cast<int8_t*>(a->codes), a->scales, static_cast<h16*>(a->hidden), a->rows, a->x_stride, a->residual_stride,
                      a->cols, a->eps};
    const int nvec = a->cols / 8;
    int v = (nvec + 32 * Q8_MAX_WARPS - 1) / (32 * Q8_MAX_WARPS);
    // More rows than SMs: three vectors per thread, so that the per-row scalars and reductions are shared by as many elements as the
    // registers allow.  With a residual two and the next row in flight are faster between 1536 and 4608 columns (2240: 87 -> 81 us for
    // 32768 rows; 4096: 19.9 -> 18.9 us for 4096), and slower outside (1152: 78 -> 86 us for 60000 rows; 12288: 113 -> 134 us for 8192).
    const int most = a->residual && a->cols > 1536 && a->cols <= 4608 ? 2 : 3;
    if (a->rows > sms)
        while (v < most && nvec > 32 * v) ++v;
    const int warps = (nvec + 32 * v - 1) / (32 * v);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto by_v = [&](auto norm, auto res) {
        constexpr bool N = decltype(norm)::value, R = decltype(res)::value;
        switch (v) {
            case 1: return launch_quant8<N, R, 1>(p, warps, sms, st);
            case 2: return launch_quant8<N, R, 2>(p, warps, sms, st);
            case 3: return launch_quant8<N, R, 3>(p, warps, sms, st);
            default: return launch_quant8<N, R, 4>(p, warps, sms, st);
        }
    };
    if (!a->weight) return by_v(std::false_type{}, std::false_type{});
    return a->residual ? by_v(std::true_type{}, std::true_type{}) : by_v(std::true_type{}, std::false_type{});
}

// The values that codes stand for: out = code * scale of its row, fp32 product, one rounding.  16 codes per thread; HBM bound at
// 3 bytes per element (18433 x 5600: 51 us = 6.1 TB/s).  INDEX: 32 bits as long as the number of 16-code pieces allows (the division that finds the row is then
// a fifth of the 64-bit one's instructions).
template <typename INDEX>
__global__ void __launch_bounds__(256)
dequantize_w8a8_kernel(const uint4* codes, const float* scales, uint4* out, INDEX total, INDEX per_row) {
    pdl_launch_dependents();
    pdl_wait();   // nothing above touches global memory
    for (INDEX i = static_cast<INDEX>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += static_cast<INDEX>(gridDim.x) * blockDim.x) {
        const uint4 c = codes[i];
        const float s = scales[i / per_row];
        const uint32_t cw[4] = {c.x, c.y, c.z, c.w};
        uint32_t o[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int w = static_cast<int>(cw[k]);
            o[2 * k] = pack2(make_float2(static_cast<float>(w << 24 >> 24) * s, static_cast<float>(w << 16 >> 24) * s));
            o[2 * k + 1] = pack2(make_float2(static_cast<float>(w << 8 >> 24) * s, static_cast<float>(w >> 24) * s));
        }
        out[2 * i] = make_uint4(o[0], o[1], o[2], o[3]);
        out[2 * i + 1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
}

int dequantize_w8a8_impl(const svdq_dequantize_w8a8_args* a, void* stream) {
    SVDQ_CHECK_ARG(a && a->codes && a->scales && a->out, "dequantize_w8a8: null pointer");
    SVDQ_CHECK_ARG(a->rows > 0 && a->cols > 0 && a->cols % 16 == 0, "dequantize_w8a8: cols (%d) must be a positive multiple of 16", a->cols);
    SVDQ_CHECK_ARG(aligned(a->codes, 16) && aligned(a->out, 16) && aligned(a->scales, 4), "dequantize_w8a8: tensors must be 16-byte aligned");
    if (int rc = check_arch()) return rc;
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    const long long per_row = a->cols / 16;
    SVDQ_CHECK_ARG(a->rows <= (1ll << 40) / per_row, "dequantize_w8a8: too many rows");
    const long long total = a->rows * per_row, want = (total + 255) / 256;
    const int grid = static_cast<int>(want < 32LL * sms ? want : 32LL * sms);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const uint4* c = static_cast<const uint4*>(a->codes);
    uint4* o = static_cast<uint4*>(a->out);
    if (total < (1ll << 31))
        return launch_q8(dequantize_w8a8_kernel<uint32_t>, grid, dim3(256), st, c, a->scales, o, static_cast<uint32_t>(total), static_cast<uint32_t>(per_row));
    return launch_q8(dequantize_w8a8_kernel<unsigned long long>, grid, dim3(256), st, c, a->scales, o, static_cast<unsigned long long>(total),
                     static_cast<unsigned long long>(per_row));
}

}  // namespace SVDQ_DT
}  // namespace svdq

#ifndef SVDQ_F16
namespace svdq {
namespace hf {
int quantize_w8a8_impl(const svdq_quantize_w8a8_args* a, void* stream);
int dequantize_w8a8_impl(const svdq_dequantize_w8a8_args* a, void* stream);
}
}  // namespace svdq

extern "C" int svdq_quantize_w8a8(const svdq_quantize_w8a8_args* a, void* stream) {
    if (a && a->dtype == SVDQ_DTYPE_FP16) return svdq::hf::quantize_w8a8_impl(a, stream);
    if (a && a->dtype != SVDQ_DTYPE_BF16) return svdq::fail(SVDQ_ERR_INVALID_ARGUMENT, "quantize_w8a8: bad dtype %d", a->dtype);
    return svdq::bf::quantize_w8a8_impl(a, stream);
}

extern "C" int svdq_dequantize_w8a8(const svdq_dequantize_w8a8_args* a, void* stream) {
    if (a && a->dtype == SVDQ_DTYPE_FP16) return svdq::hf::dequantize_w8a8_impl(a, stream);
    if (a && a->dtype != SVDQ_DTYPE_BF16) return svdq::fail(SVDQ_ERR_INVALID_ARGUMENT, "dequantize_w8a8: bad dtype %d", a->dtype);
    return svdq::bf::dequantize_w8a8_impl(a, stream);
}
#endif
