// Device helpers shared by the attention kernels: the 4-D TMA load, single-CTA kind::f16 MMAs (A in shared or tensor memory),
// their descriptors, packing and the two exponentials.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace svdq {

__device__ __forceinline__ void tma_store_4d(const void* tmap, const void* src, int x, int y, int z, int w) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
                 ::"l"(tmap), "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z), "r"(w)
                 : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const void* tmap, uint64_t* bar, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_u32(dst)), "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

// D[tmem] (+)= A[smem] * B[smem], 16-bit operands, fp32 accumulation, one CTA; in the second form A is in tensor memory: lane = row, every
// 32-bit column holds two consecutive K elements (the lower index in the lower half), so a K-step of 16 is 8 columns.
// Descriptors are given as 32-bit halves: the upper half (strides, swizzle) is a constant of the kernel and the lower half (start
// address in 16-byte units, leading byte offset) moves by small immediates, so that an unrolled issue loop needs no 64-bit
// arithmetic.  A and B share the upper half in the first form.
__device__ __forceinline__ void tc_mma_f16_lo(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc,
                                              uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_mma_f16_ts_lo(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                                 uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Instruction descriptor, kind::f16: fp32 accumulator, A and B of one 16-bit format (0 = fp16, 1 = bf16), A K-major,
// B K-major or MN-major (bit 16).
__host__ __device__ constexpr uint32_t idesc_h16(int M, int N, bool f16, bool b_mn_major) {
    return (1u << 4) | ((f16 ? 0u : 1u) << 7) | ((f16 ? 0u : 1u) << 10) | ((b_mn_major ? 1u : 0u) << 16) |
           (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

// Shared-memory descriptor of an MN-major operand under the 128-byte swizzle: 64 consecutive MN elements (128 bytes)
// per row, one row per K index, 8-row groups `sbo` bytes apart (stride byte offset), the next 64 MN elements `lbo`
// bytes on (leading byte offset).
__device__ __forceinline__ uint64_t smem_desc_sw128_mn(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((saddr & 0x3FFFF) >> 4);
    d |= static_cast<uint64_t>(lbo >> 4) << 16;
    d |= static_cast<uint64_t>(sbo >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

template <bool F16>
__device__ __forceinline__ uint32_t pack_h16(float lo, float hi) {
    uint32_t r;
    if constexpr (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// 2^x for a pair of values on the FMA pipe instead of the special-function unit: x = n + f with n = rint(x) and f in
// [-0.5, 0.5]; 2^f by a cubic (relative error 7.6e-5, a sixth of fp16's rounding step and a 25th of bf16's), n added to
// the exponent field.  Adding 1.5 * 2^23 rounds x to an integer and leaves it in the low mantissa bits.  x is clamped
// at -125 (the result is then ~2e-38 instead of less).
__device__ __forceinline__ float2 exp2_fma2(float2 x) {
    x.x = fmaxf(x.x, -125.f);
    x.y = fmaxf(x.y, -125.f);
    const float2 t = __fadd2_rn(x, make_float2(12582912.f, 12582912.f));
    const float2 n = __fadd2_rn(t, make_float2(-12582912.f, -12582912.f));
    const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
    float2 r = __ffma2_rn(f, make_float2(0.05520550534129143f, 0.05520550534129143f), make_float2(0.24261397123336792f, 0.24261397123336792f));
    r = __ffma2_rn(r, f, make_float2(0.6932547688484192f, 0.6932547688484192f));
    r = __ffma2_rn(r, f, make_float2(0.9999276995658875f, 0.9999276995658875f));
    return make_float2(__int_as_float(__float_as_int(r.x) + (__float_as_int(t.x) << 23)),
                       __int_as_float(__float_as_int(r.y) + (__float_as_int(t.y) << 23)));
}

}  // namespace svdq
