// The 128x128x128 GEMMs of the sm_100a attention kernels (attn_sm100.cu,
// attn_kv4_sm100.cu), issued by one thread.
#pragma once

#include <cstdint>

#include "sm100_ptx.h"

namespace kvp {
namespace attn_dev {

// One 128x128x128 GEMM as eight back-to-back K16 MMAs, issued in two asm
// blocks (steps 0-5, then 6-7) so the issuer can test the next GEMM's
// barriers while the first six are queued.  The descriptors of steps 1..7
// are immediate offsets of step 0's: nothing but an add sits between two MMA
// issues, and the tensor core's shallow instruction queue never runs dry
// inside a GEMM.
//   S = Q K^T: A and B K-major, 128B swizzle, two 64-column panels 16 KB
//   apart: step ks starts (ks>>2)*16384 + (ks&3)*32 bytes in, i.e. adds
//   (ks>>2)*1024 + (ks&3)*2 to the 16-byte address field.
__device__ __forceinline__ void tc_gemm_ss_head(uint32_t d_tmem, uint64_t a0, uint64_t b0, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred pf, pt;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 pf, 0, 0;\n\tsetp.eq.b32 pt, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, pf;\n\t"
        "add.s64 a, %1, 2;\n\tadd.s64 b, %2, 2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, pt;\n\t"
        "add.s64 a, %1, 4;\n\tadd.s64 b, %2, 4;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, pt;\n\t"
        "add.s64 a, %1, 6;\n\tadd.s64 b, %2, 6;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, pt;\n\t"
        "add.s64 a, %1, 1024;\n\tadd.s64 b, %2, 1024;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, pt;\n\t"
        "add.s64 a, %1, 1026;\n\tadd.s64 b, %2, 1026;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, pt;\n\t}"
        ::"r"(d_tmem), "l"(a0), "l"(b0), "r"(idesc));
}
__device__ __forceinline__ void tc_gemm_ss_tail(uint32_t d_tmem, uint64_t a0, uint64_t b0, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred pt;\n\t.reg .b64 a, b;\n\t"
        "setp.eq.b32 pt, 0, 0;\n\t"
        "add.s64 a, %1, 1028;\n\tadd.s64 b, %2, 1028;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, pt;\n\t"
        "add.s64 a, %1, 1030;\n\tadd.s64 b, %2, 1030;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, pt;\n\t}"
        ::"r"(d_tmem), "l"(a0), "l"(b0), "r"(idesc));
}
//   O (+)= P V: P from TMEM (step ks at column +8*ks), V MN-major with step
//   ks 16 rows = 2048 bytes further (+128 in the address field).
__device__ __forceinline__ void tc_gemm_ts_head(uint32_t d_tmem, uint32_t a_tmem, uint64_t b0, uint32_t idesc,
                                                uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred pf, pt;\n\t.reg .b64 b;\n\t.reg .b32 a;\n\t"
        "setp.ne.b32 pf, %4, 0;\n\tsetp.eq.b32 pt, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, pf;\n\t"
        "add.s32 a, %1, 8;\n\tadd.s64 b, %2, 128;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, pt;\n\t"
        "add.s32 a, %1, 16;\n\tadd.s64 b, %2, 256;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, pt;\n\t"
        "add.s32 a, %1, 24;\n\tadd.s64 b, %2, 384;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, pt;\n\t"
        "add.s32 a, %1, 32;\n\tadd.s64 b, %2, 512;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, pt;\n\t"
        "add.s32 a, %1, 40;\n\tadd.s64 b, %2, 640;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, pt;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b0), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void tc_gemm_ts_tail(uint32_t d_tmem, uint32_t a_tmem, uint64_t b0, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred pt;\n\t.reg .b64 b;\n\t.reg .b32 a;\n\t"
        "setp.eq.b32 pt, 0, 0;\n\t"
        "add.s32 a, %1, 48;\n\tadd.s64 b, %2, 768;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, pt;\n\t"
        "add.s32 a, %1, 56;\n\tadd.s64 b, %2, 896;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, pt;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b0), "r"(idesc));
}

// kind::f16 instruction descriptors: bf16 x bf16 -> f32 and fp16 x fp16 -> f32,
// M=128, N=128.
constexpr uint32_t idesc_bf16(bool b_mn_major) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) |
           ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

constexpr uint32_t idesc_f16(bool b_mn_major) { return idesc_bf16(b_mn_major) & ~((1u << 7) | (1u << 10)); }

}  // namespace attn_dev
}  // namespace kvp
