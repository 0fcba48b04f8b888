// The PV product of one 128-key tile as a single group of tensor-core instructions, shared by the attention
// kernels (warp-collective: the whole MMA warp executes the call and one elected lane issues).
#pragma once

#include <cstdint>

namespace vb200 {

// O_t (+)= P_t V over 128 keys: eight K=16 steps; P_t in TMEM (A advances 8 columns = 16
// packed keys per step), V MN-major (B advances 2048 bytes = 128 units per step).  Commits to
// `bar`, and also to `bar2` when use_bar2 is nonzero.
__device__ __forceinline__ void issue_pv_group(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                               uint32_t acc_first, uint32_t bar, uint32_t bar2,
                                               uint32_t use_bar2) {
  asm volatile(
      "{\n\t.reg .pred e, pf, pt, p2;\n\t.reg .b64 b1, b2, b3, b4, b5, b6, b7;\n\t"
      ".reg .b32 a1, a2, a3, a4, a5, a6, a7;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 pf, %4, 0;\n\t"
      "setp.eq.b32 pt, 0, 0;\n\t"
      "setp.ne.and.b32 p2, %7, 0, e;\n\t"
      "add.s32 a1, %1, 8;\n\tadd.s64 b1, %2, 128;\n\t"
      "add.s32 a2, %1, 16;\n\tadd.s64 b2, %2, 256;\n\t"
      "add.s32 a3, %1, 24;\n\tadd.s64 b3, %2, 384;\n\t"
      "add.s32 a4, %1, 32;\n\tadd.s64 b4, %2, 512;\n\t"
      "add.s32 a5, %1, 40;\n\tadd.s64 b5, %2, 640;\n\t"
      "add.s32 a6, %1, 48;\n\tadd.s64 b6, %2, 768;\n\t"
      "add.s32 a7, %1, 56;\n\tadd.s64 b7, %2, 896;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, pf;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a4], b4, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a5], b5, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a6], b6, %3, pt;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a7], b7, %3, pt;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t"
      "@p2 tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc_first), "r"(bar), "r"(bar2), "r"(use_bar2)
      : "memory");
}

}  // namespace vb200
