// What the attention kernels share: products of whole tiles from one election, TMEM stores, packed arithmetic of the softmax.
#pragma once
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace nxd {
namespace fa {

// Warp-uniform issue: the whole MMA warp runs the issue loop in convergent control flow and one elected lane executes the tcgen05
// instructions (sm100_ptx.cuh explains why).  One election serves the products of a whole tile and the barrier they complete; descriptors
// advance by constants.  With an election, a predicate and a new descriptor for each product the issuing warp was what a backward step
// waited for: 32 products of 32 to 64 cycles took it 2200 cycles.
#define NXD_FA_MMA "@q tcgen05.mma.cta_group::1.kind::f16 "
#define NXD_FA_BEGIN                                                                                                     \
  "{\n\t.reg .pred p, q, t;\n\t.reg .b64 a, b;\n\t.reg .b32 c;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t" \
  "setp.eq.b32 t, 0, 0;\n\t"
#define NXD_FA_COMMIT(bar) "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [" bar "];\n\t"
#define NXD_FA_SS(ia, ib) "add.s64 a, %1, " ia ";\n\tadd.s64 b, %2, " ib ";\n\t" NXD_FA_MMA "[%0], a, b, %3, t;\n\t"
#define NXD_FA_TS(ia, ib) "add.u32 c, %1, " ia ";\n\tadd.s64 b, %2, " ib ";\n\t" NXD_FA_MMA "[%0], [c], b, %3, t;\n\t"
// Eight products over 128 elements of K, both operands in shared memory; product i reads (i / 4) * 4 and (i % 4) * 1 steps (of 16 bytes) on.
template <int A4, int A1, int B4, int B1>
NXD_DEVICE void mma_ss8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t bar) {
  asm volatile(NXD_FA_BEGIN NXD_FA_MMA "[%0], %1, %2, %3, p;\n\t"
               NXD_FA_SS("%6", "%13") NXD_FA_SS("%7", "%14") NXD_FA_SS("%8", "%15") NXD_FA_SS("%9", "%16") NXD_FA_SS("%10", "%17")
               NXD_FA_SS("%11", "%18") NXD_FA_SS("%12", "%19") NXD_FA_COMMIT("%5") "}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(bar),
                 "n"(A1), "n"(2 * A1), "n"(3 * A1), "n"(A4), "n"(A4 + A1), "n"(A4 + 2 * A1), "n"(A4 + 3 * A1),
                 "n"(B1), "n"(2 * B1), "n"(3 * B1), "n"(B4), "n"(B4 + B1), "n"(B4 + 2 * B1), "n"(B4 + 3 * B1)
               : "memory");
}
// The same over 64 elements: four products.
template <int A1, int B1>
NXD_DEVICE void mma_ss4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t bar) {
  asm volatile(NXD_FA_BEGIN NXD_FA_MMA "[%0], %1, %2, %3, p;\n\t" NXD_FA_SS("%6", "%9") NXD_FA_SS("%7", "%10") NXD_FA_SS("%8", "%11")
               NXD_FA_COMMIT("%5") "}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(bar), "n"(A1), "n"(2 * A1), "n"(3 * A1), "n"(B1), "n"(2 * B1), "n"(3 * B1)
               : "memory");
}
// Four products over 64 elements of K, A in TMEM (P of the forward, Pᵀ and dSᵀ of the backward); the last two read A from A2 columns on.
template <int A2, int B1>
NXD_DEVICE void mma_ts4(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(NXD_FA_BEGIN NXD_FA_MMA "[%0], [%1], %2, %3, p;\n\t" NXD_FA_TS("8", "%5") NXD_FA_TS("%8", "%6") NXD_FA_TS("%9", "%7") "}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "n"(B1), "n"(2 * B1), "n"(3 * B1), "n"(A2), "n"(A2 + 8)
               : "memory");
}
NXD_DEVICE void tcgen05_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
NXD_DEVICE void tcgen05_st_32x16p(uint32_t taddr, const uint32_t* r) {   // first 16 registers of a larger array
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
NXD_DEVICE void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
NXD_DEVICE void tcgen05_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
NXD_DEVICE void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
NXD_DEVICE void bulk_wait_read1() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }
NXD_DEVICE void bulk_wait0() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
NXD_DEVICE uint64_t pack2u(uint32_t a, uint32_t b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b)); return r; }
NXD_DEVICE float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
NXD_DEVICE float max3_nan(float a, float b, float c) {       // NaN where one is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
NXD_DEVICE uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// columns behind `lim` to −inf: 0 after the exponential
NXD_DEVICE void fwd_mask(uint32_t (&r)[32], int lim) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (i > lim) r[i] = 0xff800000u;
}

}  // namespace fa
}  // namespace nxd
