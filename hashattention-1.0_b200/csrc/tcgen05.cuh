// Device primitives of the kernels on the 5th-generation tensor cores (sm_100a): shared-memory descriptors, tcgen05
// instructions, tensor-memory reads and writes, mbarriers with bounded waits, TMA box copies.
#pragma once

#include <cuda.h>  // CUtensorMap (the type only: the encoder is looked up at run time)

#include "common.cuh"

namespace ha {

constexpr int kTcSpinLimit = 1 << 16;   // tries of a wait ...
constexpr uint32_t kTcTryNs = 20000;    // ... each of which may suspend the thread for up to this long

__device__ __forceinline__ uint32_t tc_smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// Byte offset of 16-byte chunk `chunk` (0..7) of row `row` inside one K-half block of a K-major
// operand with 128-byte swizzle: rows are 128 B apart, 8-row groups 1024 B apart, and the chunk
// index is XORed with the row's position in its group.
__device__ __forceinline__ uint32_t tc_swizzled(uint32_t row, uint32_t chunk) {
    return (row >> 3) * 1024u + (row & 7u) * 128u + ((chunk ^ (row & 7u)) << 4);
}

// Shared-memory matrix descriptor (K-major, SWIZZLE_128B, 8-row groups 1024 B apart) in two parts: only the low word
// depends on the address, and the descriptor of a later k-step of the operand follows by adding the k-step's offset in
// 16-byte units (the sum stays inside the address field).
__device__ __forceinline__ uint32_t tc_desc_lo(uint32_t saddr) { return ((saddr >> 4) & 0x3FFFu) | (1u << 16); }
__device__ __forceinline__ uint64_t tc_desc(uint32_t lo) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(64u | (1u << 14) | (2u << 29)));
    return d;
}
// k-step ks (16 inputs = 32 bytes of the 128-byte rows, four per K-half block) of an operand, in 16-byte units
__host__ __device__ constexpr uint32_t tc_koff(uint32_t ks, uint32_t block_bytes) { return (ks >> 2) * (block_bytes >> 4) + (ks & 3) * 2; }

// Instruction descriptor: bf16 x bf16 -> fp32, both operands K-major, M = 128, N = n.
__device__ __forceinline__ uint32_t tc_idesc(uint32_t n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// The warp executes these together and one elected thread of it (the same one each time) issues. Elected inside the asm,
// the operands stay warp-uniform for the compiler.
// D (tensor memory) (+)= A (shared memory) . B (shared memory)
__device__ __forceinline__ void tc_mma_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}

// D (tensor memory) (+)= A (tensor memory: lane = row, two bf16 per column, K = 16 in 8 columns) . B (shared memory)
__device__ __forceinline__ void tc_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "}\n" ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}

// Eight products in a row, one thread elected for all of them (an election and what goes with it in front of each costs the
// issuing warp 100 clocks more). Descriptors and tensor-memory addresses step inside the asm, so that they stay warp-uniform.
// D = A . B^T over K = 128: A and B in shared memory, K-major, two blocks of 64 elements kBlock bytes apart.
template <uint32_t kBlock>
__device__ __forceinline__ void tc_mma_ss_k128(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p, q, r;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %3, %3;\n\tsetp.eq.b32 r, %3, %3;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "add.u64 a, %1, 2;\n\tadd.u64 b, %2, 2;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, r;\n\t"
        "add.u64 a, %1, 4;\n\tadd.u64 b, %2, 4;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, r;\n\t"
        "add.u64 a, %1, 6;\n\tadd.u64 b, %2, 6;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, r;\n\t"
        "add.u64 a, %1, %4;\n\tadd.u64 b, %2, %4;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, r;\n\t"
        "add.u64 a, %1, %4 + 2;\n\tadd.u64 b, %2, %4 + 2;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, r;\n\t"
        "add.u64 a, %1, %4 + 4;\n\tadd.u64 b, %2, %4 + 4;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, r;\n\t"
        "add.u64 a, %1, %4 + 6;\n\tadd.u64 b, %2, %4 + 6;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, r;\n\t"
        "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "n"(kBlock >> 4) : "memory");
}

__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile(
        "{\n\t"
        ".reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
        "}\n" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void tc_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Has phase `parity` of the mbarrier completed? (does not block)
__device__ __forceinline__ bool tc_test(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}

// Bounded wait for phase `parity` of the mbarrier; false if it ran out or another thread of the CTA gave up.
__device__ __forceinline__ bool tc_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status) {
    for (int spin = 0; spin < kTcSpinLimit; ++spin) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done) : "r"(bar), "r"(parity), "r"(kTcTryNs) : "memory");
        if (done) return true;
        if (*abort_flag != 0) return false;
    }
    report(status, HA_ERR_TIMEOUT);
    *abort_flag = 1;
    return false;
}

// The same without a time for the thread to be suspended: where a phase is usually complete or about to be, 97 clocks instead of
// 178 (a try may suspend the thread for a time that the hardware chooses, so there are more of them).
__device__ __forceinline__ bool tc_wait_soon(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status) {
    for (int spin = 0; spin < (1 << 22); ++spin) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
        if (*abort_flag != 0) return false;
    }
    report(status, HA_ERR_TIMEOUT);
    *abort_flag = 1;
    return false;
}

// The same for two mbarriers, tested together, and a whole warp, whose lanes agree before they go on.
__device__ __forceinline__ bool tc_wait_both(uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1, volatile int* abort_flag, int32_t* status) {
    for (int spin = 0; spin < (1 << 22); ++spin) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
            "and.pred p, p, q;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done) : "r"(bar0), "r"(parity0), "r"(bar1), "r"(parity1) : "memory");
        if (__all_sync(0xffffffffu, done != 0)) return true;
        if (__any_sync(0xffffffffu, *abort_flag != 0)) return false;
    }
    report(status, HA_ERR_TIMEOUT);
    *abort_flag = 1;
    return false;
}

// 16 accumulator columns of this thread's lane: issue, and the wait that makes the registers readable (it waits for
// every read the thread has issued). The wait takes the registers as operands, so that nothing that reads them can be
// scheduled in front of it.
__device__ __forceinline__ void tc_ld16_issue(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tc_ld16_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :: "memory");
}

// 16 words per thread into this thread's lane (complete after tcgen05.wait::st).
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
           "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}

// 16 words per thread, written over the columns of this thread's lane (complete after tcgen05.wait::st) or, if to_smem, as
// four 16-byte chunks of shared memory. One asm under two predicates: as two branches of the program the compiler copies
// all 16 registers for one of them.
__device__ __forceinline__ void tc_put16(uint32_t taddr, const uint32_t (&r)[16], bool to_smem, uint32_t s0, uint32_t s1, uint32_t s2, uint32_t s3) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %17, 0;\n\t"
        "@!p tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};\n\t"
        "@p st.shared.v4.b32 [%18], {%0, %1, %2, %3};\n\t"
        "@p st.shared.v4.b32 [%19], {%4, %5, %6, %7};\n\t"
        "@p st.shared.v4.b32 [%20], {%8, %9, %10, %11};\n\t"
        "@p st.shared.v4.b32 [%21], {%12, %13, %14, %15};\n\t}"
        :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
           "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
           "r"(taddr), "r"(to_smem ? 1u : 0u), "r"(s0), "r"(s1), "r"(s2), "r"(s3)
        : "memory");
}

// TMA: the box at element column x, row y of the key cache -> shared memory, bytes counted on the mbarrier (the
// copy reads this GPU's memory only and has this CTA as its single destination).
__device__ __forceinline__ void tc_tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

// two fp32 -> one word of two bf16 (round to nearest even): a in the low half, b in the high half
__device__ __forceinline__ uint32_t tc_pack_bf16(float a, float b) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
    return d;
}

}  // namespace ha
