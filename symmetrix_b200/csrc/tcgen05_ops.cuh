// Building blocks of the float32 kernels with specialised warps on the 5th-generation tensor cores (tcgen05.mma kind::tf32, row operand in tensor
// memory, the other one in shared memory): csrc/adapters_f32.cuh, csrc/grouped_f32.cuh.
#pragma once

#include "gemm_tcgen05.cuh"

namespace smx {
namespace {

// x rounded to TF32's 11 bits, half away from zero; as integers, since conversions run at a quarter of the rate.
__device__ __forceinline__ float ts_round(float x) { return __uint_as_float((__float_as_uint(x) + 0x1000u) & kTc5HiMask); }

__device__ __forceinline__ void ts_store32(uint32_t taddr, const float (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
        "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]),
        "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]), "f"(v[29]),
        "f"(v[30]), "f"(v[31])
        : "memory");
}
__device__ __forceinline__ void ts_store16(uint32_t taddr, const float (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
        "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
        : "memory");
}
__device__ __forceinline__ void ts_load32(uint32_t taddr, float (&v)[32]) {
    uint32_t u[32];
    tc5_ld32(taddr, u);
#pragma unroll
    for (int q = 0; q < 32; ++q) v[q] = __uint_as_float(u[q]);
}
__device__ __forceinline__ void ts_load16(uint32_t taddr, float (&v)[16]) {
    uint32_t u[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
          "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(taddr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int q = 0; q < 16; ++q) v[q] = __uint_as_float(u[q]);
}
// D (+)= A B with A in tensor memory and B in shared memory
__device__ __forceinline__ void ts_mma(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t"
        "}\n" ::"r"(d), "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}
// D = F32, A = B = TF32, both K-major, M = 128, N = n (a multiple of 16)
__device__ __forceinline__ uint32_t ts_idesc(int n) {
    return (1u << 4) | (2u << 7) | (2u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}
// The products of one chunk of `steps` x 8 inner values: row operand hi at column a_hi, lo at a_lo; weights hi at b_hi, lo at b_lo. The
// remainders' products come first, while the sum is small: the tensor core cuts its sums, so an addition costs up to 2^-23 of the sum.
// Descriptors of one step ahead are 32 bytes on, two units of their address field.
__device__ __forceinline__ void ts_chunk(uint32_t d, uint32_t a_hi, uint32_t a_lo, uint32_t b_hi, uint32_t b_lo, uint32_t idesc, int steps, bool accumulate) {
    const uint64_t hi = tc5_smem_desc(b_hi), lo = tc5_smem_desc(b_lo);
#pragma unroll 1
    for (int ks = 0; ks < steps; ++ks) {
        ts_mma(d, a_lo + 8 * ks, hi + 2 * ks, idesc, accumulate || ks > 0);
        ts_mma(d, a_hi + 8 * ks, lo + 2 * ks, idesc, true);
    }
#pragma unroll 1
    for (int ks = 0; ks < steps; ++ks) ts_mma(d, a_hi + 8 * ks, hi + 2 * ks, idesc, true);
}
__device__ __forceinline__ void ts_commit(unsigned long long* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// A value that is the same in all lanes, known to be so by the compiler: it can live in the uniform registers that the instructions issued by one lane
// take their operands from.
__device__ __forceinline__ int ts_uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ bool ts_elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ void ts_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ts_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ts_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Waits of a CTA's specialised warps: bounded by guard[1] polls, and given up at once when another one ran out (guard[0]).
__device__ __forceinline__ bool ts_try(uint32_t addr, unsigned parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(addr), "r"(parity) : "memory");
    return done != 0;
}
__device__ __forceinline__ bool ts_wait(unsigned long long* bar, unsigned parity, int* guard) {
    const uint32_t addr = smem_u32(bar);
#pragma unroll 1
    for (unsigned spin = 0; !ts_try(addr, parity); ++spin) {
        if ((spin & 63u) != 63u) continue;
        if (*reinterpret_cast<volatile int*>(guard)) return false;
        if (spin >= static_cast<unsigned>(guard[1])) { atomicExch(guard, 1); return false; }
    }
    return true;
}
__device__ __forceinline__ bool ts_wait_warp(unsigned long long* bar, unsigned parity, int* guard) {
    return __all_sync(0xffffffffu, ts_wait(bar, parity, guard));
}
template <int N> __device__ __forceinline__ void ts_registers_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void ts_registers_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void cp_async4(void* smem, const void* gmem) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(smem)), "l"(gmem) : "memory");
}

}  // namespace
}  // namespace smx
