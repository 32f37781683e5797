// tg_mbar.cuh — mbarriers with bounded waits, and the operands of tcgen05.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace tg {

constexpr long long WAIT_CYCLES = 2000000000ll;   // about a second

__device__ __forceinline__ uint32_t saddr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// A shared address kept in a register: otherwise every use forms it anew, from a special register
// that takes its time.
__device__ __forceinline__ uint32_t saddr_kept(const void* p) {
    uint32_t x;
    asm volatile("mov.u32 %0, %1;" : "=r"(x) : "r"(saddr(p)));
    return x;
}

__device__ __forceinline__ void mbar_init(uint64_t* m, int n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(saddr(m)), "r"(n));
}
__device__ __forceinline__ void mbar_expect(uint64_t* m, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(saddr(m)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t m) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(m) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t m, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(m), "r"(parity)
        : "memory");
    return done;
}
// Waits for the phase; false once the limit is over here or a wait has failed elsewhere in the CTA.
__device__ __forceinline__ bool mbar_wait(uint32_t m, uint32_t parity, volatile int* failed) {
    if (mbar_try(m, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try(m, parity)) {
        if (*failed) return false;
        if (clock64() - t0 > WAIT_CYCLES) {
            *failed = 1;
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ void mbar_arrive(uint64_t* m) { mbar_arrive(saddr(m)); }
__device__ __forceinline__ bool mbar_try(uint64_t* m, uint32_t parity) { return mbar_try(saddr(m), parity); }
__device__ __forceinline__ bool mbar_wait(uint64_t* m, uint32_t parity, volatile int* failed) {
    return mbar_wait(saddr(m), parity, failed);
}
// The same for what must land before the CTA may end.
__device__ __forceinline__ void mbar_drain(uint64_t* m, uint32_t parity) {
    const long long t0 = clock64();
    while (!mbar_try(m, parity) && clock64() - t0 < WAIT_CYCLES) {
    }
}

// One lane of the warp, the same every time.  The instructions of tcgen05 take their operands from
// uniform registers: with a warp in step around this, descriptors stay there, while a branch on
// the lane's number has every one moved over first (a third of the rate, measured).
__device__ __forceinline__ bool elect_one() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes;
}

// K-major operand in 128-byte swizzle: rows of 128 bytes, 8-row atoms 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}

template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t (&v)[N], uint32_t at);
template <>
__device__ __forceinline__ void tmem_ld<16>(uint32_t (&v)[16], uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(at));
}

template <>
__device__ __forceinline__ void tmem_ld<32>(uint32_t (&v)[32], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, "
                 "[%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(at));
}
__device__ __forceinline__ void tmem_st(uint32_t at, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t at, const uint32_t (&v)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
                 : "memory");
}

}  // namespace tg
