// What the tcgen05 kernels over the 8-bit cache share: bounded waits, tensor memory, operand descriptors for e4m3, copies through tensor maps.
#pragma once

#include <cuda.h>

#include "cache8.cuh"
#include "umma.cuh"

namespace smol {
namespace c8 {

// A wait that runs out (a fault of the protocol, or of the device) sets the cache's error word to 3 and the block's `stop`; every role then leaves its
// loop, what is in flight is waited for (within the same limit), and the kernel ends.
constexpr long long kWaitCycles = 2000000000;      // a second or so
__device__ __forceinline__ bool passed(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok) : "r"(umma::s2u(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __noinline__ bool slow_wait(uint64_t* bar, uint32_t parity, volatile int* stop, int32_t* err) {
    const long long begin = clock64();
#pragma unroll 1
    while (clock64() - begin < kWaitCycles) {
        if (passed(bar, parity)) return true;
        if (*stop) return false;
    }
    *stop = 1;
    atomicExch(err, 3);
    return false;
}
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* stop, int32_t* err) {
    return passed(bar, parity) || slow_wait(bar, parity, stop, err);
}
// the same for what is still in flight when a block ends
__device__ __noinline__ void drain_bar(uint64_t* bar, uint32_t parity) {
    const long long begin = clock64();
#pragma unroll 1
    while (!passed(bar, parity) && clock64() - begin < kWaitCycles) {}
}
__device__ __forceinline__ void arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(umma::s2u(bar)) : "memory"); }

template <int COLS>
__device__ __forceinline__ void tmem_take(uint32_t* dst) {      // one full warp
    static_assert(COLS >= 32 && (COLS & (COLS - 1)) == 0 && COLS <= 512, "columns of tensor memory");
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(umma::s2u(dst)), "r"((uint32_t)COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <int COLS>
__device__ __forceinline__ void tmem_give(uint32_t base) {      // the same warp
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"((uint32_t)COLS) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D fp32, A and B e4m3, 32 terms a step; a_mn / b_mn: the operand lies with its rows (A) or columns (B) contiguous
__device__ __forceinline__ constexpr uint32_t desc_e4m3(int m, int n, bool a_mn, bool b_mn) {
    return (1u << 4) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_e4m3(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
        ::"r"(d_tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// byte of byte x of row r in a tile of 128-byte rows with the 128-byte swizzle
__device__ __forceinline__ int sw128_byte(int r, int x) { return r * 128 + (((x >> 4) ^ (r & 7)) << 4) + (x & 15); }

__device__ __forceinline__ void load_box(uint32_t dst, const void* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(map), "r"(umma::s2u(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}

// NaN codes of four cleared
__device__ __forceinline__ uint32_t without_nans(uint32_t w) {
    const uint32_t nan = (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
    return w & ~(nan * 0xffu);
}
// Two f16 numbers of magnitude at most 256 as e4m3 parts: hi + lo / 16 (two codes each)
__device__ __forceinline__ void two_parts(__half2 x, uint32_t& hi, uint32_t& lo) {
    const __half2_raw raw = x;
    hi = __nv_cvt_halfraw2_to_fp8x2(raw, __NV_SATFINITE, __NV_E4M3);
    const __half2 back = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)hi, __NV_E4M3);
    // the remainder times 16: exact (eight bits at most)
    const __half2_raw rest = __hmul2(__hsub2(x, back), __float2half2_rn(16.0f));
    lo = __nv_cvt_halfraw2_to_fp8x2(rest, __NV_SATFINITE, __NV_E4M3);
}

}  // namespace c8
}  // namespace smol
