// What the tcgen05 kernels over the 8-bit cache share: bounded waits, tensor memory, operand descriptors for e4m3, copies through tensor maps.
#pragma once

#include <cuda.h>

#include "cache8_rows.cuh"
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
// the same without waiting at all: for a thread that looks at several barriers in turn
__device__ __forceinline__ bool has_passed(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
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
// by a whole warp: true if it is for every lane
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* stop, int32_t* err) {
    const bool ok = __all_sync(0xffffffffu, wait_bar(bar, parity, stop, err));
    __syncwarp();
    return ok;
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
// One lane of the warp.  The products' warp waits as a whole and issues inside `if (elected())`: issued by a thread that a branch on its index picked, a tcgen05.mma
// costs 198 cycles whatever its size, this way 75 (16 columns) to 115 (128).
__device__ __forceinline__ bool elected() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mma_e4m3(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
        ::"r"(d_tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// the same with A in tensor memory, four codes a column
__device__ __forceinline__ void mma_e4m3_weights(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}\n"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// byte of byte x of row r in a tile of 128-byte rows with the 128-byte swizzle
__device__ __forceinline__ int sw128_byte(int r, int x) { return r * 128 + (((x >> 4) ^ (r & 7)) << 4) + (x & 15); }

__device__ __forceinline__ void load_box(uint32_t dst, const void* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(map), "r"(umma::s2u(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}

constexpr float kLeastScale = 7.5231638e-37f;      // 2^-120: below every scale

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

__device__ __forceinline__ float warp_top(float v) {
    asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(v));
    return v;
}

// ---- steps of 128 positions ----
constexpr int kStep = 128, kStepBlocks = kStep / kBlock;

// The steps that rows first_pos .. last_pos see: `lead` of them from the sequence's start (the first tokens, in front of the window), then those from
// `from` up to the last visible key.
__device__ __forceinline__ Seen seen_steps(const AttendArgs& A, int first_pos, int last_pos, int kv_len) {
    Seen x;
    x.end = last_visible(A, last_pos, kv_len);
    const int steps = (x.end + kStep - 1) / kStep;
    x.from = A.window > 0 ? min(max(window_from(A, first_pos), 0) / kStep, steps) : 0;
    x.lead = A.window > 0 ? min(A.first / kStep + (A.first % kStep > 0), x.from) : 0;
    x.count = x.lead + steps - x.from;
    return x;
}
// first position of step i of a share that begins at number lo
__device__ __forceinline__ int step_place(const Seen& seen, int lo, int i) { return (lo + i < seen.lead ? lo + i : seen.from + lo + i - seen.lead) * kStep; }

// N rows of queries as they lie in memory, lane l's coordinates 4 l .. + 3 of each 128; all loads before anything is made of them (a row's after the one before it
// took 2000 cycles a row).  Lane y finds row y: offset_of(y), in elements, has a division.
template <int N, int KH, class OffsetOf>
__device__ __forceinline__ void load_queries(uint2 (&u)[N][KH], const AttendArgs& A, OffsetOf&& offset_of) {
    const int lane = threadIdx.x & 31, at = lane * 4;
    const size_t mine = offset_of(min(lane, N - 1));
    auto row_at = [&](int y) { return static_cast<const bf16*>(A.q) + __shfl_sync(0xffffffffu, mine, y); };
    if (A.q_vec) {
#pragma unroll
        for (int y = 0; y < N; ++y) {
            const bf16* q = row_at(y);
#pragma unroll
            for (int x = 0; x < KH; ++x) u[y][x] = x * 128 + at < A.c.d ? *reinterpret_cast<const uint2*>(q + x * 128 + at) : make_uint2(0u, 0u);
        }
    } else {
#pragma unroll
        for (int y = 0; y < N; ++y) {
            const unsigned short* q = reinterpret_cast<const unsigned short*>(row_at(y));
#pragma unroll
            for (int x = 0; x < KH; ++x) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = x * 128 + at + e < A.c.d ? q[x * 128 + at + e] : 0u;
                u[y][x] = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
            }
        }
    }
}
__device__ __forceinline__ void four_of(uint2 u, float (&v)[4]) { v[0] = bf_lo(u.x); v[1] = bf_hi(u.x); v[2] = bf_lo(u.y); v[3] = bf_hi(u.y); }

// What the copying warp leaves beside a stage: the scales of the step's blocks, keys' and values' (0: nothing there; the values' sign says whether a block
// holds a NaN).  With LOGS the values' are logarithms to base 2, and bit x of marks says that block x holds NaNs among its values, bit 8 + x that there is
// nothing: 512 threads that each find this out take 2 % of their time, while for few rows, whose copies are what is
// waited for, it is better left to the threads (64 sequences at up to 8192 positions 142 us; 146 with the marks, 150 with the logarithms and a vote on whether they are near).
struct StepScales {
    float2 of[kStepBlocks];
    uint32_t marks;
};

// The copying warp: keys and values of every step into a ring of NS stages (keys: KH tiles of 128 positions by 128 bytes, then VH of the values from
// column v_col on), 128-byte swizzle, in boxes of `box` positions that lie together.  Lane x < 8 looks up block x of a step; entries are loaded two steps ahead and scales one,
// so that nothing waits for them here.
template <int KH, int VH, int NS, bool LOGS>
__device__ __forceinline__ void copy_steps(const AttendArgs& A, const CUtensorMap* kmap, const CUtensorMap* vmap, int box, const Rows& W, const Seen& seen, int lo, int steps, int first_pos,
                                           unsigned char* ring, StepScales* scales, uint64_t* full, uint64_t* empty, volatile int* stop, int v_col) {
    constexpr int SB = kStep * 128 * (KH + VH);
    const int lane = threadIdx.x & 31, per = box / kBlock;
    struct Entry { int page, in_page, seen; };      // in_page < 0: nobody sees the block's box; seen: the block itself
    auto near = [&](int j, int n) { return j < seen.end && (A.window == 0 || j + n > window_from(A, first_pos) || j < A.first); };
    auto entry = [&](int i) {
        Entry e{-1, -1, 0};
        if (i < steps && lane < kStepBlocks) {
            const int j = step_place(seen, lo, i) + lane * kBlock, pg = j / A.c.page;
            if (near(j / box * box, box)) {
                e.in_page = j - pg * A.c.page;
                e.seen = near(j, kBlock);      // (the scales of places that nobody has written yet must not count)
                if (pg < A.b.max_pages) e.page = A.b.table[(size_t)W.s * A.b.max_pages + pg];
            }
        }
        return e;
    };
    auto scales_at = [&](const Entry& e) {
        if (!e.seen || e.page < 0 || e.page >= A.c.n_pages) return make_float2(0.0f, 0.0f);
        const int at = W.g * (A.c.page / kBlock) + e.in_page / kBlock;
        // (a scale that nobody has written counts as the least there is; 0 stands for no page)
        const float k = A.c.ks[(size_t)e.page * A.c.ks_page + at], v = A.c.vs[(size_t)e.page * A.c.vs_page + at];
        return make_float2(fmaxf(fabsf(k), kLeastScale), copysignf(fmaxf(fabsf(v), kLeastScale), v));
    };
    Entry now = entry(0), next = entry(1);
    float2 sc = scales_at(now);
    int issued = 0;
    for (int i = 0; i < steps; ++i) {
        const Entry after = entry(i + 2);
        const float2 sc1 = scales_at(next);
        const int st = i % NS;
        bool ok = true;
        if (i >= NS) ok = wait_bar(&empty[st], (i / NS - 1) & 1, stop, A.c.err);
        if (!__all_sync(0xffffffffu, ok)) break;
        const bool held = now.in_page >= 0 && now.page >= 0 && now.page < A.c.n_pages;
        if (now.in_page >= 0 && !held) atomicExch(A.c.err, 1);
        const bool mine = held && lane % per == 0;      // a box's first block issues it
        const int live = __popc(__ballot_sync(0xffffffffu, mine));
        if (LOGS) {
            const uint32_t marks = __ballot_sync(0xffffffffu, lane < kStepBlocks && sc.y < 0.0f) | __ballot_sync(0xffffffffu, lane < kStepBlocks && sc.x == 0.0f) << kStepBlocks;
            if (sc.x != 0.0f) sc.y = scale_log2(fabsf(sc.y));
            if (lane == 0) scales[st].marks = marks;
        }
        if (lane < kStepBlocks) scales[st].of[lane] = sc;
        __syncwarp();
        if (lane == 0) umma::bar_expect_tx(&full[st], (uint32_t)(live * box * 128 * (KH + VH)));
        __syncwarp();
        if (mine) {
            const uint32_t to = umma::s2u(ring + st * SB) + lane * kBlock * 128;
#pragma unroll
            for (int x = 0; x < KH; ++x) load_box(to + x * (kStep * 128), kmap, 128 * x, W.g * A.c.page + now.in_page, now.page, &full[st]);
#pragma unroll
            for (int x = 0; x < VH; ++x) load_box(to + (KH + x) * (kStep * 128), vmap, v_col + 128 * x, W.g * A.c.page + now.in_page, now.page, &full[st]);
        }
        issued = i + 1;
        now = next;
        next = after;
        sc = sc1;
    }
    // nothing may land in shared memory that is another's by then
    if (*stop)
        for (int i = max(issued - NS, 0); i < issued; ++i) drain_bar(&full[i % NS], (i / NS) & 1);
}

}  // namespace c8
}  // namespace smol
