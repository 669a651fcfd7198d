// Attention over the 8-bit key/value cache for few bf16 query rows per sequence (decoding), on tcgen05: the codes go from global memory to the
// tensor cores as they are, and no register ever holds one.  Included by cache8.cu.
//
// One block of threads per (NR query rows of a sequence and key/value head, key/value head, sequence, share of the keys), 128 positions a step.  With few
// rows the cache is the large operand, so both products are turned round: scores^T [128 positions x rows] = K Q^T with the step's keys as the
// 128 rows of the instruction, and result^T [dv x rows] += V^T P^T, with the values, which lie position by position, as an operand whose
// rows are contiguous.  Accumulators are a few columns of tensor memory; a thread has one position's scores of all rows, and in the end
// one column of the result.
//
// e4m3 on both sides (kind::f8f6f4).  A query, scaled by a power of two to a largest magnitude in [128, 256), is the sum of two e4m3 parts, the second 16
// times finer: four bits each and the sign of the remainder hold bf16's eight bits, down to 2^-13 of the row's largest coordinate, and 2^-23 of
// it below.  A weight exp2(s - m), times its block's value scale over the largest so far, is taken apart the same way, on 64: a relative
// error of at most 2^-9, as a weight in bf16 would have, or 2^-20 of the reference's (m: see kSlack).  Parts are columns of their own.
//
// Roles: a warp that looks pages up and issues the copies (tensor maps, 128-byte swizzle, boxes of up to 128 positions that lie together), a thread
// that issues the products, four warps for the softmax.  A NaN code is a NaN to the product even under a weight of 0: in steps with positions that
// some row does not see, and in blocks that hold a NaN, the value codes are cleaned of them in shared memory; at the end nan_columns finds the
// results that see one.
//
// What bounds it: the bytes of the cache.  On the registers' way (mma.sync, e4m3 operands made f16 by the compiler's expansion) 32 positions took 965
// instructions of a warp and 64 sequences at up to 8192 positions 227 us.
#pragma once

#include "cache8_rows.cuh"
#include "cache8_tc.cuh"

namespace smol {
namespace c8 {

constexpr int kFewStep = 128, kFewThreads = 192, kFewCopies = 4, kFewProducts = 5;      // positions a step; warps of the copies and of the products
__host__ __device__ constexpr int few_stages(int D) { return D <= 128 ? 3 : 2; }
__host__ __device__ constexpr int few_stage_bytes(int D) { return kFewStep * 2 * D; }
__host__ __device__ constexpr int few_smem(int D, int NR) { return 1024 + 2 * NR * D + 2 * 2 * NR * 128 + few_stages(D) * few_stage_bytes(D); }
__host__ __device__ constexpr int few_tmem(int D, int NR) { return 2 * NR * (2 + D / 128) <= 64 ? 64 : 128; }

struct FewBars {
    uint64_t full[3], empty[3];      // stages
    uint64_t s_full[2], s_empty[2];  // scores in tensor memory
    uint64_t p_full[2], o_full[2];   // weights in shared memory; their product done
    uint64_t q_full, drained;
    uint32_t tmem;
    int stop;
};

// The steps of 128 positions that rows first_pos .. last_pos see: `lead` of them from the sequence's start, then those from `from` on.
__device__ __forceinline__ Seen seen_steps(const AttendArgs& A, int first_pos, int last_pos, int kv_len) {
    Seen x;
    x.end = max(min(kv_len, last_pos + 1), 0);
    const int steps = (x.end + kFewStep - 1) / kFewStep;
    x.from = A.window > 0 ? min(max(first_pos - A.window + 1, 0) / kFewStep, steps) : 0;
    x.lead = A.window > 0 ? min((A.first + kFewStep - 1) / kFewStep, x.from) : 0;
    x.count = x.lead + steps - x.from;
    return x;
}

// Rows (a bit each) that see a NaN in column col of the values: blocks whose scale is negative hold them.  Rare, and slow.
template <int NR>
__device__ uint32_t nan_columns(const AttendArgs& A, const Rows& W, int col) {
    uint32_t rows = 0;
    for (int b = 0; b * kBlock < W.end; ++b) {
        const int pg = b * kBlock / A.c.page;
        const int page = pg < A.b.max_pages ? A.b.table[(size_t)W.s * A.b.max_pages + pg] : -1;
        if (page < 0 || page >= A.c.n_pages) continue;
        const int in_page = b * kBlock - pg * A.c.page;
        if (A.c.vs[(size_t)page * A.c.vs_page + W.g * (A.c.page / kBlock) + in_page / kBlock] >= 0.0f) continue;
        for (int i = 0; i < kBlock; ++i) {
            const uint8_t code = A.c.v[(size_t)page * A.c.v_page + ((size_t)W.g * A.c.page + in_page + i) * A.c.ldv + col];
            if ((code & 0x7f) != 0x7f) continue;
            for (int r = 0; r < min(W.rows, NR); ++r)
                if (sees(A, W.pos0 + (W.row0 + r) / W.Gq, b * kBlock + i, W.end)) rows |= 1u << r;
        }
    }
    return rows;
}

constexpr float kWeightUnit = 64.0f, kSlack = 2.75f;      // 64 * 2^2.75 < 448, the largest code
// whether x holds for any thread of the four softmax warps
__device__ __forceinline__ bool any_of_four(bool x) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, 1, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}\n"
        : "=r"(any) : "r"((uint32_t)x) : "memory");
    return any != 0;
}
__device__ __forceinline__ float warp_top(float v) {
    asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(v));
    return v;
}

// Column col of row r: maximum, denominator and unnormalised result of this block's share of the keys.
__device__ __forceinline__ void put_result(const AttendArgs& A, const Rows& W, int r, int col, int split, float top, float total, float v) {
    const int tok = W.t0 + (W.row0 + r) / W.Gq, h = W.g * W.Gq + (W.row0 + r) % W.Gq;
    if (A.n_splits > 1) {
        const size_t at = ((size_t)tok * A.H + h) * A.n_splits + split;
        if (col == 0) part_stats(A)[at] = make_float2(top, total);
        A.part[at * ((A.c.dv + 3) / 4 * 4) + col] = v;
    } else {
        Elem<bf16>::put(static_cast<bf16*>(A.out) + (size_t)tok * A.o_row + (size_t)h * A.o_head + col, finished(A, tok, h, col, with_sink(A, h, top, total, v)));
    }
}

// D: head sizes padded (both); NR: query rows
template <int D, int NR, bool BENT>
__global__ void __launch_bounds__(kFewThreads) attend_few_kernel(const AttendArgs A, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, int box) {
    constexpr int NS = few_stages(D), SB = few_stage_bytes(D), N = 2 * NR, HALVES = D / 128, COLS = few_tmem(D, NR);
    extern __shared__ unsigned char smem_raw[];
    __shared__ FewBars bars;
    __shared__ float s_top[2][4][NR + 1], s_rowmul[NR], s_sum[4][NR], s_r1[NR], s_r2[NR], s_slope[NR];
    __shared__ int s_pos[NR], s_bad;
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *KV = base, *Qs = KV + NS * SB, *Ps = Qs + N * D;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) { umma::bar_init(&bars.full[i], 1); umma::bar_init(&bars.empty[i], 1); }
        for (int i = 0; i < 2; ++i) {
            umma::bar_init(&bars.s_full[i], 1);
            umma::bar_init(&bars.s_empty[i], 128);
            umma::bar_init(&bars.p_full[i], 128);
            umma::bar_init(&bars.o_full[i], 1);
        }
        umma::bar_init(&bars.q_full, 128);
        umma::bar_init(&bars.drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        bars.stop = 0;
        s_bad = 0;
    }
    if (warp == kFewProducts) tmem_take<COLS>(&bars.tmem);
    dep_wait();
    const int s = blockIdx.z, g = blockIdx.y, tile = blockIdx.x / A.n_splits, split = blockIdx.x % A.n_splits;
    const int t0 = A.b.start[s], n_all = A.b.start[s + 1] - t0, n = min(n_all, A.b.max_new), pos0 = A.b.pos0[s];
    const int kv_len = A.b.kv_len ? A.b.kv_len[s] : 0x7fffffff;
    const int Gq = A.H / A.c.G, row0 = tile * NR, rows = min(n * Gq - row0, NR);
    const bool any = rows > 0 && t0 >= 0 && t0 + n_all <= A.b.T;
    const int first_pos = pos0 + row0 / Gq, last_pos = pos0 + (row0 + rows - 1) / Gq;
    Seen seen = seen_steps(A, first_pos, last_pos, kv_len);
    const Rows W{s, g, t0, row0, rows, pos0, Gq, kv_len, seen.end};
    const int share = (seen.count + A.n_splits - 1) / A.n_splits, lo = min(split * share, seen.count);
    const int steps = any ? min(lo + share, seen.count) - lo : 0;
    auto step_at = [&](int i) { return (lo + i < seen.lead ? lo + i : seen.from + lo + i - seen.lead) * kFewStep; };
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    dep_go();      // behind the allocation: a kernel set up early that wants tensor memory too must not get it first
    const uint32_t tmem = bars.tmem, tm_o = tmem + 2 * N;      // scores of even and odd steps, then the result
    volatile int* stop = &bars.stop;

    if (warp == kFewCopies) {
        // ---- copies: lane i has the step's box number i ----
        const int boxes = kFewStep / box;
        auto look_up = [&](int i) {      // page and place of this lane's box: x < 0 where nothing of it is seen
            int2 at = make_int2(-1, 0);
            if (i < steps && lane < boxes) {
                const int j = step_at(i) + lane * box, pg = j / A.c.page;
                if (j < seen.end && (A.window == 0 || j + box > first_pos - A.window + 1 || j < A.first)) {
                    at.x = pg < A.b.max_pages ? A.b.table[(size_t)s * A.b.max_pages + pg] : -1;
                    at.y = j - pg * A.c.page;
                    if (at.x < 0 || at.x >= A.c.n_pages) {
                        at.x = -1;
                        atomicExch(A.c.err, 1);
                    }
                }
            }
            return at;
        };
        int2 now = look_up(0);
        int issued = 0;
        for (int i = 0; i < steps; ++i) {
            const int2 next = look_up(i + 1);
            const int st = i % NS;
            bool ok = true;
            if (i >= NS) ok = wait_bar(&bars.empty[st], (i / NS - 1) & 1, stop, A.c.err);
            if (!__all_sync(0xffffffffu, ok)) break;
            const int live = __popc(__ballot_sync(0xffffffffu, now.x >= 0));
            if (lane == 0) umma::bar_expect_tx(&bars.full[st], (uint32_t)(live * box * 2 * D));
            __syncwarp();
            if (now.x >= 0) {
                const uint32_t to = umma::s2u(KV + st * SB) + lane * box * 128;
#pragma unroll
                for (int x = 0; x < HALVES; ++x) load_box(to + x * (kFewStep * 128), &kmap, 128 * x, g * A.c.page + now.y, now.x, &bars.full[st]);
#pragma unroll
                for (int x = 0; x < HALVES; ++x) load_box(to + (HALVES + x) * (kFewStep * 128), &vmap, 128 * x, g * A.c.page + now.y, now.x, &bars.full[st]);
            }
            issued = i + 1;
            now = next;
        }
        // nothing may land in shared memory that is another's by then
        if (*stop)
            for (int i = max(issued - NS, 0); i < issued; ++i) drain_bar(&bars.full[i % NS], (i / NS) & 1);
    } else if (warp == kFewProducts) {
        if (lane == 0 && steps > 0) {
            // ---- products ----
            const uint32_t q0 = umma::s2u(Qs), id_s = desc_e4m3(128, N, false, false), id_o = desc_e4m3(128, N, true, false);
            const int ksteps = (A.c.d + 31) / 32;
            auto values = [&](int i) {
                const int st = i % NS, b = i & 1;
                if (!wait_bar(&bars.p_full[b], (i >> 1) & 1, stop, A.c.err)) return false;
                umma::fence_after_sync();
                const uint32_t v = umma::s2u(KV + st * SB) + HALVES * (kFewStep * 128), p = umma::s2u(Ps + b * (N * 128));
#pragma unroll
                for (int x = 0; x < HALVES; ++x)
#pragma unroll
                    for (int k = 0; k < kFewStep / 32; ++k)
                        mma_e4m3(tm_o + x * N, umma::smem_desc_sw128(v + x * (kFewStep * 128) + k * 32 * 128), umma::smem_desc_sw128(p + k * 32), id_o, (i > 0 || k > 0) ? 1u : 0u);
                umma::commit(&bars.empty[st]);
                umma::commit(&bars.o_full[b]);
                return true;
            };
            bool ok = wait_bar(&bars.q_full, 0, stop, A.c.err);
            for (int i = 0; ok && i < steps; ++i) {
                const int b = i & 1, st = i % NS;
                ok = wait_bar(&bars.full[st], (i / NS) & 1, stop, A.c.err) && (i < 2 || wait_bar(&bars.s_empty[b], ((i >> 1) - 1) & 1, stop, A.c.err));
                if (!ok) break;
                umma::fence_after_sync();
                const uint32_t k0 = umma::s2u(KV + st * SB);
                for (int k = 0; k < ksteps; ++k)
                    mma_e4m3(tmem + b * N, umma::smem_desc_sw128(k0 + (k >> 2) * (kFewStep * 128) + (k & 3) * 32), umma::smem_desc_sw128(q0 + (k >> 2) * (N * 128) + (k & 3) * 32), id_s, k > 0 ? 1u : 0u);
                umma::commit(&bars.s_full[b]);
                if (i > 0) ok = values(i - 1);
            }
            if (ok) values(steps - 1);
            umma::commit(&bars.drained);      // nothing of the block's is in flight once this is through
            drain_bar(&bars.drained, 0);
        }
    } else if (steps > 0) {
        // ---- queries into shared memory: row r's first parts at row r, its second parts at row NR + r ----
        for (int r = warp; r < NR; r += 4) {
            const int row = min(row0 + r, n * Gq - 1), h = g * Gq + row % Gq;
            const bf16* q = static_cast<const bf16*>(A.q) + (size_t)(t0 + row / Gq) * A.q_row + (size_t)h * A.q_head;
            float v[HALVES][4];
            uint32_t top = 0;
#pragma unroll
            for (int x = 0; x < HALVES; ++x) {
                const int at = x * 128 + lane * 4;
                if (A.q_vec) {
                    const uint2 u = at < A.c.d ? *reinterpret_cast<const uint2*>(q + at) : make_uint2(0u, 0u);
                    v[x][0] = bf_lo(u.x); v[x][1] = bf_hi(u.x); v[x][2] = bf_lo(u.y); v[x][3] = bf_hi(u.y);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[x][e] = at + e < A.c.d ? __bfloat162float(q[at + e]) : 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(fabsf(v[x][e])));
            }
            top = __reduce_max_sync(0xffffffffu, top);
            const int e = max((int)(top >> 23) - 127, -110);      // (below: rows of less than 2^-110 keep a factor that fp32 holds)
            const float up = pow2(7 - e);
#pragma unroll
            for (int x = 0; x < HALVES; ++x) {
                uint32_t hi[2], part[2];
#pragma unroll
                for (int y = 0; y < 2; ++y) two_parts(__floats2half2_rn(v[x][2 * y] * up, v[x][2 * y + 1] * up), hi[y], part[y]);
                *reinterpret_cast<uint32_t*>(Qs + x * (N * 128) + sw128_byte(r, lane * 4)) = hi[0] | (hi[1] << 16);
                *reinterpret_cast<uint32_t*>(Qs + x * (N * 128) + sw128_byte(NR + r, lane * 4)) = part[0] | (part[1] << 16);
            }
            if (lane == 0) {
                // (a row that is not finite: every score of it is a NaN)
                s_rowmul[r] = top >= 0x7f800000u ? __int_as_float(0x7fffffff) : pow2(e - 7) * (A.scale * (BENT ? 1.0f : kLog2e));
                s_pos[r] = pos0 + row / Gq;
                if (BENT) {
                    s_r1[r] = A.r1 ? A.r1[h] : 0.0f;
                    s_r2[r] = A.r1 ? A.r2[h] : 0.0f;
                    s_slope[r] = A.slope ? A.slope[h] : 0.0f;
                }
            }
        }
        umma::fence_async_smem();
        arrive(&bars.q_full);
        auto sync4 = [&] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
        sync4();
        float rowmul[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) rowmul[r] = s_rowmul[r];

        // ---- softmax: a position per thread ----
        const int me = threadIdx.x;
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        auto page_of = [&](int i) {
            if (i >= steps) return -1;
            const int j = step_at(i) + me, pg = j / A.c.page;
            if (j >= seen.end) return -1;
            const int page = pg < A.b.max_pages ? A.b.table[(size_t)s * A.b.max_pages + pg] : -1;
            return page >= A.c.n_pages ? -1 : page;
        };
        auto scales_of = [&](int i, int page) {      // keys' and values'; (0, 0) where there is no page
            if (page < 0) return make_float2(0.0f, 0.0f);
            const int j = step_at(i) + me, at = g * (A.c.page / kBlock) + j % A.c.page / kBlock;
            return make_float2(A.c.ks[(size_t)page * A.c.ks_page + at], A.c.vs[(size_t)page * A.c.vs_page + at]);
        };
        int page = page_of(0), page1 = page_of(1);
        float2 sc = scales_of(0, page);
        float m[NR], l[NR], unit = 0.0f;      // unit: the largest value scale so far, what the result is in units of
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.0f;
        }
        for (int i = 0; i < steps; ++i) {
            const int b = i & 1, j0 = step_at(i), j = j0 + me;
            const float2 sc1 = scales_of(i + 1, page1);
            const int page2 = page_of(i + 2);
            // (a wait that has run out is not waited for again: the steps that are left go by, and nothing is written)
            wait_bar(&bars.s_full[b], (i >> 1) & 1, stop, A.c.err);
            __syncwarp();
            umma::fence_after_sync();
            float S[NR];
            {
                uint32_t v[N / 8][8];
#pragma unroll
                for (int x = 0; x < N / 8; ++x) umma::tmem_ld8_issue(tmem + b * N + 8 * x + lanes, v[x]);
                umma::tmem_ld_wait();
                const float ks = fabsf(sc.x);
#pragma unroll
                for (int r = 0; r < NR; ++r) S[r] = fmaf(__uint_as_float(v[(NR + r) / 8][r % 8]), 0.0625f, __uint_as_float(v[r / 8][r % 8])) * (rowmul[r] * ks);
            }
            umma::fence_before_sync();
            arrive(&bars.s_empty[b]);
            if (BENT) {
#pragma unroll
                for (int r = 0; r < NR; ++r) S[r] = bent_score<false>(A, S[r], s_pos[r] - j, s_r1[r], s_r2[r], s_slope[r]);
            }
            const bool whole = j0 + kFewStep <= min(first_pos + 1, seen.end) && (A.window == 0 || j0 > last_pos - A.window || j0 + kFewStep <= A.first);
            if (!whole || page < 0) {
#pragma unroll
                for (int r = 0; r < NR; ++r)
                    if (page < 0 || !sees(A, s_pos[r], j, seen.end)) S[r] = -INFINITY;
            }
            if (!whole || page < 0 || sc.y < 0.0f) {
                // this position's value codes without NaNs (they have arrived: the products of the keys have been made)
                if (sc.y < 0.0f) s_bad = 1;
                wait_bar(&bars.full[i % NS], (i / NS) & 1, stop, A.c.err);
#pragma unroll
                for (int x = 0; x < HALVES; ++x) {
                    uint4* row = reinterpret_cast<uint4*>(KV + (i % NS) * SB + (HALVES + x) * (kFewStep * 128) + me * 128);
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                        const uint4 w = row[y], z = make_uint4(without_nans(w.x), without_nans(w.y), without_nans(w.z), without_nans(w.w));
                        if (w.x != z.x || w.y != z.y || w.z != z.z || w.w != z.w) row[y] = z;
                    }
                }
            }
            // ---- The reference of a row's weights is the maximum when it was last set: a weight may be 2^kSlack, and only a step that has a larger one (or a
            // larger value scale) sets references anew, which takes the four warps' maxima and waits for the product before. ----
            const float v_unit = page < 0 ? 0.0f : fmaxf(fabsf(sc.y), 7.5231638e-37f);      // 2^-120: below every scale
            bool beyond = v_unit > unit;
#pragma unroll
            for (int r = 0; r < NR; ++r) beyond |= S[r] > m[r] + kSlack;
            if (any_of_four(beyond)) {
                float mine = warp_top(v_unit);
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float top = warp_top(S[r]);
                    mine = lane == r ? top : mine;
                }
                if (lane <= NR) s_top[b][warp][lane] = mine;
                sync4();
                float grown = unit;
#pragma unroll
                for (int w = 0; w < 4; ++w) grown = fmaxf(grown, s_top[b][w][NR]);
                const float down = grown > 0.0f ? unit / grown : 1.0f;      // powers of two
                float corr[NR];
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float mn = fmaxf(m[r], fmaxf(fmaxf(s_top[b][0][r], s_top[b][1][r]), fmaxf(s_top[b][2][r], s_top[b][3][r])));
                    const float f = mn == -INFINITY ? 1.0f : exp2_fast(m[r] - mn);
                    m[r] = mn;
                    l[r] *= f;
                    corr[r] = f * down;
                }
                unit = grown;
                if (i > 0) {
                    wait_bar(&bars.o_full[b ^ 1], ((i - 1) >> 1) & 1, stop, A.c.err);
                    __syncwarp();
                    umma::fence_after_sync();
#pragma unroll
                    for (int x = 0; x < HALVES; ++x) {
                        uint32_t v[N / 8][8];
#pragma unroll
                        for (int y = 0; y < N / 8; ++y) umma::tmem_ld8_issue(tm_o + x * N + 8 * y + lanes, v[y]);
                        umma::tmem_ld_wait();
#pragma unroll
                        for (int y = 0; y < N / 8; ++y) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[y][e] = __float_as_uint(__uint_as_float(v[y][e]) * corr[(8 * y + e) % NR]);
                            tmem_st8(tm_o + x * N + 8 * y + lanes, v[y]);
                        }
                    }
                    tmem_st_wait();
                    umma::fence_before_sync();
                }
            }
            // ---- weights: hi at row r, lo at row NR + r, this position's byte ----
            if (i >= 2) wait_bar(&bars.o_full[b], ((i - 2) >> 1) & 1, stop, A.c.err);
            const float vmul = kWeightUnit * (v_unit / fmaxf(unit, 7.5231638e-37f));
            unsigned char* P = Ps + b * (N * 128);
#pragma unroll
            for (int r = 0; r < NR; r += 2) {
                float p[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    p[e] = exp2_fast(S[r + e] - (m[r + e] == -INFINITY ? 0.0f : m[r + e]));
                    l[r + e] += p[e];
                }
                uint32_t hi, part;
                two_parts(__floats2half2_rn(p[0] * vmul, p[1] * vmul), hi, part);
                P[sw128_byte(r, me)] = (unsigned char)hi;
                P[sw128_byte(r + 1, me)] = (unsigned char)(hi >> 8);
                P[sw128_byte(NR + r, me)] = (unsigned char)part;
                P[sw128_byte(NR + r + 1, me)] = (unsigned char)(part >> 8);
            }
            umma::fence_async_smem();
            arrive(&bars.p_full[b]);
            page = page1;
            page1 = page2;
            sc = sc1;
        }
        // ---- a column of the result per thread ----
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const float total = warp_sum(l[r]);
            if (lane == 0) s_sum[warp][r] = total;
        }
        wait_bar(&bars.o_full[(steps - 1) & 1], ((steps - 1) >> 1) & 1, stop, A.c.err);
        sync4();
        umma::fence_after_sync();
        const float out_unit = unit * (1.0f / kWeightUnit);
#pragma unroll
        for (int x = 0; x < HALVES; ++x) {
            __syncwarp();
            uint32_t v[N / 8][8];
#pragma unroll
            for (int y = 0; y < N / 8; ++y) umma::tmem_ld8_issue(tm_o + x * N + 8 * y + lanes, v[y]);
            umma::tmem_ld_wait();
            const int col = x * 128 + me;
            if (col >= A.c.dv || *stop) continue;
            const uint32_t nans = s_bad ? nan_columns<NR>(A, W, col) : 0u;
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                if (r >= rows) break;
                const float total = (s_sum[0][r] + s_sum[1][r]) + (s_sum[2][r] + s_sum[3][r]);
                float o = fmaf(__uint_as_float(v[(NR + r) / 8][r % 8]), 0.0625f, __uint_as_float(v[r / 8][r % 8])) * out_unit;
                if (nans >> r & 1) o = __int_as_float(0x7fffffff);
                put_result(A, W, r, col, split, m[r], total, o);
            }
        }
    } else if (any) {
        for (int i = threadIdx.x; i < rows * A.c.dv; i += 128) put_result(A, W, i / A.c.dv, i % A.c.dv, split, -INFINITY, 0.0f, 0.0f);      // no key in this share
    }
    __syncwarp();
    umma::fence_before_sync();
    __syncthreads();
    if (warp == kFewProducts) tmem_give<COLS>(tmem);
}

}  // namespace c8
}  // namespace smol
