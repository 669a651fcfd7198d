// Attention over the 8-bit key/value cache for 9 to 64 bf16 query rows of a tree (a few drafted tokens of grouped heads), on tcgen05.  Included by cache8_quads.cu.
//
// One block of threads per (32 query rows of a sequence and key/value head, key/value head, sequence, share of the keys), 128 positions a step, two steps at a time.  With rows as
// columns of the products (cache8_few.cuh) a thread has one position of all rows, and every maximum goes through a warp and through shared memory: some 60 instructions a score.  Tiles of
// 128 rows (cache8_tiles.cuh) take 16, but pay for 128.  Here the instruction's 128 rows are the 32 query rows four times over, and each of the four copies, which are the four quarters
// of tensor memory that a warp each can read, looks at 32 of the step's positions only: a thread has one row and 32 positions, and a running softmax of its own that nobody else knows of.
// The weights are the first operand of the second product with zeros beside a copy's own 32 positions, so that a copy's result is that of its positions; the copies are joined at the end as
// shares of the keys are.  Two groups of four warps take even and odd steps' softmax, and half of the results' columns each of every step, whose running sums fit their registers so.
//
// Queries and weights are two e4m3 parts of one unit as in the tiles, relative to what a row sees in 32 positions of a step rather than in 128: a weight to 2^-9 of itself or 2^-18 of the largest term,
// since both parts are multiplied into one sum.  (The kernel for few rows has a sum for either, and 2^-22: a chain of 9 to 16 rows is answered that much more finely without a tree.)
//
// Roles: eight warps for the softmax, one that copies, one that issues the products.
//
// What bounds it: the chain of a group's two steps, 3550 cycles: products of 480 and 650 (two e4m3 parts, and a quarter of what is multiplied is wanted), their waits, a softmax of 1350 from
// scores to weights, reading results 450.  DRAM gives a step's 32 KB in 1330 an SM.  Around the steps a block takes 8000 cycles to its first scores (the batch's arrays, queries, page, scales and
// the first copy, one behind the other) and 3000 for its results.  64 sequences at up to 8192 positions, 32 and 8 heads of 128, 16 rows each 208 to 216 us (rows as columns, 16 of them, 247), 32 rows
// 213 to 217 (tiles 407), 64 rows 383; 48 of 16 rows behind windows of 4000 and 4 122 us, with soft cap, slope and sink 155; one of 48 rows of 4 heads of 64 at 2063 positions 11.4 us.
#pragma once

#include "cache8_few.cuh"
#include "cache8_launch.cuh"
#include "cache8_tiles.cuh"

namespace smol {
namespace c8 {

constexpr int kQuadSoft = 8, kQuadThreads = (kQuadSoft + 2) * 32, kQuadStages = 5, kQuadCols = 32, kQuadDim = 128;
constexpr int kQuadStage = 2 * kStep * kQuadDim, kQuadOperand = 2 * 128 * 128;      // bytes of a stage; of queries, both parts
constexpr int kQuadParts = 4, kQuadLd = kQuadDim + 4, kQuadSteps = 4;               // results that are joined in the block; steps whose softmax is remembered
__host__ __device__ constexpr int quad_smem() { return 1024 + kQuadStages * kQuadStage + kQuadOperand + kQuadSteps * kQuadParts * kQuadRows * (int)sizeof(float4); }
static_assert(kQuadParts * kQuadRows * kQuadLd * 4 <= kQuadStages * kQuadStage, "the results that are joined take the place of the stages");

struct QuadBars {
    uint64_t full[kQuadStages], empty[kQuadStages];      // stages
    uint64_t s_full[2], o_full[2];                       // of a group: scores in tensor memory; the weights' product
    uint64_t p_full[2];                                  // weights in the scores' place, and the product of the step before last read by everybody: it goes where that was
    uint64_t q_full, drained;
    uint32_t tmem;
    int stop;
};
// what is left in shared memory for the block's own join, and the cluster's (in the place of the queries)
struct QuadJoin {
    float4 part[kQuadParts][kQuadRows];      // maximum, denominator, e of the results
    float4 stat[kQuadRows];                  // the same of this block's share
    float2 finish[kQuadRows];
    size_t to[kQuadRows];
    float counts[kQuadRows][kMostCluster];
    float joint[kQuadRows * kQuadDim];
};
static_assert(sizeof(QuadJoin) <= kQuadOperand, "the join's place");

// The copying warp: keys and values of every step into a ring of stages, 128-byte swizzle, in boxes of `box` positions that lie together.  All 32 lanes look blocks up, four steps at a time and
// four ahead: an entry and then a scale that are waited for once a step cost 2000 cycles where memory is busy (64 sequences at up to 8192 positions 300 us, then 246).
__device__ __forceinline__ void quad_copies(const AttendArgs& A, const CUtensorMap* kmap, const CUtensorMap* vmap, int box, const Rows& W, const Seen& seen, int lo, int steps, int first_pos,
                                            unsigned char* ring, StepScales* scales, QuadBars& bars) {
    constexpr int AHEAD = 32 / kStepBlocks, NS = kQuadStages;
    volatile int* stop = &bars.stop;
    const int lane = threadIdx.x & 31, per = box / kBlock, block = lane % kStepBlocks, mine = lane / kStepBlocks;
    struct Entry { int page, in_page, seen; };      // in_page < 0: nobody sees the block's box; seen: the block itself
    auto near = [&](int j, int n) { return j < seen.end && (A.window == 0 || j + n > window_from(A, first_pos) || j < A.first); };
    auto entry = [&](int i) {
        Entry e{-1, -1, 0};
        if (i < steps) {
            const int j = step_place(seen, lo, i) + block * kBlock, pg = j / A.c.page;
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
    Entry now = entry(mine), next = now;
    float2 sc = scales_at(now), sc1 = sc;
    uint32_t nans = 0, holes = 0;      // of all four steps
    int issued = 0;
    for (int i = 0; i < steps; ++i) {
        const int turn = i % AHEAD, st = i % NS;
        if (turn == 0) {
            if (i > 0) {
                now = next;
                sc = sc1;
            }
            nans = __ballot_sync(0xffffffffu, sc.y < 0.0f);
            holes = __ballot_sync(0xffffffffu, sc.x == 0.0f);
            if (sc.x != 0.0f) sc.y = scale_log2(fabsf(sc.y));
            next = entry(i + AHEAD + mine);
        }
        if (turn == AHEAD / 2) sc1 = scales_at(next);
        const bool on = mine == turn, held = on && now.in_page >= 0 && now.page >= 0 && now.page < A.c.n_pages;
        if (on && now.in_page >= 0 && !held) atomicExch(A.c.err, 1);
        const bool first = held && block % per == 0;      // a box's first block issues it
        const int boxes = __popc(__ballot_sync(0xffffffffu, first));
        bool ok = true;
        if (i >= NS) ok = wait_bar(&bars.empty[st], (i / NS - 1) & 1, stop, A.c.err);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (on) scales[st].of[block] = sc;
        __syncwarp();
        if (lane == 0) {
            scales[st].marks = (nans >> turn * kStepBlocks & 0xffu) | (holes >> turn * kStepBlocks & 0xffu) << kStepBlocks;
            umma::bar_expect_tx(&bars.full[st], (uint32_t)(boxes * box * 128 * 2));
        }
        __syncwarp();
        if (first) {
            const uint32_t to = umma::s2u(ring + st * kQuadStage) + block * kBlock * 128;
            load_box(to, kmap, 0, W.g * A.c.page + now.in_page, now.page, &bars.full[st]);
            load_box(to + kStep * 128, vmap, 0, W.g * A.c.page + now.in_page, now.page, &bars.full[st]);
        }
        issued = i + 1;
    }
    // nothing may land in shared memory that is another's by then
    if (*stop)
        for (int i = max(issued - NS, 0); i < issued; ++i) drain_bar(&bars.full[i % NS], (i / NS) & 1);
}

// DV: columns of the values, padded to 64 or 128; BENT: soft cap or distance penalties
template <int DV, bool BENT>
__global__ void __launch_bounds__(kQuadThreads, 1) attend_quads_kernel(const __grid_constant__ AttendArgs A, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, int box) {
    constexpr int NS = kQuadStages;
    extern __shared__ unsigned char smem_raw[];
    __shared__ QuadBars bars;
    __shared__ StepScales s_scales[NS];
    __shared__ float s_rowmul[kQuadRows];
    __shared__ int s_row[kQuadRows], s_head[kQuadRows], s_bad;
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *KV = base, *Qs = KV + NS * kQuadStage;
    float4(*stats)[kQuadParts][kQuadRows] = reinterpret_cast<float4(*)[kQuadParts][kQuadRows]>(Qs + kQuadOperand);      // of a step: a row's maximum, what its weights are relative to on top of it, their sum
    QuadJoin& J = *reinterpret_cast<QuadJoin*>(Qs);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // ---- barriers, a thread each ----
    if (threadIdx.x < NS) {
        umma::bar_init(&bars.full[threadIdx.x], 1);
        umma::bar_init(&bars.empty[threadIdx.x], 1);
    } else if (threadIdx.x < NS + 2) {
        umma::bar_init(&bars.s_full[threadIdx.x - NS], 1);
        umma::bar_init(&bars.p_full[threadIdx.x - NS], kQuadSoft);
        umma::bar_init(&bars.o_full[threadIdx.x - NS], 2);
    } else if (threadIdx.x == NS + 2) {
        umma::bar_init(&bars.q_full, kQuadSoft);
        umma::bar_init(&bars.drained, 1);
        bars.stop = 0;
        bars.tmem = 0;      // (what it will be: all columns are taken)
        s_bad = 0;
    } else if (threadIdx.x == NS + 3) {
        asm volatile("prefetch.tensormap [%0];\n\tprefetch.tensormap [%1];" ::"l"(&kmap), "l"(&vmap) : "memory");
    }
    if (threadIdx.x <= NS + 2) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    dep_wait();
    const int s = blockIdx.z, g = blockIdx.y, tile = blockIdx.x / A.n_splits, split = blockIdx.x % A.n_splits;
    const Sequence Q(A.b, s, A.c.err);
    const int t0 = Q.t0, n_all = Q.n, n = min(n_all, A.b.max_new), pos0 = Q.pos0;
    const int kv_len = A.b.kv_len ? A.b.kv_len[s] : 0x7fffffff;
    const int Gq = A.H / A.c.G, row0 = tile * kQuadRows, rows = min(n * Gq - row0, kQuadRows);
    const bool any = rows > 0 && (long long)n_all * Gq > A.rows_over && (long long)n_all * Gq <= A.rows_most && tree_fits(A, pos0, n_all);
    if (!any) {      // (nor has any other block of the cluster: before shared and tensor memory are made use of)
        dep_go();
        return;
    }
    const TreeSpan span(A, t0 + row0 / Gq, (row0 + rows - 1) / Gq - row0 / Gq + 1, n_all, pos0);
    const int first_pos = span.first_pos, last_pos = span.last_pos, behind = span.behind;
    const Seen seen = seen_steps(A, first_pos, behind, kv_len);
    const Rows W{s, g, t0, row0, rows, pos0, Gq, kv_len, seen.end};
    const int lo = (int)((long long)split * seen.count / A.n_splits), steps = (int)((long long)(split + 1) * seen.count / A.n_splits) - lo;
    const bool clustered = A.in_cluster;
    volatile int* stop = &bars.stop;
    if (warp == kQuadSoft) {
        quad_copies(A, &kmap, &vmap, box, W, seen, lo, steps, first_pos, KV, s_scales, bars);
    } else if (warp == kQuadSoft + 1) {
        // (nobody waits for the allocation but this warp: who reads tensor memory has been told of a product)
        tmem_take<512>(&bars.tmem);
        dep_go();      // behind the allocation: a kernel set up early that wants tensor memory too must not get it first
        if (steps > 0) {
            umma::fence_before_sync();
            __syncwarp();
            umma::fence_after_sync();
            const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars.tmem), tm_o = tmem + 2 * kStep;      // scores of even and odd steps, then products likewise
            // ---- products.  A step's scores go where the weights of the step before last were, which are multiplied in front of them (products are made in the order of
            // their issue).  (Weights in shared memory instead, and scores as soon as a group has read its last ones: 260 us where this then took 246, since two operands from there are all that it gives.) ----
            const uint32_t q0 = umma::s2u(Qs), id_s = desc_e4m3(128, kStep, false, false), id_o = desc_e4m3(128, 128, false, true);
            const int ksteps = (A.c.d + 31) / 32;
            auto scores = [&](int i) {
                if (!warp_wait(&bars.full[i % NS], (i / NS) & 1, stop, A.c.err)) return false;
                if (elected()) {
                    umma::fence_after_sync();
                    const uint32_t k0 = umma::s2u(KV + i % NS * kQuadStage);
#pragma unroll
                    for (int part = 0; part < 2; ++part)
                        for (int k = 0; k < ksteps; ++k)
                            mma_e4m3(tmem + (i & 1) * kStep, umma::smem_desc_sw128(q0 + part * (128 * 128) + k * 32), umma::smem_desc_sw128(k0 + k * 32), id_s, part > 0 || k > 0 ? 1u : 0u);
                    umma::commit(&bars.s_full[i & 1]);
                }
                __syncwarp();
                return true;
            };
            bool ok = warp_wait(&bars.q_full, 0, stop, A.c.err) && scores(0) && (steps < 2 || scores(1));
            for (int i = 0; ok && i < steps; ++i) {
                const int b = i & 1;
                ok = warp_wait(&bars.p_full[b], (i >> 1) & 1, stop, A.c.err);
                if (!ok) break;
                if (elected()) {
                    umma::fence_after_sync();
                    const uint32_t v = umma::s2u(KV + i % NS * kQuadStage) + kStep * 128;
#pragma unroll
                    for (int part = 0; part < 2; ++part)
#pragma unroll
                        for (int k = 0; k < kStep / 32; ++k)
                            mma_e4m3_weights(tm_o + b * 128, tmem + b * kStep + part * (kStep / 4) + k * 8, umma::smem_desc_sw128(v + k * 32 * 128), id_o, part > 0 || k > 0 ? 1u : 0u);
                    umma::commit(&bars.empty[i % NS]);
                    umma::commit(&bars.o_full[b]);
                    arrive(&bars.o_full[b]);      // (what the group remembers of the step has been seen by this thread, and is by who waits for it)
                }
                __syncwarp();
                ok = i + 2 >= steps || scores(i + 2);
            }
            if (elected()) umma::commit(&bars.drained);      // nothing of the block's is in flight once this is through
            drain_bar(&bars.drained, 0);
        }
    } else {
        // ---- softmax: warp q of a group has the rows' copy q, positions 32 q .. + 31 of the group's steps; a row a thread ----
        const int group = warp >> 2, quad = warp & 3, my_row = min(row0 + lane, n * Gq - 1), tok = t0 + my_row / Gq, h = g * Gq + my_row % Gq, pos = tree_position(A, tok);
        if (warp == 0) {
            s_row[lane] = tok;
            s_head[lane] = h;
        }
        auto sync8 = [&] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
        // ---- queries: four rows a warp, each to its four places ----
        if (steps > 0) {
            uint2 u[4][1];
            load_queries<4, 1>(u, A, [&](int y) {
                const int row = min(row0 + warp * 4 + y, n * Gq - 1), at = row / Gq;
                return (size_t)(t0 + at) * A.q_row + (size_t)(g * Gq + row - at * Gq) * A.q_head;
            });
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int r = warp * 4 + y;
                const uint32_t w[2] = {u[y][0].x, u[y][0].y};
                // the largest magnitude, as bits: a NaN's are above infinity's
                const uint32_t most = __vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), top = __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
                const int e = max((int)(top >> 7) - 127, -110);      // (below: rows of less than 2^-110 keep a factor that fp32 holds)
                const float up = pow2(7 - e);
                uint32_t hi, rest;
                four_equal_parts(half_two(bf_lo(w[0]) * up, bf_hi(w[0]) * up), half_two(bf_lo(w[1]) * up, bf_hi(w[1]) * up), hi, rest);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    unsigned char* to = Qs + sw128_byte(x * 32 + r, lane * 4);
                    *reinterpret_cast<uint32_t*>(to) = hi;
                    *reinterpret_cast<uint32_t*>(to + 128 * 128) = rest;
                }
                // (a row that is not finite: every score of it is a NaN)
                if (lane == 0) s_rowmul[r] = top >= 0x7f80u ? __int_as_float(0x7fffffff) : pow2(e - 7) * (A.scale * (BENT ? 1.0f : kLog2e));
            }
            umma::fence_async_smem();
            __syncwarp();
            if (lane == 0) arrive(&bars.q_full);
        }
        sync8();
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const float rowmul = s_rowmul[lane], r1 = BENT && A.r1 ? A.r1[h] : 0.0f, r2 = BENT && A.r1 ? A.r2[h] : 0.0f, slope = BENT && A.slope ? A.slope[h] * kLog2e : 0.0f;
        const Bend bend(A);
        constexpr int OC = DV / 2;      // columns of the results that are this group's
        float m = -INFINITY, unit = 0.0f, l = 0.0f, o[OC];      // l in units of 2^m, o of 2^(m + unit)
#pragma unroll
        for (int c = 0; c < OC; ++c) o[c] = 0.0f;
        uint32_t tmem = 0;      // (known from the first product on)
        // a step's product, whoever brought its weights
        auto join_product = [&](int j) {
            wait_bar(&bars.o_full[j & 1], (j >> 1) & 1, stop, A.c.err);
            const float4 of = stats[j % kQuadSteps][quad][lane];
            const float m_step = of.x, unit_step = of.y, l_step = of.z;
            __syncwarp();
            umma::fence_after_sync();
            tmem = *reinterpret_cast<volatile uint32_t*>(&bars.tmem);
            // what results and denominator are relative to is the first step's, and a later one's only where they would come near fp32's end (they are below 2^90)
            if (__any_sync(0xffffffffu, m_step > m + kFarAbove || (m_step - m) + unit_step > unit + kFarAbove)) {
                const float mn = m_step > m + kFarAbove ? m_step : m, had = unit + (m - mn), has = unit_step + (m_step - mn), un = m == -INFINITY || has > had + kFarAbove ? has : had;
                const bool some = mn != -INFINITY;
                const float keep = !some || had == un ? 1.0f : m == -INFINITY ? 0.0f : exp2_fast(had - un);
                l *= !some || m == mn ? 1.0f : exp2_fast(m - mn);
                m = mn;
                unit = some ? un : unit;
#pragma unroll
                for (int c = 0; c < OC; ++c) o[c] *= keep;
            }
            l = fmaf(l_step, m_step == -INFINITY ? 0.0f : exp2_fast(m_step - m), l);
            const float add = m_step == -INFINITY ? 0.0f : exp2_fast((m_step - m) + (unit_step - unit)) * (1.0f / 256.0f);
#pragma unroll
            for (int x = 0; x < OC / 32; ++x) {
                uint32_t v[4][8];
#pragma unroll
                for (int y = 0; y < 4; ++y) umma::tmem_ld8_issue(tmem + 2 * kStep + (j & 1) * 128 + group * OC + 32 * x + 8 * y + lanes, v[y]);
                umma::tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float &o0 = o[32 * x + e], &o1 = o[32 * x + e + 1];
                    of_two(fma_two(two(__uint_as_float(v[e / 8][e % 8]), __uint_as_float(v[e / 8][e % 8 + 1])), two(add, add), two(o0, o1)), o0, o1);
                }
            }
            umma::fence_before_sync();
            __syncwarp();
            if (lane == 0 && (j & 1) != group) arrive(&bars.p_full[j & 1]);      // (the group whose step it is does when it has brought the next weights)
        };
        if (lane == 0) arrive(&bars.p_full[group ^ 1]);      // (in front of the other group's first step there is none to read)
        // A group's step i: the product of its step before, while its scores are being made, softmax and weights, and the product of the other group's step in between.
#pragma unroll 1
        for (int i = group;; i += 2) {
            const bool more = i < steps;
            uint32_t hi[8], rest[8];
            float top = -INFINITY, e = -INFINITY, total = 0.0f;
            const int st = i % NS;
            bool dirty = false;      // value codes that have been cleaned
            if (i >= 2 && i - 2 < steps) join_product(i - 2);
            if (more) {
                const int j0 = step_place(seen, lo, i), jc = j0 + quad * kQuadCols;
                // (a wait that has run out is not waited for again: the steps that are left go by, and nothing is written)
                wait_bar(&bars.full[st], (i / NS) & 1, stop, A.c.err);
                const uint32_t marks = s_scales[st].marks;
                const bool nans = marks & ((1 << kStepBlocks) - 1), holes = marks >> kStepBlocks;      // in the whole step
                float ks[2], lv[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float2 of = s_scales[st].of[quad * 2 + x];
                    ks[x] = of.x;
                    lv[x] = of.y;
                }
                wait_bar(&bars.s_full[group], (i >> 1) & 1, stop, A.c.err);
                __syncwarp();
                umma::fence_after_sync();
                tmem = *reinterpret_cast<volatile uint32_t*>(&bars.tmem);
                float S[kQuadCols];
                {
                    uint32_t v[4][8];
#pragma unroll
                    for (int x = 0; x < 4; ++x) umma::tmem_ld8_issue(tmem + group * kStep + quad * kQuadCols + 8 * x + lanes, v[x]);
                    umma::tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < kQuadCols; ++c) S[c] = __uint_as_float(v[c / 8][c % 8]);
                }
                const bool whole = !holes && j0 + kStep <= min(pos0, seen.end) && (A.window == 0 || j0 > last_pos - A.window || j0 + kStep <= A.first);
                // scores in units of log2: S times mul
                const bool direct = !BENT && whole && A.scale > 0.0f;
                float mul[2] = {rowmul * ks[0], rowmul * ks[1]};
                if (!direct) {
#pragma unroll
                    for (int c = 0; c < kQuadCols; ++c) S[c] *= mul[c / kBlock];
                    if (BENT) {
                        const float d0 = (float)(pos - jc);
                        if (jc + kQuadCols > pos0)      // (some keys are rows of the tree)
                            bend(A, S, [&](int c) { return fmaxf((float)(pos - (jc + c < seen.end ? tree_key(A, t0, pos0, jc + c) : jc + c)), 0.0f); }, [&](int) { return r1; }, [&](int) { return r2; },
                                 [&](int) { return slope; });
                        else
                            bend(A, S, [&](int c) { return fmaxf(d0 - (float)c, 0.0f); }, [&](int) { return r1; }, [&](int) { return r2; }, [&](int) { return slope; });
                    }
                    mul[0] = mul[1] = 1.0f;
                }
                if (!whole) {
                    const uint32_t mask = tree_mask(A, t0, pos0, tok, pos, jc, seen.end);
#pragma unroll
                    for (int c = 0; c < kQuadCols; ++c)
                        if (ks[c / kBlock] == 0.0f || !(mask >> c & 1u)) S[c] = -INFINITY;
                }
                if (!whole || nans) {
                    // the step's value codes without NaNs, a position a thread
                    if (nans) s_bad = 1;
                    dirty = true;
                    const int me = threadIdx.x & 127;
#pragma unroll 1
                    for (int x = 0; x < 8; ++x) {
                        uint4& at = reinterpret_cast<uint4*>(KV + st * kQuadStage + kStep * 128 + me * 128)[(x + me) & 7];      // (neighbouring threads at different banks)
                        const uint4 w = at, z = make_uint4(without_nans(w.x), without_nans(w.y), without_nans(w.z), without_nans(w.w));
                        if (w.x != z.x || w.y != z.y || w.z != z.z || w.w != z.w) at = z;
                    }
                }
                // ---- the maxima of the row's scores, and of score + log2(scale) from there ----
                float most[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float t[4] = {S[16 * x], S[16 * x + 1], S[16 * x + 2], S[16 * x + 3]};
#pragma unroll
                    for (int c = 4; c < 16; ++c) t[c % 4] = fmaxf(t[c % 4], S[16 * x + c]);
                    most[x] = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])) * mul[x];
                    top = fmaxf(top, most[x]);
                }
                const bool none = top == -INFINITY;
#pragma unroll
                for (int x = 0; x < 2; ++x) e = none ? 0.0f : fmaxf(e, (most[x] - top) + lv[x]);
                const float least = none ? 0.0f : top;
                // (value scales so far apart that weights which count in the denominator may be too small for an fp32 number; what is lost with them otherwise is below 2^-62)
                const bool far = __any_sync(0xffffffffu, !none && (e - lv[0] > kFarAbove || e - lv[1] > kFarAbove));
                if (far) {
#pragma unroll
                    for (int c = 0; c < kQuadCols; ++c) total += exp2_fast(fmaf(S[c], mul[c / kBlock], -least));
                }
                // ---- weights, times 256 ----
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    // (rounded down: not above 256 however large the scores)
                    const float over = __fadd_rd((lv[x] - e) + 8.0f, -least);
                    const uint64_t mul2 = two(mul[x], mul[x]), over2 = two(over, over);
                    uint64_t sum = two(0.0f, 0.0f);
                    uint32_t w[8];
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                        float p0, p1;
                        of_two(fma_two(two(S[16 * x + 2 * y], S[16 * x + 2 * y + 1]), mul2, over2), p0, p1);
                        p0 = exp2_fast(p0);
                        p1 = exp2_fast(p1);
                        sum = add_two(sum, two(p0, p1));
                        w[y] = half_two(p0, p1);
                    }
                    float sum0, sum1;
                    of_two(sum, sum0, sum1);
                    if (!far) total = fmaf(sum0 + sum1, exp2_fast((e - lv[x]) - 8.0f), total);
#pragma unroll
                    for (int y = 0; y < 4; ++y) four_equal_parts(w[2 * y], w[2 * y + 1], hi[4 * x + y], rest[4 * x + y]);
                }
            }
            if (more) {
                // (the rows' other copies have the other positions' weights: zeros there)
                const uint32_t P = tmem + group * kStep + lanes, zeros[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if (x == quad) {
                        tmem_st8(P + 8 * x, hi);
                        tmem_st8(P + kStep / 4 + 8 * x, rest);
                    } else {
                        tmem_st8(P + 8 * x, zeros);
                        tmem_st8(P + kStep / 4 + 8 * x, zeros);
                    }
                }
                tmem_st_wait();
                // (what is remembered is read until the step four steps on: its group has then joined the step two on, which was multiplied when everybody had joined this one)
                stats[i % kQuadSteps][quad][lane] = make_float4(top, e, total, 0.0f);
                if (dirty) umma::fence_async_smem();
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) arrive(&bars.p_full[group]);
            }
            if (i >= 1 && i - 1 < steps) join_product(i - 1);
            if (!more) break;
        }
        // ---- the copies' results are joined as shares of the keys: nothing is in flight any more, and stages and queries give their place ----
        sync8();
        if (group == 0) J.part[quad][lane] = make_float4(m, l, unit, 0.0f);
        sync8();
        float M = -INFINITY, E = -INFINITY, all = 0.0f;
#pragma unroll
        for (int x = 0; x < kQuadParts; ++x) M = fmaxf(M, J.part[x][lane].x);
#pragma unroll
        for (int x = 0; x < kQuadParts; ++x) {
            const float4 p = J.part[x][lane];
            E = fmaxf(E, p.x == -INFINITY ? -INFINITY : p.z + (p.x - M));
            // a share of no visible key weighs nothing, one of NaN scores makes its row NaN
            all = fmaf(p.y, p.x == -INFINITY ? (p.y == 0.0f ? 0.0f : p.y) : exp2_fast(p.x - M), all);
        }
        const float f = m == -INFINITY ? 0.0f : exp2_fast((unit + (m - M)) - E);
        if (warp == 0 && lane < rows) {
            if (A.n_splits == 1) {
                const Finish finish(A, h, M, all, M == -INFINITY ? 0.0f : E);
                J.finish[lane] = make_float2(finish.a, finish.b);
                J.to[lane] = (size_t)tok * A.o_row + (size_t)h * A.o_head;
            } else if (clustered) {
                J.stat[lane] = make_float4(M, all, M == -INFINITY ? 0.0f : E, 0.0f);
            } else {
                const size_t at = ((size_t)tok * A.H + h) * A.n_splits + split;
                part_stats(A)[at] = make_float4(M, all, M == -INFINITY ? 0.0f : E, 0.0f);
                J.to[lane] = at * ((A.c.dv + 3) / 4 * 4);
            }
        }
        float* results = reinterpret_cast<float*>(base);      // [part][row][kQuadLd]
        {
            float* mine = results + (quad * kQuadRows + lane) * kQuadLd + group * OC;
            if (!*stop) {
#pragma unroll
                for (int c = 0; c < OC; c += 4) *reinterpret_cast<float4*>(mine + c) = make_float4(o[c] * f, o[c + 1] * f, o[c + 2] * f, o[c + 3] * f);
                if (s_bad && quad == 0 && lane < rows) {
#pragma unroll 1
                    for (int c = 0; c < OC && group * OC + c < A.c.dv; c += 32) {
                        const uint32_t bits = nan_bits<true>(A, W, tok, pos, group * OC + c);
                        for (int x = 0; x < 32; ++x)
                            if (bits >> x & 1) mine[c + x] = __int_as_float(0x7fffffff);
                    }
                }
            }
        }
        sync8();
        if (!*stop) {
            const int pieces = (A.c.dv + 3) / 4;
#pragma unroll 1
            for (int i = threadIdx.x; i < rows * (DV / 4); i += kQuadSoft * 32) {
                const int r = i / (DV / 4), c = i % (DV / 4) * 4;
                if (c >= 4 * pieces) continue;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int x = 0; x < kQuadParts; ++x) {
                    const float4 p = *reinterpret_cast<const float4*>(results + (x * kQuadRows + r) * kQuadLd + c);
                    v.x += p.x; v.y += p.y; v.z += p.z; v.w += p.w;
                }
                if (clustered) {
                    *reinterpret_cast<float4*>(&J.joint[r * kQuadDim + c]) = v;
                } else if (A.n_splits > 1) {
                    *reinterpret_cast<float4*>(A.part + J.to[r] + c) = v;
                } else {
                    const float2 a = J.finish[r];
                    const float x[4] = {v.x * a.x * a.y, v.y * a.x * a.y, v.z * a.x * a.y, v.w * a.x * a.y};
                    bf16* to = static_cast<bf16*>(A.out) + J.to[r] + c;
                    if (A.o_vec && !A.gate && c + 4 <= A.c.dv) {
                        *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(x[0] * A.out_scale, x[1] * A.out_scale), pack_bf16(x[2] * A.out_scale, x[3] * A.out_scale));
                    } else {
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                            if (c + y < A.c.dv) to[y] = __float2bfloat16_rn(finished(A, s_row[r], s_head[r], c + y, x[y]));
                    }
                }
            }
        }
    }
    __syncwarp();
    if (clustered) {
        cluster_sync();
        if (warp < kQuadSoft && !*stop) join_shares<kQuadSoft * 32>(A, split, rows, J.stat, J.joint, kQuadDim, s_row, s_head, J.finish, J.to, J.counts);
        cluster_sync();      // nobody leaves while others read
    }
    __syncwarp();
    umma::fence_before_sync();
    __syncthreads();
    if (warp == kQuadSoft + 1) tmem_give<512>(*reinterpret_cast<volatile uint32_t*>(&bars.tmem));
}

}  // namespace c8
}  // namespace smol
