// Attention over the 8-bit key/value cache for few bf16 query rows per sequence (decoding), on tcgen05: the codes go from global memory to the
// tensor cores as they are, and no register ever holds one.  Included by cache8.cu.
//
// One block of threads per (RA query rows of a sequence and key/value head, key/value head, sequence, share of the keys), 128 positions a step.  With few
// rows the cache is the large operand, so both products are turned round: scores^T [128 positions x rows] = K Q^T with the step's keys as the
// 128 rows of the instruction, and result^T [dv x rows] += V^T P^T, with the values, which lie position by position, as an operand whose
// rows are contiguous.  Accumulators are a few columns of tensor memory; a thread has one position's scores of all rows, and in the end
// one column of the result.
//
// e4m3 on both sides (kind::f8f6f4).  A query, scaled by a power of two to a largest magnitude in [128, 256), is the sum of two e4m3 parts, the second 16
// times finer: four bits each and the sign of the remainder hold bf16's eight bits, down to 2^-13 of the row's largest coordinate, and 2^-23 of
// it below.  A weight exp2(s - m + log2(its block's value scale) - e), with the row's largest score m over the step and its largest s - m + log2(scale) e, is taken apart the
// same way, on 256: a relative error of at most 2^-9, as a weight in bf16 would have, or 2^-22 of the largest weight times scale that the row sees in the step.
// (With the scale as a factor behind exp2, over the step's largest, a value 2^20 larger that the row does not see halved the bits of its own weights.)  Parts are
// columns of their own.
//
// Roles: a warp that looks pages up and issues the copies (tensor maps, 128-byte swizzle, boxes of up to 128 positions that lie together), a warp
// that issues the products, four warps for the softmax.  A NaN code is a NaN to the product even under a weight of 0: in steps with positions that
// some row does not see, and in blocks that hold a NaN, the value codes are cleaned of them in shared memory; at the end nan_columns finds the
// results that see one.
//
// What bounds it: the bytes of the cache.  64 sequences at up to 8192 positions, 32 and 8 heads of 128: 147 us, 5.5 TB/s; one of 12 and 4 heads at 131072
// 33 us, 4.1 TB/s; 32 behind windows of 1024 17 us, and 2048 positions of 12 and 4 heads of 64 8 us, which are launch, page lookups and the join.  On the registers' way (mma.sync, e4m3 operands made f16 by the compiler's expansion) 32 positions took 965
// instructions of a warp and 64 sequences at up to 8192 positions 227 us.
#pragma once

#include "cache8_rows.cuh"
#include "cache8_tc.cuh"

namespace smol {
namespace c8 {

constexpr int kFewThreads = 192, kFewCopies = 4, kFewProducts = 5;      // warps of the copies and of the products
__host__ __device__ constexpr int few_rows(int RA) { return RA < 8 ? 8 : RA; }      // the instruction has at least 16 columns: two parts of eight rows
constexpr int kFewStages = 2;
__host__ __device__ constexpr int few_stage_bytes(int D) { return kStep * 2 * D; }
__host__ __device__ constexpr int few_smem(int D, int RA) { return 1024 + 2 * few_rows(RA) * (D + 2 * 128) + kFewStages * few_stage_bytes(D); }
__host__ __device__ constexpr int few_tmem(int D, int NR) { return 2 * NR * (2 + 2 * (D / 128)) <= 64 ? 64 : 2 * NR * (2 + 2 * (D / 128)) <= 128 ? 128 : 256; }

// blocks an SM holds: by shared memory (stages of 32 KB or 64) and registers.  Three of four rows instead of two: 64 sequences at up to 8192 positions 147 us, 160
__host__ __device__ constexpr int few_blocks(int D, int RA) { return D > 128 ? 1 : RA <= 4 ? 3 : 2; }

// What weights and results are relative to.  While the logarithms of all value scales lie within kNear of the first block's (`unit`): weights are relative to the
// row's largest score + log2(scale) =: m, results are in units of 2^m, and the denominator's terms, in units of 2^(m - unit), are the weights' times
// 2^(unit - log2(scale)): one exponential and one maximum a score.  (A weight below fp32's range counts for less than 2^-62 there.)  From the first step on that has a
// scale further away, whoever sees it, the same with an exponential and a maximum each for weights and denominator, and a unit per row: rare, and behind calls, so
// that the ordinary loop stays as short as it is (64 sequences at up to 8192 positions: 147 us, 158 with all of it in the loop, 143 without any).
constexpr float kNear = 32.0f;      // in units of log2

// the warp's largest score, and largest score - it + log2(scale)
static __device__ __noinline__ float2 apart_maxima(float s, float lv) {
    const float t = warp_top(s);
    return make_float2(t, warp_top(s - (t == -INFINITY ? 0.0f : t) + lv));
}
// (weight, the denominator's term, the row's largest score, what the weight is relative to on top of it), from the four warps' maxima
static __device__ __noinline__ float4 apart_weight(float s, float lv, const float* tops, const float* fars, int ld) {
    float top = -INFINITY, e = -INFINITY;
    for (int w = 0; w < 4; ++w) top = fmaxf(top, tops[w * ld]);
    if (top == -INFINITY) return make_float4(exp2_fast(s), exp2_fast(s), top, 0.0f);      // (0, or NaN)
    for (int w = 0; w < 4; ++w) e = fmaxf(e, fars[w * ld] + (tops[w * ld] - top));
    return make_float4(exp2_fast((s - top) + (lv - e)), exp2_fast(s - top), top, e);
}
// what results and denominator so far (in units of 2^(m + unit - 8), 2^m) and a step's count when joined
struct Apart {
    float keep, add, keep_l, add_l, unit;
    __device__ __noinline__ Apart(float m, float m_step, float unit_, float unit_step) {
        const float mn = fmaxf(m, m_step), had = m == -INFINITY ? -INFINITY : unit_ + (m - mn), has = m_step == -INFINITY ? -INFINITY : unit_step + (m_step - mn);
        unit = mn == -INFINITY ? unit_ : fmaxf(had, has);
        keep = m == -INFINITY ? 0.0f : exp2_fast(had - unit);
        add = m_step == -INFINITY ? 0.0f : exp2_fast(has - unit);
        // (a step, or all before it, of NaN scores has no maximum: its sums say so)
        keep_l = m == -INFINITY ? 1.0f : exp2_fast(m - mn);
        add_l = m_step == -INFINITY ? 1.0f : exp2_fast(m_step - mn);
    }
};

struct FewBars {
    uint64_t full[kFewStages], empty[kFewStages];      // stages
    uint64_t s_full[2], s_empty[2];  // scores in tensor memory
    uint64_t p_full[2], o_full[2];   // weights in shared memory; their product in tensor memory
    uint64_t q_full, drained;
    uint32_t tmem;
    int stop;
};

// Rows (a bit each) that see a NaN in column col of the values: blocks whose scale is negative hold them.  Rare, and slow.
template <int ROWS, bool TREE>
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
            for (int r = 0; r < min(W.rows, ROWS); ++r) {
                const int t = (W.row0 + r) / W.Gq;
                if (TREE ? tree_sees(A, W.t0, W.pos0, W.t0 + t, tree_position(A, W.t0 + t), b * kBlock + i, W.end) : sees(A, W.pos0 + t, b * kBlock + i, W.end)) rows |= 1u << r;
            }
        }
    }
    return rows;
}

__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float4 of_rank(const float4* mine, int rank) {
    uint32_t at;
    float4 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(umma::s2u(mine)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float of_rank(const float* mine, int rank) {      // the same place in another block of the cluster
    uint32_t at;
    float v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(umma::s2u(mine)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
constexpr int kMostCluster = 8;      // shares of the keys that are joined inside a cluster of blocks; more go through memory and attend_join_kernel

// What the shares of a row, with their maxima, denominators and e, count when joined, and the maximum, denominator and e of all of them.
struct SharesJoined {
    float top, total, unit, counts[kMostCluster];
    __device__ __forceinline__ SharesJoined(const float (&tops)[kMostCluster], const float (&f)[kMostCluster], const float (&e)[kMostCluster]) : top(-INFINITY), total(0.0f), unit(-INFINITY) {
        float least = INFINITY;
#pragma unroll
        for (int z = 0; z < kMostCluster; ++z) {
            top = fmaxf(top, tops[z]);
            unit = fmaxf(unit, tops[z] == -INFINITY ? -INFINITY : e[z]);
            least = fminf(least, tops[z] == -INFINITY ? INFINITY : e[z]);
        }
        if (unit - least > kNear) {      // (units far apart: not the largest, but that of the largest results)
            unit = -INFINITY;
            for (int z = 0; z < kMostCluster; ++z) unit = fmaxf(unit, tops[z] == -INFINITY ? -INFINITY : e[z] + (tops[z] - top));
        }
#pragma unroll
        for (int z = 0; z < kMostCluster; ++z) {
            // a share of no visible key weighs nothing, one of NaN scores makes its row NaN
            total = fmaf(f[z], tops[z] == -INFINITY ? (f[z] == 0.0f ? 0.0f : f[z]) : exp2_fast(tops[z] - top), total);
            counts[z] = tops[z] == -INFINITY ? 0.0f : exp2_fast((e[z] - unit) + (tops[z] - top));
        }
    }
};

// The shares of a cluster of blocks are joined: block `split` of them has rows split, split + n_splits, ...; by THREADS threads of every block.  stat, joint: a row's maximum, denominator and e in
// each block, and its unnormalised results; the other arrays are the block's own.  What the shares of a row count and what its results are multiplied by is worked out by a thread each.
template <int THREADS>
__device__ __forceinline__ void join_shares(const AttendArgs& A, int split, int rows, const float4* stat, const float* joint, int ld, const int* s_row, const int* s_head, float2* finish, size_t* to,
                                            float (*counts)[kMostCluster]) {
    const int me = threadIdx.x, count = rows > split ? (rows - split + A.n_splits - 1) / A.n_splits : 0;
    if (me < count) {
        const int r = split + me * A.n_splits, h = s_head[r];
        float top[kMostCluster], f[kMostCluster], e[kMostCluster];
#pragma unroll
        for (int z = 0; z < kMostCluster; ++z) {
            const float4 of = z < A.n_splits ? of_rank(&stat[r], z) : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
            top[z] = of.x;
            f[z] = of.y;
            e[z] = of.z;
        }
        const SharesJoined joined(top, f, e);
#pragma unroll
        for (int z = 0; z < kMostCluster; ++z) counts[me][z] = joined.counts[z];
        const Finish fin(A, h, joined.top, joined.total, joined.unit);
        finish[me] = make_float2(fin.a, fin.b);
        to[me] = (size_t)s_row[r] * A.o_row + (size_t)h * A.o_head;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
#pragma unroll 2
    for (int i = me; i < count * A.c.dv; i += THREADS) {
        const int at = i / A.c.dv, col = i - at * A.c.dv, r = split + at * A.n_splits;
        float v[kMostCluster], sum = 0.0f;
#pragma unroll
        for (int z = 0; z < kMostCluster; ++z) v[z] = z < A.n_splits ? of_rank(joint + r * ld + col, z) : 0.0f;
#pragma unroll
        for (int z = 0; z < kMostCluster; ++z) sum = fmaf(v[z], counts[at][z], sum);
        const float2 f = finish[at];
        static_cast<bf16*>(A.out)[to[at] + col] = __float2bfloat16_rn(finished(A, s_row[r], s_head[r], col, sum * f.x * f.y));
    }
}

// The same for up to four rows by four warps, whose threads each work out all of it for their own columns, the blocks' results on their way meanwhile.  (A thread a row that the others wait for
// is better from there on: 32 sequences of eight rows of 64 behind windows of 1000 23.1 us, this way (and a block's own results likewise) 24.5; of two rows, one sequence, five shares, 10.0 and 9.7, of 256 12.1 and 11.4.)
template <int D>
__device__ __forceinline__ void join_few_shares(const AttendArgs& A, int split, int rows, const float4* stat, const float* joint, const int* s_row, const int* s_head) {
    for (int r = split; r < rows; r += A.n_splits) {
        float top[kMostCluster], f[kMostCluster], e[kMostCluster], v[D / 128][kMostCluster];
#pragma unroll
        for (int z = 0; z < kMostCluster; ++z) {
            const bool on = z < A.n_splits;
            const float4 of = on ? of_rank(&stat[r], z) : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
            top[z] = of.x;
            f[z] = of.y;
            e[z] = of.z;
#pragma unroll
            for (int x = 0; x < D / 128; ++x) v[x][z] = on && threadIdx.x + 128 * x < A.c.dv ? of_rank(joint + r * D + threadIdx.x + 128 * x, z) : 0.0f;
        }
        const SharesJoined joined(top, f, e);
        const Finish fin(A, s_head[r], joined.top, joined.total, joined.unit);
#pragma unroll
        for (int x = 0; x < D / 128; ++x) {
            const int col = threadIdx.x + 128 * x;
            float sum = 0.0f;
#pragma unroll
            for (int z = 0; z < kMostCluster; ++z) sum = fmaf(v[x][z], joined.counts[z], sum);
            if (col < A.c.dv) static_cast<bf16*>(A.out)[(size_t)s_row[r] * A.o_row + (size_t)s_head[r] * A.o_head + col] = __float2bfloat16_rn(finished(A, s_row[r], s_head[r], col, sum * fin.a * fin.b));
        }
    }
}

// D: head sizes padded (both); RA: query rows; BENT: soft cap or distance penalties; TREE: rows of a tree
template <int D, int RA, bool BENT, bool TREE>
__global__ void __launch_bounds__(kFewThreads, few_blocks(D, RA)) attend_few_kernel(const AttendArgs A, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, int box) {
    constexpr int NR = few_rows(RA), NS = kFewStages, SB = few_stage_bytes(D), N = 2 * NR, HALVES = D / 128, COLS = few_tmem(D, NR);
    extern __shared__ unsigned char smem_raw[];
    __shared__ FewBars bars;
    __shared__ StepScales s_scales[NS];
    __shared__ float s_top[2][4][RA], s_rowmul[RA], s_sum[4][RA], s_r1[RA], s_r2[RA], s_slope[RA];
    __shared__ float4 s_stat[RA];      // of this block's share: maximum, denominator, e
    __shared__ float2 s_finish[RA];    // what finished results are multiplied by, and where they go
    __shared__ size_t s_to[RA];
    __shared__ float s_counts[RA][kMostCluster];      // what the shares of the keys count
    __shared__ float s_far[2][4][RA], s_step_unit[2][RA], s_unit[2][RA];      // (value scales far apart)
    __shared__ int s_apart[2];      // some thread has met one: in even and odd steps, so that the next step's is written while this one's is read
    __shared__ int s_pos[RA], s_row[RA], s_head[RA], s_bad;      // positions; the step's rows; heads
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
        asm volatile("prefetch.tensormap [%0];\n\tprefetch.tensormap [%1];" ::"l"(&kmap), "l"(&vmap) : "memory");
        bars.stop = 0;
        s_bad = s_apart[0] = s_apart[1] = 0;
    }
    if (warp == kFewProducts) tmem_take<COLS>(&bars.tmem);
    dep_wait();
    const int s = blockIdx.z, g = blockIdx.y, tile = blockIdx.x / A.n_splits, split = blockIdx.x % A.n_splits;
    const Sequence Q(A.b, s, A.c.err);
    const int t0 = Q.t0, n_all = Q.n, n = min(n_all, A.b.max_new), pos0 = Q.pos0;
    const int kv_len = A.b.kv_len ? A.b.kv_len[s] : 0x7fffffff;
    const int Gq = A.H / A.c.G, row0 = tile * RA, rows = min(n * Gq - row0, RA);
    const bool any = rows > 0 && (long long)n_all * Gq > A.rows_over && (long long)n_all * Gq <= A.rows_most && (!TREE || tree_fits(A, pos0, n_all));
    int first_pos = pos0 + row0 / Gq, last_pos = any ? pos0 + (row0 + rows - 1) / Gq : -1, behind = last_pos + 1, clear = first_pos + 1;      // clear: every row sees what is in front of it, but for the window
    if (TREE && any) {
        const TreeSpan span(A, t0 + row0 / Gq, (row0 + rows - 1) / Gq - row0 / Gq + 1, n_all, pos0);
        first_pos = span.first_pos; last_pos = span.last_pos; behind = span.behind; clear = pos0;
    }
    const Seen seen = seen_steps(A, first_pos, behind, kv_len);
    const Rows W{s, g, t0, row0, rows, pos0, Gq, kv_len, seen.end};
    const int share = (seen.count + A.n_splits - 1) / A.n_splits, lo = TREE ? (int)((long long)split * seen.count / A.n_splits) : min(split * share, seen.count);
    const int steps = any ? (TREE ? (int)((long long)(split + 1) * seen.count / A.n_splits) : min(lo + share, seen.count)) - lo : 0;
    const bool clustered = A.n_splits > 1 && A.n_splits <= kMostCluster;
    float* joint = reinterpret_cast<float*>(KV);      // [row][D], once everything has been multiplied
    // a finished row's column, and a column of this block's share of the keys: maximum, denominator, unnormalised result in units of 2^(top + e)
    auto store = [&](int r, int col, float top, float total, float e, float v) {
        const int tok = s_row[r], h = s_head[r];
        Elem<bf16>::put(static_cast<bf16*>(A.out) + (size_t)tok * A.o_row + (size_t)h * A.o_head + col, finished(A, tok, h, col, with_sink(A, h, top, total, e, v)));
    };
    auto put = [&](int r, int col, float top, float total, float e, float v) {
        if (A.n_splits == 1) {
            store(r, col, top, total, e, v);
        } else if (clustered) {
            if (col == 0) s_stat[r] = make_float4(top, total, e, 0.0f);
            joint[r * D + col] = v;
        } else {
            const size_t at = ((size_t)s_row[r] * A.H + s_head[r]) * A.n_splits + split;
            if (col == 0) part_stats(A)[at] = make_float4(top, total, e, 0.0f);
            A.part[at * ((A.c.dv + 3) / 4 * 4) + col] = v;
        }
    };
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    dep_go();      // behind the allocation: a kernel set up early that wants tensor memory too must not get it first
    const uint32_t tmem = bars.tmem, tm_o = tmem + 2 * N;      // scores of even and odd steps, then products likewise
    volatile int* stop = &bars.stop;

    if (warp == kFewCopies) {
        copy_steps<HALVES, HALVES, NS, false>(A, &kmap, &vmap, box, W, seen, lo, steps, first_pos, KV, s_scales, bars.full, bars.empty, stop, 0);
    } else if (warp == kFewProducts) {
        if (steps > 0) {
            // ---- products: whichever can be made next, so that neither the keys' waits for the weights nor the values' (and the stage they free) for the
            // next step's keys ----
            const uint32_t q0 = umma::s2u(Qs), id_s = desc_e4m3(128, N, false, false), id_o = desc_e4m3(128, N, true, false);
            const int ksteps = (A.c.d + 31) / 32;
            int scores = 0, values = 0;      // steps whose product has been issued
            long long begin = clock64();
            bool ok = warp_wait(&bars.q_full, 0, stop, A.c.err);
            while (ok && values < steps) {
                const bool keys = scores < steps && has_passed(&bars.full[scores % NS], (scores / NS) & 1) && (scores < 2 || has_passed(&bars.s_empty[scores & 1], ((scores >> 1) - 1) & 1));
                if (__all_sync(0xffffffffu, keys)) {
                    const int b = scores & 1, st = scores % NS;
                    __syncwarp();
                    if (elected()) {
                        umma::fence_after_sync();
                        const uint32_t k0 = umma::s2u(KV + st * SB);
                        for (int k = 0; k < ksteps; ++k)
                            mma_e4m3(tmem + b * N, umma::smem_desc_sw128(k0 + (k >> 2) * (kStep * 128) + (k & 3) * 32), umma::smem_desc_sw128(q0 + (k >> 2) * (N * 128) + (k & 3) * 32), id_s, k > 0 ? 1u : 0u);
                        umma::commit(&bars.s_full[b]);
                    }
                    __syncwarp();
                    ++scores;
                    begin = clock64();
                } else if (__all_sync(0xffffffffu, values < scores && has_passed(&bars.p_full[values & 1], (values >> 1) & 1))) {
                    const int b = values & 1, st = values % NS;
                    __syncwarp();
                    if (elected()) {
                        umma::fence_after_sync();
                        const uint32_t v = umma::s2u(KV + st * SB) + HALVES * (kStep * 128), p = umma::s2u(Ps + b * (N * 128));
#pragma unroll
                        for (int x = 0; x < HALVES; ++x)
#pragma unroll
                            for (int k = 0; k < kStep / 32; ++k)
                                mma_e4m3(tm_o + (b * HALVES + x) * N, umma::smem_desc_sw128(v + x * (kStep * 128) + k * 32 * 128), umma::smem_desc_sw128(p + k * 32), id_o, k > 0 ? 1u : 0u);
                        umma::commit(&bars.empty[st]);
                        umma::commit(&bars.o_full[b]);
                    }
                    __syncwarp();
                    ++values;
                    begin = clock64();
                } else if (__any_sync(0xffffffffu, *stop || clock64() - begin > kWaitCycles)) {
                    if (lane == 0 && !*stop) atomicExch(A.c.err, 3);
                    *stop = 1;
                    ok = false;
                }
            }
            if (elected()) umma::commit(&bars.drained);      // nothing of the block's is in flight once this is through
            drain_bar(&bars.drained, 0);
        }
    } else if (steps > 0) {
        // ---- queries into shared memory: row r's first parts at row r, its second parts at row NR + r ----
        uint2 u[RA / 4][HALVES];
        load_queries<RA / 4, HALVES>(u, A, [&](int y) {
            const int row = min(row0 + warp + 4 * y, n * Gq - 1), tok = row / Gq;
            return (size_t)(t0 + tok) * A.q_row + (size_t)(g * Gq + row - tok * Gq) * A.q_head;
        });
#pragma unroll
        for (int i = 0; i < RA / 4; ++i) {
            const int r = warp + 4 * i, row = min(row0 + r, n * Gq - 1), h = g * Gq + row % Gq;
            float v[HALVES][4];
            uint32_t top = 0;
#pragma unroll
            for (int x = 0; x < HALVES; ++x) {
                four_of(u[i][x], v[x]);
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
                s_row[r] = t0 + row / Gq;
                s_pos[r] = TREE ? tree_position(A, t0 + row / Gq) : pos0 + row / Gq;
                s_head[r] = h;
                if (BENT) {
                    s_r1[r] = A.r1 ? A.r1[h] : 0.0f;
                    s_r2[r] = A.r1 ? A.r2[h] : 0.0f;
                    s_slope[r] = A.slope ? A.slope[h] * kLog2e : 0.0f;
                }
            }
        }
        if (RA < NR)
            for (int i = threadIdx.x; i < 2 * (NR - RA) * (D / 4 + 2 * 32); i += 128) {      // rows that nobody has: queries and weights of zero
                const int words = D / 4 + 2 * 32, row = i / words, at = i % words, r = row < NR - RA ? RA + row : NR + row - (NR - RA) + RA;
                unsigned char* to = at < D / 4 ? Qs + at / 32 * (N * 128) + r * 128 + at % 32 * 4 : Ps + (at - D / 4) / 32 * (N * 128) + r * 128 + at % 32 * 4;
                *reinterpret_cast<uint32_t*>(to) = 0u;
            }
        umma::fence_async_smem();
        arrive(&bars.q_full);
        auto sync4 = [&] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
        sync4();
        float rowmul[RA];
#pragma unroll
        for (int r = 0; r < RA; ++r) rowmul[r] = s_rowmul[r];

        // ---- softmax: a position per thread; a column of the result per thread and half ----
        const int me = threadIdx.x;
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        const Bend bend(A);
        // (weights are multiplied as 256 times what they are: results are in units of 2^-8 of the reference's)
        float m[RA], l[RA], o[HALVES][RA];              // largest score + log2(scale), or once apart largest score; this thread's part of the denominator; results in full
        float m_step[RA], l_step[RA], unit = 0.0f;      // of the step before, whose product is not yet joined; log2 of the first block's scale
        bool apart = false, apart_step = false;
#pragma unroll
        for (int r = 0; r < RA; ++r) {
            m[r] = m_step[r] = -INFINITY;
            l[r] = l_step[r] = 0.0f;
#pragma unroll
            for (int x = 0; x < HALVES; ++x) o[x][r] = 0.0f;
        }
        auto join_product = [&](int i) {
            const int b = i & 1;
            wait_bar(&bars.o_full[b], (i >> 1) & 1, stop, A.c.err);
            __syncwarp();
            umma::fence_after_sync();
            float keep[RA], add[RA];
            if (!apart_step) {
#pragma unroll
                for (int r = 0; r < RA; ++r) {
                    const float mn = fmaxf(m[r], m_step[r]);
                    keep[r] = m[r] == mn ? 1.0f : exp2_fast(m[r] - mn);
                    add[r] = m_step[r] == -INFINITY ? 0.0f : exp2_fast(m_step[r] - mn);
                    m[r] = mn;
                    l[r] = fmaf(l_step[r], add[r], l[r] * keep[r]);
                }
            } else {
#pragma unroll
                for (int r = 0; r < RA; ++r) {
                    const Apart f(m[r], m_step[r], s_unit[b][r], s_step_unit[b][r]);
                    if (me == r) s_unit[b ^ 1][r] = f.unit;
                    keep[r] = f.keep;
                    add[r] = f.add;
                    l[r] = fmaf(l_step[r], f.add_l, l[r] * f.keep_l);
                    m[r] = fmaxf(m[r], m_step[r]);
                }
                __syncwarp();
            }
#pragma unroll
            for (int x = 0; x < HALVES; ++x) {
                uint32_t v[N / 8][8];
#pragma unroll
                for (int y = 0; y < N / 8; ++y) umma::tmem_ld8_issue(tm_o + (b * HALVES + x) * N + 8 * y + lanes, v[y]);
                umma::tmem_ld_wait();
#pragma unroll
                for (int r = 0; r < RA; ++r) o[x][r] = fmaf(fmaf(__uint_as_float(v[(NR + r) / 8][r % 8]), 0.0625f, __uint_as_float(v[r / 8][r % 8])), add[r], o[x][r] * keep[r]);
            }
            umma::fence_before_sync();
        };
        for (int i = 0; i < steps; ++i) {
            const int b = i & 1, st = i % NS, j0 = step_place(seen, lo, i), j = j0 + me;
            const int key = TREE && j >= pos0 && j < seen.end && (BENT || A.window > 0) ? tree_position(A, t0 + j - pos0) : j;      // the key's position
            // (a wait that has run out is not waited for again: the steps that are left go by, and nothing is written)
            wait_bar(&bars.full[st], (i / NS) & 1, stop, A.c.err);
            const float2 scales = s_scales[st].of[me / kBlock];
            const float ks = scales.x, vs = scales.y, lv = ks == 0.0f ? 0.0f : scale_log2(fabsf(vs));
            if (i == 0 && s_scales[0].of[0].x != 0.0f) unit = scale_log2(fabsf(s_scales[0].of[0].y));
            wait_bar(&bars.s_full[b], (i >> 1) & 1, stop, A.c.err);
            __syncwarp();
            umma::fence_after_sync();
            float S[RA];
            {
                uint32_t v[N / 8][8];
#pragma unroll
                for (int x = 0; x < N / 8; ++x) umma::tmem_ld8_issue(tmem + b * N + 8 * x + lanes, v[x]);
                umma::tmem_ld_wait();
#pragma unroll
                for (int r = 0; r < RA; ++r) S[r] = fmaf(fmaf(__uint_as_float(v[(NR + r) / 8][r % 8]), 0.0625f, __uint_as_float(v[r / 8][r % 8])), rowmul[r] * ks, BENT ? 0.0f : lv);
            }
            umma::fence_before_sync();
            arrive(&bars.s_empty[b]);
            if (BENT) {
                bend(A, S, [&](int r) { return TREE ? fmaxf((float)(s_pos[r] - key), 0.0f) : (float)(s_pos[r] - j); }, [&](int r) { return s_r1[r]; }, [&](int r) { return s_r2[r]; }, [&](int r) { return s_slope[r]; });
#pragma unroll
                for (int r = 0; r < RA; ++r) S[r] += lv;
            }
            const bool whole = j0 + kStep <= min(clear, seen.end) && (A.window == 0 || j0 > last_pos - A.window || j0 + kStep <= A.first);
            bool hidden = ks == 0.0f;      // from some row
            if (TREE && !whole) {
                // (all rows' bits on their way at once: one row after the other took 5600 cycles for 16)
                const bool there = ks != 0.0f && j < seen.end;
                const int row = j - pos0;      // of the sequence's rows (below 0: the context)
                uint32_t named[RA];
#pragma unroll
                for (int r = 0; r < RA; ++r) named[r] = there && row >= 0 ? A.tree_sees[(size_t)s_row[r] * A.tree_words + (row >> 5)] : 0xffffffffu;
#pragma unroll
                for (int r = 0; r < RA; ++r) {
                    const bool on = there && (named[r] >> (row & 31) & 1u) && (A.window == 0 || s_pos[r] - key < A.window || key < A.first);
                    hidden |= !on;
                    S[r] = on ? S[r] : -INFINITY;
                }
            } else if (!whole || hidden) {
#pragma unroll
                for (int r = 0; r < RA; ++r) {
                    const bool on = ks != 0.0f && (TREE || sees(A, s_pos[r], j, seen.end));
                    hidden |= !on;
                    S[r] = on ? S[r] : -INFINITY;
                }
            }
            if (hidden || vs < 0.0f) {
                // this position's value codes without NaNs
                if (vs < 0.0f) s_bad = 1;
#pragma unroll 1
                for (int x = 0; x < 8 * HALVES; ++x) {
                    // (neighbouring threads at different banks)
                    uint4& at = reinterpret_cast<uint4*>(KV + st * SB + (HALVES + x / 8) * (kStep * 128) + me * 128)[(x + me) & 7];
                    const uint4 w = at, z = make_uint4(without_nans(w.x), without_nans(w.y), without_nans(w.z), without_nans(w.w));
                    if (w.x != z.x || w.y != z.y || w.z != z.z || w.w != z.w) at = z;
                }
            }
            // ---- the rows' maxima over the step, of score + log2(scale) ----
            float mine = 0.0f, top[RA], sums[RA];
#pragma unroll
            for (int r = 0; r < RA; ++r) {
                const float t = warp_top(S[r]);
                mine = lane == r ? t : mine;
            }
            if (lane < RA) s_top[b][warp][lane] = mine;
            const bool apart_before = apart;
            if (ks != 0.0f && fabsf(lv - unit) > kNear) s_apart[b] = 1;
            sync4();
            apart |= s_apart[b] != 0;
            if (!apart) {
                const float counts = exp2_fast(unit - lv);
#pragma unroll
                for (int r = 0; r < RA; ++r) {
                    top[r] = fmaxf(fmaxf(s_top[b][0][r], s_top[b][1][r]), fmaxf(s_top[b][2][r], s_top[b][3][r]));
                    S[r] = exp2_fast(S[r] - (top[r] == -INFINITY ? 0.0f : top[r]));
                    sums[r] = S[r] * counts;
                }
            } else {
                if (!apart_before) {
                    if (me < RA) s_unit[b][me] = unit;
#pragma unroll
                    for (int r = 0; r < RA; ++r) {
                        m[r] -= unit;
                        m_step[r] -= unit;
                    }
                }
#pragma unroll
                for (int r = 0; r < RA; ++r) {
                    S[r] -= lv;
                    const float2 most = apart_maxima(S[r], lv);
                    if (lane == r) {
                        s_top[b][warp][r] = most.x;
                        s_far[b][warp][r] = most.y;
                    }
                }
                sync4();
#pragma unroll
                for (int r = 0; r < RA; ++r) {
                    const float4 w = apart_weight(S[r], lv, s_top[b][0] + r, s_far[b][0] + r, RA);
                    if (me == r) s_step_unit[b][r] = w.w;
                    S[r] = w.x;
                    sums[r] = w.y;
                    top[r] = w.z;
                }
            }
            // ---- weights: hi at row r, lo at row NR + r, this position's byte (the product of two steps ago, which read them, has been joined) ----
            unsigned char* P = Ps + b * (N * 128);
#pragma unroll
            for (int r = 0; r < RA; r += 2) {
                uint32_t hi, part;
                two_parts(__floats2half2_rn(S[r] * 256.0f, S[r + 1] * 256.0f), hi, part);
                P[sw128_byte(r, me)] = (unsigned char)hi;
                P[sw128_byte(r + 1, me)] = (unsigned char)(hi >> 8);
                P[sw128_byte(NR + r, me)] = (unsigned char)part;
                P[sw128_byte(NR + r + 1, me)] = (unsigned char)(part >> 8);
            }
            umma::fence_async_smem();
            arrive(&bars.p_full[b]);
            if (i > 0) join_product(i - 1);
#pragma unroll
            for (int r = 0; r < RA; ++r) {
                m_step[r] = top[r];
                l_step[r] = sums[r];
            }
            apart_step = apart;
        }
        if (apart_step) sync4();
        join_product(steps - 1);
        // ---- a column of the result per thread: written, put down as this share's, or left in shared memory for the cluster.  What a row's results are multiplied by and where they go
        // is worked out by a thread each (all rows by every thread: 11200 cycles for 16) ----
#pragma unroll
        for (int r = 0; r < RA; ++r) {
            const float total = warp_sum(l[r]);
            if (lane == 0) s_sum[warp][r] = total;
        }
        sync4();
        if (me < rows) {
            float top = 0.0f;
#pragma unroll
            for (int r = 0; r < RA; ++r) top = me == r ? m[r] : top;
            if (!apart_step) top -= unit;
            const float total = (s_sum[0][me] + s_sum[1][me]) + (s_sum[2][me] + s_sum[3][me]), e = (apart_step ? s_unit[steps & 1][me] : unit) - 8.0f;
            if (A.n_splits == 1) {
                const Finish f(A, s_head[me], top, total, e);
                s_finish[me] = make_float2(f.a, f.b);
                s_to[me] = (size_t)s_row[me] * A.o_row + (size_t)s_head[me] * A.o_head;
            } else if (clustered) {
                s_stat[me] = make_float4(top, total, e, 0.0f);
            } else {
                const size_t at = ((size_t)s_row[me] * A.H + s_head[me]) * A.n_splits + split;
                part_stats(A)[at] = make_float4(top, total, e, 0.0f);
                s_to[me] = at * ((A.c.dv + 3) / 4 * 4);
            }
        }
        sync4();
#pragma unroll
        for (int x = 0; x < HALVES; ++x) {
            const int col = x * 128 + me;
            if (col >= A.c.dv || *stop) continue;
            const uint32_t nans = s_bad ? nan_columns<RA, TREE>(A, W, col) : 0u;
            if (nans != 0u) {
#pragma unroll
                for (int r = 0; r < RA; ++r) o[x][r] = nans >> r & 1 ? __int_as_float(0x7fffffff) : o[x][r];
            }
            if (clustered || (A.n_splits == 1 && A.gate)) {
#pragma unroll
                for (int r = 0; r < RA; ++r) joint[r * D + col] = o[x][r];
            }
            if (A.n_splits == 1 && A.gate) {
#pragma unroll 1
                for (int r = 0; r < rows; ++r) {
                    const float2 f = s_finish[r];
                    static_cast<bf16*>(A.out)[s_to[r] + col] = __float2bfloat16_rn(finished(A, s_row[r], s_head[r], col, joint[r * D + col] * f.x * f.y));
                }
            } else if (A.n_splits == 1) {
#pragma unroll
                for (int r = 0; r < RA; ++r) {
                    const float2 f = s_finish[r];
                    if (r < rows) static_cast<bf16*>(A.out)[s_to[r] + col] = __float2bfloat16_rn(o[x][r] * f.x * f.y * A.out_scale);
                }
            } else if (!clustered) {
#pragma unroll
                for (int r = 0; r < RA; ++r)
                    if (r < rows) A.part[s_to[r] + col] = o[x][r];
            }
        }
    } else if (any) {
        // no key in this share
        for (int r = warp; r < RA; r += 4) {
            const int row = min(row0 + r, n * Gq - 1);
            if (lane == 0) {
                s_row[r] = t0 + row / Gq;
                s_head[r] = g * Gq + row % Gq;
            }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        for (int col = threadIdx.x; col < A.c.dv; col += 128)
            for (int r = 0; r < rows; ++r) put(r, col, -INFINITY, 0.0f, 0.0f, 0.0f);
    }
    __syncwarp();
    if (clustered) {
        cluster_sync();
        if (any && warp < 4 && !*stop) {
            if constexpr (RA <= 4) join_few_shares<D>(A, split, rows, s_stat, joint, s_row, s_head);
            else join_shares<128>(A, split, rows, s_stat, joint, D, s_row, s_head, s_finish, s_to, s_counts);
        }
        cluster_sync();      // nobody leaves while others read
    }
    __syncwarp();
    umma::fence_before_sync();
    __syncthreads();
    if (warp == kFewProducts) tmem_give<COLS>(tmem);
}

}  // namespace c8
}  // namespace smol
