// Attention over the 8-bit key/value cache for many bf16 query rows per sequence (prompts), on tcgen05.  Included by cache8.cu.
//
// One block of threads per (128 query rows of a sequence and key/value head, 128 columns of the values, key/value head, sequence, share of the keys).
// The rows are the step's tokens times the query heads that share the key/value head: what is staged once serves all of them, and a short
// portion fills a tile.  128 positions a step.  As for few rows (cache8_few.cuh) the codes go to the tensor cores as they are, and queries and
// weights are the sum of two e4m3 parts; here both parts have one unit and one accumulator, so that a product is eight instructions for 128 terms,
// as many cycles as bf16 operands would take.  That leaves a query's coordinates exact down to 2^-10 of the row's largest and 2^-18 of it
// below, and a weight's error at 2^-9, or 2^-18 of the largest weight times value scale that the row sees in the step: as for few rows the scale's logarithm is part of what is
// raised, exp2(s - m + log2(scale) - e).  (With the scale as a factor behind it, over the step's largest, a value 2^12 larger at a later position cost a row 5 %, one
// 2^18 larger all of it.)  Results are in units of 2^(m + e), the denominator, the weights' sums per block times 2^(e - log2(scale)), in units of 2^m.
//
// Roles: a warp that copies, one that issues the products, sixteen warps for the softmax: four threads per row, 32 columns of the scores and of
// the result each.  Scores are double-buffered in tensor memory, so that the next step's are multiplied while this step's are worked on, and weights
// take their place there (as the product's first operand; through shared memory a prompt of 4096 took 344 us where it then took 335); a step's product
// with the values is read back while the next one's is made, and joins the fp32 running results in registers.  Value codes that are NaN are
// cleaned away in steps that some row does not see as a whole, as for few rows.
//
// What bounds it: the softmax warps, of which an SM holds one block's (registers, and all of tensor memory).  A step of 128 rows by 128 positions takes about
// 3600 cycles, 2100 of them issuing (weights 1500 from end to end: an exponential, two roundings to codes, one back), the products 1100 beside
// them; preparing a block's queries 9000 and its results 3400 more.  4096 tokens of 32 and 8 heads of 128: 280 us, 0.49 PFLOP/s of the definition's; 7900
// behind a window of 1000, 16 and 4 heads: 206 us; trees of up to 64 rows behind up to 8192 positions, 32 sequences of 32 and 8 heads: 401 us.  Two threads a row, two groups of softmax warps in turn with others joining, and joining a product
// two steps late were all slower (331 to 379 us where this took 326).
#pragma once

#include "cache8_tc.cuh"

namespace smol {
namespace c8 {

constexpr int kTileRows = 128, kTileParts = 4, kTileCols = kStep / kTileParts, kTileSoft = 4 * kTileParts, kTileThreads = (kTileSoft + 2) * 32;
__host__ __device__ constexpr int tile_stages(int DK) { return DK <= 128 ? 3 : 2; }
__host__ __device__ constexpr int tile_stage_bytes(int DK) { return kStep * (DK + 128); }
__host__ __device__ constexpr int tile_smem(int DK) { return 1024 + 2 * kTileRows * DK + tile_stages(DK) * tile_stage_bytes(DK); }

struct TileBars {
    uint64_t full[3], empty[3];      // stages
    uint64_t s_full[2], p_full[2];   // scores in tensor memory, weights in their place
    uint64_t o_full[2];              // the weights' product in tensor memory
    uint64_t q_full, drained;
    uint32_t tmem;
    int stop;
};

// Four f16 numbers of magnitude at most 256 as e4m3 parts of one unit, hi + lo, codes in order
__device__ __forceinline__ void four_equal_parts(uint32_t x, uint32_t y, uint32_t& hi, uint32_t& lo) {
    asm("{\n\t.reg .b16 a, b, c, d;\n\t.reg .b32 f, g;\n\t"
        "cvt.rn.satfinite.e4m3x2.f16x2 a, %2;\n\tcvt.rn.satfinite.e4m3x2.f16x2 b, %3;\n\t"
        "mov.b32 %0, {a, b};\n\t"
        "cvt.rn.f16x2.e4m3x2 f, a;\n\tcvt.rn.f16x2.e4m3x2 g, b;\n\t"
        "sub.rn.f16x2 f, %2, f;\n\tsub.rn.f16x2 g, %3, g;\n\t"
        "cvt.rn.satfinite.e4m3x2.f16x2 c, f;\n\tcvt.rn.satfinite.e4m3x2.f16x2 d, g;\n\t"
        "mov.b32 %1, {c, d};\n\t}"
        : "=&r"(hi), "=&r"(lo) : "r"(x), "r"(y));
}
// two fp32 numbers in one instruction
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void of_two(uint64_t d, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d)); }
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_two(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint32_t half_two(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Columns col .. col + 31 (a bit each) of the values in which a row at `pos` sees a NaN.  Rare, and slow.
template <bool TREE>
__device__ __noinline__ uint32_t nan_bits(const AttendArgs& A, const Rows& W, int tok, int pos, int col) {
    uint32_t bits = 0;
    for (int b = 0; b * kBlock < (TREE ? W.end : min(W.end, pos + 1)); ++b) {
        const int pg = b * kBlock / A.c.page;
        const int page = pg < A.b.max_pages ? A.b.table[(size_t)W.s * A.b.max_pages + pg] : -1;
        if (page < 0 || page >= A.c.n_pages) continue;
        const int in_page = b * kBlock - pg * A.c.page;
        if (A.c.vs[(size_t)page * A.c.vs_page + W.g * (A.c.page / kBlock) + in_page / kBlock] >= 0.0f) continue;
        for (int i = 0; i < kBlock; ++i) {
            if (TREE ? !tree_sees(A, W.t0, W.pos0, tok, pos, b * kBlock + i, W.end) : !sees(A, pos, b * kBlock + i, W.end)) continue;
            const uint8_t* v = A.c.v + (size_t)page * A.c.v_page + ((size_t)W.g * A.c.page + in_page + i) * A.c.ldv + col;
            for (int c = 0; c < 32 && col + c < A.c.dv; ++c)
                if ((v[c] & 0x7f) == 0x7f) bits |= 1u << c;
        }
    }
    return bits;
}

constexpr float kFarAbove = 64.0f;      // in units of log2

// DK: key size padded; BENT: soft cap or distance penalties; TREE: rows of a tree
template <int DK, bool BENT, bool TREE>
__global__ void __launch_bounds__(kTileThreads, 1) attend_tiles_kernel(const __grid_constant__ AttendArgs A, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, int box) {
    constexpr int NS = tile_stages(DK), SB = tile_stage_bytes(DK), KH = DK / 128;
    extern __shared__ unsigned char smem_raw[];
    __shared__ TileBars bars;
    __shared__ StepScales s_scales[NS];
    __shared__ float2 s_max[2][kTileParts][kTileRows];      // a part's largest score, and largest score - it + log2(value scale)
    __shared__ float s_rowmul[kTileRows];
    __shared__ int s_bad;
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *KV = base, *Qs = KV + NS * SB;      // Qs: first parts, then second parts
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) { umma::bar_init(&bars.full[i], 1); umma::bar_init(&bars.empty[i], 1); }
        for (int i = 0; i < 2; ++i) {
            umma::bar_init(&bars.s_full[i], 1);
            umma::bar_init(&bars.p_full[i], kTileSoft);
            umma::bar_init(&bars.o_full[i], 1);
        }
        umma::bar_init(&bars.q_full, kTileSoft);
        umma::bar_init(&bars.drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];\n\tprefetch.tensormap [%1];" ::"l"(&kmap), "l"(&vmap) : "memory");
        bars.stop = 0;
        s_bad = 0;
    }
    if (warp == kTileSoft + 1) tmem_take<512>(&bars.tmem);
    dep_wait();
    const int Gq = A.H / A.c.G, v_halves = (A.c.dv + 127) / 128, tiles = gridDim.x / (A.n_splits * v_halves);
    const int split = blockIdx.x % A.n_splits, v_col = blockIdx.x / A.n_splits % v_halves * 128, tile = tiles - 1 - blockIdx.x / (A.n_splits * v_halves);      // the tiles with the most keys first
    const int s = blockIdx.z, g = blockIdx.y;
    const Sequence Q(A.b, s, A.c.err);
    const int t0 = Q.t0, n_all = Q.n, n = min(n_all, A.b.max_new), pos0 = Q.pos0;
    const int kv_len = A.b.kv_len ? A.b.kv_len[s] : 0x7fffffff;
    const int row0 = tile * kTileRows, rows = min(n * Gq - row0, kTileRows);
    const bool any = rows > 0 && (long long)n_all * Gq > A.rows_over && (long long)n_all * Gq <= A.rows_most && (!TREE || tree_fits(A, pos0, n_all));
    int first_pos = pos0 + row0 / Gq, last_pos = any ? pos0 + (row0 + rows - 1) / Gq : -1, behind = last_pos + 1, clear = first_pos + 1;      // clear: every row sees what is in front of it, but for the window
    if (TREE && any) {
        const TreeSpan span(A, t0 + row0 / Gq, (row0 + rows - 1) / Gq - row0 / Gq + 1, n_all, pos0);
        first_pos = span.first_pos; last_pos = span.last_pos; behind = span.behind; clear = pos0;
    }
    const Seen seen = seen_steps(A, first_pos, behind, kv_len);
    const Rows W{s, g, t0, row0, rows, pos0, Gq, kv_len, seen.end};
    const int share = (seen.count + A.n_splits - 1) / A.n_splits, lo = min(split * share, seen.count);
    const int steps = any ? min(lo + share, seen.count) - lo : 0;
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    dep_go();      // behind the allocation: a kernel set up early that wants tensor memory too must not get it first
    const uint32_t tmem = bars.tmem, tm_o = tmem + 2 * kStep;      // scores of even and odd steps, then products likewise
    volatile int* stop = &bars.stop;

    if (warp == kTileSoft) {
        copy_steps<KH, 1, NS, true>(A, &kmap, &vmap, box, W, seen, lo, steps, first_pos, KV, s_scales, bars.full, bars.empty, stop, v_col);
    } else if (warp == kTileSoft + 1) {
        if (steps > 0) {
            // ---- products ----
            const uint32_t q0 = umma::s2u(Qs), id_s = desc_e4m3(128, kStep, false, false), id_o = desc_e4m3(128, 128, false, true);
            const int ksteps = (A.c.d + 31) / 32;
            auto scores = [&](int i) {
                const int b = i & 1, st = i % NS;
                if (!warp_wait(&bars.full[st], (i / NS) & 1, stop, A.c.err)) return false;
                if (elected()) {
                    umma::fence_after_sync();
                    const uint32_t k0 = umma::s2u(KV + st * SB);
#pragma unroll
                    for (int part = 0; part < 2; ++part)
                        for (int k = 0; k < ksteps; ++k)
                            mma_e4m3(tmem + b * kStep, umma::smem_desc_sw128(q0 + (part * KH + (k >> 2)) * (kTileRows * 128) + (k & 3) * 32), umma::smem_desc_sw128(k0 + (k >> 2) * (kStep * 128) + (k & 3) * 32),
                                     id_s, part > 0 || k > 0 ? 1u : 0u);
                    umma::commit(&bars.s_full[b]);
                }
                __syncwarp();
                return true;
            };
            // A step's scores are multiplied behind the values of the step before last, whose weights lie where they go (products are made in the order of
            // their issue); they are wanted a whole step later.
            bool ok = warp_wait(&bars.q_full, 0, stop, A.c.err) && scores(0) && (steps < 2 || scores(1));
            for (int i = 0; ok && i < steps; ++i) {
                const int b = i & 1, st = i % NS;
                ok = warp_wait(&bars.p_full[b], (i >> 1) & 1, stop, A.c.err);
                if (!ok) break;
                if (elected()) {
                    umma::fence_after_sync();
                    const uint32_t v = umma::s2u(KV + st * SB) + KH * (kStep * 128);
#pragma unroll
                    for (int part = 0; part < 2; ++part)
#pragma unroll
                        for (int k = 0; k < kStep / 32; ++k)
                            mma_e4m3_weights(tm_o + b * 128, tmem + b * kStep + part * (kStep / 4) + k * 8, umma::smem_desc_sw128(v + k * 32 * 128), id_o, part > 0 || k > 0 ? 1u : 0u);
                    umma::commit(&bars.empty[st]);
                    umma::commit(&bars.o_full[b]);
                }
                __syncwarp();
                ok = i + 2 >= steps || scores(i + 2);
            }
            if (elected()) umma::commit(&bars.drained);      // nothing of the block's is in flight once this is through
            drain_bar(&bars.drained, 0);
        }
    } else if (steps > 0) {
        // ---- queries into shared memory, eight rows a warp, eight coordinates a lane: all loads before anything is made of them ----
        {
            constexpr int LANES = DK / 8, AT_ONCE = 32 / LANES, LOADS = 8 / AT_ONCE;      // of a row; rows of a load; loads
            const int at = lane % LANES * 8, r0 = warp * 8;
            size_t off = 0;      // (lane y finds row y, which takes a division)
            {
                const int row = min(row0 + r0 + (lane & 7), n * Gq - 1), tok = row / Gq;
                off = (size_t)(t0 + tok) * A.q_row + (size_t)(g * Gq + row - tok * Gq) * A.q_head;
            }
            uint4 u[LOADS];
#pragma unroll
            for (int y = 0; y < LOADS; ++y) {
                const bf16* q = static_cast<const bf16*>(A.q) + __shfl_sync(0xffffffffu, off, y * AT_ONCE + lane / LANES);
                u[y] = make_uint4(0u, 0u, 0u, 0u);
                if (A.q_vec == 2) {
                    if (at < A.c.d) u[y] = *reinterpret_cast<const uint4*>(q + at);
                } else {
                    auto two_at = [&](int c) {
                        const unsigned short* w = reinterpret_cast<const unsigned short*>(q);
                        return (c < A.c.d ? (uint32_t)w[c] : 0u) | (c + 1 < A.c.d ? (uint32_t)w[c + 1] << 16 : 0u);
                    };
                    u[y] = make_uint4(two_at(at), two_at(at + 2), two_at(at + 4), two_at(at + 6));
                }
            }
#pragma unroll 1
            for (int y = 0; y < LOADS; ++y) {      // (once a block: code that is fetched for it takes longer than it runs)
                const int r = r0 + y * AT_ONCE + lane / LANES;
                const uint32_t w[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
#pragma unroll
                for (int x = 1; x < LOADS; ++x) u[x - 1] = u[x];
                // the largest magnitude, as bits: a NaN's are above infinity's
                uint32_t most = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
#pragma unroll
                for (int x = LANES / 2; x > 0; x >>= 1) most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, x));
                const uint32_t top = max(most & 0xffffu, most >> 16);
                const int e = max((int)(top >> 7) - 127, -110);      // (below: rows of less than 2^-110 keep a factor that fp32 holds)
                const float up = pow2(7 - e);
                uint32_t hi[2], rest[2];
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    four_equal_parts(half_two(bf_lo(w[2 * x]) * up, bf_hi(w[2 * x]) * up), half_two(bf_lo(w[2 * x + 1]) * up, bf_hi(w[2 * x + 1]) * up), hi[x], rest[x]);
                unsigned char* to = Qs + at / 128 * (kTileRows * 128) + sw128_byte(r, at % 128);
                *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
                *reinterpret_cast<uint2*>(to + KH * (kTileRows * 128)) = make_uint2(rest[0], rest[1]);
                // (a row that is not finite: every score of it is a NaN)
                if (at == 0) s_rowmul[r] = top >= 0x7f80u ? __int_as_float(0x7fffffff) : pow2(e - 7) * (A.scale * (BENT ? 1.0f : kLog2e));
            }
        }
        umma::fence_async_smem();
        __syncwarp();
        if (lane == 0) arrive(&bars.q_full);
        asm volatile("bar.sync 5, %0;" ::"n"(kTileSoft * 32) : "memory");

        // ---- softmax: warps q, q + 4, q + 8, q + 12 share rows 32 q .. + 31; part p has columns 32 p .. + 31 of the scores and of the result ----
        const int quad = warp & 3, part = warp >> 2, row = quad * 32 + lane, my_row = min(row0 + row, n * Gq - 1), pos = TREE ? tree_position(A, t0 + my_row / Gq) : pos0 + my_row / Gq, h = g * Gq + my_row % Gq;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const float rowmul = s_rowmul[row], r1 = BENT && A.r1 ? A.r1[h] : 0.0f, r2 = BENT && A.r1 ? A.r2[h] : 0.0f, slope = BENT && A.slope ? A.slope[h] * kLog2e : 0.0f;
        const Bend bend(A);
        auto row_barrier = [&] { asm volatile("bar.sync %0, %1;" ::"r"(quad + 1), "n"(kTileParts * 32) : "memory"); };
        float m = -INFINITY, unit = 0.0f, l = 0.0f, m_step = -INFINITY, unit_step = 0.0f, l_step = 0.0f, o[kTileCols];      // l in units of 2^m, o of 2^(m + unit)
#pragma unroll
        for (int c = 0; c < kTileCols; ++c) o[c] = 0.0f;
        auto join_product = [&](int i) {
            const int b = i & 1;
            wait_bar(&bars.o_full[b], (i >> 1) & 1, stop, A.c.err);
            __syncwarp();
            umma::fence_after_sync();
            // what results and denominator are relative to is the first step's, and a later one's only where they would come near fp32's end (they are below 2^90)
            if (__any_sync(0xffffffffu, m_step > m + kFarAbove || (m_step - m) + unit_step > unit + kFarAbove)) {
                const float mn = m_step > m + kFarAbove ? m_step : m, had = unit + (m - mn), has = unit_step + (m_step - mn), un = m == -INFINITY || has > had + kFarAbove ? has : had;
                const bool some = mn != -INFINITY;
                const float keep = !some || had == un ? 1.0f : m == -INFINITY ? 0.0f : exp2_fast(had - un);
                l *= !some || m == mn ? 1.0f : exp2_fast(m - mn);
                m = mn;
                unit = some ? un : unit;
#pragma unroll
                for (int c = 0; c < kTileCols; ++c) o[c] *= keep;
            }
            l = fmaf(l_step, m_step == -INFINITY ? 0.0f : exp2_fast(m_step - m), l);
            const float add = m_step == -INFINITY ? 0.0f : exp2_fast((m_step - m) + (unit_step - unit)) * (1.0f / 256.0f);
#pragma unroll
            for (int x = 0; x < kTileCols / 32; ++x) {
                uint32_t v[4][8];
#pragma unroll
                for (int y = 0; y < 4; ++y) umma::tmem_ld8_issue(tm_o + b * 128 + part * kTileCols + 32 * x + 8 * y + lanes, v[y]);
                umma::tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float &o0 = o[32 * x + e], &o1 = o[32 * x + e + 1];
                    of_two(fma_two(two(__uint_as_float(v[e / 8][e % 8]), __uint_as_float(v[e / 8][e % 8 + 1])), two(add, add), two(o0, o1)), o0, o1);
                }
            }
            umma::fence_before_sync();
        };
        for (int i = 0; i < steps; ++i) {
            const int b = i & 1, st = i % NS, j0 = step_place(seen, lo, i), jc = j0 + part * kTileCols;
            // (a wait that has run out is not waited for again: the steps that are left go by, and nothing is written)
            wait_bar(&bars.full[st], (i / NS) & 1, stop, A.c.err);
            const uint32_t marks = s_scales[st].marks;
            const bool nans = marks & ((1 << kStepBlocks) - 1), holes = marks >> kStepBlocks;      // in the whole step
            float ks[kTileCols / kBlock], lv[kTileCols / kBlock];
#pragma unroll
            for (int x = 0; x < kTileCols / kBlock; ++x) {
                const float2 of = s_scales[st].of[part * (kTileCols / kBlock) + x];
                ks[x] = of.x;
                lv[x] = of.y;
            }
            wait_bar(&bars.s_full[b], (i >> 1) & 1, stop, A.c.err);
            __syncwarp();
            umma::fence_after_sync();
            float S[kTileCols];
            {
                uint32_t v[kTileCols / 8][8];
#pragma unroll
                for (int x = 0; x < kTileCols / 8; ++x) umma::tmem_ld8_issue(tmem + b * kStep + part * kTileCols + 8 * x + lanes, v[x]);
                umma::tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < kTileCols; ++e) S[e] = __uint_as_float(v[e / 8][e % 8]);
            }
            const bool whole = !holes && j0 + kStep <= min(clear, seen.end) && (A.window == 0 || j0 > last_pos - A.window || j0 + kStep <= A.first);
            // scores in units of log2: S times mul
            const bool direct = !BENT && whole && A.scale > 0.0f;
            float mul[kTileCols / kBlock];
#pragma unroll
            for (int x = 0; x < kTileCols / kBlock; ++x) mul[x] = rowmul * ks[x];
            if (!direct) {
#pragma unroll
                for (int e = 0; e < kTileCols; ++e) S[e] *= mul[e / kBlock];
                if (BENT) {
                    const float d0 = (float)(pos - jc);
                    if (TREE && jc + kTileCols > pos0)      // (some keys are rows of the tree)
                        bend(A, S, [&](int e) { return fmaxf((float)(pos - (jc + e < seen.end ? tree_key(A, t0, pos0, jc + e) : jc + e)), 0.0f); }, [&](int) { return r1; }, [&](int) { return r2; },
                             [&](int) { return slope; });
                    else
                        bend(A, S, [&](int e) { return TREE ? fmaxf(d0 - (float)e, 0.0f) : d0 - (float)e; }, [&](int) { return r1; }, [&](int) { return r2; }, [&](int) { return slope; });
                }
#pragma unroll
                for (int x = 0; x < kTileCols / kBlock; ++x) mul[x] = 1.0f;
            }
            if (TREE && !whole) {
                // which of the thread's keys the row's bits name (the context's all)
                const uint32_t named = tree_named(A, t0 + my_row / Gq, jc - pos0);
                const int last = seen.end - jc;
#pragma unroll
                for (int e = 0; e < kTileCols; ++e)
                    if (e >= last || ks[e / kBlock] == 0.0f || !(named >> e & 1u)) S[e] = -INFINITY;
                if (A.window > 0) {
#pragma unroll
                    for (int e = 0; e < kTileCols; ++e) {
                        const int key = e < last ? tree_key(A, t0, pos0, jc + e) : 0;
                        if (pos - key >= A.window && key >= A.first) S[e] = -INFINITY;
                    }
                }
            } else if (!whole) {
                const int far = A.window > 0 ? A.window : 0x7fffffff, last = min(pos + 1, seen.end) - jc, lead = A.first - jc, dist = pos - jc;
#pragma unroll
                for (int e = 0; e < kTileCols; ++e)
                    if (e >= last || ks[e / kBlock] == 0.0f || (dist - e >= far && e >= lead)) S[e] = -INFINITY;
            }
            if (!whole || nans) {
                // the step's value codes without NaNs, 32 bytes a thread
                if (nans) s_bad = 1;
#pragma unroll 1
                for (int x = threadIdx.x; x < kStep * 8; x += kTileSoft * 32) {
                    uint4& at = reinterpret_cast<uint4*>(KV + st * SB + KH * (kStep * 128))[x];
                    const uint4 w = at, z = make_uint4(without_nans(w.x), without_nans(w.y), without_nans(w.z), without_nans(w.w));
                    if (w.x != z.x || w.y != z.y || w.z != z.z || w.w != z.w) at = z;
                }
            }
            // ---- the row's maxima over the step: of its scores, and of score + log2(scale) from there ----
            float most[kTileCols / kBlock], top = -INFINITY, e = -INFINITY;
#pragma unroll
            for (int x = 0; x < kTileCols / kBlock; ++x) {
                float t[4] = {S[16 * x], S[16 * x + 1], S[16 * x + 2], S[16 * x + 3]};
#pragma unroll
                for (int c = 4; c < 16; ++c) t[c % 4] = fmaxf(t[c % 4], S[16 * x + c]);
                most[x] = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])) * mul[x];
                top = fmaxf(top, most[x]);
            }
#pragma unroll
            for (int x = 0; x < kTileCols / kBlock; ++x) e = fmaxf(e, top == -INFINITY ? -INFINITY : (most[x] - top) + lv[x]);
            s_max[b][part][row] = make_float2(top, e);
            row_barrier();
            {
                float2 t[kTileParts];
#pragma unroll
                for (int x = 0; x < kTileParts; ++x) {
                    t[x] = s_max[b][x][row];
                    top = fmaxf(top, t[x].x);
                }
#pragma unroll
                for (int x = 0; x < kTileParts; ++x) e = x == 0 ? t[x].y + (t[x].x - top) : fmaxf(e, t[x].y + (t[x].x - top));
            }
            const bool none = top == -INFINITY;
            if (none) e = 0.0f;
            const float base = none ? 0.0f : top;
            float total = 0.0f;      // the denominator's terms
            // (value scales so far apart that weights which count there may be too small for an fp32 number; what is lost with them otherwise is below 2^-62)
            bool far = false;
#pragma unroll
            for (int x = 0; x < kTileCols / kBlock; ++x) far |= e - lv[x] > kFarAbove;
            far = __any_sync(0xffffffffu, far && !none);
            if (far) {
#pragma unroll
                for (int c = 0; c < kTileCols; ++c) total += exp2_fast(fmaf(S[c], mul[c / kBlock], -base));
            }
            // ---- weights, times 256 ----
            // (behind the barrier all of the row's scores are in registers: weights go where they were, first parts into the first 32 columns, second parts into the next)
            const uint32_t P = tmem + b * kStep + part * (kTileCols / 4) + lanes;
            uint32_t hi[8], rest[8];
            static_assert(kTileCols == 32, "eight columns of weights a thread");
#pragma unroll
            for (int x = 0; x < kTileCols / kBlock; ++x) {
                // (rounded down: not above 256 however large the scores)
                const float over = __fadd_rd((lv[x] - e) + 8.0f, -base);
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
            tmem_st8(P, hi);
            tmem_st8(P + kStep / 4, rest);
            tmem_st_wait();
            // (value codes that were cleaned)
            if (!whole || nans) umma::fence_async_smem();
            umma::fence_before_sync();
            __syncwarp();
            if (lane == 0) arrive(&bars.p_full[b]);
            if (i > 0) join_product(i - 1);
            m_step = top;
            unit_step = e;
            l_step = total;
        }
        join_product(steps - 1);
        // ---- the row's denominator, then 32 columns a thread ----
        row_barrier();
        s_max[0][part][row].x = l;
        row_barrier();
        float total = 0.0f;
#pragma unroll
        for (int x = 0; x < kTileParts; ++x) total += s_max[0][x][row].x;
        const int col = v_col + part * kTileCols;
        if (col < A.c.dv && !__any_sync(0xffffffffu, *stop)) {
            const bool mine = row < rows;
            const int tok = t0 + my_row / Gq;
            if (s_bad && mine) {
                const uint32_t bits = nan_bits<TREE>(A, W, tok, pos, col);
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    if (bits >> c & 1) o[c] = __int_as_float(0x7fffffff);
            }
            if (A.n_splits > 1) {
                const int ld = (A.c.dv + 3) / 4 * 4;
                const size_t at = ((size_t)tok * A.H + h) * A.n_splits + split;
                if (mine && col == 0) part_stats(A)[at] = make_float4(m, total, unit, 0.0f);
                float* to = A.part + at * ld + col;
#pragma unroll
                for (int c = 0; c < kTileCols; c += 4)
                    if (mine && col + c < ld) *reinterpret_cast<float4*>(to + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
            } else {
                const Finish f(A, h, m, total, unit);      // (one division a row)
                if (A.o_vec == 2 && !A.gate) {
                    // through shared memory (the ring is done with: the last product was waited for), so that four lanes write a row's 64 bytes: a lane's own row
                    // a lane, 8 bytes at a time, cost 4000 cycles a block
                    unsigned char* tile = KV + warp * (32 * 64);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        uint32_t w[4];
#pragma unroll
                        for (int y = 0; y < 4; ++y) w[y] = pack_bf16(o[8 * x + 2 * y] * f.a * f.b * A.out_scale, o[8 * x + 2 * y + 1] * f.a * f.b * A.out_scale);
                        *reinterpret_cast<uint4*>(tile + lane * 64 + (x ^ (lane >> 1 & 3)) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    __syncwarp();
                    const int piece = lane & 3;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int l = 8 * x + (lane >> 2), at = row0 + quad * 32 + l, t = at / Gq;
                        if (quad * 32 + l >= rows || col + piece * 8 >= A.c.dv) continue;
                        bf16* to = static_cast<bf16*>(A.out) + (size_t)(t0 + t) * A.o_row + (size_t)(g * Gq + at - t * Gq) * A.o_head + col + piece * 8;
                        *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(tile + l * 64 + (piece ^ (l >> 1 & 3)) * 16);
                    }
                } else if (mine) {
                    bf16* to = static_cast<bf16*>(A.out) + (size_t)tok * A.o_row + (size_t)h * A.o_head + col;
#pragma unroll
                    for (int c = 0; c < kTileCols; ++c)
                        if (col + c < A.c.dv) to[c] = __float2bfloat16_rn(finished(A, tok, h, col + c, o[c] * f.a * f.b));
                }
            }
        }
    } else if (any) {
        // no key in this share
        for (int i = threadIdx.x; i < rows * 128; i += kTileSoft * 32) {
            const int row = i / 128, col = v_col + i % 128, tok = t0 + (row0 + row) / Gq, h = g * Gq + (row0 + row) % Gq;
            if (col >= A.c.dv) continue;
            if (A.n_splits > 1) {
                const size_t at = ((size_t)tok * A.H + h) * A.n_splits + split;
                if (col == 0) part_stats(A)[at] = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
                A.part[at * ((A.c.dv + 3) / 4 * 4) + col] = 0.0f;
            } else {
                static_cast<bf16*>(A.out)[(size_t)tok * A.o_row + (size_t)h * A.o_head + col] = __float2bfloat16_rn(0.0f);
            }
        }
    }
    __syncwarp();
    umma::fence_before_sync();
    __syncthreads();
    if (warp == kTileSoft + 1) tmem_give<512>(tmem);
}

}  // namespace c8
}  // namespace smol
