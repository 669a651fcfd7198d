// Attention over the 8-bit key/value cache for float32 queries, whatever their number, and what the kernels for bf16 share with it.  Included by cache8.cu.
//
// One block per (16 query rows of a sequence and key/value head, key/value head, sequence, share of the keys): the rows are the step's tokens
// times the query heads that share the key/value head, so that a cached row is read once for all of them.  Its four warps take the share's
// blocks of 16 positions in turn, each with a running softmax of its own, and are joined at the end.
//
// Keys and values go from global memory through a ring in shared memory into mma.sync fragments without changing hands: every lane copies
// (cp.async) exactly the 16 bytes that it multiplies later, so that no barrier stands between a copy and its use.  That is possible because the
// order of a product's terms is free -- lane c of four takes bytes 16 c .. + 15 of a key row, which is four steps of four coordinates, and the
// query fragments are laid out to match; for the values a lane holds the same DV / 8 columns of four positions, and the column index of the
// product's eight columns is the lane's group.  Codes become f16 by moving bits (cache8.cuh); queries are scaled to below 2^15 per row and
// enter as two f16 parts, weights likewise.  Scores, maxima, denominators and results are fp32.
//
// What a row's results are relative to is the largest product of weight and value scale among the keys that it sees: with m about the largest score, and e about the
// largest (s - m) + log2(scale), a weight that the product multiplies is 2^8 exp2(s - m + log2(scale) - e), so that its last bit is one of the row's own largest term,
// whatever lies beside.  (With the scale as a factor behind exp2, over the largest scale of all blocks that the tile reads, a value 2^34 larger that a row does not see
// left nothing of its own.)  The denominator is in units of 2^m, results of 2^(m + e).  Both are whole numbers, so that what goes from one unit to the
// other is a power of two and rounds nothing.
//
// What bounds it: the instructions of its fragments (legacy mma.sync: f16 products of fp32's width would take three e4m3 parts on tcgen05).  A prompt of 300 tokens, 12
// and 4 heads of 64, logarithmic penalty: 23 us, of 2000 195 us; trees of 21 rows of 3 sequences at 922 positions, 12 and 4 heads of 80 and 72, 26 us; a token each of 16 sequences at up to 8192 positions, 32 and 8 heads of 128, 153 us.
#pragma once

#include "cache8.cuh"

namespace smol {
namespace c8 {

constexpr int kRowWarps = 4, kRowTile = 16, kRowThreads = kRowWarps * 32;

__host__ __device__ constexpr int row_stage_bytes(int DK, int DV) { return kBlock * (DK + DV); }
__host__ __device__ constexpr int row_stages(int DK, int DV) { return DK + DV <= 256 ? 4 : 3; }
constexpr int kParts = 2;      // f16 parts of a query and of a weight
__host__ __device__ constexpr bool q_in_smem(int DK) { return DK * kParts > 128; }
__host__ __device__ constexpr int row_q_bytes(int DK) { return q_in_smem(DK) ? DK / 16 * kParts * 512 : 0; }
__host__ __device__ constexpr int row_join_bytes(int DV) { return kRowWarps * kRowTile * (DV + 4) * 4; }
__host__ __device__ constexpr int row_smem(int DK, int DV) {
    const int ring = kRowWarps * row_stages(DK, DV) * row_stage_bytes(DK, DV) + row_q_bytes(DK), join = row_join_bytes(DV);
    return ring > join ? ring : join;
}

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy8(uint32_t to, const void* from, bool in) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(in ? 8 : 0) : "memory");
}
template <int N> __device__ __forceinline__ void copies_left() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// The blocks of 16 positions that rows at positions from first_pos on see, which see no key from `behind` on: `lead` of them from the sequence's start (the first tokens, in
// front of the window), then those from `from` up to the last visible key.
struct Seen {
    int lead, from, count, end;      // end: one behind the last visible key
};
// one behind the last key that rows see which see no key from `behind` on; positions behind the block table's last page are reported as a page that is not there, and not walked
__device__ __forceinline__ int last_visible(const AttendArgs& A, int behind, int kv_len) {
    const int end = max(min(kv_len, behind), 0);
    if (end > A.held && threadIdx.x == 0) atomicExch(A.c.err, 1);
    return min(end, A.held);
}
// first position in the window of a row at pos (below 0: all; a row in front of the sequence's first position sees nothing, and pos - window may be no number)
__device__ __forceinline__ int window_from(const AttendArgs& A, int pos) { return max(pos, 0) - A.window + 1; }
__device__ __forceinline__ Seen seen_blocks(const AttendArgs& A, int first_pos, int behind, int kv_len) {
    Seen x;
    x.end = last_visible(A, behind, kv_len);
    const int blocks = (x.end + kBlock - 1) / kBlock;
    x.from = A.window > 0 ? min(max(window_from(A, first_pos), 0) / kBlock, blocks) : 0;
    x.lead = A.window > 0 ? min(A.first / kBlock + (A.first % kBlock > 0), x.from) : 0;
    x.count = x.lead + blocks - x.from;
    return x;
}
__device__ __forceinline__ bool sees(const AttendArgs& A, int pos, int j, int end) {
    return j <= pos && j < end && (A.window == 0 || pos - j < A.window || j < A.first);
}

// ---- rows of a tree.  What lies in the cache in front of the sequence's rows is the context, which all of them see; of the rows themselves a row sees those that its bits
// name.  Distances (window, penalties) are between positions, which are the rows' own (a key's of the context is its place); one below zero counts as zero. ----
__device__ __forceinline__ int tree_position(const AttendArgs& A, int tok) { return min(max(A.tree_pos[tok], 0), kPositions - 1); }
// smallest and largest position of rows tok .. tok + n - 1; by a whole warp
__device__ __forceinline__ int2 tree_span(const AttendArgs& A, int tok, int n) {
    int lo = kPositions, hi = 0;
    for (int i = threadIdx.x & 31; i < n; i += 32) {
        const int p = tree_position(A, tok + i);
        lo = min(lo, p);
        hi = max(hi, p);
    }
    return make_int2(__reduce_min_sync(0xffffffffu, lo), __reduce_max_sync(0xffffffffu, hi));
}
// What a block of threads with rows tok .. + n - 1 of a sequence of n_all rows behind pos0 sees: every place up to `behind`, from where the window of a row at `first_pos` begins
// (no later than the rows themselves, whose positions may be anywhere); `last_pos` is the largest position.  All of it within `whole`.
struct TreeSpan {
    int first_pos, last_pos, behind;
    __device__ __forceinline__ TreeSpan(const AttendArgs& A, int tok, int n, int n_all, int pos0) : first_pos(pos0), last_pos(pos0) {
        behind = pos0 + (int)min((long long)n_all, 32ll * A.tree_words);
        if (A.window == 0) return;
        const int2 span = tree_span(A, tok, n);
        first_pos = (int)min((long long)span.x, (long long)pos0 + A.window - 1);
        last_pos = span.y;
    }
};
// position of the key at place j, below `behind`
__device__ __forceinline__ int tree_key(const AttendArgs& A, int t0, int pos0, int j) { return j < pos0 ? j : tree_position(A, t0 + j - pos0); }
__device__ __forceinline__ bool tree_sees(const AttendArgs& A, int t0, int pos0, int tok, int pos, int j, int end) {
    if (j >= end) return false;
    const int i = j - pos0;
    if (i >= 0 && (A.tree_sees[(size_t)tok * A.tree_words + (i >> 5)] >> (i & 31) & 1u) == 0u) return false;
    if (A.window == 0) return true;
    const int key = tree_key(A, t0, pos0, j);
    return pos - key < A.window || key < A.first;
}
// which of the 32 keys from row i0 of the sequence's rows on (below 0: of the context, all of it) the bits of row tok name
__device__ __forceinline__ uint32_t tree_named(const AttendArgs& A, int tok, int i0) {
    const int w = i0 >> 5;      // (rounded down)
    const uint32_t* bits = A.tree_sees + (size_t)tok * A.tree_words;
    const uint32_t low = w < 0 ? 0xffffffffu : w < A.tree_words ? bits[w] : 0u, high = w + 1 < 0 ? 0xffffffffu : w + 1 < A.tree_words ? bits[w + 1] : 0u;
    return __funnelshift_r(low, high, i0 & 31);
}
// which of the 32 keys from place jc on row tok sees; by a whole warp, whose lanes find a key's position each.  (A call, so that the loops around it keep their registers.)
static __device__ __noinline__ uint32_t tree_mask(const AttendArgs& A, int t0, int pos0, int tok, int pos, int jc, int end) {
    uint32_t mask = tree_named(A, tok, jc - pos0);
    if (end < jc + 32) mask = end <= jc ? 0u : mask & (1u << (end - jc)) - 1u;
    if (A.window > 0) {
        // of the context's places: those behind the window's beginning, and the first ones
        const long long from = (long long)pos - A.window + 1 - jc, first = (long long)A.first - jc;
        uint32_t near = (from <= 0 ? 0xffffffffu : from < 32 ? 0xffffffffu << from : 0u) | (first >= 32 ? 0xffffffffu : first > 0 ? (1u << first) - 1u : 0u);
        if (jc + 32 > pos0) {      // of the rows' own: by their positions, which a lane each has found
            const int at = jc + (threadIdx.x & 31), mine = at < end ? tree_key(A, t0, pos0, at) : 0;
#pragma unroll 1
            for (int e = max(pos0 - jc, 0); e < min(end - jc, 32); ++e) {      // (a loop: code that is fetched for a few steps takes longer than it runs, 5500 cycles unrolled)
                const int key = __shfl_sync(0xffffffffu, mine, e);
                const bool on = pos - key < A.window || key < A.first;
                near = on ? near | 1u << e : near & ~(1u << e);
            }
        }
        mask &= near;
    }
    return mask;
}
// Sequences of a tree lie behind a context of no fewer than zero positions.
__device__ __forceinline__ bool tree_fits(const AttendArgs& A, int pos0, int n) {
    if (pos0 >= 0) return true;
    if (n > 0 && threadIdx.x == 0) atomicExch(A.c.err, 2);
    return false;
}

// What follows the scaled product, in units of log2: soft cap and distance penalties, with the library's functions (float32).
__device__ __forceinline__ float bent_score(const AttendArgs& A, float s, int dist, float r1, float r2, float slope) {
    if (A.softcap > 0.0f) s = A.softcap * tanhf(s / A.softcap);
    const float d = (float)max(dist, 0);
    if (A.r1) s -= r1 * log1pf(r2 * d);
    return (s - slope * d) * kLog2e;
}
// The same with the hardware's (bf16): cap tanh(s / cap) log2 e = c - 2 c / (2^(s in) + 1) with c = cap log2 e and in = 2 log2 e / cap, and r ln(x) log2 e = r log2(x);
// slope comes in units of log2.  (Of a distance below zero, that is hidden anyway, a NaN is made.)
// That difference is off by some 2^-22 of the cap however small the score is: 6e-5 of a weight at a cap of 256, little beside a weight's own 2^-9, but 0.1 at 1e6.
// Above, scores below a quarter of the cap take tanh's series, cap tanh(x) = s (1 - x^2 / 3 + 2 x^4 / 15 - 17 x^6 / 315 + 62 x^8 / 2835) with x = s / cap, whose next
// term is below 2^-25 there; the others are off by at most 2^-20 of themselves either way.
constexpr float kCapOfDifference = 256.0f;
struct Bend {
    float in, c;
    __device__ __forceinline__ explicit Bend(const AttendArgs& A) : in(A.softcap > 0.0f ? fminf(2.0f * kLog2e / A.softcap, 3e38f) : 0.0f), c(fminf(A.softcap * kLog2e, 3.4e38f)) {}
    // N scores; dist(e), r1(e), r2(e), slope(e): of score e.  A loop per option: with the options looked at in every score, a step of the tiles took 7500 cycles.
    template <int N, class Dist, class R1, class R2, class Slope>
    __device__ __forceinline__ void operator()(const AttendArgs& A, float (&s)[N], Dist&& dist, R1&& r1, R2&& r2, Slope&& slope) const {
        if (A.softcap > kCapOfDifference) {
            const float inv = 1.0f / A.softcap;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float x = s[e] * inv, t = x * x, far = c * fmaf(-2.0f, __fdividef(1.0f, exp2_fast(s[e] * in) + 1.0f), 1.0f), l = s[e] * kLog2e;
                const float p = fmaf(fmaf(fmaf(62.0f / 2835.0f, t, -17.0f / 315.0f), t, 2.0f / 15.0f), t, -1.0f / 3.0f);
                s[e] = t < 0.0625f ? fmaf(l * t, p, l) : far;
            }
        } else if (c > 0.0f) {
#pragma unroll
            for (int e = 0; e < N; ++e) s[e] = fmaf(-2.0f * c, __fdividef(1.0f, exp2_fast(s[e] * in) + 1.0f), c);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) s[e] *= kLog2e;
        }
        if (A.r1) {
#pragma unroll
            for (int e = 0; e < N; ++e) s[e] = fmaf(-r1(e), log2_fast(fmaf(r2(e), dist(e), 1.0f)), s[e]);
        }
        if (A.slope) {
#pragma unroll
            for (int e = 0; e < N; ++e) s[e] = fmaf(-slope(e), dist(e), s[e]);
        }
    }
};

template <class T> struct Elem;
template <> struct Elem<float> {
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};
template <> struct Elem<bf16> {
    static __device__ __forceinline__ void put(bf16* p, float v) { *p = __float2bfloat16_rn(v); }
};

__device__ __forceinline__ float finished(const AttendArgs& A, int t, int h, int c, float v) {
    v *= A.out_scale;
    if (A.gate) v /= 1.0f + expf(-A.gate[(size_t)t * A.gate_row + (size_t)h * A.c.dv + c]);
    return v;
}

// What a row's unnormalised results, in units of 2^(top + e), are multiplied by: by a, then by b.  The denominator is total, in units of 2^top, and the sink's
// part.  Nothing visible: no weights, and the result is zero.  (In two steps: 2^e over the sink's part alone may be no fp32 number where result and quotient are.)
struct Finish {
    float a, b;
    __device__ __forceinline__ Finish(const AttendArgs& A, int h, float top, float total, float e) {
        const float sink = A.sink ? A.sink[h] * kLog2e : -INFINITY, M = fmaxf(sink, top);
        const float all = fmaf(total, top == -INFINITY ? 1.0f : exp2_fast(top - M), M == -INFINITY ? 0.0f : exp2_fast(sink - M));
        const float x = top == -INFINITY ? 0.0f : e + (top - M), half = floorf(0.5f * x);      // (whole numbers stay whole: their powers are exact)
        a = exp2_fast(half);
        b = all == 0.0f ? 1.0f : exp2_fast(x - half) / all;
    }
};
__device__ __forceinline__ float with_sink(const AttendArgs& A, int h, float top, float total, float e, float v) {
    const Finish f(A, h, top, total, e);
    return v * f.a * f.b;
}

// Blocks of scale sign < 0 hold NaN codes, which the products took for 480: a row that sees one of them becomes NaN, all of it where a key holds
// one, the value's column otherwise (mark(row, column)).  Rare, and slow.
template <bool TREE, class Mark>
__device__ void mark_nans(const AttendArgs& A, int s, int g, int t0, int row0, int rows, int pos0, int Gq, int kv_len, Mark mark) {
    for (int r = 0; r < rows; ++r) {
        const int tok = t0 + (row0 + r) / Gq, pos = TREE ? tree_position(A, tok) : pos0 + (row0 + r) / Gq, end = TREE ? kv_len : min(kv_len, pos + 1);
        for (int b = 0; b * kBlock < end; ++b) {
            const int pg = b * kBlock / A.c.page;
            const int page = pg < A.b.max_pages ? A.b.table[(size_t)s * A.b.max_pages + pg] : -1;
            if (page < 0 || page >= A.c.n_pages) continue;
            const int in_page = b * kBlock - pg * A.c.page, at = g * (A.c.page / kBlock) + in_page / kBlock;
            const bool kbad = A.c.ks[(size_t)page * A.c.ks_page + at] < 0.0f, vbad = A.c.vs[(size_t)page * A.c.vs_page + at] < 0.0f;
            if (!kbad && !vbad) continue;
            for (int i = 0; i < kBlock; ++i) {
                if (TREE ? !tree_sees(A, t0, pos0, tok, pos, b * kBlock + i, kv_len) : !sees(A, pos, b * kBlock + i, kv_len)) continue;
                const size_t row = (size_t)g * A.c.page + in_page + i;
                const uint8_t *k = A.c.k + (size_t)page * A.c.k_page + row * A.c.ldk, *v = A.c.v + (size_t)page * A.c.v_page + row * A.c.ldv;
                if (kbad)
                    for (int c = threadIdx.x; c < A.c.d; c += blockDim.x)
                        if ((k[c] & 0x7f) == 0x7f)
                            for (int o = 0; o < A.c.dv; ++o) mark(r, o);
                if (vbad)
                    for (int c = threadIdx.x; c < A.c.dv; c += blockDim.x)
                        if ((v[c] & 0x7f) == 0x7f) mark(r, c);
            }
        }
    }
}

// What the rows of a block of threads are: rows row0 .. row0 + rows - 1 of sequence s (token by token, the heads of key/value head g within one).
struct Rows {
    int s, g, t0, row0, rows, pos0, Gq, kv_len, end;
};
template <int ROWS>
struct Join {
    float max[kRowWarps][ROWS], sum[kRowWarps][ROWS], weight[kRowWarps][ROWS], top[ROWS], total[ROWS], unit[ROWS];      // weight: e of the warps' results, then what these count
    int bad;
};
__host__ __device__ constexpr int join_ld(int DV) { return DV + 4; }

// The four warps' maxima, sums and unnormalised results join[(warp * ROWS + row) * LD + column], joined and finished, or written as this share's part.
template <int ROWS, int LD, bool TREE>
__device__ __forceinline__ void join_rows(const AttendArgs& A, Join<ROWS>& J, float* join, const Rows& W, int split) {
    if (threadIdx.x < ROWS) {
        const int row = threadIdx.x;
        const float M = fmaxf(fmaxf(J.max[0][row], J.max[1][row]), fmaxf(J.max[2][row], J.max[3][row]));
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) {
            // a row of NaN scores has no maximum: its sums say so
            const float f = J.max[w][row] == -INFINITY ? (J.sum[w][row] == 0.0f ? 0.0f : J.sum[w][row]) : exp2_fast(J.max[w][row] - M);
            total = fmaf(J.sum[w][row], f, total);
        }
        float e[kRowWarps], E = -INFINITY;      // (a warp that has seen nothing: -infinity)
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) {
            e[w] = J.max[w][row] == -INFINITY ? -INFINITY : J.weight[w][row] + (J.max[w][row] - M);
            E = fmaxf(E, e[w]);
        }
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) J.weight[w][row] = e[w] == -INFINITY ? 0.0f : exp2_fast(e[w] - E);
        J.top[row] = M;
        J.total[row] = total;
        J.unit[row] = E;
    }
    __syncthreads();
    if (J.bad) {
        mark_nans<TREE>(A, W.s, W.g, W.t0, W.row0, W.rows, W.pos0, W.Gq, min(W.kv_len, W.end), [&](int row, int col) { join[row * LD + col] = __int_as_float(0x7fffffff); });      // (times whatever weight: NaN)
        __syncthreads();
    }
    for (int i = threadIdx.x; i < W.rows * A.c.dv; i += kRowThreads) {
        const int row = i / A.c.dv, col = i - row * A.c.dv, tok = W.t0 + (W.row0 + row) / W.Gq, h = W.g * W.Gq + (W.row0 + row) % W.Gq;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) v = fmaf(join[(w * ROWS + row) * LD + col], J.weight[w][row], v);
        if (A.n_splits > 1) {
            const size_t at = ((size_t)tok * A.H + h) * A.n_splits + split;
            if (col == 0) part_stats(A)[at] = make_float4(J.top[row], J.total[row], J.unit[row], 0.0f);
            A.part[at * ((A.c.dv + 3) / 4 * 4) + col] = v;
        } else {
            static_cast<float*>(A.out)[(size_t)tok * A.o_row + (size_t)h * A.o_head + col] = finished(A, tok, h, col, with_sink(A, h, J.top[row], J.total[row], J.unit[row], v));
        }
    }
}

// DK, DV: head sizes padded; BENT: soft cap or distance penalties; TREE: rows of a tree
template <int DK, int DV, bool BENT, bool TREE>
__global__ void __launch_bounds__(kRowThreads) attend_rows_kernel(const AttendArgs A) {
    constexpr int KP = DK / 64, VB = DV / 8, NS = row_stages(DK, DV), SB = row_stage_bytes(DK, DV), KS = DK / 16;
    constexpr bool QS = q_in_smem(DK);
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ Join<kRowTile> J;
    dep_wait();
    dep_go();
    const int s = blockIdx.z, g = blockIdx.y, tile = blockIdx.x / A.n_splits, split = blockIdx.x % A.n_splits;
    const Sequence Q(A.b, s, A.c.err);
    const int t0 = Q.t0, n = min(Q.n, A.b.max_new), pos0 = Q.pos0;
    const int Gq = A.H / A.c.G, row0 = tile * kRowTile, rows = min(n * Gq - row0, kRowTile);
    if (rows <= 0 || (TREE && !tree_fits(A, pos0, n))) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int kv_len = A.b.kv_len ? A.b.kv_len[s] : 0x7fffffff;
    int first_pos = pos0 + row0 / Gq, last_pos = pos0 + (row0 + rows - 1) / Gq, behind = last_pos + 1, clear = first_pos + 1;      // clear: every row sees what is in front of it, but for the window
    if (TREE) {
        const TreeSpan span(A, t0 + row0 / Gq, (row0 + rows - 1) / Gq - row0 / Gq + 1, Q.n, pos0);
        first_pos = span.first_pos; last_pos = span.last_pos; behind = span.behind; clear = pos0;
    }
    const Seen seen = seen_blocks(A, first_pos, behind, kv_len);
    const int share = (seen.count + A.n_splits - 1) / A.n_splits, b_lo = min(split * share, seen.count), b_hi = min(b_lo + share, seen.count);
    const int mine = b_hi - b_lo > warp ? (b_hi - b_lo - warp + kRowWarps - 1) / kRowWarps : 0;      // blocks of this warp: b_lo + warp, + 4, ...
    const Rows W{s, g, t0, row0, rows, pos0, Gq, kv_len, seen.end};
    if (threadIdx.x == 0) J.bad = 0;

    // where the warp's blocks are: lane i knows block number i of 32 (`now`), and of the 32 that follow
    struct Place { int page, in_page; float ks, lv; };      // lv: log2 of the values' scale
    bool bad = false;
    auto block_of = [&](int i) { const int x = b_lo + warp + i * kRowWarps; return x < seen.lead ? x : seen.from + x - seen.lead; };
    auto look_up = [&](int i0) {
        Place p;
        p.page = -1; p.in_page = 0; p.ks = 0.0f; p.lv = 0.0f;
        if (i0 + lane < mine) {
            const int j = block_of(i0 + lane) * kBlock, pg = j / A.c.page;
            p.page = pg < A.b.max_pages ? A.b.table[(size_t)s * A.b.max_pages + pg] : -1;
            p.in_page = j - pg * A.c.page;
            if (p.page < 0 || p.page >= A.c.n_pages) {
                p.page = -1;
                atomicExch(A.c.err, 1);
            } else {
                const int at = g * (A.c.page / kBlock) + p.in_page / kBlock;
                p.ks = A.c.ks[(size_t)p.page * A.c.ks_page + at];
                const float vs = A.c.vs[(size_t)p.page * A.c.vs_page + at];
                p.lv = scale_log2(fmaxf(fabsf(vs), 7.5231638e-37f));      // 2^-120: below every scale
                bad |= p.ks < 0.0f || vs < 0.0f;
            }
        }
        return p;
    };
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (NS * SB) + lane * 16;
    // a block's copies: pieces KP per key row (two rows a lane), then the lane's columns of four value rows
    auto copy_block = [&](int i, const Place& p) {
        const int page = __shfl_sync(0xffffffffu, p.page, i & 31), in_page = __shfl_sync(0xffffffffu, p.in_page, i & 31);
        const bool live = i < mine && page >= 0;
        const uint32_t to = ring + (i % NS) * SB;
        const uint8_t* k = A.c.k + (size_t)max(page, 0) * A.c.k_page + ((size_t)g * A.c.page + in_page) * A.c.ldk;
        const uint8_t* v = A.c.v + (size_t)max(page, 0) * A.c.v_page + ((size_t)g * A.c.page + in_page) * A.c.ldv;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < KP; ++y) {
                const int at = (c + 4 * y) * 16;
                const bool in = live && at < A.c.ldk;
                copy16(to + (x * KP + y) * 512, in ? k + (size_t)(r + 8 * x) * A.c.ldk + at : A.c.k, in);
            }
        // positions 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const uint8_t* row = v + (size_t)(2 * c + (x & 1) + 8 * (x >> 1)) * A.c.ldv;
            if (VB == 8) {
                const bool in = live && r * 8 < A.c.ldv;
                copy8(to - lane * 8 + kBlock * DK + x * 256, in ? row + r * 8 : A.c.v, in);
            } else {
#pragma unroll
                for (int y = 0; y < VB / 16; ++y) {
                    const int at = r * VB + 16 * y;
                    const bool in = live && at < A.c.ldv;
                    copy16(to + kBlock * DK + (x * (VB / 16) + y) * 512, in ? row + at : A.c.v, in);
                }
            }
        }
        copies_end();
    };
    Place now = look_up(0), next = look_up(32);
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) copy_block(i, now);

    // ---- queries: fragments of rows r and r + 8, scaled so that the largest magnitude lies in [2^14, 2^15) ----
    float rowmul[2];
    uint32_t qa[QS ? 1 : KS][QS ? 1 : kParts][4];
    uint4* qs = reinterpret_cast<uint4*>(smem + kRowWarps * NS * SB);
    {
        const float* q[2];
        float up[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int row = min(row0 + r + 8 * x, n * Gq - 1);
            q[x] = static_cast<const float*>(A.q) + (size_t)(t0 + row / Gq) * A.q_row + (size_t)(g * Gq + row % Gq) * A.q_head;
            uint32_t top = 0;
            for (int k = c; k < A.c.d; k += 4) top = max(top, __float_as_uint(fabsf(q[x][k])));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // (2^(14 - e) for a largest magnitude of m 2^e: within fp32 for e from -110 to 127; smaller rows are scaled by 2^124)
            const int e = max((int)(top >> 23) - 127, -110);
            up[x] = pow2(14 - e);
            rowmul[x] = top >= 0x7f800000u ? __int_as_float(0x7fffffff) : pow2(e - 14) * (A.scale * kCodeUnit * (BENT ? 1.0f : kLog2e));
        }
        auto fragment = [&](int k, uint32_t (&part)[kParts][4]) {
            // step k: word k % 4 of the lane's piece c + 4 (k / 4); its bytes 1 and 3, then 0 and 2
            const int at = ((k / 4) * 4 + c) * 16 + (k % 4) * 4;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = at + e < A.c.d ? q[x][at + e] * up[x] : 0.0f;
                const uint32_t odd = pack_f16(v[1], v[3]), even = pack_f16(v[0], v[2]);
                part[0][x] = odd;
                part[0][2 + x] = even;
                {
                    const float2 o = unpack_f16(odd), z = unpack_f16(even);
                    part[1][x] = pack_f16(v[1] - o.x, v[3] - o.y);
                    part[1][2 + x] = pack_f16(v[0] - z.x, v[2] - z.y);
                }
            }
        };
        if constexpr (QS) {
            for (int k = warp; k < KS; k += kRowWarps) {
                uint32_t part[kParts][4];
                fragment(k, part);
#pragma unroll
                for (int p = 0; p < kParts; ++p) qs[(k * kParts + p) * 32 + lane] = make_uint4(part[p][0], part[p][1], part[p][2], part[p][3]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < KS; ++k) fragment(k, qa[k]);
        }
    }
    __syncthreads();

    float r1[2], r2[2], slope[2];
    int pos[2], tok[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int row = min(row0 + r + 8 * x, n * Gq - 1), h = g * Gq + row % Gq;
        tok[x] = t0 + row / Gq;
        pos[x] = TREE ? tree_position(A, t0 + row / Gq) : pos0 + row / Gq;
        r1[x] = BENT && A.r1 ? A.r1[h] : 0.0f;
        r2[x] = BENT && A.r1 ? A.r2[h] : 0.0f;
        slope[x] = BENT && A.slope ? A.slope[h] : 0.0f;
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, unit[2] = {-INFINITY, -INFINITY};      // l is in units of 2^m, o of 2^(m + unit)
    float o[VB][4];
#pragma unroll
    for (int t = 0; t < VB; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][e] = 0.0f;

    for (int i = 0; i < mine; ++i) {
        if (i > 0 && (i & 31) == 0) {
            now = next;
            next = look_up(i + 32);
        }
        {
            const int ahead = i + NS - 1;
            copy_block(ahead, (ahead & ~31) == (i & ~31) ? now : next);
        }
        const int page = __shfl_sync(0xffffffffu, now.page, i & 31);
        const float ks = __shfl_sync(0xffffffffu, now.ks, i & 31), lv = __shfl_sync(0xffffffffu, now.lv, i & 31);
        copies_left<NS - 1>();
        if (page < 0) continue;
        const unsigned char* st = smem + warp * (NS * SB) + (i % NS) * SB;
        // ---- scores of 16 rows and 16 positions ----
        float sc[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int y = 0; y < KP; ++y) {
            uint4 w[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) w[x] = *reinterpret_cast<const uint4*>(st + (x * KP + y) * 512 + lane * 16);
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                uint32_t a[kParts][4];
#pragma unroll
                for (int p = 0; p < kParts; ++p) {
                    if constexpr (QS) {
                        const uint4 u = qs[((y * 4 + z) * kParts + p) * 32 + lane];
                        a[p][0] = u.x; a[p][1] = u.y; a[p][2] = u.z; a[p][3] = u.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) a[p][e] = qa[y * 4 + z][p][e];
                    }
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const uint32_t word = z == 0 ? w[x].x : z == 1 ? w[x].y : z == 2 ? w[x].z : w[x].w;
                    const uint32_t b0 = odd_codes(word), b1 = even_codes(word);
#pragma unroll
                    for (int p = 0; p < kParts; ++p) mma_f16_16816(sc[x], a[p][0], a[p][1], a[p][2], a[p][3], b0, b1);
                }
            }
        }
        // ---- running softmax, in units of log2; a lane has positions 2c, 2c + 1, 2c + 8, 2c + 9 of rows r and r + 8 ----
        const int j0 = block_of(i) * kBlock + 2 * c;
        const float km = fabsf(ks);
        const bool whole = j0 - 2 * c + kBlock <= min(clear, seen.end) && (A.window == 0 || j0 - 2 * c > last_pos - A.window || j0 - 2 * c + kBlock <= A.first);
        float p[2][4], top[2];
        int key[4];                // positions of the keys
        uint32_t named[2];         // the block's keys that the rows' bits name
        if (TREE) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = j0 + (e & 1) + 8 * (e >> 1);
                key[e] = !whole && j >= pos0 && j < seen.end ? tree_position(A, t0 + j - pos0) : j;
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) named[x] = whole ? 0xffffffffu : tree_named(A, tok[x], j0 - 2 * c - pos0);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const float mul = rowmul[x] * km;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = j0 + (e & 1) + 8 * (e >> 1);
                float v = sc[e >> 1][2 * x + (e & 1)] * mul;
                if (BENT) v = bent_score(A, v, pos[x] - (TREE ? key[e] : j), r1[x], r2[x], slope[x]);
                const bool on = whole || (TREE ? j < seen.end && (named[x] >> (j - j0 + 2 * c) & 1u) && (A.window == 0 || pos[x] - key[e] < A.window || key[e] < A.first) : sees(A, pos[x], j, seen.end));
                p[x][e] = on ? v : -INFINITY;
            }
            top[x] = fmaxf(fmaxf(p[x][0], p[x][1]), fmaxf(p[x][2], p[x][3]));
            top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
            top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1] || (top[0] - m[0]) + lv > unit[0] || (top[1] - m[1]) + lv > unit[1])) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float mn = fmaxf(m[x], ceilf(top[x]));
                if (mn == -INFINITY) continue;
                const float had = unit[x] + (m[x] - mn), un = fmaxf(had, ceilf((top[x] - mn) + lv)), keep = exp2_fast(had - un);
                l[x] *= exp2_fast(m[x] - mn);
                m[x] = mn;
                unit[x] = un;
#pragma unroll
                for (int t = 0; t < VB; ++t) {
                    o[t][2 * x] *= keep;
                    o[t][2 * x + 1] *= keep;
                }
            }
        }
        uint32_t pa[kParts][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const bool none = m[x] == -INFINITY;
            const float base = none ? 0.0f : m[x], away = none ? 0.0f : unit[x] - lv;
            // The denominator's terms are the weights' times 2^away, unless weights that count in it may be too small for an fp32 number (what is lost with them otherwise
            // is below 2^-62 of it).
            float sum = 0.0f;
            if (away > 64.0f) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += exp2_fast(p[x][e] - base);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) p[x][e] = exp2_fast((p[x][e] - base) - away);
            if (!(away > 64.0f)) sum = ((p[x][0] + p[x][1]) + (p[x][2] + p[x][3])) * exp2_fast(away);
            l[x] += sum;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const float a = p[x][2 * y] * kCodeUnit, b = p[x][2 * y + 1] * kCodeUnit;
                pa[0][x + 2 * y] = pack_f16(a, b);
                {
                    const float2 h = unpack_f16(pa[0][x + 2 * y]);
                    pa[1][x + 2 * y] = pack_f16(a - h.x, b - h.y);
                }
            }
        }
        // ---- weights x values: column of the product = lane group r', VB columns of it a lane ----
#pragma unroll
        for (int y = 0; y < VB / 4; y += VB == 8 ? 2 : 4) {
            uint32_t w[4][4];      // words of the four positions' rows
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                if (VB == 8) {
                    const uint2 u = *reinterpret_cast<const uint2*>(st + kBlock * DK + x * 256 + lane * 8);
                    w[x][0] = u.x; w[x][1] = u.y; w[x][2] = 0; w[x][3] = 0;
                } else {
                    const uint4 u = *reinterpret_cast<const uint4*>(st + kBlock * DK + (x * (VB / 16) + y / 4) * 512 + lane * 16);
                    w[x][0] = u.x; w[x][1] = u.y; w[x][2] = u.z; w[x][3] = u.w;
                }
            }
#pragma unroll
            for (int z = 0; z < (VB == 8 ? 2 : 4); ++z) {
                // columns 4 z .. + 3 of positions 2c and 2c + 1, and of 2c + 8 and 2c + 9: (second, first | second, first), (fourth, third | ...)
                const uint32_t a01 = __byte_perm(w[0][z], w[1][z], 0x4501), a23 = __byte_perm(w[0][z], w[1][z], 0x6723);
                const uint32_t b01 = __byte_perm(w[2][z], w[3][z], 0x4501), b23 = __byte_perm(w[2][z], w[3][z], 0x6723);
                const int t = (y + z) * 4;
#pragma unroll
                for (int pp = 0; pp < kParts; ++pp) {
                    mma_f16_16816(o[t], pa[pp][0], pa[pp][1], pa[pp][2], pa[pp][3], odd_codes(a01), odd_codes(b01));
                    mma_f16_16816(o[t + 1], pa[pp][0], pa[pp][1], pa[pp][2], pa[pp][3], even_codes(a01), even_codes(b01));
                    mma_f16_16816(o[t + 2], pa[pp][0], pa[pp][1], pa[pp][2], pa[pp][3], odd_codes(a23), odd_codes(b23));
                    mma_f16_16816(o[t + 3], pa[pp][0], pa[pp][1], pa[pp][2], pa[pp][3], even_codes(a23), even_codes(b23));
                }
            }
        }
    }
    copies_left<0>();
    // ---- the warps' results are joined ----
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
        if (c == 0) {
            J.max[warp][r + 8 * x] = m[x];
            J.sum[warp][r + 8 * x] = l[x];
            J.weight[warp][r + 8 * x] = unit[x];
        }
    }
    if (bad) J.bad = 1;
    __syncthreads();      // everybody's copies are used up: the ring becomes the results' place
    constexpr int LD = join_ld(DV);
    float* join = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float* to = join + (warp * kRowTile + r + 8 * x) * LD + (2 * c + e) * VB;
#pragma unroll
            for (int t = 0; t < VB; t += 4)
                *reinterpret_cast<float4*>(to + t) = make_float4(o[t][2 * x + e], o[t + 1][2 * x + e], o[t + 2][2 * x + e], o[t + 3][2 * x + e]);
        }
    join_rows<kRowTile, LD, TREE>(A, J, join, W, split);
}

// A block of threads per (token, head): joins the shares of the keys, and the sink.  Latency is all there is to it, so everything a warp needs is
// on its way at once: the shares' maxima first, then eight shares' results at a time, dealt out to the eight warps.
constexpr int kJoinWarps = 8;
template <class T>
__global__ void __launch_bounds__(kJoinWarps * 32) attend_join_kernel(const AttendArgs A) {
    __shared__ float4 s_acc[kJoinWarps][kMaxDim / 4];
    const int unit = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = unit / A.H, h = unit % A.H;
    dep_wait();
    dep_go();
    // rows in front of the first sequence, behind the last or behind max_new of their own are nobody's
    int lo = 0, hi = A.b.S;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (A.b.start[mid] <= t) lo = mid;
        else hi = mid;
    }
    const Sequence Q(A.b, lo, A.c.err);
    if (t < Q.t0 || t - Q.t0 >= min(Q.n, A.b.max_new) || (long long)Q.n * (A.H / A.c.G) <= A.rows_over || (A.tree_pos && !tree_fits(A, Q.pos0, 0))) return;      // (whoever has no shares)
    const int pieces = (A.c.dv + 3) / 4;
    const float4* stat = part_stats(A) + (size_t)unit * A.n_splits;      // maximum, denominator, e of the results
    const float4* part = reinterpret_cast<const float4*>(A.part) + (size_t)unit * A.n_splits * pieces;
    float4 st[kMaxSplits / 32];
    float M = -INFINITY, E = -INFINITY;
#pragma unroll
    for (int x = 0; x < kMaxSplits / 32; ++x) {
        st[x] = lane + 32 * x < A.n_splits ? stat[lane + 32 * x] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        M = fmaxf(M, st[x].x);
    }
    M = warp_max(M);
    float total = 0.0f;
#pragma unroll
    for (int x = 0; x < kMaxSplits / 32; ++x) {
        // a share of no visible key weighs nothing, one of NaN scores makes its row NaN
        total = fmaf(st[x].y, st[x].x == -INFINITY ? (st[x].y == 0.0f ? 0.0f : st[x].y) : exp2_fast(st[x].x - M), total);
        st[x].z = st[x].x == -INFINITY ? -INFINITY : st[x].z + (st[x].x - M);
        E = fmaxf(E, st[x].z);
    }
    E = warp_max(E);
#pragma unroll
    for (int x = 0; x < kMaxSplits / 32; ++x) st[x].z = st[x].z == -INFINITY ? 0.0f : exp2_fast(st[x].z - E);
    float4 acc[kMaxDim / 128];
#pragma unroll
    for (int e = 0; e < kMaxDim / 128; ++e) acc[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int x = 0; x < kMaxSplits / 32; ++x) {
        if (32 * x >= A.n_splits) break;
#pragma unroll
        for (int i = 0; i < 32 / kJoinWarps; ++i) {
            const int z = 32 * x + i * kJoinWarps + warp;
            const float f = __shfl_sync(0xffffffffu, st[x].z, z & 31);
#pragma unroll
            for (int e = 0; e < kMaxDim / 128; ++e)
                if (z < A.n_splits && lane + 32 * e < pieces) {
                    const float4 v = part[(size_t)z * pieces + lane + 32 * e];
                    acc[e].x = fmaf(v.x, f, acc[e].x);
                    acc[e].y = fmaf(v.y, f, acc[e].y);
                    acc[e].z = fmaf(v.z, f, acc[e].z);
                    acc[e].w = fmaf(v.w, f, acc[e].w);
                }
        }
    }
#pragma unroll
    for (int e = 0; e < kMaxDim / 128; ++e) s_acc[warp][lane + 32 * e] = acc[e];
    __syncthreads();
    const Finish finish(A, h, M, warp_sum(total), E);
    const float* flat = reinterpret_cast<const float*>(s_acc);
    for (int col = threadIdx.x; col < A.c.dv; col += kJoinWarps * 32) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) v += flat[w * kMaxDim + col];
        Elem<T>::put(static_cast<T*>(A.out) + (size_t)t * A.o_row + (size_t)h * A.o_head + col, finished(A, t, h, col, v * finish.a * finish.b));
    }
}

}  // namespace c8
}  // namespace smol
