// What moves inside the 8-bit key/value cache: rows of an accepted path, whole pages; and the layout of a tree of drafted rows.  Included by cache8_drafts.cu.
#pragma once

#include "cache8_tc.cuh"

namespace smol {
namespace c8 {

// ---- trees ----
// Of every row's parent among the rows of its sequence (-1: it follows the context): its position, the context's length and its depth, and a bit for itself and every row on
// its way up.  A parent comes in front of its children, so that 32 rows that follow one another know their ways among themselves after five doublings
// (in registers), and what is left is a hop per 32 rows in front of them: word w of a row is the ways among rows 32 w .. + 31 of the row in them that the hops reach.
// Latency is all there is to it: 1.7 us for 64 trees of 64 rows, 1.4 for one of 25.
constexpr int kTreeRows = 4096;      // most rows of a sequence
struct TreeArgs {
    Batch b;
    const int32_t* parents;
    int32_t* positions;
    uint32_t* sees;
    int words;
    int32_t* err;
};
__global__ void __launch_bounds__(1024) tree_kernel(const TreeArgs A) {
    __shared__ uint32_t s_mask[kTreeRows];      // rows among the row's 32 that are on its way
    __shared__ int s_up[kTreeRows];             // the row in front of these that its way goes on with (-1: none)
    dep_wait();
    dep_go();
    const Sequence Q(A.b, blockIdx.x, A.err);
    if (Q.n == 0) return;
    if (Q.pos0 < 0 || Q.n > A.b.max_new) {
        if (threadIdx.x == 0) atomicExch(A.err, 2);
        return;
    }
    for (int i0 = threadIdx.x & ~31; i0 < Q.n; i0 += blockDim.x) {
        const int lane = threadIdx.x & 31, i = i0 + lane;
        int parent = i < Q.n ? A.parents[Q.t0 + i] : -1;
        if (parent < -1 || parent >= i) {
            atomicExch(A.err, 2);
            parent = -1;
        }
        uint32_t mask = 1u << lane;
        int up = parent;      // below i0: outside; otherwise the lane that the mask's way goes on with
#pragma unroll
        for (int x = 0; x < 5; ++x) {
            const int from = up >= i0 ? up - i0 : lane;
            const uint32_t more = __shfl_sync(0xffffffffu, mask, from);
            const int next = __shfl_sync(0xffffffffu, up, from);
            mask |= more;
            up = up >= i0 ? next : up;
        }
        if (i < Q.n) {
            s_mask[i] = mask;
            s_up[i] = up;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < Q.n; i += blockDim.x) {
        uint32_t* sees = A.sees + (size_t)(Q.t0 + i) * A.words;
        int at = i, depth = 0;
        for (int w = A.words - 1; w >= 0; --w) {
            uint32_t word = 0;
            if (at >= 0 && at >> 5 == w) {
                word = s_mask[at];
                at = s_up[at];
            }
            sees[w] = word;
            depth += __popc(word);
        }
        A.positions[Q.t0 + i] = Q.pos0 + depth - 1;
    }
}

// ---- caches of several layers, all of one shape ----
constexpr int kMoveLayers = 32;      // of a launch
struct Layer {
    uint8_t *k, *v;
    float *ks, *vs;
    int32_t* err;
};
struct Layers {
    Cache c;      // the shape (its pointers are the first layer's)
    int n;
    Layer of[kMoveLayers];
};

// ---- rows ----
// Rows rows[s][0] < rows[s][1] < ... < rows[s][counts[s] - 1] behind pos0[s] become the rows pos0[s], pos0[s] + 1, ...: written as an append of the values that they have would
// write them.  A warp per (layer, head, sequence) takes the blocks of 16 positions that rows go to one after the other, keys and values at once.  A block's rows are in registers before
// any of it is written, and rows of later blocks come from behind it, so that nothing is overwritten that is still to be read.
//
// A code changes only where the scale does: rows whose block had the scale that they get are copied.  A block that holds older rows keeps its scale while no
// row comes from a larger one (codes are at most 448, so that a row's values are at most 448 times its old scale); otherwise, and in a block of kept rows alone, the largest magnitude is found.
// What bounds it: the instructions that look for a magnitude and rescale (0.56 of the issue slots, 660 a warp), and a chain of three loads (counts and rows, pages, codes and scales).  Up to 7 of 64
// rows of 64 sequences in 28 layers of 8 heads of 128: 14.7 us (a warp for keys and one for values 35.6, in float32 throughout 19.6); one sequence in 12 layers of 4 heads of 64 3.4.
struct KeepArgs {
    Layers l;
    const int32_t *pos0, *table, *rows, *counts;
    int S, max_pages, most;
};
// Sixteen codes times f.  In f16 where that is exact before the one rounding: codes are multiples of 2^-9 below 2^9, f a power of two from 2^-14 (products are multiples of 2^-23)
// to 2^15 (what passes f16 passes 448 too).  (In float32 it is sixteen conversions more, of which an SM makes sixteen a cycle.)
__device__ __forceinline__ uint4 rescaled(uint4 codes, float f) {
    uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
    const uint32_t bits = __float_as_uint(f);
    if ((bits & 0x7fffffu) == 0u && bits >= (127u - 14u) << 23 && bits <= (127u + 15u) << 23) {
        const __half2 f2 = __float2half2_rn(f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t part[2];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const __half2_raw raw = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i] >> 16 * z & 0xffffu), __NV_E4M3);
                part[z] = __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(__hmul2(__half2(raw), f2)), __NV_SATFINITE, __NV_E4M3);
            }
            w[i] = part[0] | part[1] << 16;
        }
    } else {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
            const float4 v = from_e4m3x4(codes.x);
            const uint32_t q = to_e4m3x4(v.x * f, v.y * f, v.z * f, v.w * f);
            codes = make_uint4(codes.y, codes.z, codes.w, q);
        }
        return codes;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
constexpr int kKeepWarps = 4;
// PASSES of 16 / PASSES rows, 2 PASSES lanes a row of 16 codes each, as in append_kernel
template <int PASSES>
__global__ void __launch_bounds__(kKeepWarps * 32) keep_kernel(const __grid_constant__ KeepArgs A) {
    constexpr int LANES = 2 * PASSES, ROWS = 32 / LANES;
    dep_wait();
    dep_go();
    const Cache& c = A.l.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, piece = lane % LANES, sub = lane / LANES;
    const int g = blockIdx.x * kKeepWarps + warp, s = blockIdx.y;
    if (g >= c.G) return;
    const Layer& L = A.l.of[blockIdx.z];
    const int32_t *rows = A.rows + (size_t)s * A.most, *table = A.table + (size_t)s * A.max_pages;
    const int pos0 = A.pos0[s], count = A.counts[s];
    int r = lane < A.most ? rows[lane] : 0, before = lane > 0 && lane < A.most ? rows[lane - 1] : -1;      // (with the counts, not behind them)
    // ---- what the arrays say, before anything is made of it ----
    int wrong = pos0 < 0 || pos0 >= kPositions || count < 0 || count > A.most ? 2 : 0;
    if (wrong == 0)
        for (int i = lane; i < count; i += 32) {
            if (i >= 32) {
                r = rows[i];
                before = rows[i - 1];
            }
            if (r < i || r <= before || r >= kPositions - pos0) {      // (rows that ascend from 0 on are not below their number: what a lane reads here, it has checked by itself)
                wrong = 2;
            } else {
                const int from = (pos0 + r) / c.page, to = (pos0 + i) / c.page;      // (0 <= to <= from)
                const int a = from < A.max_pages ? table[from] : -1, b = from < A.max_pages ? table[to] : -1;
                if ((unsigned)a >= (unsigned)c.n_pages || (unsigned)b >= (unsigned)c.n_pages) wrong = max(wrong, 1);
            }
        }
    wrong = __reduce_max_sync(0xffffffffu, wrong);
    if (wrong > 0) {
        if (lane == 0) atomicExch(L.err, wrong);
        return;
    }
    if (count == 0) return;
    const int blocks = g * (c.page / kBlock);
    for (int block = pos0 / kBlock; block <= (pos0 + count - 1) / kBlock; ++block) {
        const int p0 = block * kBlock, lo = max(pos0 - p0, 0), hi = min(pos0 + count - p0, kBlock);
        // lane r: where row r of the block comes from
        int from_page = 0, from_row = 0;
        const bool mine = lane >= lo && lane < hi;
        bool moves = lo == 0;      // (rows that stay where they are, in a block whose scale has to stay: nothing to do)
        if (mine) {
            const int p = pos0 + rows[p0 + lane - pos0], pg = p / c.page;
            from_page = table[pg];
            from_row = p - pg * c.page;
            moves |= p != p0 + lane;
        }
        if (!__any_sync(0xffffffffu, moves)) continue;
        const int pg = p0 / c.page, page = table[pg], in_page = p0 - pg * c.page;
        uint4 x[2][PASSES];
        float scale[2], had[2];      // lane r: of row r's block; of this block
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int ld = z ? c.ldv : c.ldk;
            const uint8_t* row = (z ? L.v : L.k) + (size_t)from_page * (z ? c.v_page : c.k_page) + ((size_t)g * c.page + from_row) * ld;
#pragma unroll
            for (int y = 0; y < PASSES; ++y) {
                if (y * ROWS >= hi || (y + 1) * ROWS <= lo) continue;
                const int r = y * ROWS + sub;
                const uint8_t* at = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), r));
                x[z][y] = make_uint4(0u, 0u, 0u, 0u);
                if (r >= lo && r < hi && piece * 16 < ld) x[z][y] = *reinterpret_cast<const uint4*>(at + piece * 16);
            }
            const float* scales = (z ? L.vs : L.ks) + blocks;
            const size_t stride = z ? c.vs_page : c.ks_page;
            scale[z] = mine ? scales[(size_t)from_page * stride + from_row / kBlock] : 0.0f;
            had[z] = scales[(size_t)page * stride + in_page / kBlock];
        }
        __syncwarp();      // every lane has read the block
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int ld = z ? c.ldv : c.ldk;
            uint8_t* const to = (z ? L.v : L.k) + (size_t)page * (z ? c.v_page : c.k_page) + ((size_t)g * c.page + in_page) * ld;
            const int Eold = lo > 0 ? min(max((int)((__float_as_uint(had[z]) >> 23) & 0xffu) - 127, kLeastExp), kMostExp) : kLeastExp;
            int E = Eold;
            bool nan = lo > 0 && had[z] < 0.0f;
            if (lo == 0 || __any_sync(0xffffffffu, fabsf(scale[z]) > pow2(Eold) || scale[z] < 0.0f)) {
                float top = 0.0f;
                const bool marked = __any_sync(0xffffffffu, scale[z] < 0.0f);      // some row may hold a NaN
#pragma unroll
                for (int y = 0; y < PASSES; ++y) {
                    if (y * ROWS >= hi || (y + 1) * ROWS <= lo) continue;
                    // magnitudes order as codes do
                    uint32_t w[4] = {x[z][y].x, x[z][y].y, x[z][y].z, x[z][y].w}, most = 0;
                    if (marked) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t clean = without_nans(w[i]);
                            nan |= clean != w[i];
                            w[i] = clean;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) most = __vmaxu2(most, __vmaxu2(w[i] & 0x007f007fu, w[i] >> 8 & 0x007f007fu));
                    most = max(most & 0xffffu, most >> 16);
                    top = fmaxf(top, from_e4m3x4(most).x * fabsf(__shfl_sync(0xffffffffu, scale[z], y * ROWS + sub)));
                }
                const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
                nan = __any_sync(0xffffffffu, nan);
                // bits: m 2^e, 1 <= m < 2, and 448 = 1.75 2^8
                E = max(Eold, min((int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), kMostExp));
            }
            if (E > Eold && lo > 0) {
                // older rows' codes follow the scale that grows
                const float down = pow2(max(Eold - E, -126));
                for (int r = sub; r < lo; r += ROWS)
                    if (piece * 16 < ld) {
                        uint4* old = reinterpret_cast<uint4*>(to + (size_t)r * ld + piece * 16);
                        const uint4 w = *old;
                        *old = rescaled(w, down);
                    }
            }
            // lane r: of row r.  (From 2^18 on the row is zeros: the least code, 2^-9, would pass 448.  The quotient of two scales may be no fp32 number, and zeros times infinity NaN.)
            const float f = fminf(fabsf(scale[z]) * pow2(-E), pow2(18));
            const bool same = __all_sync(0xffffffffu, !mine || f == 1.0f);
#pragma unroll
            for (int y = 0; y < PASSES; ++y) {
                if (y * ROWS >= hi || (y + 1) * ROWS <= lo) continue;
                const int r = y * ROWS + sub;
                const float fr = same ? 1.0f : __shfl_sync(0xffffffffu, f, r);
                if (r >= lo && r < hi && piece * 16 < ld) *reinterpret_cast<uint4*>(to + (size_t)r * ld + piece * 16) = fr == 1.0f ? x[z][y] : rescaled(x[z][y], fr);
            }
            if (lane == 0) (z ? L.vs : L.ks)[(size_t)page * (z ? c.vs_page : c.ks_page) + blocks + in_page / kBlock] = nan ? -pow2(E) : pow2(E);
        }
        __syncwarp();
    }
}

// ---- pages ----
// Codes and scales of pages pair[i].x into pages pair[i].y, of every layer.  A block of threads per (16 KB of codes, or a page's scales; pair; layer), all of its loads at once.
// What bounds it: DRAM.  128 pages of 64 positions of 8 heads of 128 in 28 layers, 471 MB read and written: 141 us, 6.7 TB/s; one page of 4 heads of 64 in 12 layers 1.6 us.  Pairs travel as the
// launch's arguments, so that nothing is copied to the device in front of it and a wrong page is refused on the host.
constexpr int kCopyThreads = 256, kCopyLoads = 4, kCopyBytes = kCopyThreads * kCopyLoads * 16, kCopyPairs = 512;
struct CopyArgs {
    Layers l;
    int k_parts, v_parts;      // blocks of threads of a page's keys and values
    int2 pair[kCopyPairs];
};
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyArgs A) {
    dep_wait();
    dep_go();
    const Cache& c = A.l.c;
    const Layer& L = A.l.of[blockIdx.z];
    const int2 pair = A.pair[blockIdx.y];
    const int part = blockIdx.x;
    if (part < A.k_parts + A.v_parts) {
        const bool value = part >= A.k_parts;
        const size_t stride = value ? c.v_page : c.k_page, bytes = (size_t)c.G * c.page * (value ? c.ldv : c.ldk);
        const uint8_t* from = (value ? L.v : L.k) + (size_t)pair.x * stride;
        uint8_t* to = (value ? L.v : L.k) + (size_t)pair.y * stride;
        const size_t at = (size_t)(value ? part - A.k_parts : part) * kCopyBytes + threadIdx.x * 16;
        uint4 x[kCopyLoads];
#pragma unroll
        for (int i = 0; i < kCopyLoads; ++i)
            if (at + i * (kCopyThreads * 16) < bytes) x[i] = *reinterpret_cast<const uint4*>(from + at + i * (kCopyThreads * 16));
#pragma unroll
        for (int i = 0; i < kCopyLoads; ++i)
            if (at + i * (kCopyThreads * 16) < bytes) *reinterpret_cast<uint4*>(to + at + i * (kCopyThreads * 16)) = x[i];
    } else {
        const int n = c.G * (c.page / kBlock);
        for (int i = threadIdx.x; i < 2 * n; i += kCopyThreads) {
            const bool value = i >= n;
            const size_t stride = value ? c.vs_page : c.ks_page;
            float* s = (value ? L.vs : L.ks) + (value ? i - n : i);
            s[(size_t)pair.y * stride] = s[(size_t)pair.x * stride];
        }
    }
}

}  // namespace c8
}  // namespace smol
