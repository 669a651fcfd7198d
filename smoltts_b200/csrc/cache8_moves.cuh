// What moves inside the 8-bit key/value cache: rows of an accepted path, whole pages; and the layout of a tree of drafted rows.  Included by cache8_drafts.cu.
#pragma once

#include "cache8_tc.cuh"

namespace smol {
namespace c8 {

// ---- trees ----
// Of every row's parent among the rows of its sequence (-1: it follows the context): its position, the context's length and its depth, and a bit for itself and every row on
// its way up.  A parent comes in front of its children, so that 32 rows that follow one another know their ways among themselves after five doublings
// (in registers), and what is left is a hop per 32 rows in front of them: word w of a row is the ways among rows 32 w .. + 31 of the row in them that the hops reach.
// Latency is all there is to it.
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
// write them.  A warp per (layer, keys or values, sequence, head) takes the blocks of 16 positions that rows go to one after the other: a block's rows are in registers before any of it
// is written, and rows of later blocks come from behind it, so that nothing is overwritten that is still to be read.
// What bounds it: latency, a chain of four loads (count, rows, page, codes and scales).
struct KeepArgs {
    Layers l;
    const int32_t *pos0, *table, *rows, *counts;
    int S, max_pages, most;
};
constexpr int kKeepWarps = 4;
// PASSES of 16 / PASSES rows, 2 PASSES lanes a row of 16 codes each, as in append_kernel
template <int PASSES>
__global__ void __launch_bounds__(kKeepWarps * 32) keep_kernel(const __grid_constant__ KeepArgs A) {
    constexpr int LANES = 2 * PASSES, ROWS = 32 / LANES;
    dep_wait();
    dep_go();
    const Cache& c = A.l.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, piece = lane % LANES, sub = lane / LANES;
    const int unit = blockIdx.x * kKeepWarps + warp, s = blockIdx.y;      // unit: layer, head, keys or values
    if (unit >= A.l.n * c.G * 2) return;
    const Layer& L = A.l.of[unit / (c.G * 2)];
    const int g = unit / 2 % c.G;
    const bool value = unit & 1;
    const int32_t *rows = A.rows + (size_t)s * A.most, *table = A.table + (size_t)s * A.max_pages;
    const int pos0 = A.pos0[s], count = A.counts[s];
    // ---- what the arrays say, before anything is made of it ----
    auto page_of = [&](int p) {
        const int pg = p / c.page;
        return pg < A.max_pages ? table[pg] : -1;
    };
    int wrong = pos0 < 0 || pos0 >= kPositions || count < 0 || count > A.most ? 2 : 0;
    if (wrong == 0)
        for (int i = lane; i < count; i += 32) {
            const int r = rows[i], before = i > 0 ? rows[i - 1] : -1;
            if (r <= before || r >= kPositions - pos0) wrong = 2;
            else if ((unsigned)page_of(pos0 + i) >= (unsigned)c.n_pages || (unsigned)page_of(pos0 + r) >= (unsigned)c.n_pages) wrong = max(wrong, 1);
        }
    wrong = __reduce_max_sync(0xffffffffu, wrong);
    if (wrong > 0) {
        if (lane == 0) atomicExch(L.err, wrong);
        return;
    }
    if (count == 0) return;
    const int ld = value ? c.ldv : c.ldk;
    uint8_t* const codes = value ? L.v : L.k;
    float* const scales = value ? L.vs : L.ks;
    const size_t page_bytes = value ? c.v_page : c.k_page, page_scales = value ? c.vs_page : c.ks_page;
    const int blocks_of_page = c.page / kBlock;
    for (int block = pos0 / kBlock; block <= (pos0 + count - 1) / kBlock; ++block) {
        const int p0 = block * kBlock, lo = max(pos0 - p0, 0), hi = min(pos0 + count - p0, kBlock);
        // lane r: where row r of the block comes from
        size_t at = 0;
        float scale = 0.0f;
        if (lane >= lo && lane < hi) {
            const int p = pos0 + rows[p0 + lane - pos0], pg = p / c.page, page = table[pg], in_page = p - pg * c.page;
            at = (size_t)page * page_bytes + ((size_t)g * c.page + in_page) * ld;
            scale = scales[(size_t)page * page_scales + g * blocks_of_page + in_page / kBlock];
        }
        const int pg = p0 / c.page, page = table[pg], in_page = p0 - pg * c.page;
        float* const to_scale = scales + (size_t)page * page_scales + g * blocks_of_page + in_page / kBlock;
        uint8_t* const to = codes + (size_t)page * page_bytes + ((size_t)g * c.page + in_page) * ld;
        uint4 x[PASSES];
        float factor[PASSES];
        float top = 0.0f;
        bool nan = false;
#pragma unroll
        for (int y = 0; y < PASSES; ++y) {
            const int r = y * ROWS + sub;
            const size_t from = __shfl_sync(0xffffffffu, at, r);
            factor[y] = fabsf(__shfl_sync(0xffffffffu, scale, r));
            x[y] = make_uint4(0u, 0u, 0u, 0u);
            if (r >= lo && r < hi && piece * 16 < ld) x[y] = *reinterpret_cast<const uint4*>(codes + from + piece * 16);
        }
#pragma unroll
        for (int y = 0; y < PASSES; ++y) {
            // magnitudes order as codes do
            const uint32_t w[4] = {x[y].x, x[y].y, x[y].z, x[y].w};
            uint32_t most = 0;
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                const uint32_t clean = without_nans(w[z]);
                nan |= clean != w[z];
                most = __vmaxu4(most, clean & 0x7f7f7f7fu);
            }
            most = __vmaxu4(most, most >> 16);
            most = max(most & 0xffu, most >> 8 & 0xffu);
            top = fmaxf(top, from_e4m3x4(most).x * factor[y]);
        }
        const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
        nan = __any_sync(0xffffffffu, nan);
        // bits: m 2^e, 1 <= m < 2, and 448 = 1.75 2^8
        int E = min(max((int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), kLeastExp), kMostExp);
        if (lo > 0) {
            // older rows: the scale does not shrink under them, and their codes follow it when it grows
            const float had = *to_scale;
            const int Eold = min(max((int)((__float_as_uint(had) >> 23) & 0xffu) - 127, kLeastExp), kMostExp);
            nan |= had < 0.0f;
            if (E > Eold) {
                const float down = pow2(max(Eold - E, -126));
                for (int r = sub; r < lo; r += ROWS)
                    if (piece * 16 < ld) {
                        uint4* old = reinterpret_cast<uint4*>(to + (size_t)r * ld + piece * 16);
                        const uint4 w = *old;
                        auto again = [&](uint32_t q) {
                            const float4 v = from_e4m3x4(q);
                            return to_e4m3x4(v.x * down, v.y * down, v.z * down, v.w * down);
                        };
                        *old = make_uint4(again(w.x), again(w.y), again(w.z), again(w.w));
                    }
            }
            E = max(E, Eold);
        }
        __syncwarp();      // every lane has read the block, and its scale
        const float up = pow2(-E);
#pragma unroll
        for (int y = 0; y < PASSES; ++y) {
            const int r = y * ROWS + sub;
            if (r < lo || r >= hi || piece * 16 >= ld) continue;
            const float f = factor[y] * up;
            auto again = [&](uint32_t q) {
                const float4 v = from_e4m3x4(q);
                return to_e4m3x4(v.x * f, v.y * f, v.z * f, v.w * f);
            };
            *reinterpret_cast<uint4*>(to + (size_t)r * ld + piece * 16) = make_uint4(again(x[y].x), again(x[y].y), again(x[y].z), again(x[y].w));
        }
        if (lane == 0) *to_scale = nan ? -pow2(E) : pow2(E);
        __syncwarp();
    }
}

// ---- pages ----
// Codes and scales of pages pair[i].x into pages pair[i].y, of every layer.  A block of threads per (16 KB of codes, or a page's scales; pair; layer), all of its loads at once.
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
