// Launches of the 8-bit key/value cache's attention: which kernel takes which rows, with what grid.  Included by cache8.cu (rows whose positions are their places) and
// cache8_drafts.cu (rows of a tree).
#pragma once

#include <algorithm>
#include <atomic>
#include <utility>

#include "cache8_few.cuh"
#include "cache8_rows.cuh"
#include "cache8_tiles.cuh"
#include "tmap_host.h"

namespace smol {
namespace c8 {

// Every kernel here begins with the wait for the kernel in front of it, so all of them may be set up early.
template <class... P, class... X>
static cudaError_t launch_cluster(int cluster, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, X&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(std::forward<X>(args))...);
}
template <class... P, class... X>
static cudaError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, X&&... args) {
    return launch_cluster(1, kernel, grid, block, smem, st, std::forward<X>(args)...);
}

// Shared memory above 48 KB, a few of which are static, is asked for once per kernel and device.
template <class K>
static cudaError_t more_smem(K kernel, int bytes, std::atomic<uint64_t>& asked) {
    if (bytes <= 40 * 1024) return cudaSuccess;
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return e;
    if (dev < 64 && (asked.load() >> dev & 1)) return cudaSuccess;
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return e;
    if (dev < 64) asked.fetch_or(1ull << dev);
    return cudaSuccess;
}

// Query rows of a sequence and key/value head up to which the kernel for few rows takes them: it reads the keys once per 16 rows and shares them out finely, the
// tiles pay for 128 rows whatever they hold.  Both measured, few rows / tiles, 8 heads of 128: 16 sequences at 4096 positions with 16 rows 54 / 72 us,
// 24 rows 86 / 74, 32 rows 88 / 74; 64 at 2048 84 / 140, 164 / 141, 161 / 143; one at 32768 30 / 43, 49 / 44, 50 / 44.  Where all of it is too little
// to fill the GPU the keys' shares are what counts: one at 2048 with 32 rows 16.6 / 16.6, with 64 18.1 / 19.6, with 96 33 / 21.
constexpr int kFewMost = 16, kFewMostSmall = 64;
constexpr long long kSmall = 1 << 16;      // sequences times heads times positions (16384: the last of these; 262144: the one at 32768)
// Rows of a tree that the kernel for 32 rows takes (cache8_quads.cuh), and otherwise one of those for few or many.  64 sequences at up to 8192 positions, 8 heads of 128, few / 32 rows / tiles: 8 rows 168 / 208 /
// 399 us, 16 rows 247 / 208 / 399, 32 rows 485 / 213 / 408, 64 rows - / 383 / 400.  (It has no form for rows without a tree.)
constexpr int kQuadLeast = 8, kQuadMost = 64, kQuadRows = 32;
inline bool quads_serve(const AttendArgs& A, bool f32) {
    const long long rows = A.b.max_new * (long long)(A.H / A.c.G);
    return A.tree_pos && !f32 && std::max(A.c.d, A.c.dv) <= 128 && rows > kQuadLeast && rows <= kQuadMost;
}
inline bool tiles_serve(const AttendArgs& A, bool f32) {
    if (quads_serve(A, f32)) return false;
    const long long rows = A.b.max_new * (long long)(A.H / A.c.G), most = (long long)A.b.S * A.c.G * A.b.max_len <= kSmall ? kFewMostSmall : kFewMost;
    return !f32 && rows > most;
}

// query rows of a block of threads
static int row_tile(const AttendArgs& A, bool f32) {
    const long long rows = A.b.max_new * (long long)(A.H / A.c.G);
    return f32 ? kRowTile : quads_serve(A, f32) ? kQuadRows : rows <= 4 ? 4 : rows <= 8 ? 8 : tiles_serve(A, f32) ? kTileRows : 16;
}
static int row_tiles(const AttendArgs& A, bool f32) { return (int)((A.b.max_new * (long long)(A.H / A.c.G) + row_tile(A, f32) - 1) / row_tile(A, f32)); }

// Rows of a head's codes, page by page: boxes of 128 bytes by `box` positions; bytes behind the row read as zeros.
static bool codes_map(CUtensorMap* map, const uint8_t* base, int ld, size_t page_bytes, const Cache& c, int box) {
    TensorMapEncodeTiledFn encode = tensor_map_encoder();
    if (!encode) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)ld, (cuuint64_t)c.G * c.page, (cuuint64_t)c.n_pages}, strides[2] = {(cuuint64_t)ld, (cuuint64_t)page_bytes};
    const cuuint32_t boxes[3] = {128u, (cuuint32_t)box, 1u}, ones[3] = {1u, 1u, 1u};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(base), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// positions that lie together and begin at a multiple of themselves: the largest power of two that divides the page, at most a step's
static int box_of(const Cache& c) { return std::min(c.page & -c.page, kStep); }

// A block of 32 rows has an SM to itself, and a cluster's blocks have to lie in one part of the GPU: more than some 96 of them are not held at once (16 clusters of 8, 64 rows behind
// 32768 positions: 78 us; in nine shares through memory 40).
constexpr int kQuadClusters = 96;
static bool joins_in_cluster(const AttendArgs& A, int splits, bool f32) {
    if (quads_serve(A, f32) && (long long)A.b.S * A.c.G * row_tiles(A, f32) * splits > kQuadClusters) return false;
    return !f32 && !tiles_serve(A, f32) && splits > 1 && splits <= kMostCluster;
}

template <int D, int RA, bool BENT, bool TREE>
static cudaError_t few_as(const AttendArgs& A, cudaStream_t st) {
    static std::atomic<uint64_t> asked{0};
    constexpr int bytes = few_smem(D, RA);
    if (cudaError_t e = more_smem(attend_few_kernel<D, RA, BENT, TREE>, bytes, asked)) return e;
    CUtensorMap kmap, vmap;
    const int box = box_of(A.c);
    if (!codes_map(&kmap, A.c.k, A.c.ldk, A.c.k_page, A.c, box) || !codes_map(&vmap, A.c.v, A.c.ldv, A.c.v_page, A.c, box)) return cudaErrorInvalidValue;
    return launch_cluster(joins_in_cluster(A, A.n_splits, false) ? A.n_splits : 1, attend_few_kernel<D, RA, BENT, TREE>, dim3(row_tiles(A, false) * A.n_splits, A.c.G, A.b.S), kFewThreads, bytes, st, A, kmap,
                          vmap, box);
}
template <int D, int RA, bool TREE>
static cudaError_t few_of(const AttendArgs& A, cudaStream_t st) { return plain_scores(A) ? few_as<D, RA, false, TREE>(A, st) : few_as<D, RA, true, TREE>(A, st); }
template <int D, bool TREE>
static cudaError_t few_rows(const AttendArgs& A, cudaStream_t st) {
    if (row_tile(A, false) == 4) return few_of<D, 4, TREE>(A, st);
    if (row_tile(A, false) == 8) return few_of<D, 8, TREE>(A, st);
    if constexpr (TREE && D <= 128) return cudaErrorInvalidValue;      // (the kernel for 32 rows)
    else return few_of<D, 16, TREE>(A, st);
}
template <bool TREE>
static cudaError_t attend_few(const AttendArgs& A, cudaStream_t st) { return std::max(A.c.d, A.c.dv) <= 128 ? few_rows<128, TREE>(A, st) : few_rows<256, TREE>(A, st); }

template <int D, bool BENT, bool TREE>
static cudaError_t rows_as(const AttendArgs& A, cudaStream_t st) {
    static std::atomic<uint64_t> asked{0};
    constexpr int bytes = row_smem(D, D);
    if (cudaError_t e = more_smem(attend_rows_kernel<D, D, BENT, TREE>, bytes, asked)) return e;
    return launch(attend_rows_kernel<D, D, BENT, TREE>, dim3(row_tiles(A, true) * A.n_splits, A.c.G, A.b.S), kRowThreads, bytes, st, A);
}
template <int D, bool TREE>
static cudaError_t rows_of(const AttendArgs& A, cudaStream_t st) { return plain_scores(A) ? rows_as<D, false, TREE>(A, st) : rows_as<D, true, TREE>(A, st); }
template <bool TREE>
static cudaError_t attend_rows(const AttendArgs& A, cudaStream_t st) {
    const int d = std::max(A.c.d, A.c.dv);
    return d <= 64 ? rows_of<64, TREE>(A, st) : d <= 128 ? rows_of<128, TREE>(A, st) : rows_of<256, TREE>(A, st);
}

template <int DK, bool BENT, bool TREE>
static cudaError_t tiles_as(const AttendArgs& A, cudaStream_t st) {
    static std::atomic<uint64_t> asked{0};
    constexpr int bytes = tile_smem(DK);
    if (cudaError_t e = more_smem(attend_tiles_kernel<DK, BENT, TREE>, bytes, asked)) return e;
    CUtensorMap kmap, vmap;
    const int box = box_of(A.c);
    if (!codes_map(&kmap, A.c.k, A.c.ldk, A.c.k_page, A.c, box) || !codes_map(&vmap, A.c.v, A.c.ldv, A.c.v_page, A.c, box)) return cudaErrorInvalidValue;
    return launch(attend_tiles_kernel<DK, BENT, TREE>, dim3(row_tiles(A, false) * ((A.c.dv + 127) / 128) * A.n_splits, A.c.G, A.b.S), kTileThreads, bytes, st, A, kmap, vmap, box);
}
template <bool TREE>
static cudaError_t attend_tiles(const AttendArgs& A, cudaStream_t st) {
    if (A.c.d <= 128) return plain_scores(A) ? tiles_as<128, false, TREE>(A, st) : tiles_as<128, true, TREE>(A, st);
    return plain_scores(A) ? tiles_as<256, false, TREE>(A, st) : tiles_as<256, true, TREE>(A, st);
}

}  // namespace c8
}  // namespace smol
