// Drafting and forking on the 8-bit key/value cache: attention of rows of a tree, trees' layouts, rows and pages that move.
#include <new>
#include <vector>

#include "../../include/smoltts_b200_lm.h"
#include "cache8_launch.cuh"
#include "cache8_moves.cuh"
#include "lm_report.h"

#define SMOL_OK 0
#define SMOL_ERR_INVALID (-1)
#define SMOL_ERR_CUDA (-3)
#define SMOL_ERR_CAPACITY (-5)

namespace smol {
namespace c8 {

using lm::report;

cudaError_t attend_tree_few(const AttendArgs& A, cudaStream_t st) {
    return quads_serve(A, false) ? attend_tree_quads(A, st) : attend_few<true>(A, st);
}
cudaError_t attend_tree_tiles(const AttendArgs& A, cudaStream_t st) { return attend_tiles<true>(A, st); }
cudaError_t attend_tree_rows(const AttendArgs& A, cudaStream_t st) { return attend_rows<true>(A, st); }

// Caches first .. of `n` as layers of one launch: all of the first one's shape, and none twice.
static int layers_of(const SmolLmCache8* caches, int n, const char* me) {
    Cache shape, c;
    for (int i = 0; i < n; ++i) {
        if (int rc = cache_of(&caches[i], i == 0 ? shape : c, me)) return rc;
        if (i == 0) continue;
        if (c.n_pages != shape.n_pages || c.page != shape.page || c.G != shape.G || c.d != shape.d || c.dv != shape.dv || c.k_page != shape.k_page || c.v_page != shape.v_page ||
            c.ks_page != shape.ks_page || c.vs_page != shape.vs_page)
            return report(SMOL_ERR_INVALID, me, "caches of different shapes");
        for (int j = 0; j < i; ++j)
            if (caches[j].k == caches[i].k || caches[j].v == caches[i].v || caches[j].k_scale == caches[i].k_scale || caches[j].v_scale == caches[i].v_scale)
                return report(SMOL_ERR_INVALID, me, "a cache comes twice");
    }
    return SMOL_OK;
}
static void take_layers(Layers& l, const SmolLmCache8* caches, int n, const char* me) {
    cache_of(caches, l.c, me);
    l.n = n;
    for (int i = 0; i < n; ++i) l.of[i] = Layer{static_cast<uint8_t*>(caches[i].k), static_cast<uint8_t*>(caches[i].v), caches[i].k_scale, caches[i].v_scale, caches[i].err};
}

static cudaError_t keep(const KeepArgs& A, cudaStream_t st) {
    const int ld = std::max(A.l.c.ldk, A.l.c.ldv);
    const dim3 grid((A.l.c.G + kKeepWarps - 1) / kKeepWarps, A.S, A.l.n);
    return ld <= 64 ? launch(keep_kernel<2>, grid, kKeepWarps * 32, 0, st, A) : ld <= 128 ? launch(keep_kernel<4>, grid, kKeepWarps * 32, 0, st, A) : launch(keep_kernel<8>, grid, kKeepWarps * 32, 0, st, A);
}

// Whether the pages are there, no page is written twice, and none is read that is written.
static int pairs_of(const int32_t* src, const int32_t* dst, int n, int n_pages, const char* me) {
    for (int i = 0; i < n; ++i)
        if (src[i] < 0 || src[i] >= n_pages || dst[i] < 0 || dst[i] >= n_pages) return report(SMOL_ERR_INVALID, me, "a page outside the cache");
    const char* twice = "a page is written twice, or read and written";
    if (n <= 32) {
        for (int i = 0; i < n; ++i)
            for (int j = 0; j < n; ++j)
                if (src[j] == dst[i] || (j != i && dst[j] == dst[i])) return report(SMOL_ERR_INVALID, me, twice);
        return SMOL_OK;
    }
    try {
        std::vector<bool> written((size_t)n_pages, false);
        for (int i = 0; i < n; ++i) {
            if (written[dst[i]]) return report(SMOL_ERR_INVALID, me, twice);
            written[dst[i]] = true;
        }
        for (int i = 0; i < n; ++i)
            if (written[src[i]]) return report(SMOL_ERR_INVALID, me, twice);
    } catch (const std::bad_alloc&) {
        return report(SMOL_ERR_CAPACITY, me, "out of host memory");
    }
    return SMOL_OK;
}

}  // namespace c8
}  // namespace smol

using namespace smol::c8;
using smol::lm::report;

extern "C" int smol_lm_cache8_tree(const SmolLmCache8Tree* a, void* stream) {
    const char* me = "smol_lm_cache8_tree";
    if (!a || !a->seq_start || !a->seq_pos0 || !a->parents || !a->positions || !a->sees || !a->err) return report(SMOL_ERR_INVALID, me, "null argument");
    if (a->n_tokens < 1 || a->n_seqs < 1 || a->max_new < 1) return report(SMOL_ERR_INVALID, me, "n_tokens, n_seqs and max_new must be positive");
    if (a->max_new > kTreeRows) return report(SMOL_ERR_CAPACITY, me, "more than 4096 rows of a sequence");
    if (a->words < (a->max_new + 31) / 32) return report(SMOL_ERR_INVALID, me, "fewer words than max_new bits");
    TreeArgs A{};
    A.b.start = a->seq_start; A.b.pos0 = a->seq_pos0; A.b.S = a->n_seqs; A.b.T = a->n_tokens; A.b.max_new = a->max_new;
    A.parents = a->parents; A.positions = a->positions; A.sees = a->sees; A.words = a->words; A.err = a->err;
    const cudaError_t e = launch(tree_kernel, a->n_seqs, std::min(1024, (a->max_new + 31) / 32 * 32), 0, static_cast<cudaStream_t>(stream), A);
    return e == cudaSuccess ? SMOL_OK : report(SMOL_ERR_CUDA, me, cudaGetErrorString(e));
}

extern "C" int smol_lm_cache8_keep(const SmolLmCache8* caches, int32_t n_caches, const SmolLmCache8Keep* a, void* stream) {
    const char* me = "smol_lm_cache8_keep";
    if (!caches || !a || n_caches < 1) return report(SMOL_ERR_INVALID, me, "null argument, or no cache");
    if (int rc = layers_of(caches, n_caches, me)) return rc;
    if (!a->seq_pos0 || !a->block_table || !a->rows || !a->counts) return report(SMOL_ERR_INVALID, me, "null array");
    if (a->n_seqs < 1 || a->max_pages < 1 || a->max_keep < 1) return report(SMOL_ERR_INVALID, me, "n_seqs, max_pages and max_keep must be positive");
    if (a->n_seqs > 65535) return report(SMOL_ERR_CAPACITY, me, "more than 65535 sequences");
    KeepArgs A{};
    A.pos0 = a->seq_pos0; A.table = a->block_table; A.rows = a->rows; A.counts = a->counts;
    A.S = a->n_seqs; A.max_pages = a->max_pages; A.most = a->max_keep;
    for (int i = 0; i < n_caches; i += kMoveLayers) {
        take_layers(A.l, caches + i, std::min(n_caches - i, kMoveLayers), me);
        if (cudaError_t e = keep(A, static_cast<cudaStream_t>(stream))) return report(SMOL_ERR_CUDA, me, cudaGetErrorString(e));
    }
    return SMOL_OK;
}

extern "C" int smol_lm_cache8_copy_pages(const SmolLmCache8* caches, int32_t n_caches, const int32_t* src, const int32_t* dst, int32_t n_pairs, void* stream) {
    const char* me = "smol_lm_cache8_copy_pages";
    if (!caches || n_caches < 1 || n_pairs < 0 || (n_pairs > 0 && (!src || !dst))) return report(SMOL_ERR_INVALID, me, "null argument, or no cache");
    if (int rc = layers_of(caches, n_caches, me)) return rc;
    if (int rc = pairs_of(src, dst, n_pairs, caches[0].n_pages, me)) return rc;
    CopyArgs A;
    for (int i = 0; i < n_caches; i += kMoveLayers) {
        take_layers(A.l, caches + i, std::min(n_caches - i, kMoveLayers), me);
        const Cache& c = A.l.c;
        const size_t rows = (size_t)c.G * c.page;
        A.k_parts = (int)((rows * c.ldk + kCopyBytes - 1) / kCopyBytes);
        A.v_parts = (int)((rows * c.ldv + kCopyBytes - 1) / kCopyBytes);
        for (int j = 0; j < n_pairs; j += kCopyPairs) {
            const int n = std::min(n_pairs - j, kCopyPairs);
            for (int x = 0; x < n; ++x) A.pair[x] = make_int2(src[j + x], dst[j + x]);
            if (cudaError_t e = launch(copy_pages_kernel, dim3(A.k_parts + A.v_parts + 1, n, A.l.n), kCopyThreads, 0, static_cast<cudaStream_t>(stream), A))
                return report(SMOL_ERR_CUDA, me, cudaGetErrorString(e));
        }
    }
    return SMOL_OK;
}
