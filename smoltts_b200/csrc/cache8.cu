// The 8-bit key/value cache: launches and the C entries of include/smoltts_b200_lm.h.
#include <algorithm>
#include <atomic>

#include "../../include/smoltts_b200_lm.h"
#include "cache8.cuh"
#include "cache8_append.cuh"
#include "cache8_launch.cuh"
#include "lm_report.h"

#define SMOL_OK 0
#define SMOL_ERR_INVALID (-1)
#define SMOL_ERR_CUDA (-3)
#define SMOL_ERR_UNSUPPORTED (-4)
#define SMOL_ERR_CAPACITY (-5)

namespace smol {
namespace c8 {

using lm::report;

template <class T, int PASSES, bool ODD>
static cudaError_t append_placed(const AppendArgs& A, dim3 grid, cudaStream_t st) {
    return A.places ? launch(append_kernel<T, PASSES, ODD, true>, grid, kAppendThreads, 0, st, A) : launch(append_kernel<T, PASSES, ODD, false>, grid, kAppendThreads, 0, st, A);
}
template <class T, int PASSES>
static cudaError_t append_of(const AppendArgs& A, dim3 grid, cudaStream_t st) { return A.pairs % 8 == 0 ? append_placed<T, PASSES, false>(A, grid, st) : append_placed<T, PASSES, true>(A, grid, st); }
template <class T>
static cudaError_t append_as(const AppendArgs& A, int n_sms, cudaStream_t st) {
    const int blocks = (A.b.max_new + 2 * kBlock - 2) / kBlock, units = 2 * A.c.G + A.H, warps = kAppendThreads / 32;
    // a block of threads per 16 positions while that fills the SMs a few times; its heads are shared out over several where it does not (10671 tokens of 48 heads,
    // 753 blocks: 54 us in two shares, 58 in one, 58 in four)
    const int most = (units + warps - 1) / warps, z = std::min<long long>(most, std::max<long long>(1, (8ll * n_sms + (long long)blocks * A.b.S - 1) / ((long long)blocks * A.b.S)));
    const dim3 grid(blocks, A.b.S, z);
    const int ld = std::max(A.c.ldk, A.c.ldv);
    return ld <= 64 ? append_of<T, 2>(A, grid, st) : ld <= 128 ? append_of<T, 4>(A, grid, st) : append_of<T, 8>(A, grid, st);
}
cudaError_t append(const AppendArgs& A, bool f32, int n_sms, int* launches, cudaStream_t st) {
    *launches += 1;
    return f32 ? append_as<float>(A, n_sms, st) : append_as<bf16>(A, n_sms, st);
}

// shares of the keys: one block of threads each
static int splits_for(const AttendArgs& A, bool f32, int n_sms) {
    const bool tiles = tiles_serve(A, f32);
    const long long halves = tiles ? (A.c.dv + 127) / 128 : 1, base = (long long)A.b.S * A.c.G * row_tiles(A, f32) * halves;      // blocks of a share
    long long keys = A.b.max_len;
    if (A.window > 0) keys = std::min(keys, (long long)A.window + A.b.max_new + A.first + 2 * kBlock);
    // As many shares as the SMs hold blocks at once, none of less than 256 keys (a token of 12 heads at 2048 positions, appended and
    // attended to: 10.9 us; with shares of 128, which are one step, 11.5; of 512 12.7).  More blocks than are held at once wait for whole others: one sequence at
    // 131072 34 us in 111 shares, 43 in 128.
    const int held = f32 ? 2 : tiles || quads_serve(A, f32) ? 1 : few_blocks(std::max(A.c.d, A.c.dv), row_tile(A, false));
    // (float32 rows of a tree: 64, a block of 16 for each of a block of threads' warps.  3 sequences of 63 rows at 922 positions 25.6 us, with 256 29.4; one of 12 rows 13.2 and 19.3)
    const long long slots = (long long)held * n_sms, least = f32 && A.tree_pos ? 64 : 256;
    auto at_once = [&](long long blocks) { return std::max(1ll, std::min({slots / blocks, (keys + least - 1) / least, (long long)kMaxSplits})); };
    long long want = at_once(base);
    // Rows of a tree, a little more than a cluster joins: eight, without the launch that joins shares in memory.  On the device that is within 0.9 us either way (4 to 32 rows of 8 heads of 128 at
    // 2100 to 4000 positions; 48 rows of 4 heads of 64 at 2063 11.4 us, in nine 12.3), on the host 3 us less.
    if (A.tree_pos && want > kMostCluster && want <= 2 * kMostCluster && joins_in_cluster(A, kMostCluster, f32)) want = kMostCluster;
    if (halves == 1) return (int)want;
    // Values of more than 128 columns take two blocks a tile, and so at most half as many shares at once: often fewer SMs at work, where two rounds of shorter shares may
    // take less time for all that they and their join cost.  In keys, with a block's own start at 512 and the join at 2048: 300 rows of 16 and 8 heads, 80 blocks, one share /
    // three at 4000 positions 75 / 90 us, at 6000 107 / 110, at 8000 134 / 127, at 20000 316 / 247; 420 rows, 112 blocks, one / two at 8000 134 / 176, at 32000 488 / 530.
    auto walk = [&](long long shares) { return (base * shares + slots - 1) / slots * ((keys + shares - 1) / shares + 512) + (shares > 1 ? 2048 : 0); };
    const long long more = at_once(base / halves);
    return (int)(walk(more) < walk(want) ? more : want);
}

// A batch whose sequences may bring anything from one row to many: those of few rows go to the kernel for few rows, which shares their keys out.  With short
// contexts (a tile walks 2048 positions in 35 us), one sequence, or as many rows as if all brought max_new, that is not worth a launch (8 us of 77 where it finds
// nothing to do: 16 sequences of 6 rows at 4096 positions).
static bool mixed(const AttendArgs& A, bool f32) {
    return tiles_serve(A, f32) && A.b.S > 1 && A.b.T < (long long)A.b.S * A.b.max_new && A.b.max_len > 2048 && A.H / A.c.G <= kFewMost && A.rows_most > kFewMost;
}

size_t attend_bytes(const AttendArgs& A, bool f32, int n_sms) {
    const int splits = splits_for(A, f32, n_sms);
    return splits == 1 || joins_in_cluster(A, splits, f32) ? 0 : (part_floats(A, splits) + 4ull * A.b.T * A.H * splits) * sizeof(float);
}
// There are shares only while blocks (of at most 128 rows) times shares are no more than the SMs hold, 3 each of at most 16 rows or 1 of 128.
size_t attend_bytes_most(int dv) { return (size_t)256 * kTileRows * ((dv + 3) / 4 * 4 + 4) * sizeof(float); }

cudaError_t attend(AttendArgs A, bool f32, int n_sms, void* workspace, int* launches, cudaStream_t st) {
    AttendArgs few = A;
    const bool two = mixed(A, f32);
    if (two) A.rows_over = kFewMost;
    A.n_splits = splits_for(A, f32, n_sms);
    A.part = static_cast<float*>(workspace);
    A.in_cluster = joins_in_cluster(A, A.n_splits, f32);
    if (cudaError_t e = A.tree_pos ? (f32 ? attend_tree_rows(A, st) : tiles_serve(A, f32) ? attend_tree_tiles(A, st) : attend_tree_few(A, st))
                                   : (f32 ? attend_rows<false>(A, st) : tiles_serve(A, f32) ? attend_tiles<false>(A, st) : attend_few<false>(A, st)))
        return e;
    *launches += 1;
    if (A.n_splits > 1 && !A.in_cluster) {
        *launches += 1;
        if (cudaError_t e = f32 ? launch(attend_join_kernel<float>, A.b.T * A.H, kJoinWarps * 32, 0, st, A) : launch(attend_join_kernel<bf16>, A.b.T * A.H, kJoinWarps * 32, 0, st, A)) return e;
    }
    if (!two) return cudaSuccess;
    few.rows_most = kFewMost;
    few.b.max_new = kFewMost / (A.H / A.c.G);
    few.n_splits = std::min(splits_for(few, f32, n_sms), kMostCluster);      // (joined without the workspace, which the tiles' shares may be in)
    // Nor does it go by kQuadClusters, which is about clusters against shares through memory: fewer shares are what is left here, and slower.  Trees of 16 rows beside one of 85, 8 heads of 128,
    // 8 shares / as many as make 96 blocks: one sequence at 32768 positions 60 / 70 us, two 76 / 95, seven at 8192 in two shares / one 76 / 96.
    few.part = nullptr;
    few.in_cluster = few.n_splits > 1;
    *launches += 1;
    return A.tree_pos ? attend_tree_few(few, st) : attend_few<false>(few, st);
}

// ---------------------------------------------------------------------------------------------------------------------

static bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

static int n_sms_of_device(int* n) {
    static std::atomic<int> known[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && dev < 64 && known[dev].load() > 0) { *n = known[dev].load(); return SMOL_OK; }
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return report(SMOL_ERR_CUDA, "8-bit cache", cudaGetErrorString(e));
    if (dev < 64) known[dev].store(*n);
    return SMOL_OK;
}

// whether rows of n elements are whole groups of eight on 16-byte boundaries, or of four as one load
static bool whole_eights(const void* p, size_t row, size_t head, int n, bool f32) { return n % 8 == 0 && (row | head) * (f32 ? 4 : 2) % 16 == 0 && aligned(p, 16); }
static bool whole_fours(const void* p, size_t row, size_t head, int n, bool f32) { return n % 4 == 0 && row % 4 == 0 && head % 4 == 0 && aligned(p, f32 ? 16 : 8); }
void note_alignment(AppendArgs& A, bool f32) {
    A.k_vec = whole_eights(A.k, A.k_row, A.k_head, A.c.d, f32);
    A.v_vec = whole_eights(A.v, A.v_row, A.v_head, A.c.dv, f32);
    A.q_vec = A.H == 0 || (whole_eights(A.q, A.q_row, A.q_head, A.c.d, f32) && whole_eights(A.q_out, A.o_row, A.o_head, A.c.d, f32));
}
void note_alignment(AttendArgs& A, bool f32) {
    A.q_vec = whole_eights(A.q, A.q_row, A.q_head, A.c.d, f32) ? 2 : whole_fours(A.q, A.q_row, A.q_head, A.c.d, f32) ? 1 : 0;
    A.o_vec = whole_eights(A.out, A.o_row, A.o_head, A.c.dv, f32) ? 2 : whole_fours(A.out, A.o_row, A.o_head, A.c.dv, f32) ? 1 : 0;
    A.held = (int)std::min<long long>((long long)A.b.max_pages * A.c.page, kPositions);
}

int cache_of(const SmolLmCache8* s, Cache& c, const char* me) {
    if (!s->k || !s->v || !s->k_scale || !s->v_scale || !s->err) return report(SMOL_ERR_INVALID, me, "null pointer in the cache");
    if (s->n_pages < 1 || s->page_size < kBlock || s->page_size % kBlock) return report(SMOL_ERR_INVALID, me, "page_size must be a multiple of 16, with at least one page");
    if (s->kv_heads < 1 || s->dim < 1 || s->vdim < 1) return report(SMOL_ERR_INVALID, me, "kv_heads, dim and vdim must be positive");
    if (s->dim > kMaxDim || s->vdim > kMaxDim) return report(SMOL_ERR_UNSUPPORTED, me, "head sizes above 256");
    if ((long long)s->kv_heads * s->page_size > 0x7fffffffll) return report(SMOL_ERR_UNSUPPORTED, me, "a page of more than 2^31 - 1 rows");      // (heads times positions: coordinates of the copies)
    if (s->kv_heads > 65535) return report(SMOL_ERR_UNSUPPORTED, me, "more than 65535 key/value heads");
    c.ldk = (s->dim + 15) / 16 * 16;
    c.ldv = (s->vdim + 15) / 16 * 16;
    const size_t scales = (size_t)s->kv_heads * (s->page_size / kBlock);
    c.k_page = s->k_page ? s->k_page : (size_t)s->kv_heads * s->page_size * c.ldk;
    c.v_page = s->v_page ? s->v_page : (size_t)s->kv_heads * s->page_size * c.ldv;
    c.ks_page = s->k_scale_page ? s->k_scale_page : scales;
    c.vs_page = s->v_scale_page ? s->v_scale_page : scales;
    if (!aligned(s->k, 16) || !aligned(s->v, 16) || c.k_page % 16 || c.v_page % 16 || !aligned(s->k_scale, 4) || !aligned(s->v_scale, 4))
        return report(SMOL_ERR_INVALID, me, "codes must lie on 16-byte boundaries, page by page");
    c.k = static_cast<uint8_t*>(s->k); c.v = static_cast<uint8_t*>(s->v); c.ks = s->k_scale; c.vs = s->v_scale;
    c.n_pages = s->n_pages; c.page = s->page_size; c.G = s->kv_heads; c.d = s->dim; c.dv = s->vdim; c.err = s->err;
    return SMOL_OK;
}
static int batch_of(const SmolLmCache8Batch* s, Batch& b, const char* me) {
    if (!s->seq_start || !s->seq_pos0 || !s->block_table) return report(SMOL_ERR_INVALID, me, "null array");
    if (s->n_seqs < 1 || s->n_tokens < 1 || s->max_pages < 1 || s->max_new < 1 || s->max_len < 1) return report(SMOL_ERR_INVALID, me, "n_seqs, n_tokens, max_pages, max_new and max_len must be positive");
    if (s->n_seqs > 65535) return report(SMOL_ERR_CAPACITY, me, "more than 65535 sequences");
    if (s->max_new > (1 << 24)) return report(SMOL_ERR_CAPACITY, me, "max_new above 2^24");
    b.start = s->seq_start; b.pos0 = s->seq_pos0; b.table = s->block_table; b.kv_len = s->kv_len;
    b.S = s->n_seqs; b.T = s->n_tokens; b.max_pages = s->max_pages; b.max_new = std::min(s->max_new, s->n_tokens); b.max_len = s->max_len;
    return SMOL_OK;
}
static int attend_of(const SmolLmCache8* c, const SmolLmCache8Batch* b, const SmolLmCache8Attend* a, AttendArgs& A, bool pointers) {
    const char* me = "smol_lm_cache8_attend";
    if (!c || !b || !a) return report(SMOL_ERR_INVALID, me, "null argument");
    if (int rc = cache_of(c, A.c, me)) return rc;
    if (int rc = batch_of(b, A.b, me)) return rc;
    if (a->dtype != SMOL_LM_BF16 && a->dtype != SMOL_LM_F32) return report(SMOL_ERR_INVALID, me, "dtype must be 0 (bf16) or 1 (f32)");
    if (a->heads < 1 || a->heads % A.c.G) return report(SMOL_ERR_INVALID, me, "heads must be a multiple of kv_heads");
    if ((long long)A.b.max_new * (a->heads / A.c.G) > (1ll << 30) || (long long)A.b.T * a->heads > (1ll << 31) - 64)
        return report(SMOL_ERR_CAPACITY, me, "more query rows than 32 bits count");
    if (a->window < 0 || a->first < 0 || !(a->softcap >= 0.0f) || a->softcap > 3.4e38f) return report(SMOL_ERR_INVALID, me, "window, first and softcap must not be negative, and softcap finite");
    if (!a->dist_r1 != !a->dist_r2) return report(SMOL_ERR_INVALID, me, "dist_r1 and dist_r2 come together");
    if (pointers && (!a->q || !a->out)) return report(SMOL_ERR_INVALID, me, "null queries or results");
    const bool f32 = a->dtype == SMOL_LM_F32;
    A.q = a->q; A.out = a->out; A.q_row = a->q_row; A.q_head = a->q_head; A.o_row = a->out_row; A.o_head = a->out_head;
    A.H = a->heads; A.window = a->window; A.first = a->first; A.scale = a->scale; A.softcap = a->softcap;
    A.sink = a->sink; A.slope = a->dist_slope; A.r1 = a->dist_r1; A.r2 = a->dist_r2; A.gate = a->gate; A.gate_row = a->gate_row; A.out_scale = a->out_scale;
    A.part = nullptr; A.n_splits = 1;
    A.rows_over = 0; A.rows_most = 0x7fffffff;
    A.tree_pos = a->tree_positions; A.tree_sees = a->tree_sees; A.tree_words = a->tree_words;
    if (!A.tree_pos != !A.tree_sees) return report(SMOL_ERR_INVALID, me, "tree_positions and tree_sees come together");
    if (A.tree_pos && A.tree_words < 1) return report(SMOL_ERR_INVALID, me, "a tree needs words of bits");
    note_alignment(A, f32);
    return SMOL_OK;
}

}  // namespace c8
}  // namespace smol

using namespace smol::c8;
using smol::lm::report;

extern "C" int smol_lm_cache8_append(const SmolLmCache8* cache, const SmolLmCache8Batch* batch, const SmolLmCache8Append* a, void* stream) {
    const char* me = "smol_lm_cache8_append";
    if (!cache || !batch || !a) return report(SMOL_ERR_INVALID, me, "null argument");
    AppendArgs A{};
    if (int rc = cache_of(cache, A.c, me)) return rc;
    if (int rc = batch_of(batch, A.b, me)) return rc;
    if (a->dtype != SMOL_LM_BF16 && a->dtype != SMOL_LM_F32) return report(SMOL_ERR_INVALID, me, "dtype must be 0 (bf16) or 1 (f32)");
    if (!a->k || !a->v || !a->q != !a->q_out || (a->q && a->heads < 1)) return report(SMOL_ERR_INVALID, me, "null keys or values, or queries without heads or a place to go");
    if (a->rot_dims < 0 || a->rot_dims % 2 || a->rot_dims > A.c.d || (a->rot_dims > 0 && !a->freq)) return report(SMOL_ERR_INVALID, me, "rot_dims must be even and at most dim, with frequencies");
    const bool f32 = a->dtype == SMOL_LM_F32;
    A.k = a->k; A.v = a->v; A.q = a->q; A.q_out = a->q_out;
    A.k_row = a->k_row; A.k_head = a->k_head; A.v_row = a->v_row; A.v_head = a->v_head;
    A.q_row = a->q_row; A.q_head = a->q_head; A.o_row = a->q_out_row; A.o_head = a->q_out_head;
    A.H = a->q ? a->heads : 0; A.freq = a->freq; A.pairs = a->rot_dims / 2; A.half = a->rot_half; A.mult = a->rot_mult;
    if (a->n_axes < 0 || (a->positions ? a->n_axes < 1 : a->n_axes > 0 || a->axis)) return report(SMOL_ERR_INVALID, me, "positions come with the number of their axes, and axes with positions");
    A.places = a->positions; A.axis = a->axis; A.n_axes = a->n_axes;
    note_alignment(A, f32);
    int n_sms = 0, launches = 0;
    if (int rc = n_sms_of_device(&n_sms)) return rc;
    const cudaError_t e = append(A, f32, n_sms, &launches, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SMOL_OK : report(SMOL_ERR_CUDA, me, cudaGetErrorString(e));
}

extern "C" int smol_lm_cache8_workspace_bytes(const SmolLmCache8* cache, const SmolLmCache8Batch* batch, const SmolLmCache8Attend* a, size_t* bytes) {
    if (!bytes) return report(SMOL_ERR_INVALID, "smol_lm_cache8_workspace_bytes", "null argument");
    AttendArgs A{};
    if (int rc = attend_of(cache, batch, a, A, false)) return rc;
    int n_sms = 0;
    if (int rc = n_sms_of_device(&n_sms)) return rc;
    *bytes = attend_bytes(A, a->dtype == SMOL_LM_F32, n_sms);
    return SMOL_OK;
}

extern "C" int smol_lm_cache8_attend(const SmolLmCache8* cache, const SmolLmCache8Batch* batch, const SmolLmCache8Attend* a, void* workspace, size_t workspace_bytes, void* stream) {
    AttendArgs A{};
    if (int rc = attend_of(cache, batch, a, A, true)) return rc;
    int n_sms = 0, launches = 0;
    if (int rc = n_sms_of_device(&n_sms)) return rc;
    const bool f32 = a->dtype == SMOL_LM_F32;
    const size_t need = attend_bytes(A, f32, n_sms);
    if (need > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < need)) return report(SMOL_ERR_CAPACITY, "smol_lm_cache8_attend", "workspace too small or not on a 16-byte boundary");
    const cudaError_t e = attend(A, f32, n_sms, workspace, &launches, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SMOL_OK : report(SMOL_ERR_CUDA, "smol_lm_cache8_attend", cudaGetErrorString(e));
}
