// Attention of 9 to 64 rows of a tree over the 8-bit key/value cache: launches.  (A source of its own, which is compiled beside the others.)
#include "cache8_launch.cuh"
#include "cache8_quads.cuh"

namespace smol {
namespace c8 {

template <int DV, bool BENT>
static cudaError_t quads_as(const AttendArgs& A, cudaStream_t st) {
    static std::atomic<uint64_t> asked{0};
    if (cudaError_t e = more_smem(attend_quads_kernel<DV, BENT>, quad_smem(), asked)) return e;
    CUtensorMap kmap, vmap;
    const int box = box_of(A.c);
    if (!codes_map(&kmap, A.c.k, A.c.ldk, A.c.k_page, A.c, box) || !codes_map(&vmap, A.c.v, A.c.ldv, A.c.v_page, A.c, box)) return cudaErrorInvalidValue;
    return launch_cluster(A.in_cluster ? A.n_splits : 1, attend_quads_kernel<DV, BENT>, dim3(row_tiles(A, false) * A.n_splits, A.c.G, A.b.S), kQuadThreads, quad_smem(), st, A,
                          kmap, vmap, box);
}
template <int DV>
static cudaError_t quads_of(const AttendArgs& A, cudaStream_t st) { return plain_scores(A) ? quads_as<DV, false>(A, st) : quads_as<DV, true>(A, st); }
cudaError_t attend_tree_quads(const AttendArgs& A, cudaStream_t st) { return A.c.dv <= 64 ? quads_of<64>(A, st) : quads_of<128>(A, st); }

}  // namespace c8
}  // namespace smol
