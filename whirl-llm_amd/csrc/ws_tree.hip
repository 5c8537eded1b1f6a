// The kernels of ws_tree.h, a translation unit of its own.
#define WS_NO_NAMED_KERNELS
#include "ws_tree.h"

namespace ws {

namespace {
// vectors of a workgroup's share, by its build (the longest rows are 262144 vectors, of 64 parts at most)
constexpr uint32_t kSmall = 4u * 256u, kMost = 12u * 256u, kWide = 9u * 512u;
static_assert((1048575u / Elem<0>::kPer + 63u) / 64u + 8u <= kWide);

template <int DT, bool MASK, int T, int NV, int WAVES>
void verify(hipStream_t s, const TreeVerifyArgs& a) {
    hipLaunchKernelGGL((tree_draw_kernel<DT, MASK, T, NV, WAVES>), grid_of(a.parts, a.n_seq), dim3(T), 0, s, a);
}
template <int DT, bool MASK>
void of_size(hipStream_t s, const TreeVerifyArgs& a) {
    hipLaunchKernelGGL((tree_rows_kernel<DT, MASK>), grid_of(a.row_parts, a.levels * a.n_seq), dim3(kRowThreads), 0, s, a);
    if (a.per <= kSmall) verify<DT, MASK, 256, 4, 4>(s, a);
    else if (a.per <= kMost) verify<DT, MASK, 256, 12, 2>(s, a);
    else verify<DT, MASK, 512, 9, 2>(s, a);
}
}  // namespace

int prepare_tree() {
    hipFuncAttributes fa;
    return static_cast<int>(hipFuncGetAttributes(&fa, reinterpret_cast<const void*>(&tree_stage_kernel)));
}

uint32_t tree_most_share() { return kMost; }

int launch_tree_stage(hipStream_t stream, const TreeStageArgs& a) {
    hipLaunchKernelGGL(tree_stage_kernel, dim3(a.n_seq), dim3(64), 0, stream, a);
    return static_cast<int>(hipGetLastError());
}

int launch_tree_verify(hipStream_t stream, int dtype, const TreeVerifyArgs& a) {
    if (dtype == 0) a.R.allow ? of_size<0, true>(stream, a) : of_size<0, false>(stream, a);
    else a.R.allow ? of_size<1, true>(stream, a) : of_size<1, false>(stream, a);
    return static_cast<int>(hipGetLastError());
}

}  // namespace ws
