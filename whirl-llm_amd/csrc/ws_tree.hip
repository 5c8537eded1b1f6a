// The kernels of ws_tree.h, a translation unit of its own.
#define WS_NO_NAMED_KERNELS
#include "ws_tree.h"

namespace ws {

namespace {
// Vectors of a thread of the middle build: as many as leave three workgroups a compute unit (two of bf16, whose vectors have twice the powers). 256 rows of 50257 fp32, masked: 12 (five workgroups a
// row) 46 us, 17 (three, which all run at once) 41.
template <int DT>
constexpr uint32_t kMiddle = DT == 0 ? 17u : 12u;
// (the longest rows, in 64 parts, fit it)
static_assert((1048575u / Elem<0>::kPer + 63u) / 64u + 8u <= kMiddle<0> * kDrawThreads && (1048575u / Elem<1>::kPer + 63u) / 64u + 8u <= kMiddle<1> * kDrawThreads);
constexpr uint32_t kSmall = 4u;

template <int DT, bool MASK, int NV, int WAVES>
void draw(hipStream_t s, const TreeVerifyArgs& a) {
    hipLaunchKernelGGL((tree_draw_kernel<DT, MASK, NV, WAVES>), grid_of(a.parts, a.n_seq), dim3(kDrawThreads), 0, s, a);
}
template <int DT, bool MASK>
void of_size(hipStream_t s, const TreeVerifyArgs& a) {
    hipLaunchKernelGGL((tree_rows_kernel<DT, MASK>), grid_of(a.row_parts, a.levels * a.n_seq), dim3(kRowThreads), 0, s, a);
    if (a.per <= kSmall * kDrawThreads) draw<DT, MASK, kSmall, 4>(s, a);
    else draw<DT, MASK, kMiddle<DT>, DT == 0 ? 3 : 2>(s, a);
}
}  // namespace

int prepare_tree() {
    hipFuncAttributes fa;
    return static_cast<int>(hipFuncGetAttributes(&fa, reinterpret_cast<const void*>(&tree_stage_kernel)));
}

uint32_t tree_most_share(int dtype) { return kDrawThreads * (dtype == 0 ? kMiddle<0> : kMiddle<1>); }

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
