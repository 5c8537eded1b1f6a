// The kernels of ws_cache.h, a translation unit of its own.
#define WS_NO_NAMED_KERNELS
#include "ws_cache.h"

namespace ws {

int prepare_cache() {
    hipFuncAttributes fa;
    return static_cast<int>(hipFuncGetAttributes(&fa, reinterpret_cast<const void*>(&cache_reserve_kernel)));
}

int launch_cache_reserve(hipStream_t stream, const PagesArgs& a) {
    hipLaunchKernelGGL(cache_reserve_kernel, dim3(1), dim3(WS_BLOCK), 0, stream, a);
    return static_cast<int>(hipGetLastError());
}

int launch_cache_fork(hipStream_t stream, const PagesArgs& a) {
    hipLaunchKernelGGL(cache_fork_kernel, dim3(1), dim3(WS_BLOCK), 0, stream, a);
    if (const int e = static_cast<int>(hipGetLastError()); e != 0) return e;
    hipLaunchKernelGGL(cache_copy_kernel, dim3(a.n, a.C.layers, 2), dim3(kMoveThreads), 0, stream, a);
    return static_cast<int>(hipGetLastError());
}

int launch_cache_release(hipStream_t stream, const PagesArgs& a) {
    hipLaunchKernelGGL(cache_release_kernel, dim3(1), dim3(WS_BLOCK), 0, stream, a);
    return static_cast<int>(hipGetLastError());
}

int launch_cache_keep(hipStream_t stream, const KeepArgs& a) {
    hipLaunchKernelGGL(cache_keep_kernel, dim3(a.n_seq, a.C.layers, 2), dim3(kMoveThreads), 0, stream, a);
    return static_cast<int>(hipGetLastError());
}

}  // namespace ws
