// The kernels of ws_loss.h, a translation unit of its own.
#define WS_NO_NAMED_KERNELS
#include "ws_loss.h"

namespace ws {

namespace {
constexpr uint32_t kScoreThreads = 256u, kGradThreads = 256u, kGradVectors = 4u;

template <int DT, bool ENT, bool MASK, bool POLICY>
void score(hipStream_t stream, const ScoreArgs& a) {
    hipLaunchKernelGGL((score_rows_kernel<DT, ENT, MASK, POLICY, kScoreThreads>), dim3(a.R.rows * a.parts), dim3(kScoreThreads), 0, stream, a);
}
template <int DT, bool ENT, bool MASK>
void grad(hipStream_t stream, const GradArgs& a) {
    hipLaunchKernelGGL((grad_rows_kernel<DT, ENT, MASK, kGradThreads, kGradVectors>), dim3(a.R.rows * a.chunks), dim3(kGradThreads), 0, stream, a);
}
template <int DT, bool ENT, bool SLOPE, bool MASK>
void rows(hipStream_t stream, const RowsArgs& b) {
    const uint32_t vectors = b.S.R.vocab / Elem<DT>::kPer;
    if (vectors <= 20u * 256u) hipLaunchKernelGGL((policy_rows_kernel<DT, ENT, SLOPE, MASK, 256, 20>), dim3(b.S.R.rows), dim3(256), 0, stream, b);
    else if (vectors <= 20u * 512u) hipLaunchKernelGGL((policy_rows_kernel<DT, ENT, SLOPE, MASK, 512, 20>), dim3(b.S.R.rows), dim3(512), 0, stream, b);
    else hipLaunchKernelGGL((policy_rows_kernel<DT, ENT, SLOPE, MASK, 1024, 19>), dim3(b.S.R.rows), dim3(1024), 0, stream, b);
}
template <template <int, bool, bool> class F, class... A>
void by_kind(int dtype, bool ent, bool mask, A&&... a) {
    if (dtype == 0) {
        if (ent) mask ? F<0, true, true>::go(a...) : F<0, true, false>::go(a...);
        else mask ? F<0, false, true>::go(a...) : F<0, false, false>::go(a...);
    } else {
        if (ent) mask ? F<1, true, true>::go(a...) : F<1, true, false>::go(a...);
        else mask ? F<1, false, true>::go(a...) : F<1, false, false>::go(a...);
    }
}
template <int DT, bool ENT, bool MASK>
struct Score {
    static void go(hipStream_t s, const ScoreArgs& a) { score<DT, ENT, MASK, false>(s, a); }
};
template <int DT, bool ENT, bool MASK>
struct ScorePolicy {
    static void go(hipStream_t s, const ScoreArgs& a) { score<DT, ENT, MASK, true>(s, a); }
};
template <int DT, bool ENT, bool MASK>
struct Grad {
    static void go(hipStream_t s, const GradArgs& a) { grad<DT, ENT, MASK>(s, a); }
};
template <int DT, bool ENT, bool MASK>
struct Rows {
    static void go(hipStream_t s, const RowsArgs& b, bool slope) {
        if constexpr (ENT) {
            if (slope) return rows<DT, true, true, MASK>(s, b);
        }
        rows<DT, ENT, false, MASK>(s, b);
    }
};
}  // namespace

uint32_t loss_grad_chunks(int dtype, uint32_t vocab) {
    const uint32_t vectors = vocab / (dtype == 0 ? 4u : 8u), each = kGradThreads * kGradVectors;
    return vectors ? (vectors + each - 1u) / each : 1u;
}
uint32_t loss_threads() { return kScoreThreads; }

int launch_score(hipStream_t stream, int dtype, const ScoreArgs& a, bool policy) {
    if (policy) by_kind<ScorePolicy>(dtype, a.entropy != nullptr, a.R.allow != nullptr, stream, a);
    else by_kind<Score>(dtype, a.entropy != nullptr, a.R.allow != nullptr, stream, a);
    return static_cast<int>(hipGetLastError());
}

int launch_grad(hipStream_t stream, int dtype, const GradArgs& a) {
    by_kind<Grad>(dtype, a.d_entropy != nullptr, a.R.allow != nullptr, stream, a);
    return static_cast<int>(hipGetLastError());
}

int launch_policy_rows(hipStream_t stream, int dtype, const RowsArgs& b, bool slope) {
    by_kind<Rows>(dtype, b.S.entropy != nullptr, b.S.R.allow != nullptr, stream, b, slope);
    return static_cast<int>(hipGetLastError());
}

int launch_policy(hipStream_t stream, const PolicyArgs& a, unsigned groups) {
    hipLaunchKernelGGL(policy_kernel<512>, dim3(groups), dim3(512), 0, stream, a);
    return static_cast<int>(hipGetLastError());
}

int launch_preference(hipStream_t stream, const PreferenceArgs& a, unsigned groups) {
    hipLaunchKernelGGL(preference_kernel<512>, dim3(groups), dim3(512), 0, stream, a);
    return static_cast<int>(hipGetLastError());
}

}  // namespace ws
