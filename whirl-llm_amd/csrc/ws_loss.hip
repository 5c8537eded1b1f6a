// The kernels of ws_loss.h, a translation unit of its own.
#define WS_NO_NAMED_KERNELS
#include "ws_loss.h"

namespace ws {

namespace {
constexpr uint32_t kScoreThreads = 256u, kGradThreads = 256u, kGradVectors = 2u, kPolicyThreads = 1024u;
// vectors of a workgroup's share: up to the first a wave takes them, up to the second and third 256 threads of policy_rows_kernel, beyond it 512 (fp32 rows that 64 parts of the third
// do not hold: 400 x 786 400 on one side of the border 589 us, x 786 416 on the other 707)
constexpr uint32_t kLeastShare = 4u * 64u, kSmallShare = 4u * 256u, kMostShare = 12u * 256u, kWideShare = 12u * 512u;
// (the longest rows that the entry points take, in vectors, and the 64 parts that can meet)
static_assert((1048575u / Elem<0>::kPer + 7u + 63u) / 64u + 7u <= kWideShare && (1048575u / Elem<1>::kPer + 7u + 63u) / 64u + 7u <= kMostShare);

template <int DT, bool ENT, bool MASK>
struct Score {
    static void go(hipStream_t s, const ScoreArgs& a) {
        if (a.per <= kLeastShare) hipLaunchKernelGGL((score_rows_kernel<DT, ENT, MASK, 64>), grid_of(a.parts, a.R.rows), dim3(64), 0, s, a);
        else hipLaunchKernelGGL((score_rows_kernel<DT, ENT, MASK, kScoreThreads>), grid_of(a.parts, a.R.rows), dim3(kScoreThreads), 0, s, a);
    }
};
template <int DT, bool ENT, bool MASK>
struct Grad {
    static void go(hipStream_t s, const GradArgs& a) {
        constexpr uint32_t each = kGradThreads * kGradVectors;
        const uint32_t chunks = (a.R.vocab / Elem<DT>::kPer + 7u + each - 1u) / each;  // (the vectors of a row: RowSpan)
        hipLaunchKernelGGL((grad_rows_kernel<DT, ENT, MASK, kGradThreads, kGradVectors>), grid_of(chunks, a.R.rows), dim3(kGradThreads), 0, s, a);
    }
};
// the builds of policy_rows_kernel: threads, vectors a thread
template <int DT, bool ENT, bool SLOPE, bool MASK, int T, int NV, int WAVES>
void rows(hipStream_t s, const RowsArgs& a) {
    hipLaunchKernelGGL((policy_rows_kernel<DT, ENT, SLOPE, MASK, T, NV, WAVES>), grid_of(a.parts, a.R.rows), dim3(T), 0, s, a);
}
template <int DT, bool ENT, bool MASK>
struct Rows {
    template <bool SLOPE>
    static void of_size(hipStream_t s, const RowsArgs& a) {
        const uint32_t share = a.per;
        if (share <= kLeastShare && a.parts == 1u) rows<DT, ENT, SLOPE, MASK, 64, 4, 6>(s, a);
        else if (share <= kSmallShare) rows<DT, ENT, SLOPE, MASK, 256, 4, 6>(s, a);
        else if (DT != 0 || share <= kMostShare) rows<DT, ENT, SLOPE, MASK, 256, 12, 5>(s, a);
        else if constexpr (DT == 0) rows<DT, ENT, SLOPE, MASK, 512, 12, 4>(s, a);
    }
    static void go(hipStream_t s, const RowsArgs& a, bool slope) {
        if constexpr (ENT) {
            if (slope) return of_size<true>(s, a);
        }
        of_size<false>(s, a);
    }
};
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
}  // namespace

// loads this file's kernels on the current device (the first launch would; under capture there is nothing left to do then)
int prepare_loss() {
    hipFuncAttributes fa;
    return static_cast<int>(hipFuncGetAttributes(&fa, reinterpret_cast<const void*>(&policy_kernel<kPolicyThreads>)));
}

uint32_t loss_most_share() { return kMostShare; }

int launch_score(hipStream_t stream, int dtype, const ScoreArgs& a) {
    by_kind<Score>(dtype, a.entropy != nullptr, a.R.allow != nullptr, stream, a);
    return static_cast<int>(hipGetLastError());
}

int launch_grad(hipStream_t stream, int dtype, const GradArgs& a) {
    by_kind<Grad>(dtype, a.d_entropy != nullptr, a.R.allow != nullptr, stream, a);
    return static_cast<int>(hipGetLastError());
}

int launch_policy_rows(hipStream_t stream, int dtype, const RowsArgs& a, bool slope) {
    by_kind<Rows>(dtype, a.entropy != nullptr, a.R.allow != nullptr, stream, a, slope);
    return static_cast<int>(hipGetLastError());
}

int launch_policy(hipStream_t stream, const PolicyArgs& a, unsigned groups) {
    hipLaunchKernelGGL(policy_kernel<kPolicyThreads>, dim3(groups), dim3(kPolicyThreads), 0, stream, a);
    return static_cast<int>(hipGetLastError());
}

int launch_preference(hipStream_t stream, const PreferenceArgs& a, unsigned groups) {
    hipLaunchKernelGGL(preference_kernel<512>, dim3(groups), dim3(512), 0, stream, a);
    return static_cast<int>(hipGetLastError());
}

}  // namespace ws
