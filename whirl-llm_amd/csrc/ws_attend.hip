// The kernels of ws_attend.h, a translation unit of its own.
#define WS_NO_NAMED_KERNELS
#include "ws_attend.h"

namespace ws {

namespace {
struct Build {
    int dtype;
    uint32_t dim, cols;  // head_dim and columns up to which it is taken
    uint32_t each;       // workgroups a compute unit
    uint64_t part_floats;
    uint32_t subs;
    void (*run)(hipStream_t, const AttendArgs&);
};
template <int DT, int DP, int MS, int WM, int OCC>
void launch(hipStream_t s, const AttendArgs& a) {
    hipLaunchKernelGGL((attend_kernel<DT, DP, MS, WM, OCC>), dim3(a.groups), dim3(kAttendThreads), 0, s, a);
    hipLaunchKernelGGL((attend_join_kernel<DT, DP, MS, WM>), dim3(a.groups, MS * WM), dim3(64 * kJoinWavesOf<WM>), 0, s, a);
}
template <int DT, int DP, int MS, int WM, int OCC>
constexpr Build build(uint32_t cols) {
    return Build{DT, DP, cols, OCC, AttendShape<DT, DP, MS, WM>::kPartFloats, MS * WM, &launch<DT, DP, MS, WM, OCC>};
}
constexpr uint32_t kAny = 0xffffffffu;
// Which build, by the columns of a sequence's kv head: the quickest of those below. us, 16 sequences of 8192 positions, 8 kv heads, four waves apart / one tile of columns / two tiles:
//   128 bf16: 16 columns 117 / 121 / 141, 20 143 / 121 / 141, 64 205 / 125 / 146, 68 464 / 155 / 146, 256 - / 269 / 202;  64 bf16: 16 52 / 55 / 58, 20 65 / 56 / 59, 64 145 / 56 / 62, 68 209 / 80 / 64
//   (4 columns of 64 sequences of 2200 59 / 55, of 256 of 1000 116 / 102, of one of 4096 15.2 / 14.7: no waves apart);
//   256 bf16: 16 192 / 232, 32 210 / 237, 36 529 / 241;  64 fp32: 16 116 / 118 / 182, 32 145 / 167 / 182, 36 299 / 170 / 288, 68 472 / 336 / 293;
//   128 fp32: 4 and 16 columns 189 / 200, 32 268 / 305, 64 - / 315, 4 of one sequence of 4096 24 / 27 (four waves apart take a unit's registers alone: a build more for a twentieth, not kept);
//   256 fp32: 4 to 16 columns 823 / 701, 32 1469 / 708 (four waves apart spill 275 registers)
constexpr Build kBuilds[] = {
    build<1, 64, 1, 4, 2>(64), build<1, 64, 2, 4, 2>(kAny),
    build<1, 128, 1, 1, 2>(16), build<1, 128, 1, 4, 2>(64), build<1, 128, 2, 4, 2>(kAny),
    build<1, 256, 1, 1, 1>(32), build<1, 256, 1, 4, 1>(kAny),
    build<0, 64, 1, 1, 2>(32), build<0, 64, 1, 4, 2>(64), build<0, 64, 2, 4, 2>(kAny),
    build<0, 128, 1, 4, 2>(kAny), build<0, 256, 1, 4, 1>(kAny),
};
}  // namespace

int prepare_attend() {
    hipFuncAttributes fa;
    return static_cast<int>(hipFuncGetAttributes(&fa, reinterpret_cast<const void*>(&attend_kernel<1, 128, 1, 1, 2>)));
}

AttendPlan attend_plan(int dtype, uint32_t head_dim, uint32_t cols, uint32_t compute_units) {
    AttendPlan p{};
    for (const Build& b : kBuilds) {
        if (b.dtype == dtype && head_dim <= b.dim && cols <= b.cols) {
            p.build = static_cast<uint32_t>(&b - kBuilds);
            p.groups = compute_units * b.each;
            p.part_bytes = uint64_t{p.groups} * 2u * b.part_floats * 4u;
            p.bytes = p.part_bytes + uint64_t{p.groups} * sizeof(AttendRun);
            return p;
        }
    }
    return p;
}

int launch_attend(hipStream_t stream, const AttendPlan& plan, const AttendArgs& a) {
    kBuilds[plan.build].run(stream, a);
    return static_cast<int>(hipGetLastError());
}

}  // namespace ws
