// qt_pattn8.hip — the kernels of attention over a quantised paged cache, with and without trees of drafted tokens.
#include "qt_pattn.h"

template <typename QT, int HD, bool TREE>
static hipError_t launch(const AttArgs &a, const AttPlan &plan, hipStream_t st) {
    const dim3 grid((unsigned)(plan.slots * a.nkv), a.splits);
    if (plan.kind == ATT_ONE && plan.stream) return qt_launch(k_att_one<QT, QtE4m3, HD, true, true, TREE>, grid, dim3(64 * ATT_WV), 0, st, a);
    if constexpr (sizeof(typename QT::elem) == 2)
        if (plan.kind == ATT_TILE) return qt_launch(k_att_tile<QT, HD, true, QtE4m3, TREE>, grid, dim3(256), 0, st, a);
    return qt_launch(k_att_one<QT, QtE4m3, HD, true, false, TREE>, grid, dim3(64 * ATT_WV), 0, st, a);
}
template <typename QT> static hipError_t launch_hd(const AttArgs &a, const AttPlan &plan, int hd, bool tree, hipStream_t st) {
    if (tree) return hd == 128 ? launch<QT, 128, true>(a, plan, st) : launch<QT, 64, true>(a, plan, st);
    return hd == 128 ? launch<QT, 128, false>(a, plan, st) : launch<QT, 64, false>(a, plan, st);
}

hipError_t att_launch_codes(const AttArgs &a, const AttPlan &plan, int dtype, int hd, bool tree, hipStream_t st) {
    if (dtype == QWEN_HIP_DT_F32) return launch_hd<QtF32>(a, plan, hd, tree, st);
    if (dtype == QWEN_HIP_DT_BF16) return launch_hd<QtBf16>(a, plan, hd, tree, st);
    return launch_hd<QtF16>(a, plan, hd, tree, st);
}
