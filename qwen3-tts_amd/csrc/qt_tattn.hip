// qt_tattn.hip — the kernels of attention for trees of drafted tokens over a paged cache of 16 bits.
#include "qt_pattn.h"

template <typename QT, int HD> static hipError_t launch(const AttArgs &a, const AttPlan &plan, hipStream_t st) {
    typedef typename std::conditional<std::is_same<QT, QtF32>::value, QtBf16, QT>::type KT;
    const dim3 grid((unsigned)(plan.slots * a.nkv), a.splits);
    if (plan.kind == ATT_ONE && plan.stream) return qt_launch(k_att_one<QT, KT, HD, true, true, true>, grid, dim3(64 * ATT_WV), 0, st, a);
    if constexpr (sizeof(typename QT::elem) == 2)
        if (plan.kind == ATT_TILE) return qt_launch(k_att_tile<QT, HD, true, QT, true>, grid, dim3(256), 0, st, a);
    return qt_launch(k_att_one<QT, KT, HD, true, false, true>, grid, dim3(64 * ATT_WV), 0, st, a);
}

hipError_t att_launch_tree(const AttArgs &a, const AttPlan &plan, int dtype, int hd, hipStream_t st) {
    if (dtype == QWEN_HIP_DT_F32) return hd == 128 ? launch<QtF32, 128>(a, plan, st) : launch<QtF32, 64>(a, plan, st);
    if (dtype == QWEN_HIP_DT_BF16) return hd == 128 ? launch<QtBf16, 128>(a, plan, st) : launch<QtBf16, 64>(a, plan, st);
    return hd == 128 ? launch<QtF16, 128>(a, plan, st) : launch<QtF16, 64>(a, plan, st);
}
