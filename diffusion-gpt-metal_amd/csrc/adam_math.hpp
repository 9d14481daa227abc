// AdamW of one element, shared by the kernels of one tensor (train.hip) and of
// many (adam_many.hip), so that their results are the same bits.
#pragma once

#include <hip/hip_runtime.h>

namespace dgm {

struct AdamArgs {
    float lr, b1, b2, eps, wd, invBC1, invBC2;
};

// One element of adamw (metal/kernels.metal:795-801), literally.
__device__ __forceinline__ void adam_elem(float& w, float g, float& m, float& v, const AdamArgs& a) {
#pragma clang fp contract(off)
    const float mi = a.b1 * m + (1.0f - a.b1) * g;
    const float vi = a.b2 * v + (1.0f - a.b2) * g * g;
    m = mi;
    v = vi;
    const float upd = (mi * a.invBC1) / (sqrtf(vi * a.invBC2) + a.eps);
    w -= a.lr * (upd + a.wd * w);
}

}  // namespace dgm
