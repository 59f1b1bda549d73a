// Device pieces shared by the rotary kernels (gsp_pool_ops.hip, gsp_mrope.hip).
#pragma once

#include <hip/hip_runtime.h>

namespace gsp {

// Cosine and sine of a pair's angle, position times rate, times the rotation's
// scale.  The angle is formed and reduced to [-pi, pi] in fp64, so it stays
// exact at long positions; cosine and sine are fp32.  A scale of 1 leaves them
// exact.
__device__ inline void rope_angle(double pos, double rate, float mscale, float* c, float* s) {
    const double ang = pos * rate;
    const double r = ang - 6.283185307179586 * rint(ang * 0.15915494309189535);
    float sn, cn;
    sincosf((float)r, &sn, &cn);
    *c = cn * mscale;
    *s = sn * mscale;
}

__device__ inline void rope_turn(float x0, float x1, float c, float s, float* y0, float* y1) {
    *y0 = x0 * c - x1 * s;
    *y1 = x0 * s + x1 * c;
}

template <typename KT>
__device__ inline void store4(KT* p, const float4& x) {
    if constexpr (sizeof(KT) == 4) {
        *reinterpret_cast<float4*>(p) = x;
    } else {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        h4 h = {(_Float16)x.x, (_Float16)x.y, (_Float16)x.z, (_Float16)x.w};
        *reinterpret_cast<h4*>(p) = h;
    }
}

}  // namespace gsp
