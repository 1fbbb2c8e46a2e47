// One element's Adam / AdamW update and its scalars, for the flat buffer (adam.hip)
// and for many tensors at once (adam_multi.hip).
#pragma once

#include "common.hpp"

#include <cmath>

namespace nott {
namespace adam {

struct AdamScalars {
    float beta1, beta2, one_m_b1, one_m_b2;
    float wd, decay;          // decay = 1 - lr*wd (AdamW)
    float neg_step;           // -(lr / bc1)
    float bc2_sqrt;           // sqrt(bc2)
    float eps;
};

// MODE 0: no weight decay; 1: Adam (L2 added to the gradient); 2: AdamW (decoupled).
template <int MODE>
__device__ __forceinline__ void adam_elem(float& p, float g, float& m, float& v, const AdamScalars& s) {
    // Only the explicit fmaf calls may fuse; p·decay must round before the
    // final add, as it does in the reference.
#pragma clang fp contract(off)
    if (MODE == 2) p = p * s.decay;
    if (MODE == 1) g = __builtin_fmaf(p, s.wd, g);
    const float mb = m * s.beta1;
    m = __builtin_fmaf(g, s.one_m_b1, mb);
    const float vb = v * s.beta2;
    const float ag = s.one_m_b2 * g;
    v = __builtin_fmaf(ag, g, vb);
    const float denom = __builtin_sqrtf(v) / s.bc2_sqrt + s.eps;
    const float num = s.neg_step * m;
    p = p + num / denom;
}

// The host's scalar set, written once for the device form: the same double
// arithmetic as nott_adam_step, rounded to float at the same places.
__host__ __device__ inline AdamScalars make_scalars(double lr, double beta1, double beta2, double eps, double wd,
                                                    int64_t step) {
    const double bc1 = 1.0 - pow(beta1, (double)step);
    const double bc2 = 1.0 - pow(beta2, (double)step);
    AdamScalars s;
    s.beta1 = (float)beta1;
    s.beta2 = (float)beta2;
    s.one_m_b1 = (float)(1.0 - beta1);
    s.one_m_b2 = (float)(1.0 - beta2);
    s.wd = (float)wd;
    s.decay = (float)(1.0 - lr * wd);
    s.neg_step = (float)(-(lr / bc1));
    s.bc2_sqrt = (float)sqrt(bc2);
    s.eps = (float)eps;
    return s;
}

// Device form of the host's scalar set: advances the step count held in
// device memory and forms the bias corrections from it and from the
// hyper-parameters {lr, beta1, beta2, eps, weight_decay} read at launch time.
static __global__ void adam_prep_kernel(const double* __restrict__ hp, nott_adam_device_state* __restrict__ st) {
    const int64_t t = st->step + 1;
    st->step = t;
    const AdamScalars s = make_scalars(hp[0], hp[1], hp[2], hp[3], hp[4], t);
    static_assert(sizeof(AdamScalars) <= sizeof(st->reserved), "scalar block size");
    *reinterpret_cast<AdamScalars*>(st->reserved) = s;
}

}  // namespace adam
}  // namespace nott
