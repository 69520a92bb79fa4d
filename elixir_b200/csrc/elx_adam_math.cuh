// Part of the elixir_b200 CUDA library (C ABI: include/elixir_b200.h): what the update kernels share, whatever the
// form their moments are held in.
#pragma once

#include "elx_common.cuh"

namespace elx {

// Per-group constants derived once per CTA from ElxHyper and the device step counter.
struct GroupK {
    float lr, beta1, omb1, beta2, omb2, eps;
    float wd_l2;   // weight decay added to the gradient (L2 mode), 0 in decoupled mode
    float wd_w;    // weight decay added to the update (decoupled mode), 0 in L2 mode
    float bc1, bc2, rbc1, rbc2;
};

static __device__ __noinline__ GroupK derive_group(const ElxHyper& h, int step) {
    GroupK k;
    k.lr = h.lr;
    k.beta1 = h.beta1;
    k.beta2 = h.beta2;
    k.omb1 = 1.0f - h.beta1;
    k.omb2 = 1.0f - h.beta2;
    k.eps = h.eps;
    k.wd_l2 = h.adamw_mode ? 0.0f : h.weight_decay;
    k.wd_w = h.adamw_mode ? h.weight_decay : 0.0f;
    double bc1 = 1.0, bc2 = 1.0;
    if (h.bias_correction) {
        // 1 - beta^t evaluated in double from the fp32 betas, then rounded to fp32
        bc1 = 1.0 - pow(static_cast<double>(h.beta1), static_cast<double>(step));
        bc2 = 1.0 - pow(static_cast<double>(h.beta2), static_cast<double>(step));
    }
    k.bc1 = static_cast<float>(bc1);
    k.bc2 = static_cast<float>(bc2);
    k.rbc1 = static_cast<float>(1.0 / bc1);
    k.rbc2 = static_cast<float>(1.0 / bc2);
    return k;
}

// IEEE division and square root whose zero operands never reach the instruction sequence: __fdiv_rn and
// __fsqrt_rn handle a zero (like a denormal) on a slow path that a whole warp takes when one lane needs it, and
// states with many exact zeros -- moments of parameters that never had a gradient -- made a launch take twice as
// long (14.2 ms against 7.2 ms on an all-zero state).  For x = +-0 and y > 0 (inf included) the quotient is x itself,
// and the square root of +-0 is itself: the same bits as the plain operations, for every input.
__device__ __forceinline__ float div_or_zero(float x, float y) {
    const bool zero = x == 0.0f && y > 0.0f;
    const float q = __fdiv_rn(zero ? 1.0f : x, y);
    return zero ? x : q;
}
__device__ __forceinline__ float sqrt_or_zero(float x) {
    const bool zero = x == 0.0f;
    const float r = __fsqrt_rn(zero ? 1.0f : x);
    return zero ? x : r;
}

// How the gradient is unscaled in this launch.
enum { kNoDiv = 0, kMulInv = 1, kTrueDiv = 2 };

}  // namespace elx
