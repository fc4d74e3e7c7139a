// snn_update.h -- one element of the optimizers' updates: the kernels of snn_train.hip and, with the gradient scaled by the clipping
// coefficient besides, those of snn_clip.hip.
#pragma once
#include <hip/hip_runtime.h>

// torch.optim.Adam with L2 weight decay; bc1, bc2_sqrt: 1 - beta1^step, sqrt(1 - beta2^step)
__device__ __forceinline__ void adam_update(float gi, float* __restrict__ p, float* __restrict__ m, float* __restrict__ v, int64_t i, float lr,
                                            float beta1, float beta2, float eps, float weight_decay, float bc1, float bc2_sqrt)
{
    const float pi = p[i];
    if (weight_decay != 0.0f) gi = fmaf(weight_decay, pi, gi);
    const float mi = m[i] + (gi - m[i]) * (1.0f - beta1);          // lerp, as torch
    const float vi = beta2 * v[i] + (1.0f - beta2) * gi * gi;
    m[i] = mi;
    v[i] = vi;
    const float denom = sqrtf(vi) / bc2_sqrt + eps;
    p[i] = pi - (lr / bc1) * (mi / denom);
}
// torch.optim.SGD with momentum, dampening 0, no Nesterov
__device__ __forceinline__ void sgd_update(float gi, float* __restrict__ p, float* __restrict__ buf, int64_t i, float lr, float momentum,
                                           float weight_decay, int first)
{
    const float pi = p[i];
    if (weight_decay != 0.0f) gi = fmaf(weight_decay, pi, gi);
    if (momentum != 0.0f) {
        gi = first ? gi : fmaf(momentum, buf[i], gi);      // the first step copies the gradient into the buffer
        buf[i] = gi;
    }
    p[i] = pi - lr * gi;
}
