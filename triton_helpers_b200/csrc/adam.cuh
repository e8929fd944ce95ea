// Adam's update of one element and the packets it is done in, for the kernels that walk tensors.
#pragma once

#include "common.cuh"

namespace th {
namespace {

struct AdamScalars {
    float lr, beta1, beta2, eps;
    float bias1, bias2_sqrt;  // 1 - beta1^t, sqrt(1 - beta2^t)
    float grad_scale;         // multiplies the stored gradient (1 / loss scale / world size)
    int zero_grad;            // write zeros back into the gradient buffer
};

// One element.  A gradient that is not finite (a 16-bit sum that overflowed, a NaN from upstream)
// leaves the parameter and both moments as they were and is counted in `skipped`: one bad element
// must not turn into inf / inf = NaN in the parameter and poison every later step.
template <typename T>
__device__ __forceinline__ T adam_one(T p, T g_in, float &m, float &v, const AdamScalars &a, int &skipped) {
    const float g = to_float<T>(g_in) * a.grad_scale;
    if (!isfinite(g)) {
        ++skipped;
        return p;
    }
    m = a.beta1 * m + (1.f - a.beta1) * g;
    v = a.beta2 * v + (1.f - a.beta2) * g * g;
    const float denom = sqrtf(v) / a.bias2_sqrt + a.eps;
    return from_float<T>(to_float<T>(p) - (a.lr / a.bias1) * (m / denom));
}

// Adds n to the count of elements passed over, which stays at 2^31 - 1 (a step of 100 M parameters whose norm is not finite counts them all).  A thread adds only
// after it has seen less, 4096 at a time: with the 148 x 2048 threads that run at once the unsigned word stays below 2^31 + 1.3e9, and whoever
// takes it past the most brings it back.
__device__ __forceinline__ void count_skipped(int *total, int n) {
    constexpr unsigned kMost = 0x7fffffffu;
    unsigned *at = reinterpret_cast<unsigned *>(total);
    while (n > 0 && *reinterpret_cast<volatile unsigned *>(at) < kMost) {
        const unsigned piece = static_cast<unsigned>(min(n, 4096));
        if (atomicAdd(at, piece) + piece > kMost) atomicMin(at, kMost);
        n -= static_cast<int>(piece);
    }
}

// Elements of a parameter in one 16-byte packet, and the matching moments (float32: four, for twice the threads and half their
// registers of eight: 3.3 M parameters 34.2 -> 26.4 us)
template <typename T>
constexpr int kPacket = 16 / sizeof(T);
template <typename T>
struct __align__(16) Packet16 {
    T v[kPacket<T>];
};
template <int N>
struct __align__(16) Moments {
    float v[N];
};

}  // namespace
}  // namespace th
