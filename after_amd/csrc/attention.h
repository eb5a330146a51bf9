// What the attention kernels of attention.hip and kv4.hip share.
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>

namespace after {

// |scale| log2 e, for exponentials to the base 2; infinite beyond 2.35e38, which callers refuse.  Never 0, so that a masked score,
// -inf, stays -inf: with the smallest positive number in its place every score of 32 bits is within 2^-21 of 0.
inline float scale_log2(float scale) { return std::fmax(std::fabs(scale) * 1.44269504088896340736f, 0x1p-149f); }

// A softmax's running maximum is a product rounded to 32 bits, round(top * scale2), and fmaf(score, scale2, -maximum) rounds no
// product: at the largest score the two are up to 2^-24 of the maximum apart, more than an exponential's range holds from 2^32 on.
// Beyond this maximum, where that is 1/4, products are rounded before the difference.
constexpr float kFarTop = 0x1p22f;
__device__ __forceinline__ float scaled_below(float s, float scale2, float maximum) {
#pragma clang fp contract(off)
    const float x = s * scale2;
    return x - maximum;
}

// What a query's sum of exponentials divides by: nothing seen gives zeros, but where every score is -inf, 0 / 0 is NaN
__device__ __forceinline__ float inverse_sum(float sum, bool sees) { return sum == 0.f ? (sees ? NAN : 0.f) : 1.f / sum; }

}  // namespace after
