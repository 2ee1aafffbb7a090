// paged_quant.hpp -- a row of a key/value cache in 8 bits: the dims of one head at
// one position as codes, and the byte of their step.
//
//   s(b) = (8 + b % 8) 2^(b / 8 - 22),  b = the smallest byte in [0, 207] with
//   127 s(b) >= max|x|;  c = clamp(round(x / s), -127, 127) + 128;  x' = (c - 128) s
//
// round is half away from zero, as in the int8 schemes.  The step has four
// significant bits, so a value has eleven: the matrix products take it as f16
// without a rounding and without a factor per key afterwards.  That costs up to an
// eighth (4.5% on average) of the step max|x| / 127 would be.  Steps range from
// 2^-19 (rows below 2.4e-4) to 120 (up to 15240).
#pragma once

#include "common.hpp"

namespace gfh {
namespace paged {

constexpr int kMaxStep = 207;
// fp32 bits of s(b): (b + kStepBits) << 20
constexpr int kStepBits = (127 + 3 - 22) * 8;

__device__ __forceinline__ float step_of(int b) { return __uint_as_float((uint32_t)(min(b, kMaxStep) + kStepBits) << 20); }

// The byte for a row's largest magnitude.
__device__ __forceinline__ int step_byte(float most) {
    // a guess from the product, off by one where it rounds over a step; 127 s is exact
    const uint32_t x = __float_as_uint(most * (1.0f / 127.0f));
    int b = min(max((int)((x + 0xfffffu) >> 20) - kStepBits, 0), kMaxStep);
    b -= b > 0 && 127.0f * step_of(b - 1) >= most;
    b += b < kMaxStep && 127.0f * step_of(b) < most;
    return b;
}

// (a NaN counts as 0)
__device__ __forceinline__ uint32_t code_of(float x, float step) {
    const float y = roundf(x / step);
    return (uint32_t)(128 + (y != y ? 0 : (int)fminf(fmaxf(y, -127.0f), 127.0f)));
}

}  // namespace paged
}  // namespace gfh
