// quantize.cuh — the quantiser's arithmetic (quantize.cu, linear_i8.cu).
#pragma once

#include "block.cuh"

namespace ppdl {

// x / s rounded half to even, as the real quotient rounds, for a finite
// |x| <= about 200 s and s in [2^-64, 2^128): the FP32 product with 1 / s
// may land on the wrong side of a half, so the remainder of the rounded
// value decides.  r = x - q s is exact: x and q s are whole multiples of
// half a unit in the last place of s, and |r| is at most about s.
__device__ __forceinline__ int quantize(float x, float s, float inv) {
    float q = rintf(x * inv);
    const float r = __fmaf_rn(-q, s, x), h = 0.5f * s;
    const bool odd = ((int)q & 1) != 0;
    if (r > h || (r == h && odd)) q += 1.0f;
    if (r < -h || (r == -h && odd)) q -= 1.0f;
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

// What a row is divided by: its scale from the largest |x| (as the bits of
// |x|, whose unsigned order puts infinities and NaNs on top).  Scales below
// 2^-64 quantise x 2^64 by s 2^64, both exact, so that 1 / s is finite.
struct Divisor {
    float s, su, up, inv;
    bool usable;
    __device__ explicit Divisor(unsigned amax) {
        s = __fdiv_rn(__uint_as_float(amax), 127.0f);
        usable = s > 0.0f && amax < 0x7f800000u;
        up = s < 0x1p-64f ? 0x1p64f : 1.0f;
        su = s * up;
        inv = usable ? __frcp_rn(su) : 0.0f;
    }
    __device__ __forceinline__ int operator()(float x) const {
        return usable ? quantize(x * up, su, inv) : 0;
    }
};

}  // namespace ppdl
