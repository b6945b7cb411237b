// rotary.cu — rotary positions with several axes (time, height, width, ...)
// on queries and keys.
//
// Pair i of the first `rotated` values of every head is turned by the angle
// pos[axis(i)] * freq[i]; `sections` says how many consecutive pairs each
// axis turns.  The pair is (x[i], x[i + rotated / 2]), or (x[2i], x[2i + 1])
// when interleaved.  The inverse turns back, which is also the backward pass
// (the transpose of a rotation).
//
// The angle of a far position needs more than 32 bits: position times
// frequency is taken in turns (revolutions) in 64 bits, whole turns are
// dropped, and only the fraction in [-1/2, 1/2] goes through the FP32 sine
// and cosine.
#include "block.cuh"
#include "block.h"

namespace ppdl {

namespace {

// (cos, sin) of pair i at a token whose positions start at element `at`
__device__ __forceinline__ float2 turn_of(const RotaryArgs &a, long long at, int i) {
    int axis = 0, end = a.sections[0];
    while (axis < a.axes - 1 && i >= end) end += a.sections[++axis];
    const long long j = at + axis * a.pos_as;
    const double p = a.pos_bytes == 8 ? (double)((const long long *)a.pos)[j]
                                      : (double)((const int *)a.pos)[j];
    double t = p * a.freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
    t -= rint(t);
    float s, c;
    sincospif(2.0f * (float)t, &s, &c);
    return make_float2(c, a.inverse ? -s : s);
}

// One block per token.
template <typename T>
__global__ void rotary_token_kernel(RotaryArgs a) {
    pdl_begin();
    pdl_trigger();
    extern __shared__ float2 turn[];
    const int pairs = a.rotated / 2;
    const int b = blockIdx.x / a.length, t = blockIdx.x % a.length;
    for (int i = threadIdx.x; i < pairs; i += blockDim.x)
        turn[i] = turn_of(a, b * a.pos_bs + t * a.pos_ts, i);
    __syncthreads();
    for (int s = 0; s < 2; s++) {
        const RotaryHeads &h = a.h[s];
        const T *in = (const T *)h.in + b * h.in_bs + t * h.in_ts;
        T *out = (T *)h.out + b * h.out_bs + t * h.out_ts;
        const int per = pairs + a.dim - a.rotated;
        for (int u = threadIdx.x; u < h.heads * per; u += blockDim.x) {
            const int head = u / per, i = u - head * per;
            const T *p = in + head * h.in_hs;
            T *o = out + head * h.out_hs;
            if (i >= pairs) {
                o[pairs + i] = p[pairs + i];
                continue;
            }
            const int ia = a.interleaved ? 2 * i : i, ib = a.interleaved ? 2 * i + 1 : i + pairs;
            const float2 cs = turn[i];
            const float va = to_float(p[ia]), vb = to_float(p[ib]);
            o[ia] = from_float<T>(va * cs.x - vb * cs.y);
            o[ib] = from_float<T>(vb * cs.x + va * cs.y);
        }
    }
}

}  // namespace

Status launch_rotary(const RotaryArgs &a, cudaStream_t st) {
    const long long tokens = (long long)a.batch * a.length;
    if (tokens == 0) return OK;
    if (tokens > 0x7fffffffLL) return ERR_SHAPE;
    return with_type(a.type, [&](auto t) {
        using T = decltype(t);
        pdl_launch(rotary_token_kernel<T>, (unsigned)tokens, 128, (size_t)a.rotated / 2 * 8, st, a);
        return cuda_status();
    });
}

}  // namespace ppdl
