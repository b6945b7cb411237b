// quantize.cu — 8-bit rows with a scale each: scale = max |x| / 127,
// q = x / scale rounded half to even on the exact quotient.
#include "block.cuh"
#include "block.h"

namespace ppdl {

namespace {

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

// One block per row: the largest |x| (as the bits of |x|, whose unsigned
// order puts infinities and NaNs on top), then the quotients.  Scales below
// 2^-64 quantise x 2^64 by s 2^64, both exact, so that 1 / s is finite.
template <typename T>
__global__ void quantize_rows_kernel(const T *x, long long ldx, int K, int8_t *q, long long ldq,
                                     float *scale) {
    pdl_begin();
    __shared__ unsigned sh[32];
    const long long row = blockIdx.x;
    x += row * ldx;
    q += row * ldq;
    unsigned m = 0;
    for (int i = threadIdx.x; i < K; i += blockDim.x)
        m = max(m, __float_as_uint(fabsf(to_float(x[i]))));
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = m;
    __syncthreads();
    m = 0;
    for (int i = 0; i < (int)(blockDim.x >> 5); i++) m = max(m, sh[i]);
    const float s = __fdiv_rn(__uint_as_float(m), 127.0f);
    if (threadIdx.x == 0) scale[row] = s;
    const bool usable = s > 0.0f && m < 0x7f800000u;
    const float up = s < 0x1p-64f ? 0x1p64f : 1.0f;
    const float su = s * up, inv = usable ? __frcp_rn(su) : 0.0f;
    for (int i = threadIdx.x; i < K; i += blockDim.x)
        q[i] = usable ? (int8_t)quantize(to_float(x[i]) * up, su, inv) : (int8_t)0;
}

}  // namespace

Status launch_quantize_rows(const Rows &x, int type, long long rows, int K, int8_t *q,
                            long long ldq, float *scale, cudaStream_t st) {
    if (rows == 0) return OK;
    if (rows < 0 || rows > 0x7fffffffLL || K <= 0) return ERR_SHAPE;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        pdl_launch(quantize_rows_kernel<T>, (unsigned)rows, K >= 1024 ? 256 : 128, 0, st,
                   (const T *)x.p, x.ld, K, q, ldq, scale);
        return cuda_status();
    });
}

}  // namespace ppdl
