// linear_i8.cu — linear layers in 8-bit integers with a scale for each token
// (row of the activations) and each channel (row of the weights):
//
//   y(m, n) = act(sum_k q(m, k) w(n, k) * q_scale[m] * w_scale[n] + bias[n]) + res(m, n)
//
// and the quantiser that makes q and q_scale from FP32 / BF16 / FP16 rows.
// The integer sums are exact (at most 131071 products of at most 128 x 128: below 2^31).
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

// One thread per output, 16 x 16 outputs a block, 64 bytes of k at a time
// through shared memory, four products an instruction.
template <typename T>
__global__ void __launch_bounds__(256) linear_i8_simt_kernel(LinearI8Args a) {
    pdl_begin();
    __shared__ int sq[16][17], sw[16][17];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const long long m0 = (long long)blockIdx.y * 16;
    const int n0 = blockIdx.x * 16;
    auto word = [&](const int8_t *p, int k) {  // bytes k .. k + 3 of a row, zero past K
        int v = 0;
        for (int j = 0; j < 4; j++)
            if (k + j < a.K) v |= (int)(uint8_t)p[k + j] << (8 * j);
        return v;
    };
    int acc = 0;
    for (int k0 = 0; k0 < a.K; k0 += 64) {
        const int k = k0 + 4 * tx;
        sq[ty][tx] = m0 + ty < a.M ? word(a.q + (m0 + ty) * a.ldq, k) : 0;
        sw[ty][tx] = n0 + ty < a.N ? word(a.w + (long long)(n0 + ty) * a.ldw, k) : 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 16; j++) acc = __dp4a(sq[ty][j], sw[tx][j], acc);
        __syncthreads();
    }
    const long long m = m0 + ty;
    const int n = n0 + tx;
    if (m >= a.M || n >= a.N) return;
    float v = (float)acc * a.q_scale[m] * a.w_scale[n];
    if (a.bias) v += a.bias[n];
    v = act_apply(v, a.act);
    if (a.res.p) v += to_float(((const T *)a.res.p)[m * a.res.ld + n]);
    ((T *)a.y.p)[m * a.y.ld + n] = from_float<T>(v);
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

Status launch_linear_i8(const LinearI8Args &a, cudaStream_t st) {
    if (a.M == 0) return OK;
    if (a.M < 0 || a.N <= 0 || a.K <= 0 || cdiv(a.M, 16) > 65535) return ERR_SHAPE;
    return with_type(a.type, [&](auto t) {
        using T = decltype(t);
        pdl_launch(linear_i8_simt_kernel<T>, dim3(cdiv(a.N, 16), cdiv(a.M, 16)), 256, 0, st, a);
        return cuda_status();
    });
}

}  // namespace ppdl
