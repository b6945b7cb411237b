// layernorm.cu — layer norm over rows, forward and backward.
//
//   forward   s = x (+ res, rounded to the element type),
//             mean = sum s / D, var = sum (s - mean)^2 / D,
//             rstd = 1 / sqrt(var + eps), y = (s - mean) rstd w + b
//   backward  xh = (x - mean) rstd, g = dy w,
//             dx = rstd (g - mean(g) - xh mean(g xh)) (+ dsum),
//             dw = sum over rows of dy xh, db = sum over rows of dy
//
// All sums are FP32.  The forward's sum with a residual is rounded to the
// element type before the statistics are taken, whether or not it is stored,
// so that the backward pass (which reads the stored sum) differentiates the
// function that ran.  The variance is the sum of squared deviations from the
// mean, not a difference of moments, so a large common offset costs nothing.
#include "block.cuh"
#include "block.h"

namespace ppdl {

namespace {

template <typename WT>
__device__ __forceinline__ float weight_at(const WT *w, long long i, float none) {
    return w ? to_float(w[i]) : none;
}

// One block per row, any width: the row is read once for the mean, once for
// the variance and once for the output.
template <typename T, typename WT>
__global__ void layernorm_row_kernel(const T *x, long long ldx, const T *res, long long ldres, T *y,
                                     long long ldy, T *sum, long long ldsum, const WT *w,
                                     const WT *b, float *mean_out, float *rstd_out, int D,
                                     float eps) {
    pdl_begin();
    __shared__ float sh[32];
    const long long row = blockIdx.x;
    x += row * ldx;
    y += row * ldy;
    if (res) res += row * ldres;
    if (sum) sum += row * ldsum;
    auto value = [&](int i) {
        const float v = to_float(x[i]);
        return res ? to_float(from_float<T>(v + to_float(res[i]))) : v;
    };
    float s = 0.0f;
    for (int i = threadIdx.x; i < D; i += blockDim.x) s += value(i);
    const float mean = block_sum(s, sh) / (float)D;
    s = 0.0f;
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
        const float d = value(i) - mean;
        s += d * d;
    }
    const float rstd = 1.0f / sqrtf(block_sum(s, sh) / (float)D + eps);
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
        const float v = value(i);
        if (sum) sum[i] = from_float<T>(v);
        y[i] = from_float<T>((v - mean) * rstd * weight_at(w, i, 1.0f) + weight_at(b, i, 0.0f));
    }
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
}

// dx, one block per row, any width.
template <typename T, typename WT>
__global__ void layernorm_dx_row_kernel(const T *dy, long long lddy, const T *x, long long ldx,
                                        const T *dsum, long long lddsum, T *dx, long long lddx,
                                        const WT *w, const float *mean_in, const float *rstd_in,
                                        int D) {
    pdl_begin();
    __shared__ float sh[32];
    const long long row = blockIdx.x;
    dy += row * lddy;
    x += row * ldx;
    dx += row * lddx;
    if (dsum) dsum += row * lddsum;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
        const float g = to_float(dy[i]) * weight_at(w, i, 1.0f);
        s1 += g;
        s2 += g * ((to_float(x[i]) - mean) * rstd);
    }
    const float m1 = block_sum(s1, sh) / (float)D, m2 = block_sum(s2, sh) / (float)D;
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
        const float g = to_float(dy[i]) * weight_at(w, i, 1.0f);
        const float xh = (to_float(x[i]) - mean) * rstd;
        float v = (g - m1 - xh * m2) * rstd;
        if (dsum) v += to_float(dsum[i]);
        dx[i] = from_float<T>(v);
    }
}

// Column sums of dy xh and dy over the row chunk blockIdx.y, one column per
// thread, into part[chunk][2][D].
template <typename T>
__global__ void layernorm_dw_column_kernel(const T *dy, long long lddy, const T *x, long long ldx,
                                           const float *mean, const float *rstd, long long rows,
                                           int D, long long chunk, float *part) {
    pdl_begin();
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= D) return;
    const long long r0 = blockIdx.y * chunk, r1 = min(rows, r0 + chunk);
    float sw = 0.0f, sb = 0.0f;
    for (long long r = r0; r < r1; r++) {
        const float g = to_float(dy[r * lddy + c]);
        sw += g * ((to_float(x[r * ldx + c]) - mean[r]) * rstd[r]);
        sb += g;
    }
    part[((long long)blockIdx.y * 2) * D + c] = sw;
    part[((long long)blockIdx.y * 2 + 1) * D + c] = sb;
}

// dw, db = the parts' sums, in part order
template <typename WT>
__global__ void layernorm_dw_sum_kernel(const float *part, int parts, int D, WT *dw, WT *db) {
    pdl_begin();
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= D) return;
    WT *out = blockIdx.y ? db : dw;
    if (!out) return;
    float s = 0.0f;
    for (int p = 0; p < parts; p++) s += part[((long long)p * 2 + blockIdx.y) * D + c];
    out[c] = from_float<WT>(s);
}

constexpr int kMaxParts = 296;
int row_parts(long long rows) { return (int)(rows < kMaxParts ? rows : kMaxParts); }

// f(T{}, WT{}) for the element types of rows and weights
template <typename F>
Status with_types(int type, int w_type, F f) {
    return with_type(type, [&](auto t) {
        if (w_type == T_F32) return f(t, float{});
        return f(t, t);
    });
}

template <typename T>
T *ptr(const Rows &r) { return (T *)r.p; }

}  // namespace

Status launch_layernorm(const LayerNormArgs &a, cudaStream_t st) {
    if (a.rows == 0) return OK;
    if (a.rows < 0 || a.rows > 0x7fffffffLL || a.D <= 0) return ERR_SHAPE;
    return with_types(a.type, a.w_type, [&](auto t, auto wt) {
        using T = decltype(t);
        using WT = decltype(wt);
        const int threads = a.D >= 1024 ? 256 : 128;
        pdl_launch(layernorm_row_kernel<T, WT>, (unsigned)a.rows, threads, 0, st,
                   (const T *)a.x.p, a.x.ld, (const T *)a.res.p, a.res.ld, ptr<T>(a.y), a.y.ld,
                   ptr<T>(a.sum), a.sum.ld, (const WT *)a.weight, (const WT *)a.bias, a.mean,
                   a.rstd, a.D, a.eps);
        return cuda_status();
    });
}

long long layernorm_backward_work(long long rows, int D) {
    if (rows <= 0 || D <= 0) return 0;
    return 2LL * row_parts(rows) * D;
}

Status launch_layernorm_backward(const LayerNormBackwardArgs &a, cudaStream_t st) {
    if (a.rows < 0 || a.rows > 0x7fffffffLL || a.D <= 0) return ERR_SHAPE;
    if (a.rows == 0 && !a.dweight && !a.dbias) return OK;
    return with_types(a.type, a.w_type, [&](auto t, auto wt) {
        using T = decltype(t);
        using WT = decltype(wt);
        int parts = 0;
        if (a.rows > 0) {
            pdl_launch(layernorm_dx_row_kernel<T, WT>, (unsigned)a.rows, a.D >= 1024 ? 256 : 128, 0,
                       st, (const T *)a.dy.p, a.dy.ld, (const T *)a.x.p, a.x.ld,
                       (const T *)a.dsum.p, a.dsum.ld, ptr<T>(a.dx), a.dx.ld, (const WT *)a.weight,
                       a.mean, a.rstd, a.D);
            if (!a.dweight && !a.dbias) return cuda_status();
            const long long chunk = (a.rows + row_parts(a.rows) - 1) / row_parts(a.rows);
            parts = (int)((a.rows + chunk - 1) / chunk);
            pdl_launch(layernorm_dw_column_kernel<T>, dim3(cdiv(a.D, 128), parts), 128, 0, st,
                       (const T *)a.dy.p, a.dy.ld, (const T *)a.x.p, a.x.ld, a.mean, a.rstd, a.rows,
                       a.D, chunk, a.work);
        }
        if (a.dweight || a.dbias)
            pdl_launch(layernorm_dw_sum_kernel<WT>, dim3(cdiv(a.D, 128), 2), 128, 0, st, a.work,
                       parts, a.D, (WT *)a.dweight, (WT *)a.dbias);
        return cuda_status();
    });
}

}  // namespace ppdl
