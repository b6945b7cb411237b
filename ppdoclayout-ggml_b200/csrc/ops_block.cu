// ops_block.cu — the C ABI of the transformer-block operators (layer norm,
// 8-bit integer linear layers, rotary positions; include/ppdl_ops.h).
//
// Every argument is checked on the host; nothing is launched for a call that
// is refused.
#include <cmath>
#include <cstdio>

#include "../../include/ppdl_ops.h"
#include "block.cuh"
#include "block.h"

namespace ppdl {
void set_op_error(const char *msg);
}

namespace {

int refuse(const char *msg) {
    ppdl::set_op_error(msg);
    return PPDL_ERR_SHAPE;
}

int status_of(ppdl::Status s, const char *shape_msg) {
    switch (s) {
        case ppdl::OK: return PPDL_OK;
        case ppdl::ERR_SHAPE: return refuse(shape_msg);
        case ppdl::ERR_UNSUPPORTED:
            ppdl::set_op_error("unsupported form");
            return PPDL_ERR_UNSUPPORTED;
        default: ppdl::set_op_error("CUDA launch failed"); return PPDL_ERR_CUDA;
    }
}

// p aligned to an element of `size` bytes
bool aligned(const void *p, int size) { return ((uintptr_t)p & (uintptr_t)(size - 1)) == 0; }

// rows of D elements at p, ld apart; a null p passes when `optional`
bool rows_ok(const void *p, long long ld, long long rows, int D, int type, bool optional = false) {
    if (!p) return optional || rows == 0;
    return aligned(p, ppdl::elem_size(type)) && (rows <= 1 || ld >= D);
}

// The rows that ppdl_linear_i8_dynamic quantises
struct Dynamic {
    const void *x;
    long long ldx;
    int type;
};

// ppdl_linear_i8; with `dynamic`, q and q_scale are workspace that its rows
// are first quantised into, unless the product's kernel quantises them itself
int linear_i8(const int8_t *q, long long ldq, const float *q_scale, const int8_t *w, long long ldw,
              const float *w_scale, const float *bias, const void *res, long long ldres, int type,
              int act, int M, int N, int K, void *y, long long ldy, void *stream,
              const Dynamic *dynamic) {
    ppdl::set_op_error("");
    if (!ppdl::elem_type_ok(type) || act < 0 || act > 3)
        return refuse("linear_i8: unknown element type or activation");
    if (M < 0 || N <= 0 || K <= 0 || K > 131071) return refuse("linear_i8: bad sizes (K 1..131071)");
    if (!rows_ok(y, ldy, M, N, type) || !rows_ok(res, ldres, M, N, type, true) ||
        (M && (!q || !w || !q_scale || !w_scale)) || !aligned(q_scale, 4) || !aligned(w_scale, 4) ||
        !aligned(bias, 4) || !aligned(q, 16) || !aligned(w, 16) ||
        (M > 1 && (ldq < K || ldq % 16)) || (N > 1 && (ldw < K || ldw % 16)))
        return refuse("linear_i8: null or misaligned pointer, rows closer than their width, or q / "
                      "w rows not on 16-byte strides");
    // a single row's stride is never stepped
    if (M == 1) ldq = (K + 15LL) / 16 * 16;
    if (N == 1) ldw = (K + 15LL) / 16 * 16;
    ppdl::LinearI8Args a;
    a.q = q; a.ldq = ldq; a.q_scale = q_scale; a.w = w; a.ldw = ldw; a.w_scale = w_scale;
    a.bias = bias; a.res = {res, ldres}; a.y = {y, ldy};
    a.type = type; a.act = act; a.M = M; a.N = N; a.K = K;
    if (dynamic) {
        const Dynamic &d = *dynamic;
        if (!ppdl::elem_type_ok(d.type) || !rows_ok(d.x, d.ldx, M, K, d.type))
            return refuse("linear_i8_dynamic: unknown element type, null or misaligned rows, or "
                          "rows closer than K elements");
        ppdl::Status s = ppdl::OK;
        if (ppdl::launch_linear_i8_few({d.x, d.ldx}, d.type, a, (cudaStream_t)stream, &s))
            return status_of(s, "linear_i8_dynamic: sizes too large");
        s = ppdl::launch_quantize_rows({d.x, d.ldx}, d.type, M, K, (int8_t *)q, ldq,
                                       (float *)q_scale, (cudaStream_t)stream);
        if (s != ppdl::OK) return status_of(s, "linear_i8_dynamic: sizes too large");
    }
    return status_of(ppdl::launch_linear_i8(a, (cudaStream_t)stream), "linear_i8: sizes too large");
}

// True when the results of some heads certainly share memory: heads of dim
// values nearer to one another than that, or equal steps of two dimensions.
bool results_overlap(const ppdl_rotary_heads &h, int batch, int length, int dim) {
    const long long n[3] = {batch, length, h.heads};
    const long long step[3] = {h.out_batch, h.out_token, h.out_head};
    for (int i = 0; i < 3; i++) {
        if (n[i] < 2) continue;
        if (step[i] < dim && step[i] > -dim) return true;
        for (int j = 0; j < i; j++)
            if (n[j] > 1 && (step[i] == step[j] || step[i] + step[j] == 0)) return true;
    }
    return false;
}

// True when heads turned in place would be written where others are read.
bool moved_in_place(const ppdl_rotary_heads &h, int batch, int length) {
    return h.in == h.out &&
           ((batch > 1 && h.in_batch != h.out_batch) || (length > 1 && h.in_token != h.out_token) ||
            (h.heads > 1 && h.in_head != h.out_head));
}

}  // namespace

extern "C" {

PPDL_OPS_API int ppdl_layernorm(const void *x, long long ldx, const void *res, long long ldres,
                                const void *weight, const void *bias, int type, int w_type,
                                long long rows, int D, float eps, void *y, long long ldy, void *sum,
                                long long ldsum, float *mean, float *rstd, void *stream) {
    ppdl::set_op_error("");
    if (!ppdl::elem_type_ok(type) || (w_type != type && w_type != PPDL_F32))
        return refuse("layernorm: unknown element type, or weights neither of the rows' type nor FP32");
    if (rows < 0 || D <= 0 || !(eps >= 0.0f) || std::isinf(eps))
        return refuse("layernorm: bad sizes or eps");
    if (sum && !res) return refuse("layernorm: a sum needs a residual");
    if (!rows_ok(x, ldx, rows, D, type) || !rows_ok(y, ldy, rows, D, type) ||
        !rows_ok(res, ldres, rows, D, type, true) || !rows_ok(sum, ldsum, rows, D, type, true) ||
        !aligned(weight, ppdl::elem_size(w_type)) || !aligned(bias, ppdl::elem_size(w_type)) ||
        !aligned(mean, 4) || !aligned(rstd, 4))
        return refuse("layernorm: null or misaligned pointer, or rows closer than D elements");
    ppdl::LayerNormArgs a;
    a.x = {x, ldx}; a.res = {res, ldres}; a.y = {y, ldy}; a.sum = {sum, ldsum};
    a.weight = weight; a.bias = bias; a.mean = mean; a.rstd = rstd;
    a.rows = rows; a.D = D; a.type = type; a.w_type = w_type; a.eps = eps;
    return status_of(ppdl::launch_layernorm(a, (cudaStream_t)stream), "layernorm: too many rows");
}

PPDL_OPS_API long long ppdl_layernorm_backward_workspace(long long rows, int D) {
    return ppdl::layernorm_backward_work(rows, D);
}

PPDL_OPS_API int ppdl_layernorm_backward(const void *dy, long long lddy, const void *x,
                                         long long ldx, const void *weight, const float *mean,
                                         const float *rstd, const void *dsum, long long lddsum,
                                         int type, int w_type, long long rows, int D, void *dx,
                                         long long lddx, void *dweight, void *dbias, float *work,
                                         void *stream) {
    ppdl::set_op_error("");
    if (!ppdl::elem_type_ok(type) || (w_type != type && w_type != PPDL_F32))
        return refuse("layernorm_backward: unknown element type, or weights neither of the rows' "
                      "type nor FP32");
    if (rows < 0 || D <= 0) return refuse("layernorm_backward: bad sizes");
    const int ws = ppdl::elem_size(w_type);
    if (!rows_ok(dy, lddy, rows, D, type) || !rows_ok(x, ldx, rows, D, type) ||
        !rows_ok(dx, lddx, rows, D, type) || !rows_ok(dsum, lddsum, rows, D, type, true) ||
        (rows && (!mean || !rstd)) || !aligned(mean, 4) || !aligned(rstd, 4) ||
        !aligned(weight, ws) || !aligned(dweight, ws) || !aligned(dbias, ws))
        return refuse("layernorm_backward: null or misaligned pointer, or rows closer than D "
                      "elements");
    if (rows && (dweight || dbias) && (!work || !aligned(work, 16)))
        return refuse("layernorm_backward: the weights' gradients need a 16-byte aligned workspace");
    ppdl::LayerNormBackwardArgs a;
    a.dy = {dy, lddy}; a.x = {x, ldx}; a.dsum = {dsum, lddsum}; a.dx = {dx, lddx};
    a.weight = weight; a.mean = mean; a.rstd = rstd; a.dweight = dweight; a.dbias = dbias;
    a.rows = rows; a.D = D; a.type = type; a.w_type = w_type; a.work = work;
    return status_of(ppdl::launch_layernorm_backward(a, (cudaStream_t)stream),
                     "layernorm_backward: too many rows");
}

PPDL_OPS_API int ppdl_quantize_rows_i8(const void *x, long long ldx, int type, long long rows,
                                       int K, int8_t *q, long long ldq, float *scale,
                                       void *stream) {
    ppdl::set_op_error("");
    if (!ppdl::elem_type_ok(type)) return refuse("quantize_rows_i8: unknown element type");
    if (rows < 0 || K <= 0) return refuse("quantize_rows_i8: bad sizes");
    if (!rows_ok(x, ldx, rows, K, type) || (rows && (!q || !scale)) || !aligned(scale, 4) ||
        !aligned(q, 16) || (rows > 1 && (ldq < K || ldq % 16)))
        return refuse("quantize_rows_i8: null or misaligned pointer, rows closer than K elements, "
                      "or q rows not on 16-byte strides");
    return status_of(ppdl::launch_quantize_rows({x, ldx}, type, rows, K, q, ldq, scale,
                                                (cudaStream_t)stream),
                     "quantize_rows_i8: too many rows");
}

PPDL_OPS_API int ppdl_linear_i8(const int8_t *q, long long ldq, const float *q_scale,
                                const int8_t *w, long long ldw, const float *w_scale,
                                const float *bias, const void *res, long long ldres, int type,
                                int act, int M, int N, int K, void *y, long long ldy,
                                void *stream) {
    return linear_i8(q, ldq, q_scale, w, ldw, w_scale, bias, res, ldres, type, act, M, N, K, y, ldy,
                     stream, nullptr);
}

namespace {
// work: M rows of 8-bit values on 16-byte strides, then M scales
long long row_bytes(int K) { return (K + 15LL) / 16 * 16; }
long long scales_at(int M, int K) { return (long long)M * row_bytes(K); }
}  // namespace

PPDL_OPS_API long long ppdl_linear_i8_dynamic_workspace(int M, int K) {
    if (M <= 0 || K <= 0) return 0;
    return scales_at(M, K) + 4LL * M;
}

PPDL_OPS_API int ppdl_linear_i8_dynamic(const void *x, long long ldx, int x_type, const int8_t *w,
                                        long long ldw, const float *w_scale, const float *bias,
                                        const void *res, long long ldres, int type, int act, int M,
                                        int N, int K, void *y, long long ldy, void *work,
                                        void *stream) {
    ppdl::set_op_error("");
    if (M > 0 && (!work || !aligned(work, 16)))
        return refuse("linear_i8_dynamic: null or misaligned workspace");
    if (M < 0 || K <= 0) return refuse("linear_i8_dynamic: bad sizes");
    int8_t *q = (int8_t *)work;
    const Dynamic rows = {x, ldx, x_type};
    return linear_i8(q, row_bytes(K), (const float *)(q + scales_at(M, K)), w, ldw, w_scale, bias,
                     res, ldres, type, act, M, N, K, y, ldy, stream, &rows);
}

PPDL_OPS_API int ppdl_rotary(const ppdl_rotary_heads *q, const ppdl_rotary_heads *k, int type,
                             int batch, int length, int dim, int rotated, const void *positions,
                             int position_bytes, long long axis_stride, long long batch_stride,
                             long long token_stride, int axes, const int32_t *sections,
                             const double *freq, int interleaved, int inverse, void *stream) {
    ppdl::set_op_error("");
    if (!ppdl::elem_type_ok(type)) return refuse("rotary: unknown element type");
    if (batch < 0 || length < 0 || dim <= 0 || dim > 1024 || rotated < 2 || rotated > dim ||
        rotated % 2)
        return refuse("rotary: bad sizes (heads of 1..1024 values, an even number of them turned)");
    if (axes < 1 || axes > ppdl::kMaxAxes || !sections)
        return refuse("rotary: one to four axes");
    if (position_bytes != 4 && position_bytes != 8)
        return refuse("rotary: positions are 32-bit or 64-bit integers");
    const bool some = batch > 0 && length > 0;
    if (!aligned(positions, position_bytes) || !aligned(freq, 8) || (some && (!positions || !freq)))
        return refuse("rotary: null or misaligned positions or frequencies");
    ppdl::RotaryArgs a;
    long long pairs = 0;
    for (int i = 0; i < axes; i++) {
        if (sections[i] < 0) return refuse("rotary: a negative section");
        a.sections[i] = sections[i];
        pairs += sections[i];
    }
    if (pairs != rotated / 2) return refuse("rotary: the sections do not add up to the turned pairs");
    const ppdl_rotary_heads *h[2] = {q, k};
    for (int i = 0; i < 2; i++) {
        if (!h[i] || h[i]->heads == 0) continue;
        if (h[i]->heads < 0 || h[i]->heads > 65535 || (some && (!h[i]->in || !h[i]->out)) ||
            !aligned(h[i]->in, ppdl::elem_size(type)) || !aligned(h[i]->out, ppdl::elem_size(type)))
            return refuse("rotary: bad number of heads, or null or misaligned heads");
        if (some && (results_overlap(*h[i], batch, length, dim) ||
                     moved_in_place(*h[i], batch, length)))
            return refuse("rotary: results that overlap, or heads turned in place with other "
                          "strides");
        if (some && i == 1 && a.h[0].heads && a.h[0].out == h[1]->out)
            return refuse("rotary: queries and keys turned into the same place");
        ppdl::RotaryHeads &o = a.h[i];
        o.in = h[i]->in; o.out = h[i]->out; o.heads = h[i]->heads;
        o.in_bs = h[i]->in_batch; o.in_ts = h[i]->in_token; o.in_hs = h[i]->in_head;
        o.out_bs = h[i]->out_batch; o.out_ts = h[i]->out_token; o.out_hs = h[i]->out_head;
    }
    a.type = type; a.batch = batch; a.length = length; a.dim = dim; a.rotated = rotated;
    a.pos = positions; a.pos_bytes = position_bytes;
    a.pos_as = axis_stride; a.pos_bs = batch_stride; a.pos_ts = token_stride;
    a.axes = axes; a.freq = freq; a.interleaved = interleaved != 0; a.inverse = inverse != 0;
    return status_of(ppdl::launch_rotary(a, (cudaStream_t)stream), "rotary: too many tokens");
}

}  // extern "C"
