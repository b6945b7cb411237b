// block.h — launchers of the transformer-block operators: layer norm
// (layernorm.cu), 8-bit integer linear layers (linear_i8.cu) and rotary
// positions (rotary.cu).
//
// Every launcher enqueues on `st`, allocates nothing and returns a
// ppdl::Status.  Rows lie `ld` elements apart; elements of a row are
// contiguous.
#pragma once

#include <stdint.h>

#include "common.cuh"

namespace ppdl {

// rows of a matrix of element type `type`
struct Rows {
    const void *p = nullptr;
    long long ld = 0;
};

struct LayerNormArgs {
    Rows x, res, y, sum;  // res and sum may be null
    const void *weight = nullptr, *bias = nullptr;  // of w_type; may be null (1 / 0)
    float *mean = nullptr, *rstd = nullptr;         // may be null
    long long rows = 0;
    int D = 0, type = 0, w_type = 0;
    float eps = 0.0f;
};
Status launch_layernorm(const LayerNormArgs &a, cudaStream_t st);

struct LayerNormBackwardArgs {
    Rows dy, x, dsum, dx;                   // dsum may be null
    const void *weight = nullptr;           // of w_type; may be null (1)
    const float *mean = nullptr, *rstd = nullptr;
    void *dweight = nullptr, *dbias = nullptr;  // of w_type; may be null
    long long rows = 0;
    int D = 0, type = 0, w_type = 0;
    float *work = nullptr;                  // layernorm_backward_work() floats
};
Status launch_layernorm_backward(const LayerNormBackwardArgs &a, cudaStream_t st);
long long layernorm_backward_work(long long rows, int D);
// the backward pass' device error flag, as tc_error_fetch_and_clear()
int row_error_fetch_and_clear();

// q[m][k] = x[m][k] / scale[m] rounded half to even, scale[m] = amax / 127
Status launch_quantize_rows(const Rows &x, int type, long long rows, int K, int8_t *q,
                            long long ldq, float *scale, cudaStream_t st);

struct LinearI8Args {
    const int8_t *q = nullptr, *w = nullptr;  // [M][K], [N][K]
    long long ldq = 0, ldw = 0;
    const float *q_scale = nullptr, *w_scale = nullptr, *bias = nullptr;
    Rows res, y;
    int type = 0, act = 0;
    int M = 0, N = 0, K = 0;
};
Status launch_linear_i8(const LinearI8Args &a, cudaStream_t st);
// The same on rows x of x_type in place of q, quantised in the kernel: for a
// few short rows (false: not these, nothing was launched).
bool launch_linear_i8_few(const Rows &x, int x_type, const LinearI8Args &a, cudaStream_t st,
                          Status *status);
// its device error flag, as tc_error_fetch_and_clear()
int linear_error_fetch_and_clear();

struct RotaryHeads {
    const void *in = nullptr;
    void *out = nullptr;
    int heads = 0;
    long long in_bs = 0, in_ts = 0, in_hs = 0, out_bs = 0, out_ts = 0, out_hs = 0;
};
constexpr int kMaxAxes = 4;
struct RotaryArgs {
    RotaryHeads h[2];  // queries and keys (heads 0: none)
    int type = 0, batch = 0, length = 0, dim = 0, rotated = 0;
    const void *pos = nullptr;
    int pos_bytes = 8;  // 4 or 8
    long long pos_as = 0, pos_bs = 0, pos_ts = 0;
    int axes = 1, sections[kMaxAxes] = {};
    const double *freq = nullptr;
    int interleaved = 0, inverse = 0;
};
Status launch_rotary(const RotaryArgs &a, cudaStream_t st);

}  // namespace ppdl
