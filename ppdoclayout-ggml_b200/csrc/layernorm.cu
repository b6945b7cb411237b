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
//
// Memory bounds all of it: a few operations a value, and every value is read
// and written once.  Measured (copy rate 6.54 TB/s): forward 52500 x 256 FP32
// with residual, stored sum and statistics 33.6 us (98 % of it), 8192 x 4096
// BF16 30.1 (68 %), backward 16384 x 4096 BF16 87.2 (71 %), 52500 x 256 FP32
// 34 (73 %); one row of 4096 3.1 us, 2400 x 256 backward 8 us in two kernels,
// which is latency.  Rows in registers for what has few rows or is narrow;
// rings of bulk copies where more bytes have to be in flight than registers
// hold; groups of rows through shared memory where rows are no whole vectors;
// one value at a time for the rest.
#include <initializer_list>
#include <type_traits>

#include "block.cuh"
#include "block.h"
#include "rows.cuh"
#include "tc_ptx.cuh"

namespace ppdl {

namespace {

template <typename WT>
__device__ __forceinline__ float weight_at(const WT *w, long long i, float none) {
    return w ? to_float(w[i]) : none;
}

// One block per row, any width (rows too wide for registers): read once for the
// mean, and again, from L2, for the variance and for the output.  (The column
// is unsigned: its last step passes 2^31 - 1 where D is next to it.)
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
    auto value = [&](unsigned i) {
        const float v = to_float(x[i]);
        return res ? to_float(from_float<T>(v + to_float(res[i]))) : v;
    };
    float s = 0.0f;
    for (unsigned i = threadIdx.x; i < (unsigned)D; i += blockDim.x) s += value(i);
    const float mean = block_sum(s, sh) / (float)D;
    s = 0.0f;
    for (unsigned i = threadIdx.x; i < (unsigned)D; i += blockDim.x) {
        const float d = value(i) - mean;
        s += d * d;
    }
    const float rstd = rsqrtf(block_sum(s, sh) / (float)D + eps);
    for (unsigned i = threadIdx.x; i < (unsigned)D; i += blockDim.x) {
        const float v = value(i);
        if (sum) sum[i] = from_float<T>(v);
        y[i] = from_float<T>((v - mean) * rstd * weight_at(w, i, 1.0f) + weight_at(b, i, 0.0f));
    }
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
}

// Rows of whole 16-byte vectors in registers: TPR threads hold a row of at
// most TPR * NE values, a block has as many rows as fit 128 threads (one,
// when TPR is more).  One pass over memory.  (Blocks of 512 share an SM in
// twos: 2048 x 16384 BF16 55 -> 37 us; smaller ones spill for it and lose.)
template <typename T, typename WT, int TPR, int NE>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, TPR == 512 ? 2 : 1)
layernorm_vector_kernel(const T *x, long long ldx, const T *res, long long ldres, T *y,
                        long long ldy, T *sum, long long ldsum, const WT *w, const WT *b,
                        float *mean_out, float *rstd_out, long long rows, int D, float eps) {
    using Tile = PairTile<T, TPR, NE>;
    pdl_begin();
    pdl_trigger();
    __shared__ __align__(16) float sh[2][32];
    constexpr int kRows = TPR < 128 ? 128 / TPR : 1, kHalf = Tile::kVec / 2;
    const int lane = threadIdx.x % TPR;
    long long row = (long long)blockIdx.x * kRows + threadIdx.x / TPR;
    // rows past the end repeat the last one (its threads take part in the
    // shuffles) and store nothing
    const bool real = row < rows;
    if (!real) row = rows - 1;
    typename Tile::Raw r;
    Tile::load(r, x + row * ldx, D, lane);
    if (res) {
        typename Tile::Raw q;
        Tile::load(q, res + row * ldres, D, lane);
#pragma unroll
        for (int j = 0; j < NE / 2; j++)
            Tile::set_pair(r, j, add2(Tile::pair(r, j), Tile::pair(q, j)));
    }
    float2 t = both(0.0f);
#pragma unroll
    for (int j = 0; j < NE / 2; j++) t = add2(t, Tile::pair(r, j));
    float s[1] = {t.x + t.y};
    team_sums<TPR>(s, sh[0], threadIdx.x / TPR);
    const float mean = s[0] / (float)D;
    t = both(0.0f);
#pragma unroll
    for (int i = 0; i < Tile::kVecs; i++)
        // a vector past D holds zeros and takes no part
        if (Tile::column(i, lane) < D) {
#pragma unroll
            for (int j = i * kHalf; j < (i + 1) * kHalf; j++) {
                const float2 v = add2(Tile::pair(r, j), both(-mean));
                t = fma2(v, v, t);
            }
        }
    s[0] = t.x + t.y;
    team_sums<TPR>(s, sh[1], threadIdx.x / TPR);
    const float rstd = rsqrtf(s[0] / (float)D + eps);
    if (!real) return;
    if (sum) Tile::store(sum + row * ldsum, r, D, lane);
    const bool wide_w = sizeof(WT) * Tile::kVec >= 16 && ((uintptr_t)w & 15) == 0;
    const bool wide_b = sizeof(WT) * Tile::kVec >= 16 && ((uintptr_t)b & 15) == 0;
#pragma unroll
    for (int i = 0; i < Tile::kVecs; i++) {
        float2 pw[kHalf], pb[kHalf];
        Tile::vector_params(pw, w, 1.0f, i, D, lane, wide_w);
        Tile::vector_params(pb, b, 0.0f, i, D, lane, wide_b);
#pragma unroll
        for (int k = 0; k < kHalf; k++) {
            const float2 v = add2(Tile::pair(r, i * kHalf + k), both(-mean));
            Tile::set_pair(r, i * kHalf + k, fma2(mul2(v, both(rstd)), pw[k], pb[k]));
        }
    }
    Tile::store(y + row * ldy, r, D, lane);
    if (lane == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
}

// The same for rows of any alignment, value by value.
template <typename T, typename WT, int TPR, int NE>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR)
layernorm_tile_kernel(const T *x, long long ldx, const T *res, long long ldres, T *y,
                      long long ldy, T *sum, long long ldsum, const WT *w, const WT *b,
                      float *mean_out, float *rstd_out, long long rows, int D, float eps) {
    using Tile = RowTile<T, TPR, NE>;
    pdl_begin();
    pdl_trigger();
    __shared__ __align__(16) float sh[2][32];
    constexpr int kRows = TPR < 128 ? 128 / TPR : 1;
    const int lane = threadIdx.x % TPR;
    long long row = (long long)blockIdx.x * kRows + threadIdx.x / TPR;
    // rows past the end repeat the last one (its threads take part in the
    // shuffles) and store nothing
    const bool real = row < rows;
    if (!real) row = rows - 1;
    typename Tile::Raw r;
    Tile::load(r, x + row * ldx, D, lane);
    if (res) {
        typename Tile::Raw q;
        Tile::load(q, res + row * ldres, D, lane);
#pragma unroll
        for (int j = 0; j < NE; j++) r.v[j] = from_float<T>(to_float(r.v[j]) + to_float(q.v[j]));
    }
    float v[NE], s[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < NE; j++) {
        v[j] = to_float(r.v[j]);
        s[0] += v[j];
    }
    team_sums<TPR>(s, sh[0], threadIdx.x / TPR);
    const float mean = s[0] / (float)D;
    s[0] = 0.0f;
#pragma unroll
    for (int j = 0; j < NE; j++) {
        v[j] -= mean;
        if (Tile::inside(j, D, lane)) s[0] += v[j] * v[j];
    }
    team_sums<TPR>(s, sh[1], threadIdx.x / TPR);
    const float rstd = rsqrtf(s[0] / (float)D + eps);
    if (!real) return;
    if (sum) Tile::store(sum + row * ldsum, r, D, lane);
    float p[NE];
    Tile::load_params(p, w, 1.0f, D, lane);
#pragma unroll
    for (int j = 0; j < NE; j++) v[j] = v[j] * rstd * p[j];
    Tile::load_params(p, b, 0.0f, D, lane);
#pragma unroll
    for (int j = 0; j < NE; j++) r.v[j] = from_float<T>(v[j] + p[j]);
    Tile::store(y + row * ldy, r, D, lane);
    if (lane == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
}

__device__ int g_row_error = 0;

// Persistent blocks with their rows coming through rings in shared memory
// (RowRing), weights and biases in registers: for many wide 16-bit rows of
// whole 16-byte vectors.  8192 x 4096 BF16 take 30.1 us, 68 % of copy
// bandwidth: what bounds them is the chain of a row (two sums over 8 warps,
// about 270 instructions a warp) with two rows on an SM at a time; more rows
// in smaller registers spilled, and a load from local memory queues behind
// the stores to y.
constexpr int ring_threads(int tpr) { return tpr < 256 ? 256 : tpr; }
constexpr int ring_blocks(int tpr) { return tpr > 256 ? 1 : 2; }
template <typename T, typename WT, int TPR, int NE>
__global__ void __launch_bounds__(ring_threads(TPR), ring_blocks(TPR))
layernorm_ring_kernel(const T *x, long long ldx, const T *res, long long ldres, T *y,
                      long long ldy, T *sum, long long ldsum, const WT *w, const WT *b,
                      float *mean_out, float *rstd_out, long long rows, int D, float eps,
                      int stages) {
    using Tile = PairTile<T, TPR, NE>;
    constexpr int kThreads = ring_threads(TPR), kHalf = Tile::kVec / 2;
    using Rows = RowRing<T, TPR, NE, kThreads, 2>;
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ typename Rows::Shared shared;
    __shared__ __align__(16) float sh[2][kThreads / 32];
    const int lane = threadIdx.x % TPR, team = threadIdx.x / TPR;
    Rows ring;
    ring.setup({x, res}, {ldx, ldres}, ring_smem, &shared, &g_row_error, rows, D, stages);
    pdl_begin();
    pdl_trigger();
    ring.start();
    float2 pw[NE / 2], pb[NE / 2];
    Tile::load_params(pw, w, 1.0f, D, lane);
    Tile::load_params(pb, b, 0.0f, D, lane);
    const float inv_d = 1.0f / (float)D;
    y += ring.first * ldy;
    if (sum) sum += ring.first * ldsum;
    if (mean_out) mean_out += ring.first;
    if (rstd_out) rstd_out += ring.first;
    const long long ystep = ring.step * ldy, sumstep = ring.step * ldsum;
    for (int it = 0; it < ring.iters; it++, ring.at.next()) {
        ring.wait();
        typename Tile::Raw r;
        Tile::load(r, ring.row(0), D, lane);
        if (res) {
            typename Tile::Raw q;
            Tile::load(q, ring.row(1), D, lane);
#pragma unroll
            for (int j = 0; j < NE / 2; j++)
                Tile::set_pair(r, j, add2(Tile::pair(r, j), Tile::pair(q, j)));
        }
        float2 v[NE / 2], t = both(0.0f);
#pragma unroll
        for (int j = 0; j < NE / 2; j++) {
            v[j] = Tile::pair(r, j);
            t = add2(t, v[j]);
        }
        const bool real = it < ring.mine && ring.good;
        if (sum && real) Tile::store(sum, r, D, lane);
        float s[1] = {t.x + t.y};
        team_sums<TPR>(s, sh[0], team);
        ring.refill();
        const float mean = s[0] * inv_d;
        t = both(0.0f);
#pragma unroll
        for (int i = 0; i < Tile::kVecs; i++) {
            // a vector past D holds zeros and takes no part
            if (Tile::column(i, lane) < D) {
#pragma unroll
                for (int j = i * kHalf; j < (i + 1) * kHalf; j++) {
                    v[j] = add2(v[j], both(-mean));
                    t = fma2(v[j], v[j], t);
                }
            }
        }
        s[0] = t.x + t.y;
        team_sums<TPR>(s, sh[1], team);
        const float rstd = rsqrtf(s[0] * inv_d + eps);
        if (real) {
#pragma unroll
            for (int j = 0; j < NE / 2; j++)
                Tile::set_pair(r, j, fma2(mul2(v[j], both(rstd)), pw[j], pb[j]));
            Tile::store(y, r, D, lane);
            if (lane == 0) {
                if (mean_out) *mean_out = mean;
                if (rstd_out) *rstd_out = rstd;
            }
        }
        y += ystep;
        if (sum) sum += sumstep;
        if (mean_out) mean_out += ring.step;
        if (rstd_out) rstd_out += ring.step;
    }
    ring.finish();
}

// Dense rows that are no whole 16-byte vectors, groups of them through shared
// memory (GroupRing), TPR threads a row, weights and biases in registers.
// Row by row, a warp's loads are of one value a lane, 16-bit ones 64 bytes for
// a whole instruction (16771 x 2001 BF16 48.7 us, so 38.8, 53 % of the copy
// rate: the barriers' latency bounds it now).
constexpr int kGroupThreads = 512, kGroupMaxRows = 128;
template <typename T, typename WT, int TPR, int NP>
__global__ void __launch_bounds__(kGroupThreads, 1)
layernorm_group_kernel(const T *x, const T *res, T *y, T *sum, const WT *w, const WT *b,
                       float *mean_out, float *rstd_out, long long rows, int D, float eps,
                       int rows_at, int stages) {
    using Tile = WordTile<T, TPR, NP>;
    using Groups = GroupRing<T, 2>;
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ typename Groups::Shared shared;
    __shared__ __align__(16) float sh[2][kGroupThreads / 32];
    // an even number of teams: a team's rows start in the same half of a word
    const int lane = threadIdx.x % TPR, team = threadIdx.x / TPR, teams = blockDim.x / TPR;
    const Tile tile(lane, team & D & 1, D);
    Groups ring;
    ring.setup({x, res}, ring_smem, &shared, &g_row_error, rows, D, rows_at, stages);
    pdl_begin();
    pdl_trigger();
    ring.start();
    float2 pw[NP], pb[NP];
    tile.load_params(pw, w, 1.0f);
    tile.load_params(pb, b, 0.0f);
    const float inv_d = 1.0f / (float)D;
    for (int it = 0; it < ring.iters; it++) {
        ring.wait();
        const int count = ring.count(ring.group);
        const long long row0 = ring.group * rows_at;
        for (int q0 = 0; q0 < count; q0 += teams) {
            const int q = q0 + team;
            const bool real = q < count;
            T *row = ring.buffer(0) + q * D;
            typename Tile::Raw r = {};
            if (real) {
                tile.load(r, row);
                if (res) {
                    T *other = ring.buffer(1) + q * D;
                    typename Tile::Raw o;
                    tile.load(o, other);
#pragma unroll
                    for (int j = 0; j < NP; j++)
                        Tile::set_pair(r, j, add2(Tile::pair(r, j), Tile::pair(o, j)));
                    if (sum) tile.store(other, r);
                }
            }
            float2 v[NP], t = both(0.0f);
#pragma unroll
            for (int j = 0; j < NP; j++) {
                v[j] = Tile::pair(r, j);
                t = add2(t, v[j]);
            }
            float s[1] = {t.x + t.y};
            team_sums<TPR>(s, sh[0], team);
            const float mean = s[0] * inv_d;
            t = both(0.0f);
#pragma unroll
            for (int j = 0; j < NP; j++) {
                v[j] = add2(v[j], both(-mean));
                if (!tile.inside(j, 0)) v[j].x = 0.0f;
                if (!tile.inside(j, 1)) v[j].y = 0.0f;
                t = fma2(v[j], v[j], t);
            }
            s[0] = t.x + t.y;
            team_sums<TPR>(s, sh[1], team);
            const float rstd = rsqrtf(s[0] * inv_d + eps);
            if (!real) continue;
#pragma unroll
            for (int j = 0; j < NP; j++)
                Tile::set_pair(r, j, fma2(mul2(v[j], both(rstd)), pw[j], pb[j]));
            tile.store(row, r);
            if (lane == 0 && ring.good) {
                if (mean_out) mean_out[row0 + q] = mean;
                if (rstd_out) rstd_out[row0 + q] = rstd;
            }
        }
        ring.store(it, 0, y, 1, sum);
    }
    ring.finish();
}

// xh = (x - mean) rstd, the difference first: x rstd - mean rstd costs an
// instruction less, but the rounding of mean rstd is u |mean| rstd whatever
// the difference, and the product can pass FP32's range.
__device__ __forceinline__ float2 normalised(float2 x, float mean, float rstd) {
    return mul2(add2(x, both(-mean)), both(rstd));
}

// dx = rstd (g - mean(g) - xh mean(g xh)), xh as (x - mean) rstd with rstd
// taken to its factor: m1 = -mean(g) rstd, m2 = -mean(g xh) rstd.
__device__ __forceinline__ float2 dx_of(float2 x, float mean, float rstd, float2 g, float2 m1,
                                        float2 m2) {
    return fma2(fma2(add2(x, both(-mean)), m2, g), both(rstd), m1);
}

// A row's places past D hold x = 0 and g = 0, which add nothing to the row's
// sums as long as xh = -mean rstd is finite there; where it is not, the sum of
// g xh is taken again without them.
__device__ __forceinline__ bool zero_overflows(float mean, float rstd) {
    return !(fabsf(mean * rstd) < INFINITY);
}

// dx, one block per row, any width (unsigned columns as above).
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
    for (unsigned i = threadIdx.x; i < (unsigned)D; i += blockDim.x) {
        const float g = to_float(dy[i]) * weight_at(w, i, 1.0f);
        s1 += g;
        s2 += g * ((to_float(x[i]) - mean) * rstd);
    }
    const float m1 = block_sum(s1, sh) / (float)D, m2 = block_sum(s2, sh) / (float)D;
    for (unsigned i = threadIdx.x; i < (unsigned)D; i += blockDim.x) {
        const float g = to_float(dy[i]) * weight_at(w, i, 1.0f);
        const float xh = (to_float(x[i]) - mean) * rstd;
        float v = (g - m1 - xh * m2) * rstd;
        if (dsum) v += to_float(dsum[i]);
        dx[i] = from_float<T>(v);
    }
}

// dx, one block of TPR threads per row of at most TPR * NE values, read once.
// VEC: whole 16-byte vectors at aligned places.
template <typename T, typename WT, int TPR, int NE, bool VEC>
__global__ void __launch_bounds__(TPR, 1024 / TPR)
layernorm_dx_tile_kernel(const T *dy, long long lddy, const T *x, long long ldx, const T *dsum,
                         long long lddsum, T *dx, long long lddx, const WT *w,
                         const float *mean_in, const float *rstd_in, int D) {
    pdl_begin();
    pdl_trigger();
    __shared__ float sh[32];
    const int lane = threadIdx.x;
    const long long row = blockIdx.x;
    const float mean = mean_in[row], rstd = rstd_in[row], inv_d = 1.0f / (float)D;
    if constexpr (VEC) {
        using Tile = PairTile<T, TPR, NE>;
        constexpr int kHalf = Tile::kVec / 2;
        typename Tile::Raw rx, rd;
        Tile::load(rx, x + row * ldx, D, lane);
        Tile::load(rd, dy + row * lddy, D, lane);
        const bool wide = sizeof(WT) * Tile::kVec >= 16 && ((uintptr_t)w & 15) == 0;
        float2 g[NE / 2], t0 = both(0.0f), t1 = both(0.0f);
#pragma unroll
        for (int i = 0; i < Tile::kVecs; i++) {
            float2 p[kHalf];
            Tile::vector_params(p, w, 1.0f, i, D, lane, wide);
#pragma unroll
            for (int k = 0; k < kHalf; k++) {
                const int j = i * kHalf + k;
                g[j] = mul2(Tile::pair(rd, j), p[k]);
                t0 = add2(t0, g[j]);
                t1 = fma2(g[j], normalised(Tile::pair(rx, j), mean, rstd), t1);
            }
        }
        if (zero_overflows(mean, rstd)) {
            t1 = both(0.0f);
#pragma unroll
            for (int j = 0; j < NE / 2; j++)
                if (Tile::pair_column(j, lane) < D)
                    t1 = fma2(g[j], normalised(Tile::pair(rx, j), mean, rstd), t1);
        }
        const float s0 = block_sum(t0.x + t0.y, sh), s1 = block_sum(t1.x + t1.y, sh);
        const float2 m1 = both(-s0 * inv_d * rstd), m2 = both(-s1 * inv_d * rstd);
        if (dsum) Tile::load(rd, dsum + row * lddsum, D, lane);
#pragma unroll
        for (int j = 0; j < NE / 2; j++) {
            float2 v = dx_of(Tile::pair(rx, j), mean, rstd, g[j], m1, m2);
            if (dsum) v = add2(v, Tile::pair(rd, j));
            Tile::set_pair(rx, j, v);
        }
        Tile::store(dx + row * lddx, rx, D, lane);
    } else {
        using Tile = RowTile<T, TPR, NE>;
        typename Tile::Raw rx, rd;
        Tile::load(rx, x + row * ldx, D, lane);
        Tile::load(rd, dy + row * lddy, D, lane);
        float g[NE], t0 = 0.0f, t1 = 0.0f;
        Tile::load_params(g, w, 1.0f, D, lane);
#pragma unroll
        for (int j = 0; j < NE; j++) {
            g[j] *= to_float(rd.v[j]);
            t0 += g[j];
            t1 += g[j] * ((to_float(rx.v[j]) - mean) * rstd);
        }
        if (zero_overflows(mean, rstd)) {
            t1 = 0.0f;
#pragma unroll
            for (int j = 0; j < NE; j++)
                if (Tile::inside(j, D, lane)) t1 += g[j] * ((to_float(rx.v[j]) - mean) * rstd);
        }
        const float m1 = block_sum(t0, sh) * inv_d, m2 = block_sum(t1, sh) * inv_d;
        if (dsum) Tile::load(rd, dsum + row * lddsum, D, lane);
#pragma unroll
        for (int j = 0; j < NE; j++) {
            float v = (g[j] - m1 - (to_float(rx.v[j]) - mean) * rstd * m2) * rstd;
            if (dsum) v += to_float(rd.v[j]);
            rx.v[j] = from_float<T>(v);
        }
        Tile::store(dx + row * lddx, rx, D, lane);
    }
}

// Column sums of dy xh and dy over the row chunk blockIdx.y and the 32 * NE
// columns of blockIdx.x, into part[chunk][2][D]: 8 warps take the chunk's rows
// in turn, NE columns a lane.
template <typename T, int NE, bool VEC>
__global__ void __launch_bounds__(256)
layernorm_dw_column_kernel(const T *dy, long long lddy, const T *x, long long ldx,
                           const float *mean, const float *rstd, long long rows, int D,
                           long long chunk, float *part) {
    pdl_begin();
    pdl_trigger();
    __shared__ float red[2][8][32 * NE];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = blockIdx.x * 32 * NE;
    const int left = D - c0;  // the warps' rows are the columns from c0 on
    const long long r0 = blockIdx.y * chunk, r1 = min(rows, r0 + chunk);
    using Tile = std::conditional_t<VEC, PairTile<T, 32, NE>, RowTile<T, 32, NE>>;
    float sw[NE], sb[NE];
#pragma unroll
    for (int j = 0; j < NE; j++) sw[j] = sb[j] = 0.0f;
    dy += c0;
    x += c0;
#pragma unroll 2
    for (long long r = r0 + warp; r < r1; r += 8) {
        typename Tile::Raw rx, rd;
        Tile::load(rx, x + r * ldx, left, lane);
        Tile::load(rd, dy + r * lddy, left, lane);
        const float m = mean[r], s = rstd[r];
#pragma unroll
        for (int j = 0; j < NE; j++) {
            float g, v;
            if constexpr (VEC) {
                g = j % 2 ? Tile::pair(rd, j / 2).y : Tile::pair(rd, j / 2).x;
                v = j % 2 ? Tile::pair(rx, j / 2).y : Tile::pair(rx, j / 2).x;
            } else {
                g = to_float(rd.v[j]);
                v = to_float(rx.v[j]);
            }
            sw[j] += g * ((v - m) * s);
            sb[j] += g;
        }
    }
#pragma unroll
    for (int j = 0; j < NE; j++) {
        int c;
        if constexpr (VEC) c = Tile::pair_column(j / 2, lane) + j % 2;
        else c = Tile::column(j, lane);
        red[0][warp][c] = sw[j];
        red[1][warp][c] = sb[j];
    }
    __syncthreads();
    part += (long long)blockIdx.y * 2 * D + c0;
    for (int t = threadIdx.x; t < 2 * 32 * NE; t += 256) {
        const int which = t / (32 * NE), c = t % (32 * NE);
        if (c >= left) continue;
        float sum = 0.0f;
        for (int q = 0; q < 8; q++) sum += red[which][q][c];
        part[(long long)which * D + c] = sum;
    }
}

// The whole backward pass in one reading of dy and x: TPR threads hold a row
// of at most TPR * NE values, a block of kThreads goes through rows
// blockIdx.x * kRows, + gridDim.x * kRows, ... and keeps its share of the
// weights' gradients in registers, column by column.  The next rows are
// loaded while the present ones are summed.  part[block][2][D] takes the
// block's sums (null: no weights' gradients).
constexpr int bwd_threads(int tpr) { return tpr < 256 ? 256 : tpr; }
template <typename T, typename WT, int TPR, int NE>
__global__ void __launch_bounds__(bwd_threads(TPR), TPR > 256 ? 1 : 2)
layernorm_bwd_tile_kernel(const T *dy, long long lddy, const T *x, long long ldx, const T *dsum,
                          long long lddsum, T *dx, long long lddx, const WT *w,
                          const float *mean_in, const float *rstd_in, long long rows, int D,
                          float *part) {
    using Tile = RowTile<T, TPR, NE>;
    constexpr int kThreads = bwd_threads(TPR), kRows = kThreads / TPR;
    __shared__ __align__(16) float sh[2][kThreads / 32 * 2];
    __shared__ float red[kRows > 1 ? kThreads * NE : 1];
    pdl_begin();
    pdl_trigger();
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
    float p[NE], dw[NE], db[NE];
    Tile::load_params(p, w, 1.0f, D, lane);
#pragma unroll
    for (int j = 0; j < NE; j++) dw[j] = db[j] = 0.0f;

    typename Tile::Raw rx, rdy;
    float mean = 0.0f, rstd = 0.0f;
    // rows past the end are zeros with no spread: they add nothing, where a
    // repeated row with a zero factor would add NaNs for its infinities
    auto load = [&](long long row) {
        const bool real = kRows == 1 || row < rows;  // a block of one row stops before
        const long long at = real ? row : rows - 1;
        const int width = real ? D : 0;
        Tile::load(rx, x + at * ldx, width, lane);
        Tile::load(rdy, dy + at * lddy, width, lane);
        mean = real ? mean_in[at] : 0.0f;
        rstd = real ? rstd_in[at] : 0.0f;
    };
    const long long step = (long long)gridDim.x * kRows;
    long long row = (long long)blockIdx.x * kRows + group;
    int parity = 0;
    load(row);
    for (long long base = (long long)blockIdx.x * kRows; base < rows;
         base += step, row += step, parity ^= 1) {
        const bool real = kRows == 1 || row < rows;
        const float m = mean, r = rstd;
        float xh[NE], g[NE];
#pragma unroll
        for (int j = 0; j < NE; j++) {
            xh[j] = (to_float(rx.v[j]) - m) * r;
            g[j] = to_float(rdy.v[j]);
        }
        if (zero_overflows(m, r)) {
#pragma unroll
            for (int j = 0; j < NE; j++)
                if (!Tile::inside(j, D, lane)) xh[j] = 0.0f;
        }
        if (base + step < rows) load(row + step);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < NE; j++) {
            dw[j] += g[j] * xh[j];
            db[j] += g[j];
            g[j] *= p[j];
            s[0] += g[j];
            s[1] += g[j] * xh[j];
        }
        typename Tile::Raw out;
        if (dsum && real) Tile::load(out, dsum + row * lddsum, D, lane);
        team_sums<TPR>(s, sh[parity], group);
        const float m1 = s[0] / (float)D, m2 = s[1] / (float)D;
        if (real) {
#pragma unroll
            for (int j = 0; j < NE; j++) {
                float v = (g[j] - m1 - xh[j] * m2) * r;
                if (dsum) v += to_float(out.v[j]);
                out.v[j] = from_float<T>(v);
            }
            Tile::store(dx + row * lddx, out, D, lane);
        }
    }
    if (!part) return;
    part += (long long)blockIdx.x * 2 * D;
    if constexpr (kRows == 1) {
#pragma unroll
        for (int j = 0; j < NE; j++) {
            const int c = Tile::column(j, lane);
            if (c < D) {
                part[c] = dw[j];
                part[D + c] = db[j];
            }
        }
    } else {
        // the block's row groups, in order
        for (int which = 0; which < 2; which++) {
#pragma unroll
            for (int j = 0; j < NE; j++)
                red[(group * NE + j) * TPR + lane] = which ? db[j] : dw[j];
            __syncthreads();
            for (int t = threadIdx.x; t < TPR * NE; t += kThreads) {
                const int j = t / TPR, l = t % TPR;
                const int c = Tile::column(j, l);
                if (c < D) {
                    float sum = 0.0f;
                    for (int q = 0; q < kRows; q++) sum += red[q * NE * TPR + t];
                    part[which * D + c] = sum;
                }
            }
            __syncthreads();
        }
    }
}

// The same with the rows coming through rings in shared memory, as in
// layernorm_ring_kernel.
template <typename T, typename WT, int TPR, int NE>
__global__ void __launch_bounds__(ring_threads(TPR), ring_blocks(TPR))
layernorm_bwd_ring_kernel(const T *dy, long long lddy, const T *x, long long ldx, const T *dsum,
                          long long lddsum, T *dx, long long lddx, const WT *w,
                          const float *mean_in, const float *rstd_in, long long rows, int D,
                          float *part, int stages) {
    using Tile = PairTile<T, TPR, NE>;
    constexpr int kThreads = ring_threads(TPR);
    using Rows = RowRing<T, TPR, NE, kThreads, 3>;
    constexpr int kRows = Rows::kRows;
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ typename Rows::Shared shared;
    __shared__ __align__(16) float sh[2][kThreads / 32 * 2];
    const int lane = threadIdx.x % TPR, team = threadIdx.x / TPR;
    Rows ring;
    ring.setup({x, dy, dsum}, {ldx, lddy, lddsum}, ring_smem, &shared, &g_row_error, rows, D,
               stages);
    pdl_begin();
    pdl_trigger();
    ring.start();
    float2 p[NE / 2], dw[NE / 2], db[NE / 2];
    Tile::load_params(p, w, 1.0f, D, lane);
#pragma unroll
    for (int j = 0; j < NE / 2; j++) dw[j] = db[j] = both(0.0f);
    const float inv_d = 1.0f / (float)D;
    // the rows' statistics, two iterations ahead: a load queues behind the
    // stores before it
    float mean[2] = {}, rstd[2] = {};
    mean_in += ring.first;
    rstd_in += ring.first;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        if (k < ring.mine) {
            mean[k] = *mean_in;
            rstd[k] = *rstd_in;
        }
        mean_in += ring.step;
        rstd_in += ring.step;
    }
    dx += ring.first * lddx;
    const long long dxstep = ring.step * lddx;
    for (int it = 0; it < ring.iters; it++, ring.at.next(), dx += dxstep) {
        ring.wait();
        const float r = rstd[0], m = mean[0];
        mean[0] = mean[1];
        rstd[0] = rstd[1];
        if (it + 2 < ring.mine) {
            mean[1] = *mean_in;
            rstd[1] = *rstd_in;
        }
        mean_in += ring.step;
        rstd_in += ring.step;
        const bool real = it < ring.mine;
        typename Tile::Raw rx, rdy, out;
        // xh and g rstd + dsum are kept in place of x, g and dsum, which nothing
        // is spilled for (4096 x 8192 FP32 89.4 us, with the three kept 108);
        // 16-bit rows of 512 threads take x - mean twice (8192 x 8192 BF16
        // 94.2 us, 96.0 with xh kept)
        constexpr bool kKeep = sizeof(T) == 4 || TPR < 512;
        float2 xh[kKeep ? NE / 2 : 1], g[NE / 2], t0 = both(0.0f), t1 = both(0.0f);
        if (real) {
            Tile::load(rx, ring.row(0), D, lane);
            Tile::load(rdy, ring.row(1), D, lane);
            if (dsum) Tile::load(out, ring.row(2), D, lane);
#pragma unroll
            for (int j = 0; j < NE / 2; j++) {
                // (a vector past D, all zeros, keeps its zeros: xh stays finite)
                const float off = Tile::column(j / (Tile::kVec / 2), lane) < D ? m : 0.0f;
                const float2 h = normalised(Tile::pair(rx, j), off, r);
                const float2 d = Tile::pair(rdy, j);
                dw[j] = fma2(d, h, dw[j]);
                db[j] = add2(db[j], d);
                g[j] = mul2(d, p[j]);
                t0 = add2(t0, g[j]);
                t1 = fma2(g[j], h, t1);
                if constexpr (kKeep) {
                    xh[j] = h;
                    g[j] = mul2(g[j], both(r));
                    if (dsum) g[j] = add2(g[j], Tile::pair(out, j));
                }
            }
        }
        float s[2] = {t0.x + t0.y, t1.x + t1.y};
        team_sums<TPR>(s, sh[it & 1], team);
        ring.refill();
        const float2 m1 = both(-s[0] * inv_d * r), m2 = both(-s[1] * inv_d * r);
        if (real && ring.good) {
#pragma unroll
            for (int j = 0; j < NE / 2; j++) {
                float2 v;
                if constexpr (kKeep) {
                    v = add2(g[j], fma2(xh[j], m2, m1));
                } else {
                    v = dx_of(Tile::pair(rx, j), m, r, g[j], m1, m2);
                    if (dsum) v = add2(v, Tile::pair(out, j));
                }
                Tile::set_pair(out, j, v);
            }
            Tile::store(dx, out, D, lane);
        }
    }
    ring.finish();
    if (!part) return;
    part += (long long)blockIdx.x * 2 * D;
    if constexpr (kRows == 1) {
#pragma unroll
        for (int j = 0; j < NE / 2; j++) {
            const int c = Tile::pair_column(j, lane);
            if (c < D) {
                part[c] = dw[j].x;
                part[c + 1] = dw[j].y;
                part[D + c] = db[j].x;
                part[D + c + 1] = db[j].y;
            }
        }
    } else {
        // the block's rows' sums in order, through the ring (all copies landed)
        float2 *red = reinterpret_cast<float2 *>(ring_smem);
        for (int which = 0; which < 2; which++) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NE / 2; j++)
                red[(team * (NE / 2) + j) * TPR + lane] = which ? db[j] : dw[j];
            __syncthreads();
            for (int t = threadIdx.x; t < TPR * NE / 2; t += kThreads) {
                const int c = Tile::pair_column(t / TPR, t % TPR);
                if (c < D) {
                    float2 sum = both(0.0f);
                    for (int q = 0; q < kRows; q++) sum = add2(sum, red[q * (NE / 2) * TPR + t]);
                    part[which * D + c] = sum.x;
                    part[which * D + c + 1] = sum.y;
                }
            }
        }
    }
}

// The same for dense rows that are no whole 16-byte vectors, groups of them
// through shared memory as in layernorm_group_kernel.
template <typename T, typename WT, int TPR, int NP>
__global__ void __launch_bounds__(kGroupThreads, 1)
layernorm_bwd_group_kernel(const T *dy, const T *x, const T *dsum, T *dx, const WT *w,
                           const float *mean_in, const float *rstd_in, long long rows, int D,
                           float *part, int rows_at, int stages) {
    using Tile = WordTile<T, TPR, NP>;
    using Groups = GroupRing<T, 3>;
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ typename Groups::Shared shared;
    __shared__ __align__(16) float sh[2][kGroupThreads / 32 * 2];
    __shared__ float2 stats[2][kGroupMaxRows];  // the present group's and the next one's
    // an even number of teams: a team's rows start in the same half of a word
    const int lane = threadIdx.x % TPR, team = threadIdx.x / TPR, teams = blockDim.x / TPR;
    const Tile tile(lane, team & D & 1, D);
    Groups ring;
    ring.setup({x, dy, dsum}, ring_smem, &shared, &g_row_error, rows, D, rows_at, stages);
    pdl_begin();
    pdl_trigger();
    ring.start();
    float2 p[NP], dw[NP], db[NP];
    tile.load_params(p, w, 1.0f);
#pragma unroll
    for (int j = 0; j < NP; j++) dw[j] = db[j] = both(0.0f);
    // thread q looks after row q's statistics, a group ahead
    float2 next = both(0.0f);
    auto look = [&](long long group) {
        const long long row = group * rows_at + threadIdx.x;
        if ((int)threadIdx.x < rows_at && row < rows) next = make_float2(mean_in[row], rstd_in[row]);
    };
    look(ring.group);
    const float inv_d = 1.0f / (float)D;
    int parity = 0;
    for (int it = 0; it < ring.iters; it++) {
        if ((int)threadIdx.x < rows_at) stats[it & 1][threadIdx.x] = next;
        look(ring.group + gridDim.x);
        ring.wait();
        __syncthreads();
        const int count = ring.count(ring.group);
        for (int q0 = 0; q0 < count; q0 += teams, parity ^= 1) {
            const int q = q0 + team;
            const bool real = q < count;
            T *row = ring.buffer(0) + q * D;
            typename Tile::Raw rx = {}, rd = {};
            float2 xh[NP], g[NP], t0 = both(0.0f), t1 = both(0.0f);
            float r = 0.0f;
            if (real) {
                tile.load(rx, row);
                tile.load(rd, ring.buffer(1) + q * D);
                const float m = stats[it & 1][q].x;
                r = stats[it & 1][q].y;
#pragma unroll
                for (int j = 0; j < NP; j++) {
                    // (a place outside the row, a zero, keeps it: xh stays finite)
                    const float2 c = fma2(tile.ones(j), both(-m), Tile::pair(rx, j));
                    xh[j] = mul2(c, both(r));
                    const float2 d = Tile::pair(rd, j);
                    dw[j] = fma2(d, xh[j], dw[j]);
                    db[j] = add2(db[j], d);
                    g[j] = mul2(d, p[j]);
                    t0 = add2(t0, g[j]);
                    t1 = fma2(g[j], xh[j], t1);
                }
            }
            float s[2] = {t0.x + t0.y, t1.x + t1.y};
            team_sums<TPR>(s, sh[parity], team);
            if (!real) continue;
            const float2 m1 = both(-s[0] * inv_d * r), m2 = both(-s[1] * inv_d * r);
            if (dsum) tile.load(rd, ring.buffer(2) + q * D);
#pragma unroll
            for (int j = 0; j < NP; j++) {
                float2 v = fma2(g[j], both(r), fma2(xh[j], m2, m1));
                if (dsum) v = add2(v, Tile::pair(rd, j));
                Tile::set_pair(rx, j, v);
            }
            tile.store(row, rx);
        }
        ring.store(it, 0, dx, 0, nullptr);
    }
    ring.finish();
    if (!part) return;
    part += (long long)blockIdx.x * 2 * D;
    // the teams' sums in order, through the ring (all its copies are done)
    float *red = reinterpret_cast<float *>(ring_smem);
    for (int which = 0; which < 2; which++) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NP; j++)
            reinterpret_cast<float2 *>(red)[(team * NP + j) * TPR + lane] = which ? db[j] : dw[j];
        __syncthreads();
        for (int c = threadIdx.x; c < D; c += blockDim.x) {
            float total = 0.0f;
            for (int q = 0; q < teams; q++)
                total += red[q * NP * TPR * 2 + Tile::place(c, q & D & 1)];
            part[which * D + c] = total;
        }
    }
}

// dw (blockIdx.y 0) and db (1): the parts' sums, 32 columns a block, 8
// threads a column, each every eighth part, then the 8 in order.
template <typename WT>
__global__ void __launch_bounds__(256) layernorm_dw_sum_kernel(const float *part, int parts, int D,
                                                               WT *dw, WT *db) {
    pdl_begin();
    pdl_trigger();
    __shared__ float sh[8][32];
    WT *out = blockIdx.y ? db : dw;
    if (!out) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (c < D) {
        const float *p = part + (long long)blockIdx.y * D + c;
#pragma unroll 8
        for (int q = warp; q < parts; q += 8) s += p[(long long)q * 2 * D];
    }
    sh[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < D) {
        for (int q = 1; q < 8; q++) s += sh[q][lane];
        out[c] = from_float<WT>(s);
    }
}

// blocks that keep column sums, at most: two on each of 148 SMs
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

// the ring kernels: SMs, shared memory of a block's ring, and the threads of
// a row of D values, NE each
constexpr int kSms = 148;
constexpr int ring_bytes(int tpr) { return 216 * 1024 / ring_blocks(tpr) - 4096; }
template <int NE, typename F>
bool ring_dispatch(int D, F f) {
    if (D <= 4 * NE) return f(Int<4>{});
    if (D <= 8 * NE) return f(Int<8>{});
    if (D <= 16 * NE) return f(Int<16>{});
    if (D <= 32 * NE) return f(Int<32>{});
    if (D <= 64 * NE) return f(Int<64>{});
    if (D <= 128 * NE) return f(Int<128>{});
    if (D <= 256 * NE) return f(Int<256>{});
    if (D <= 512 * NE) return f(Int<512>{});
    return false;
}

// How groups of rows are taken by teams of tpr threads: whole 16-byte vectors
// together, a row for every team, and 8 KB (a shorter copy is not worth its
// barrier).  `read` matrices go through the ring, of at least 3 stages: one in
// work, one leaving, one coming.  `most` blocks of 256 threads on an SM, when
// their rings fit, or two, or one of 512: a block that waits at its barriers
// leaves the SM to the others (50000 x 1153 FP16 forward 63 us with three,
// with one 90; backward 200000 x 257 BF16 108 with two, with one 142).  False when a matrix is neither
// null nor dense and 16-byte aligned, or nothing fits.
struct Groups {
    int rows_at, stages, threads;
    unsigned grid;
    size_t smem;
};
constexpr int kGroupSmem = 212 * 1024;
bool group_shape(Groups &g, std::initializer_list<const Rows *> all, int read, long long rows,
                 int D, int size, int tpr, int most) {
    for (const Rows *m : all)
        if (m->p && ((uintptr_t)m->p & 15 || (rows > 1 && m->ld != D))) return false;
    for (int blocks = tpr > kGroupThreads / 4 ? 1 : most; blocks > 0; blocks--) {
        const int threads = blocks > 1 ? kGroupThreads / 2 : kGroupThreads;
        int at = threads / tpr;
        while (at <= kGroupMaxRows &&
               ((long long)at * D * size % 16 || (long long)at * D * size < 8192))
            at *= 2;
        const long long stage = (long long)read * at * D * size;
        const long long fit = (blocks == 1 ? kGroupSmem : blocks == 2 ? 110 * 1024 : 72 * 1024) / stage;
        if (at > kGroupMaxRows || fit < 3) continue;
        g.rows_at = at;
        g.stages = fit > kRingStages ? kRingStages : (int)fit;
        g.threads = threads;
        const long long groups = (rows + at - 1) / at;
        g.grid = (unsigned)(groups < kSms * blocks ? groups : kSms * blocks);
        g.smem = (size_t)g.stages * stage;
        return true;
    }
    return false;
}
// f(TPR, NP) with the fewest places for rows of D (NARROW: from 33 on, else
// from 257 on) that keeps WordTile's promise
template <bool NARROW, typename F>
bool group_dispatch(int D, F &&f) {
    if constexpr (NARROW) {
        if (D <= 80) return f(Int<8>{}, Int<5>{});
        if (D <= 160) return f(Int<16>{}, Int<5>{});
    }
    if (D <= 320) return f(Int<32>{}, Int<5>{});
    if (D <= 512) return f(Int<32>{}, Int<8>{});
    if (D <= 640) return f(Int<64>{}, Int<5>{});
    if (D <= 1024) return f(Int<64>{}, Int<8>{});
    if (D <= 1280) return f(Int<128>{}, Int<5>{});
    if (D <= 2048) return f(Int<128>{}, Int<8>{});
    if (D <= 2560) return f(Int<256>{}, Int<5>{});
    if (D <= 4096) return f(Int<256>{}, Int<8>{});
    return false;
}

template <typename T>
T *ptr(const Rows &r) { return (T *)r.p; }

}  // namespace

int row_error_fetch_and_clear() {
    int h = 0, zero = 0;
    cudaMemcpyFromSymbol(&h, g_row_error, sizeof(int));
    if (h) cudaMemcpyToSymbol(g_row_error, &zero, sizeof(int));
    return h;
}

Status launch_layernorm(const LayerNormArgs &a, cudaStream_t st) {
    if (a.rows == 0) return OK;
    if (a.rows < 0 || a.rows > 0x7fffffffLL || a.D <= 0) return ERR_SHAPE;
    return with_types(a.type, a.w_type, [&](auto t, auto wt) {
        using T = decltype(t);
        using WT = decltype(wt);
        const int size = (int)sizeof(T);
        const bool vec = vector_rows(a.x.p, a.x.ld, a.rows, a.D, size) &&
                         vector_rows(a.res.p, a.res.ld, a.rows, a.D, size) &&
                         vector_rows(a.y.p, a.y.ld, a.rows, a.D, size) &&
                         vector_rows(a.sum.p, a.sum.ld, a.rows, a.D, size);
        auto tile = [&](auto tpr, auto ne, auto vector) {
            constexpr int TPR = decltype(tpr)::value, NE = decltype(ne)::value;
            constexpr int kThreads = TPR < 128 ? 128 : TPR;
            constexpr bool VEC = decltype(vector)::value != 0;
            auto kernel = [&] {
                if constexpr (VEC) return layernorm_vector_kernel<T, WT, TPR, NE>;
                else return layernorm_tile_kernel<T, WT, TPR, NE>;
            }();
            pdl_launch(kernel, (unsigned)cdiv(a.rows, kThreads / TPR), kThreads, 0, st,
                       (const T *)a.x.p, a.x.ld, (const T *)a.res.p, a.res.ld, ptr<T>(a.y), a.y.ld,
                       ptr<T>(a.sum), a.sum.ld, (const WT *)a.weight, (const WT *)a.bias, a.mean,
                       a.rstd, a.rows, a.D, a.eps);
            return cuda_status();
        };
        constexpr int kRingNE = 16;
        auto ring = [&](auto tpr) {
            constexpr int TPR = decltype(tpr)::value, kThreads = ring_threads(TPR);
            using Rows = RowRing<T, TPR, kRingNE, kThreads, 2>;
            auto kernel = layernorm_ring_kernel<T, WT, TPR, kRingNE>;
            const long long stage = Rows::block_stage(a.res.p ? 2 : 1, a.D);
            const int stages = ring_stages(ring_bytes(TPR), stage);
            constexpr int kBlocks = kSms * ring_blocks(TPR);
            // at least 4 rows for each place in a block, or the tile's blocks
            // are done before the rings are set up
            if (a.rows < 4LL * kBlocks * Rows::kRows || stages < 2 ||
                !smem_attr_once((const void *)kernel, ring_bytes(TPR)))
                return false;
            pdl_launch(kernel, (unsigned)kBlocks, kThreads, (size_t)(stages * stage), st,
                       (const T *)a.x.p, a.x.ld, (const T *)a.res.p, a.res.ld, ptr<T>(a.y), a.y.ld,
                       ptr<T>(a.sum), a.sum.ld, (const WT *)a.weight, (const WT *)a.bias, a.mean,
                       a.rstd, a.rows, a.D, a.eps, stages);
            return true;
        };
        // wide 16-bit rows gain from the rings (16384 x 2000 28.8 us, 31.6
        // without; 4096 x 8192 33.0 / 36.8); shorter ones do not (20000 x 768
        // 17.9 / 16.2), nor do FP32 ones (52500 x 256 36.9 / 33.7)
        if constexpr (sizeof(T) == 2) {
            if (vec && a.D > 1024 &&
                (a.D <= 2048 ? ring(Int<128>{}) : a.D <= 4096 ? ring(Int<256>{})
                 : a.D <= 8192 ? ring(Int<512>{}) : false))
                return cuda_status();
        }
        auto group = [&](auto tpr, auto np) {
            constexpr int TPR = decltype(tpr)::value, NP = decltype(np)::value;
            Groups g;
            auto kernel = layernorm_group_kernel<T, WT, TPR, NP>;
            if (!group_shape(g, {&a.x, &a.res, &a.y, &a.sum}, a.res.p ? 2 : 1, a.rows, a.D, size,
                             TPR, NP > 5 ? 2 : 3) ||
                !smem_attr_once((const void *)kernel, kGroupSmem))
                return false;
            pdl_launch(kernel, g.grid, g.threads, g.smem, st, (const T *)a.x.p,
                       (const T *)a.res.p, ptr<T>(a.y), ptr<T>(a.sum), (const WT *)a.weight,
                       (const WT *)a.bias, a.mean, a.rstd, a.rows, a.D, a.eps, g.rows_at, g.stages);
            return true;
        };
        // other dense rows through groups (16771 x 2001 BF16 38.8 us, by the
        // tile 48.7; 29104 x 1153 40.2 / 49.9; 52350 x 641 FP32 56.6 / 85.5),
        // unless they are narrow (200000 x 100 BF16 33.0 / 31.4) or few (2043 x
        // 257 3.6 / 2.5; the switch is below the crossover: 3640 x 1153, a
        // group's, 8.9 / 7.5), or FP32 with a residual (29101 x 1153 96 / 80:
        // three stages of two matrices leave one block an SM)
        if (!vec && a.D > 256 && a.rows * a.D >= 1 << 22 && !(sizeof(T) == 4 && a.res.p) &&
            group_dispatch<false>(a.D, group))
            return cuda_status();
        // the smallest tile that holds the row, in vectors 64 bytes a thread
        // (rows up to 256 values half of that)
        constexpr int NE = sizeof(T) == 2 ? 32 : 16, F = sizeof(T) == 2 ? 1 : 2;
        constexpr Int<1> vector;
        constexpr Int<0> single;
        bool some = true;
        if (vec) {
            if (a.D <= 64) tile(Int<4>{}, Int<16>{}, vector);
            else if (a.D <= 128) tile(Int<8>{}, Int<16>{}, vector);
            else if (a.D <= 256) tile(Int<16>{}, Int<16>{}, vector);
            else if (a.D <= 512) tile(Int<16 * F>{}, Int<NE>{}, vector);
            else if (a.D <= 1024) tile(Int<32 * F>{}, Int<NE>{}, vector);
            else if (a.D <= 2048) tile(Int<64 * F>{}, Int<NE>{}, vector);
            else if (a.D <= 4096) tile(Int<128 * F>{}, Int<NE>{}, vector);
            else if (a.D <= 8192) tile(Int<256 * F>{}, Int<NE>{}, vector);
            else if (a.D <= 16384) tile(Int<512 * F>{}, Int<NE>{}, vector);
            else if (a.D <= 1024 * NE && sizeof(T) == 2) tile(Int<1024>{}, Int<NE>{}, vector);
            else some = false;
        } else {
            if (a.D <= 64) tile(Int<4>{}, Int<16>{}, single);
            else if (a.D <= 128) tile(Int<8>{}, Int<16>{}, single);
            else if (a.D <= 256) tile(Int<16>{}, Int<16>{}, single);
            else if (a.D <= 320) tile(Int<32>{}, Int<10>{}, single);
            else if (a.D <= 512) tile(Int<32>{}, Int<16>{}, single);
            else if (a.D <= 640) tile(Int<64>{}, Int<10>{}, single);
            else if (a.D <= 1024) tile(Int<64>{}, Int<16>{}, single);
            else if (a.D <= 1280) tile(Int<128>{}, Int<10>{}, single);
            else if (a.D <= 2048) tile(Int<128>{}, Int<16>{}, single);
            else if (a.D <= 2560) tile(Int<256>{}, Int<10>{}, single);
            else if (a.D <= 4096) tile(Int<256>{}, Int<16>{}, single);
            else if (a.D <= 5120) tile(Int<512>{}, Int<10>{}, single);
            else if (a.D <= 8192) tile(Int<512>{}, Int<16>{}, single);
            else if (a.D <= 10240) tile(Int<1024>{}, Int<10>{}, single);
            else if (a.D <= 16384) tile(Int<1024>{}, Int<16>{}, single);
            else some = false;
        }
        if (some) return cuda_status();
        pdl_launch(layernorm_row_kernel<T, WT>, (unsigned)a.rows, 512, 0, st,
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
        const int size = (int)sizeof(T);
        const bool vec = vector_rows(a.dy.p, a.dy.ld, a.rows, a.D, size) &&
                         vector_rows(a.x.p, a.x.ld, a.rows, a.D, size) &&
                         vector_rows(a.dx.p, a.dx.ld, a.rows, a.D, size) &&
                         vector_rows(a.dsum.p, a.dsum.ld, a.rows, a.D, size);
        const bool grads = a.dweight || a.dbias;
        int parts = 0;
        auto tile = [&](auto tpr, auto ne) {
            constexpr int TPR = decltype(tpr)::value, NE = decltype(ne)::value;
            constexpr int kThreads = bwd_threads(TPR), kRows = kThreads / TPR;
            auto kernel = layernorm_bwd_tile_kernel<T, WT, TPR, NE>;
            const int most = TPR > 256 ? kMaxParts / 2 : kMaxParts;
            const long long blocks = (a.rows + kRows - 1) / kRows;
            parts = (int)(blocks < most ? blocks : most);
            pdl_launch(kernel, (unsigned)parts, kThreads, 0, st, (const T *)a.dy.p, a.dy.ld,
                       (const T *)a.x.p, a.x.ld, (const T *)a.dsum.p, a.dsum.ld, ptr<T>(a.dx),
                       a.dx.ld, (const WT *)a.weight, a.mean, a.rstd, a.rows, a.D,
                       grads ? a.work : nullptr);
        };
        auto ring = [&](auto tpr, auto ne) {
            constexpr int TPR = decltype(tpr)::value, NE = decltype(ne)::value, kThreads = ring_threads(TPR);
            using Rows = RowRing<T, TPR, NE, kThreads, 3>;
            auto kernel = layernorm_bwd_ring_kernel<T, WT, TPR, NE>;
            const long long stage = Rows::block_stage(a.dsum.p ? 3 : 2, a.D);
            const int stages = ring_stages(ring_bytes(TPR), stage);
            if (stages < 2 || !smem_attr_once((const void *)kernel, ring_bytes(TPR))) return false;
            const long long reduce = Rows::kRows > 1 ? kThreads * NE * 4 : 0;
            const long long smem = stages * stage > reduce ? stages * stage : reduce;
            const long long blocks = (a.rows + Rows::kRows - 1) / Rows::kRows;
            constexpr int kBlocks = kSms * ring_blocks(TPR);
            parts = (int)(blocks < kBlocks ? blocks : kBlocks);
            pdl_launch(kernel, (unsigned)parts, kThreads, (size_t)smem, st, (const T *)a.dy.p,
                       a.dy.ld, (const T *)a.x.p, a.x.ld, (const T *)a.dsum.p, a.dsum.ld,
                       ptr<T>(a.dx), a.dx.ld, (const WT *)a.weight, a.mean, a.rstd, a.rows, a.D,
                       grads ? a.work : nullptr, stages);
            return true;
        };
        auto group = [&](auto tpr, auto np) {
            constexpr int TPR = decltype(tpr)::value, NP = decltype(np)::value;
            Groups g;
            auto kernel = layernorm_bwd_group_kernel<T, WT, TPR, NP>;
            if (!group_shape(g, {&a.x, &a.dy, &a.dsum, &a.dx}, a.dsum.p ? 3 : 2, a.rows, a.D, size,
                             TPR, 2) ||
                !smem_attr_once((const void *)kernel, kGroupSmem))
                return false;
            parts = (int)g.grid;
            const size_t reduce = (size_t)g.threads * NP * 8;
            pdl_launch(kernel, g.grid, g.threads, g.smem > reduce ? g.smem : reduce, st,
                       (const T *)a.dy.p, (const T *)a.x.p, (const T *)a.dsum.p, ptr<T>(a.dx),
                       (const WT *)a.weight, a.mean, a.rstd, a.rows, a.D, grads ? a.work : nullptr,
                       g.rows_at, g.stages);
            return true;
        };
        // two vectors a thread: 16 values of 16 bits or 8 of 32 (with 16, FP32
        // rows spill; wider than 4096 they have to)
        constexpr int kNE = 32 / (int)sizeof(T);
        // dense rows that are no vectors go through groups (50000 x 1153 FP16
        // 95.5 us, 142 by the tile; FP32 122 / 171; 200000 x 79 BF16 36 / 73;
        // 16761 x 1001 34 / 36.4), unless they are narrow (200000 x 51 BF16 36 /
        // 26) or few (the switch is below the crossover: 4191 x 1001, a
        // group's, 17.7 / 14.9)
        const bool done =
            a.rows == 0 ||
            (vec ? ring_dispatch<kNE>(a.D, [&](auto tpr) { return ring(tpr, Int<kNE>{}); }) ||
                       (sizeof(T) == 4 && a.D > 4096 && a.D <= 8192 && ring(Int<512>{}, Int<16>{}))
                 : a.D > 64 && a.rows * a.D >= 1 << 22 && group_dispatch<true>(a.D, group));
        if (done) {
        } else if (a.D <= 64) {
            tile(Int<8>{}, Int<8>{});
        } else if (a.D <= 256) {
            tile(Int<32>{}, Int<8>{});
        } else if (a.D <= 320) {
            tile(Int<64>{}, Int<5>{});
        } else if (a.D <= 512) {
            tile(Int<64>{}, Int<8>{});
        } else if (a.D <= 640) {
            tile(Int<128>{}, Int<5>{});
        } else if (a.D <= 1024) {
            tile(Int<128>{}, Int<8>{});
        } else if (a.D <= 1280) {
            tile(Int<256>{}, Int<5>{});
        } else if (a.D <= 2048) {
            tile(Int<256>{}, Int<8>{});
        } else if (a.D <= 2560) {
            tile(Int<512>{}, Int<5>{});
        } else if (a.D <= 4096) {
            tile(Int<512>{}, Int<8>{});
        } else {
            // two readings: dx row by row, the weights' gradients column by
            // column (14000 x 4097 BF16 208 us, in one reading with 1024
            // threads a row and one block an SM 397; 100 x 5001 FP32 7.8 / 12)
            auto dx = [&](auto kernel, int threads) {
                pdl_launch(kernel, (unsigned)a.rows, threads, 0, st, (const T *)a.dy.p, a.dy.ld,
                           (const T *)a.x.p, a.x.ld, (const T *)a.dsum.p, a.dsum.ld, ptr<T>(a.dx),
                           a.dx.ld, (const WT *)a.weight, a.mean, a.rstd, a.D);
            };
            auto column = [&](auto kernel, int ne) {
                // some 8 blocks of 8 warps an SM, at least 16 chunks of rows
                const long long across = (a.D + 32 * ne - 1) / (32 * ne);
                const long long want = (8 * kSms + across - 1) / across;
                const long long most = row_parts(a.rows);
                const long long n = want < 16 ? 16 : want, cut = n < most ? n : most;
                const long long chunk = (a.rows + cut - 1) / cut;
                parts = (int)((a.rows + chunk - 1) / chunk);
                pdl_launch(kernel, dim3((unsigned)across, parts), 256, 0, st, (const T *)a.dy.p,
                           a.dy.ld, (const T *)a.x.p, a.x.ld, a.mean, a.rstd, a.rows, a.D, chunk,
                           a.work);
            };
            if (vec && a.D <= 16384) dx(layernorm_dx_tile_kernel<T, WT, 1024, 16, true>, 1024);
            else if (!vec && a.D <= 5120) dx(layernorm_dx_tile_kernel<T, WT, 512, 10, false>, 512);
            else if (!vec && a.D <= 8192) dx(layernorm_dx_tile_kernel<T, WT, 512, 16, false>, 512);
            else if (!vec && a.D <= 10240) dx(layernorm_dx_tile_kernel<T, WT, 1024, 10, false>, 1024);
            else if (!vec && a.D <= 16384) dx(layernorm_dx_tile_kernel<T, WT, 1024, 16, false>, 1024);
            else dx(layernorm_dx_row_kernel<T, WT>, 512);
            constexpr int kVec = 16 / (int)sizeof(T);
            if (grads && vec) column(layernorm_dw_column_kernel<T, kVec, true>, kVec);
            else if (grads) column(layernorm_dw_column_kernel<T, 4, false>, 4);
        }
        if (grads)
            pdl_launch(layernorm_dw_sum_kernel<WT>, dim3(cdiv(a.D, 32), 2), 256, 0, st, a.work,
                       parts, a.D, (WT *)a.dweight, (WT *)a.dbias);
        return cuda_status();
    });
}

}  // namespace ppdl
