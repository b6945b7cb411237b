// quantize.cu — 8-bit rows with a scale each: scale = max |x| / 127,
// q = x / scale rounded half to even on the exact quotient.
//
// Memory bounds it (a row stays in registers between its maximum and its
// quotients): 8192 x 8192 BF16 46 us, 4.4 TB/s; 52500 x 256 FP32 10.5 us, its
// input partly in L2.
#include "block.cuh"
#include "block.h"
#include "quantize.cuh"
#include "rows.cuh"

namespace ppdl {

namespace {

template <int TPR>
__device__ __forceinline__ unsigned row_max(unsigned m, unsigned *sh) {
    constexpr int kWidth = TPR < 32 ? TPR : 32;
#pragma unroll
    for (int o = kWidth / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if constexpr (TPR > 32) {
        if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = m;
        __syncthreads();
        sh += threadIdx.x / TPR * (TPR / 32);  // the row's warps
#pragma unroll
        for (int w = 0; w < TPR / 32; w++) m = max(m, sh[w]);
    }
    return m;
}

// The bits of the largest |v| of a word of values (two 16-bit ones, or one).
template <typename T>
struct AbsMax {
    uint32_t m = 0;
    __device__ __forceinline__ void add(uint32_t w) { m = max(m, w & 0x7fffffffu); }
    __device__ __forceinline__ unsigned bits() const { return m; }
};
template <>
struct AbsMax<__nv_bfloat16> {
    uint32_t m = 0;
    __device__ __forceinline__ void add(uint32_t w) { m = __vmaxu2(m, w & 0x7fff7fffu); }
    __device__ __forceinline__ unsigned bits() const { return max(m & 0xffffu, m >> 16) << 16; }
};
template <>
struct AbsMax<__half> {
    uint32_t m = 0;
    __device__ __forceinline__ void add(uint32_t w) { m = __vmaxu2(m, w & 0x7fff7fffu); }
    __device__ __forceinline__ unsigned bits() const {
        return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(m & 0xffffu, m >> 16))));
    }
};

// Rows of whole 16-byte vectors in registers.  The quotient is first taken
// as x (1 / s), off by at most 127 x 2^-23 = 1.6e-5, and rounded by adding
// 1.5 x 2^23, which leaves the whole number in the low byte.  Values that
// close to a half decide on their remainders, pair by pair: in 16-bit rows
// half the largest value (63.5 steps) alone makes them common, one in some
// hundreds, so that most warps have one and few pairs do.
template <typename T, int TPR, int NE>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, 1024 / (TPR < 128 ? 128 : TPR))
quantize_vector_kernel(const T *x, long long ldx, long long rows, int K, int8_t *q, long long ldq,
                       float *scale) {
    using Tile = PairTile<T, TPR, NE>;
    pdl_begin();
    pdl_trigger();
    __shared__ unsigned sh[32];
    constexpr int kRows = TPR < 128 ? 128 / TPR : 1, kWords = Tile::kVecs * 4;
    const int lane = threadIdx.x % TPR;
    long long row = (long long)blockIdx.x * kRows + threadIdx.x / TPR;
    const bool real = row < rows;
    if (!real) row = rows - 1;
    typename Tile::Raw r;
    Tile::load(r, x + row * ldx, K, lane);
    AbsMax<T> most;
#pragma unroll
    for (int k = 0; k < kWords; k++) most.add(Tile::word(r, k));
    const Divisor d(row_max<TPR>(most.bits(), sh));
    if (!real) return;
    if (lane == 0) scale[row] = d.s;
    q += row * ldq;
    constexpr float kNear = 0.49998f;
    const float2 inv = both(d.inv), magic = both(12582912.0f);
    // the rounded pair's bits, and how far its quotients are from whole numbers
    auto round_pair = [&](int j, float2 &m) {
        const float2 t = mul2(Tile::pair(r, j), inv);
        m = add2(t, magic);
        const float2 off = add2(t, sub2(magic, m));
        return fmaxf(fabsf(off.x), fabsf(off.y));
    };
    float far = 0.0f;
    uint32_t out[NE / 4];
#pragma unroll
    for (int j = 0; j < NE / 2; j += 2) {
        float2 m0, m1;
        far = fmaxf(far, round_pair(j, m0));
        far = fmaxf(far, round_pair(j + 1, m1));
        const uint32_t lo = __byte_perm(__float_as_uint(m0.x), __float_as_uint(m0.y), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(m1.x), __float_as_uint(m1.y), 0x0040);
        out[j / 2] = __byte_perm(lo, hi, 0x5410);
    }
    auto exact_pair = [&](int j) {
        const float2 v = Tile::pair(r, j);
        const uint32_t b = (uint32_t)(d(v.x) & 255) | (uint32_t)(d(v.y) & 255) << 8;
        out[j / 2] = __byte_perm(out[j / 2], b, j & 1 ? 0x5410 : 0x3254);
    };
    if (!d.usable || d.up != 1.0f) {
        // zeros, infinities and NaNs, or a scale below 2^-64
#pragma unroll
        for (int j = 0; j < NE / 2; j++) exact_pair(j);
    } else if (far > kNear) {
#pragma unroll
        for (int j = 0; j < NE / 2; j++) {
            float2 m;
            if (round_pair(j, m) > kNear) exact_pair(j);
        }
    }
#pragma unroll
    for (int i = 0; i < Tile::kVecs; i++) {
        const int c = Tile::column(i, lane);
        if (c >= K) continue;
        if constexpr (Tile::kVec == 8)
            *reinterpret_cast<uint2 *>(q + c) = make_uint2(out[2 * i], out[2 * i + 1]);
        else
            *reinterpret_cast<uint32_t *>(q + c) = out[i];
    }
}

// Rows in registers, any alignment; a thread's neighbouring values leave as
// one store of 4 bytes.
template <typename T, int TPR, int NE>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR)
quantize_tile_kernel(const T *x, long long ldx, long long rows, int K, int8_t *q, long long ldq,
                     float *scale) {
    using Tile = RowTile<T, TPR, NE, 4>;
    pdl_begin();
    pdl_trigger();
    __shared__ unsigned sh[32];
    constexpr int kRows = TPR < 128 ? 128 / TPR : 1;
    const int lane = threadIdx.x % TPR;
    long long row = (long long)blockIdx.x * kRows + threadIdx.x / TPR;
    const bool real = row < rows;
    if (!real) row = rows - 1;
    typename Tile::Raw r;
    Tile::load(r, x + row * ldx, K, lane);
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < NE; j++) m = max(m, __float_as_uint(fabsf(to_float(r.v[j]))));
    const Divisor d(row_max<TPR>(m, sh));
    if (!real) return;
    if (lane == 0) scale[row] = d.s;
    q += row * ldq;
#pragma unroll
    for (int i = 0; i < Tile::kVecs; i++) {
        const int c = Tile::column(i, lane);
        unsigned w[Tile::kVec / 4];
#pragma unroll
        for (int h = 0; h < Tile::kVec / 4; h++) {
            w[h] = 0;
#pragma unroll
            for (int e = 0; e < 4; e++)
                w[h] |= (unsigned)(d(to_float(r.v[i * Tile::kVec + 4 * h + e])) & 255) << (8 * e);
        }
        if (c + Tile::kVec <= K) {
            *reinterpret_cast<unsigned *>(q + c) = w[0];
        } else {
#pragma unroll
            for (int e = 0; e < Tile::kVec; e++)
                if (c + e < K) q[c + e] = (int8_t)(w[e / 4] >> (8 * (e % 4)));
        }
    }
}

// One block per row, any width (rows too wide for registers): read once for
// the scale and again, from L2, for the quotients.
template <typename T>
__global__ void quantize_row_kernel(const T *x, long long ldx, int K, int8_t *q, long long ldq,
                                    float *scale) {
    pdl_begin();
    pdl_trigger();
    __shared__ unsigned sh[32];
    const long long row = blockIdx.x;
    x += row * ldx;
    q += row * ldq;
    unsigned m = 0;
    for (int i = threadIdx.x; i < K; i += blockDim.x)
        m = max(m, __float_as_uint(fabsf(to_float(x[i]))));
    const Divisor d(row_max<512>(m, sh));
    if (threadIdx.x == 0) scale[row] = d.s;
    for (int i = threadIdx.x; i < K; i += blockDim.x) q[i] = (int8_t)d(to_float(x[i]));
}

}  // namespace

Status launch_quantize_rows(const Rows &x, int type, long long rows, int K, int8_t *q,
                            long long ldq, float *scale, cudaStream_t st) {
    if (rows == 0) return OK;
    if (rows < 0 || rows > 0x7fffffffLL || K <= 0) return ERR_SHAPE;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const bool vec = vector_rows(x.p, x.ld, rows, K, (int)sizeof(T));
        auto tile = [&](auto tpr, auto ne) {
            constexpr int TPR = decltype(tpr)::value, NE = decltype(ne)::value;
            constexpr int kThreads = TPR < 128 ? 128 : TPR;
            pdl_launch(quantize_tile_kernel<T, TPR, NE>, (unsigned)cdiv(rows, kThreads / TPR), kThreads, 0, st,
                       (const T *)x.p, x.ld, rows, K, q, ldq, scale);
            return cuda_status();
        };
        auto vectors = [&](auto tpr) {
            constexpr int TPR = decltype(tpr)::value, NE = 64 / (int)sizeof(T);
            constexpr int kThreads = TPR < 128 ? 128 : TPR;
            pdl_launch(quantize_vector_kernel<T, TPR, NE>, (unsigned)cdiv(rows, kThreads / TPR),
                       kThreads, 0, st, (const T *)x.p, x.ld, rows, K, q, ldq, scale);
            return cuda_status();
        };
        if (vec) {
            constexpr int NE = 64 / (int)sizeof(T);
            if (K <= 4 * NE) return vectors(Int<4>{});
            if (K <= 8 * NE) return vectors(Int<8>{});
            if (K <= 16 * NE) return vectors(Int<16>{});
            if (K <= 32 * NE) return vectors(Int<32>{});
            if (K <= 64 * NE) return vectors(Int<64>{});
            if (K <= 128 * NE) return vectors(Int<128>{});
            if (K <= 256 * NE) return vectors(Int<256>{});
            if (K <= 512 * NE) return vectors(Int<512>{});
            if (K <= 1024 * NE) return vectors(Int<1024>{});
        }
        if (K <= 64) return tile(Int<8>{}, Int<8>{});
        if (K <= 256) return tile(Int<32>{}, Int<8>{});
        if (K <= 512) return tile(Int<32>{}, Int<16>{});
        if (K <= 1024) return tile(Int<32>{}, Int<32>{});
        if (K <= 2048) return tile(Int<128>{}, Int<16>{});
        if (K <= 4096) return tile(Int<256>{}, Int<16>{});
        if (K <= 8192) return tile(Int<512>{}, Int<16>{});
        if (K <= 16384) return tile(Int<1024>{}, Int<16>{});
        pdl_launch(quantize_row_kernel<T>, (unsigned)rows, 512, 0, st, (const T *)x.p, x.ld, K, q,
                   ldq, scale);
        return cuda_status();
    });
}

}  // namespace ppdl
