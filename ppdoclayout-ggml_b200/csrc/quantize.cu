// quantize.cu — 8-bit rows with a scale each: scale = max |x| / 127,
// q = x / scale rounded half to even on the exact quotient.
//
// A row stays in registers between its maximum and its quotients.  FP32 rows
// are bound by memory: 20000 x 4096 68 us, 6.0 TB/s; 52500 x 256 10.5 us, the
// input partly in L2; odd ones, 50000 x 1153, 52 us, 5.6 TB/s.  16-bit rows have
// twice as many values a byte: 8192 x 8192 BF16 46 us, 4.4 TB/s, issue slots 62 %
// and the ALU 58 % busy, waits for memory the largest stall; 50000 x 1153 FP16
// 59 us.
#include <type_traits>

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

// Values of a row at any alignment, loaded one by one, held by TPR threads as
// quads of neighbouring columns, whose results are whole words: quads lane,
// lane + TPR, ...  (16-bit values as shifted words, three to a quad, and the
// row's ends one by one, took 86 us for 50000 x 1153 FP16, so 59; bulk copies
// of whole groups of rows through shared memory 74.)
template <typename T, int TPR, int NE>
struct QuadTile {
    static constexpr int kVec = 4, kVecs = NE / 4;
    struct Raw {
        uint32_t u[NE * (int)sizeof(T) / 4];
    };
    static __device__ __forceinline__ int column(int i, int lane) { return (i * TPR + lane) * 4; }
    // what lies past D is zero
    static __device__ __forceinline__ void load(Raw &r, const T *row, int D, int lane) {
        if constexpr (sizeof(T) == 2) {
            const uint16_t *v = reinterpret_cast<const uint16_t *>(row);
#pragma unroll
            for (int j = 0; j < NE / 2; j++) {
                const int c = column(j / 2, lane) + j % 2 * 2;
                r.u[j] = 0;
                if (c < D) r.u[j] = v[c];
                if (c + 1 < D) r.u[j] |= (uint32_t)v[c + 1] << 16;
            }
        } else {
#pragma unroll
            for (int j = 0; j < NE; j++) {
                r.u[j] = 0;
                const int c = column(j / 4, lane) + j % 4;
                if (c < D) r.u[j] = __float_as_uint(row[c]);
            }
        }
    }
    static __device__ __forceinline__ uint32_t word(const Raw &r, int k) { return r.u[k]; }
    static __device__ __forceinline__ float2 pair(const Raw &r, int j) {
        if constexpr (sizeof(T) == 2) return unpack2<T>(r.u[j]);
        else return make_float2(__uint_as_float(r.u[2 * j]), __uint_as_float(r.u[2 * j + 1]));
    }
};

// A row's values, held as pairs (PairTile, QuadTile), by d.  The quotient is
// first taken as x (1 / s), off by at most 127 x 2^-23 = 1.6e-5, and rounded
// by adding 1.5 x 2^23, which leaves the whole number in the low byte.  Values
// that close to a half decide on their remainders, pair by pair: in 16-bit
// rows half the largest value (63.5 steps) alone makes them common, one in
// some hundreds, so that most warps have one and few pairs do.
template <typename Tile, int NE, bool VEC>
__device__ __forceinline__ void quantize_pairs(const typename Tile::Raw &r, const Divisor &d, int K,
                                               int8_t *q, int lane) {
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
        if constexpr (Tile::kVec == 8) {
            *reinterpret_cast<uint2 *>(q + c) = make_uint2(out[2 * i], out[2 * i + 1]);
        } else if (VEC || c + 4 <= K) {
            *reinterpret_cast<uint32_t *>(q + c) = out[i];
        } else {
            for (int e = 0; c + e < K; e++) q[c + e] = (int8_t)(out[i] >> (8 * e));
        }
    }
}

// Rows in registers, of whole 16-byte vectors (VEC) or at any alignment.
template <typename T, int TPR, int NE, bool VEC>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, 1024 / (TPR < 128 ? 128 : TPR))
quantize_kernel(const T *x, long long ldx, long long rows, int K, int8_t *q, long long ldq,
                       float *scale) {
    using Tile = std::conditional_t<VEC, PairTile<T, TPR, NE>, QuadTile<T, TPR, NE>>;
    pdl_begin();
    pdl_trigger();
    __shared__ unsigned sh[32];
    constexpr int kRows = TPR < 128 ? 128 / TPR : 1, kWords = NE * (int)sizeof(T) / 4;
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
    quantize_pairs<Tile, NE, VEC>(r, d, K, q, lane);
}

// One block per row, any width (rows too wide for registers): read once for
// the scale and again, from L2, for the quotients.  (The column is unsigned:
// its last step passes 2^31 - 1 where K is next to it.)
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
    for (unsigned i = threadIdx.x; i < (unsigned)K; i += blockDim.x)
        m = max(m, __float_as_uint(fabsf(to_float(x[i]))));
    const Divisor d(row_max<512>(m, sh));
    if (threadIdx.x == 0) scale[row] = d.s;
    for (unsigned i = threadIdx.x; i < (unsigned)K; i += blockDim.x)
        q[i] = (int8_t)d(to_float(x[i]));
}

}  // namespace

Status launch_quantize_rows(const Rows &x, int type, long long rows, int K, int8_t *q,
                            long long ldq, float *scale, cudaStream_t st) {
    if (rows == 0) return OK;
    if (rows < 0 || rows > 0x7fffffffLL || K <= 0) return ERR_SHAPE;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const bool vec = vector_rows(x.p, x.ld, rows, K, (int)sizeof(T));
        auto tile = [&](auto tpr, auto ne, auto vector) {
            constexpr int TPR = decltype(tpr)::value, NE = decltype(ne)::value;
            constexpr int kThreads = TPR < 128 ? 128 : TPR;
            pdl_launch(quantize_kernel<T, TPR, NE, decltype(vector)::value != 0>,
                       (unsigned)cdiv(rows, kThreads / TPR), kThreads, 0, st, (const T *)x.p, x.ld,
                       rows, K, q, ldq, scale);
            return cuda_status();
        };
        // 64 or 48 bytes a thread in vectors (10000 x 2560 BF16 21.0 us, with
        // 64 alone 24.0); one by one, the tile with the fewest places left
        // empty (200000 x 257 BF16 69 us by 384 places, by 512 132)
        constexpr Int<1> vector;
        constexpr Int<0> single;
        if (vec) {
            constexpr int kNE = 64 / (int)sizeof(T), kLess = kNE / 4 * 3, kMore = kNE / 4 * 5;
            auto by = [&](auto tpr) {
                constexpr int TPR = decltype(tpr)::value;
                if constexpr (TPR >= 16 && TPR < 1024 && TPR * kNE != 4096) {
                    if (K <= TPR * kLess) return tile(tpr, Int<kLess>{}, vector);
                }
                return tile(tpr, Int<kNE>{}, vector);
            };
            if (K <= 4 * kNE) return by(Int<4>{});
            if (K <= 8 * kNE) return by(Int<8>{});
            if (K <= 16 * kNE) return by(Int<16>{});
            if (K <= 32 * kNE) return by(Int<32>{});
            if (K <= 64 * kNE) return by(Int<64>{});
            if (K > 2048 && K <= 2560) return tile(Int<2560 / kMore>{}, Int<kMore>{}, vector);
            if (K <= 128 * kNE) return by(Int<128>{});
            if (K <= 256 * kNE) return by(Int<256>{});
            if (K <= 512 * kNE) return by(Int<512>{});
            if (K <= 1024 * kNE) return by(Int<1024>{});
        }
        if (K <= 64) return tile(Int<8>{}, Int<8>{}, single);
        if (K <= 128) return tile(Int<8>{}, Int<16>{}, single);
        if (K <= 256) return tile(Int<16>{}, Int<16>{}, single);
        if (K <= 384) return tile(Int<32>{}, Int<12>{}, single);
        if (K <= 512) return tile(Int<32>{}, Int<16>{}, single);
        if (K <= 768) return tile(Int<32>{}, Int<24>{}, single);
        if (K <= 1024) return tile(Int<32>{}, Int<32>{}, single);
        if (K <= 1280) return tile(Int<64>{}, Int<20>{}, single);
        if (K <= 2048) return tile(Int<128>{}, Int<16>{}, single);
        if (K <= 2560) return tile(Int<128>{}, Int<20>{}, single);
        if (K <= 4096) return tile(Int<256>{}, Int<16>{}, single);
        if (K <= 5120) return tile(Int<256>{}, Int<20>{}, single);
        if (K <= 8192) return tile(Int<512>{}, Int<16>{}, single);
        if (K <= 10240) return tile(Int<512>{}, Int<20>{}, single);
        if (K <= 16384) return tile(Int<1024>{}, Int<16>{}, single);
        pdl_launch(quantize_row_kernel<T>, (unsigned)rows, 512, 0, st, (const T *)x.p, x.ld, K, q,
                   ldq, scale);
        return cuda_status();
    });
}

}  // namespace ppdl
