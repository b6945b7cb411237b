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
//
// Memory bounds it, once the turns are made once a token and not once a
// head: 8 x 2500 tokens of 16 + 16 heads x 64 FP32 50.7 us (99 % of the copy
// rate), 4 x 4096 tokens of 32 + 8 heads x 128 BF16 62.6 (82 %); 64 new
// tokens of 32 + 8 heads 2.4 us, which is latency.
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

// Heads as 16-byte vectors.  A block has `tokens` tokens: it first fills a
// table of their turns in shared memory — one 64-bit angle and one sine and
// cosine a token and pair, for all heads — then its threads go through the
// units: a unit is a vector of first values and the vector of their partners
// (interleaved: two neighbouring vectors), or one vector past the turned
// values.  The first unit's loads are issued before the table.
struct RotaryUnits {
    int tokens, turned, all;  // tokens a block; turned and all units of a head
    FastDiv per_token, per_head, pairs, length;
};

template <typename T>
__device__ __forceinline__ void unpack_vector(float (&v)[16 / sizeof(T)], uint4 u) {
    if constexpr (sizeof(T) == 2) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = unpack2<T>(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    } else {
        v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y);
        v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack_vector(const float (&v)[16 / sizeof(T)]) {
    if constexpr (sizeof(T) == 2)
        return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                          pack2<T>(v[6], v[7]));
    else
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                          __float_as_uint(v[3]));
}

template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_vector_kernel(RotaryArgs a, RotaryUnits g) {
    pdl_begin();
    pdl_trigger();
    constexpr int V = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) float2 turn[];
    const int pairs = a.rotated / 2, all_tokens = a.batch * a.length;
    const int first = blockIdx.x * g.tokens, here = min(g.tokens, all_tokens - first);
    const int units = here * (a.h[0].heads + a.h[1].heads) * g.all;

    struct Unit {
        uint4 lo, hi;
        T *out;
        int table, second;  // first pair in the table; values to the second vector (0: none)
    };
    auto load = [&](int u) {
        Unit r;
        const int t = g.per_token.div(u), in_token = u - t * (int)g.per_token.d;
        int head = g.per_head.div(in_token);
        const int k = in_token - head * g.all;
        const int token = first + t, b = g.length.div(token);
        const long long at = token - b * a.length;
        const bool keys = head >= a.h[0].heads;
        const RotaryHeads &h = a.h[keys ? 1 : 0];
        if (keys) head -= a.h[0].heads;
        int column;
        if (k >= g.turned) {
            column = a.rotated + (k - g.turned) * V;
            r.second = 0;
        } else {
            column = INTERLEAVED ? 2 * k * V : k * V;
            r.second = INTERLEAVED ? V : pairs;
        }
        // (interleaved heads whose turned values are an odd number of vectors
        // end in a unit of one)
        const bool two = r.second && (!INTERLEAVED || column + V < a.rotated);
        r.table = k >= g.turned ? -1 : t * pairs + k * V;
        if (INTERLEAVED && r.second && !two) r.second = 0;
        const T *in = (const T *)h.in + b * h.in_bs + at * h.in_ts + head * h.in_hs + column;
        r.out = (T *)h.out + b * h.out_bs + at * h.out_ts + head * h.out_hs + column;
        r.lo = *reinterpret_cast<const uint4 *>(in);
        if (two) r.hi = *reinterpret_cast<const uint4 *>(in + r.second);
        return r;
    };
    Unit next = {};
    if ((int)threadIdx.x < units) next = load(threadIdx.x);
    for (int i = threadIdx.x; i < here * pairs; i += 256) {
        const int t = g.pairs.div(i), token = first + t, b = g.length.div(token);
        turn[i] = turn_of(a, b * a.pos_bs + (token - b * a.length) * a.pos_ts, i - t * pairs);
    }
    __syncthreads();
    for (int u = threadIdx.x; u < units; u += 256) {
        Unit r = next;
        if (u + 256 < units) next = load(u + 256);
        if (r.table >= 0) {
            const float2 *cs = turn + r.table;
            float x[V], y[V];
            unpack_vector<T>(x, r.lo);
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    const float2 w = cs[i / 2];
                    y[i] = x[i] * w.x - x[i + 1] * w.y;
                    y[i + 1] = x[i + 1] * w.x + x[i] * w.y;
                }
                r.lo = pack_vector<T>(y);
                if (r.second) {
                    unpack_vector<T>(x, r.hi);
#pragma unroll
                    for (int i = 0; i < V; i += 2) {
                        const float2 w = cs[V / 2 + i / 2];
                        y[i] = x[i] * w.x - x[i + 1] * w.y;
                        y[i + 1] = x[i + 1] * w.x + x[i] * w.y;
                    }
                    r.hi = pack_vector<T>(y);
                }
            } else {
                float p[V], q[V];
                unpack_vector<T>(y, r.hi);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float2 w = cs[i];
                    p[i] = x[i] * w.x - y[i] * w.y;
                    q[i] = y[i] * w.x + x[i] * w.y;
                }
                r.lo = pack_vector<T>(p);
                r.hi = pack_vector<T>(q);
            }
        }
        *reinterpret_cast<uint4 *>(r.out) = r.lo;
        if (r.second) *reinterpret_cast<uint4 *>(r.out + r.second) = r.hi;
    }
}

// One block per token, one value pair a thread: any alignment.
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

// whole 16-byte vectors: pointers, strides and the parts of a head
bool vector_heads(const RotaryArgs &a, int size) {
    const int v = 16 / size;
    if (a.dim % v || a.rotated % v || (!a.interleaved && a.rotated / 2 % v)) return false;
    for (const RotaryHeads &h : a.h) {
        if (!h.heads) continue;
        const long long steps[6] = {a.batch > 1 ? h.in_bs : 0, a.length > 1 ? h.in_ts : 0,
                                    h.heads > 1 ? h.in_hs : 0, a.batch > 1 ? h.out_bs : 0,
                                    a.length > 1 ? h.out_ts : 0, h.heads > 1 ? h.out_hs : 0};
        for (long long s : steps)
            if (s % v) return false;
        if ((uintptr_t)h.in & 15 || (uintptr_t)h.out & 15) return false;
    }
    return true;
}

}  // namespace

Status launch_rotary(const RotaryArgs &a, cudaStream_t st) {
    const long long tokens = (long long)a.batch * a.length;
    if (tokens == 0) return OK;
    if (tokens > 0x7fffffffLL) return ERR_SHAPE;
    const int heads = a.h[0].heads + a.h[1].heads;
    if (heads == 0) return OK;
    return with_type(a.type, [&](auto t) {
        using T = decltype(t);
        constexpr int V = 16 / (int)sizeof(T);
        const int pairs = a.rotated / 2;
        // values past the turned ones stay as they are when turned in place
        bool in_place = true;
        for (const RotaryHeads &h : a.h) in_place = in_place && (!h.heads || h.in == h.out);
        RotaryUnits g;
        g.turned = a.interleaved ? cdiv(a.rotated, 2 * V) : pairs / V;
        g.all = g.turned + (in_place ? 0 : (a.dim - a.rotated) / V);
        const long long per_token = (long long)heads * g.all;
        if (vector_heads(a, (int)sizeof(T)) && per_token < (1 << 20)) {
            // about four units a thread, as long as all SMs have blocks
            // (4 x 4096 tokens of 40 heads x 128 BF16 62.6 us, with one token
            // a block 82.6; of 5 heads x 32 15.3 / 131)
            long long per = 1024 / per_token;
            if (per > tokens / (8 * 148)) per = tokens / (8 * 148);
            if (per > 4096 / pairs) per = 4096 / pairs;  // 32 KB of table
            g.tokens = per < 1 ? 1 : (int)per;
            g.per_token = FastDiv((uint32_t)per_token);
            g.per_head = FastDiv((uint32_t)g.all);
            g.pairs = FastDiv((uint32_t)pairs);
            g.length = FastDiv((uint32_t)a.length);
            auto kernel = a.interleaved ? rotary_vector_kernel<T, true>
                                        : rotary_vector_kernel<T, false>;
            pdl_launch(kernel, (unsigned)cdiv(tokens, g.tokens), 256, (size_t)g.tokens * pairs * 8,
                       st, a, g);
            return cuda_status();
        }
        pdl_launch(rotary_token_kernel<T>, (unsigned)tokens, 128, (size_t)a.rotated / 2 * 8, st, a);
        return cuda_status();
    });
}

}  // namespace ppdl
