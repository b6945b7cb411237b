// linear_i8.cu — linear layers in 8-bit integers with a scale for each token
// (row of the activations) and each channel (row of the weights), on the
// 5th-generation tensor cores:
//
//   y(m, n) = act(sum_k q(m, k) w(n, k) * q_scale[m] * w_scale[n] + bias[n]) + res(m, n)
//
// The integer sums are exact: at most 131071 products of at most 128 x 128
// stay below 2^31, in any order.
//
// The product is computed transposed: the MMA's M dimension is 128 output
// channels (the weights are its A operand), its N dimension BT tokens.  A
// TMEM lane is then one channel, so that in the epilogue the 32 lanes of a
// warp hold 32 neighbouring channels of one token: rows of y (and of the
// residual) are read and written in whole segments straight from registers,
// with no pass through shared memory, and a lane's channel scale and bias
// stay in registers for the whole tile.  It also makes a single token cheap:
// only the N dimension shrinks (to 16).
//
// One CTA of 12 warps: warp 0 loads 128-byte wide k-blocks of both operands
// by TMA (128-byte swizzle) into a ring of stages, warp 1 issues
// tcgen05.mma kind::i8 (four K = 32 steps a block) into one of two TMEM
// accumulators, warps 4-11 (two per lane quadrant, each half the tokens) run
// the epilogue of one tile while the next is accumulated.
//
// Two forms.  Whole-K: a persistent grid over the tiles.  Split-K, for few
// tiles: a cluster shares a tile's k-blocks; every CTA puts its partial
// sums into its own shared memory, and after a cluster barrier each CTA adds
// up its share of the tokens over its peers and finishes it.  Integer sums
// do not depend on the order, so both forms give the same bits.
//
// One or two tokens in 16 or 32 bits are quantised by the split form itself:
// while its weights are on their way, every CTA finds the rows' largest
// values and quantises its own k-blocks into shared memory, which saves a
// launch.
//
// Measured: 8192 cubed BF16 410-440 us (2.5-2.7 POP/s, the power cap at work),
// 4096 cubed 53 us (2.6), 52500 x 256 -> 1536 FP32 58.6 us (the result's bytes:
// 6.5 TB/s), one token of 4096 -> 4096 9.8 us quantised in the call (the weights'
// 16.8 MB take 2.6; launch, two trips to memory, the second behind the
// quantisation, and the cluster exchange the rest), 2400 x 256 -> 1024 FP32 6.2
// us (latency).
//
// Every mbarrier wait is bounded; on expiry the kernel raises a device error
// flag, all roles drain out and TMEM is released (ppdl_op_device_error).
#include <cuda.h>

#include "block.cuh"
#include "block.h"
#include "gemm_tc.h"
#include "quantize.cuh"
#include "tc_ptx.cuh"

namespace ppdl {

namespace {

__device__ int g_linear_error = 0;

constexpr int kFeat = 128;  // channels per tile (MMA M)
constexpr int kBK = 128;    // k per stage: one 128-byte swizzle row
constexpr int kWarpTma = 0, kWarpMma = 1, kWarpScale = 2, kWarpEpi = 4;
// barriers, TMEM address, abort flag and whether two tiles' scales are
// ordinary; then those scales: 128 of channels, 128 biases and up to 256 of
// tokens each
constexpr int kScaleFloats = 512;
constexpr int kCtrlBytes = 256 + 2 * kScaleFloats * 4;
constexpr int kAbortAt = 204, kOrdinaryAt = 208;
constexpr int kSmemMax = 227 * 1024;
constexpr int kABytes = kFeat * kBK;

// The forms of the kernel.
enum Form : int {
    WHOLE = 0,  // a CTA per tile, persistent
    PAIR = 1,   // two CTAs per tile of 256 channels, persistent
    SPLIT = 2   // a cluster per tile, its k-blocks shared out
};

// epilogue warps: a multiple of 4, one or more per TMEM lane quadrant, each
// with its share of the tile's tokens
constexpr int epi_warps(int bt, int form) { return form != SPLIT && bt >= 128 ? 16 : 8; }
constexpr int threads(int bt, int form) { return 32 * (kWarpEpi + epi_warps(bt, form)); }
// token rows of a stage: a CTA of a pair loads half of them
constexpr int load_tokens(int bt, int form) { return form == PAIR ? bt / 2 : bt; }
constexpr int stage_bytes(int bt, int form) { return kABytes + load_tokens(bt, form) * kBK; }
// stages in the ring: what fits beside the control block and the alignment
// slack, at most 8; the split form keeps to 4 so that two CTAs share an SM
constexpr int stages(int bt, int form) {
    const int fit = (kSmemMax - kCtrlBytes - 1024) / stage_bytes(bt, form);
    const int most = form == SPLIT ? 4 : 8;
    return fit < most ? fit : most;
}
constexpr int smem_bytes(int bt, int form) {
    return kCtrlBytes + 1024 + stages(bt, form) * stage_bytes(bt, form);
}
// the quantising form: a ring of weights alone, and this CTA's k-blocks of
// quantised tokens behind it
constexpr int kFuseBlocks = 16;
constexpr int fuse_smem(int bt) {
    return kCtrlBytes + 1024 + stages(bt, SPLIT) * kABytes + kFuseBlocks * bt * kBK;
}
constexpr uint32_t tmem_cols(int bt, int form) {
    const int c = form == SPLIT ? bt : 2 * bt;
    return c < 32 ? 32 : c;
}

struct Args {
    int M, N, kblocks;
    int f_tiles, t_tiles, tiles;
    FastDiv group;  // by the tiles of a whole group
    int kps;  // split form: k-blocks per CTA of the cluster
    int act;
    int pairs;  // 16-bit rows of y and res start on 4 bytes
    const float *q_scale, *w_scale, *bias;
    const void *res;
    void *y;
    long long ldres, ldy;
    const void *x;  // quantising form: M rows of K values
    long long ldx;
    int K;
};

__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
    return mbar_wait_bounded(bar, parity, abort_flag, &g_linear_error);
}

// D (TMEM) (+)= A (shared) * B (shared), 8-bit signed, K = 32
__device__ __forceinline__ void umma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// The same over a CTA pair: 256 rows of A, each CTA holding 128 of them and
// half of B's rows, each CTA's TMEM the sums of its own rows.
__device__ __forceinline__ void umma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// arrives at the barrier of both CTAs of the pair
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}
// a load into this CTA's shared memory that reports to the leader's barrier
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap *tm, uint32_t bar,
                                                 int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
// mbar_arrive_relaxed at another CTA's barrier
__device__ __forceinline__ void mbar_arrive_relaxed_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
                 : "memory");
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// the same shared-memory address in the cluster's CTA `rank`
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ int4 peer_load(uint32_t addr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ int peer_load1(uint32_t addr) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

// tile index -> (channel tile, token tile): token tiles in groups of 8, the
// group's channel tiles outer, so that the CTAs that run at one time share
// both operands in L2
constexpr int kGroup = 8;
__device__ __forceinline__ void tile_of(const Args &a, int tile, int &ft, int &tt) {
    const int g = a.group.div(tile), r = tile - g * (kGroup * a.f_tiles);
    const int width = min(kGroup, a.t_tiles - g * kGroup);
    ft = width == kGroup ? r / kGroup : r / width;
    tt = g * kGroup + r - ft * width;
}

// A sum under its two scales, plus the bias.  The scales are multiplied first
// (they are the same for a whole row or column), unless their product leaves
// FP32's normal range: a small one would lose digits of a result that is a
// normal number, an infinite one make a NaN of a sum of zero.  The larger
// scale then goes first: the sum, below 2^31, times it overflows only where
// the result does (a product below 2^-126 with a factor of at least 2^-149
// leaves less than 2^23 for the other).  Without a branch, the split form's
// epilogue gains 0.2 us (64 x 4096 -> 4096 9.75, with one 9.9).
__device__ __forceinline__ float scaled(float acc, float sx, float sw, float bias) {
    const float s = __fmul_rn(sx, sw);
    const bool normal = fabsf(s) >= 0x1p-126f && fabsf(s) < INFINITY;
    const bool x_first = fabsf(sx) > fabsf(sw);
    const float first = normal ? 1.0f : x_first ? sx : sw;
    const float second = normal ? s : x_first ? sw : sx;
    return __fmaf_rn(__fmul_rn(acc, first), second, bias);
}
// Two such scales have a normal product, or one of them is zero.
__device__ __forceinline__ bool ordinary_scale(float s) {
    return s == 0.0f || (fabsf(s) >= 0x1p-62f && fabsf(s) <= 0x1p63f);
}

// What follows the sum, with every rounding written out (the residual's sum
// by __fadd_rn as well), so that all forms give the same bits: scaled() for
// ordinary scales.  acc is rounded to FP32 (2^-24 relative).
template <int C, int ACT>
__device__ __forceinline__ void finish_all(float (&v)[C], const uint32_t (&acc)[C], const float *sx,
                                           float sw, float bias) {
    const float2 sw2 = both(sw), bias2 = both(bias);
#pragma unroll
    for (int j = 0; j < C; j += 4) {
        const float4 s = *reinterpret_cast<const float4 *>(sx + j);
        const float2 s01 = mul2(make_float2(s.x, s.y), sw2), s23 = mul2(make_float2(s.z, s.w), sw2);
        const float2 a01 = make_float2((float)(int)acc[j], (float)(int)acc[j + 1]);
        const float2 a23 = make_float2((float)(int)acc[j + 2], (float)(int)acc[j + 3]);
        const float2 v01 = fma2(a01, s01, bias2), v23 = fma2(a23, s23, bias2);
        v[j] = act_keep_nan(v01.x, ACT);
        v[j + 1] = act_keep_nan(v01.y, ACT);
        v[j + 2] = act_keep_nan(v23.x, ACT);
        v[j + 3] = act_keep_nan(v23.y, ACT);
    }
}

// Epilogue of C tokens t0 .. t0 + C - 1 of channel n (one per lane).  No
// branch depends on a value, so that the C chains of conversion, scale,
// activation and store overlap: with 2 to 4 warps a scheduler there is
// little else to hide their latency.  EDGE: some of the tokens or lanes lie
// past y, their loads and stores are predicated off.
template <typename T, int C, int ACT, bool RES, bool EDGE>
__device__ __forceinline__ void epilogue_chunk(const Args &a, const uint32_t (&acc)[C], int t0,
                                               int n, float sw, float bias, const float *sx,
                                               int lane) {
    float v[C];
    const int tokens = EDGE ? a.M - t0 : C;
    if constexpr (sizeof(T) == 2) {
        if (a.pairs && (!EDGE || n - lane + 32 <= a.N)) {
            // lane pairs exchange values, so that the even lane holds token j
            // and the odd lane token j + 1 of two neighbouring channels: one
            // 4-byte store (and residual load) per lane and pair of tokens
            const int odd = lane & 1;
            const long long first = t0 + odd, nn = n - odd;
            uint32_t r[RES ? C / 2 : 1];
            if constexpr (RES) {
                const T *rp = (const T *)a.res + first * a.ldres + nn;
#pragma unroll
                for (int j = 0; j < C; j += 2, rp += 2 * a.ldres) {
                    r[j / 2] = 0;
                    if (!EDGE || j + odd < tokens)
                        r[j / 2] = *reinterpret_cast<const uint32_t *>(rp);
                }
            }
            finish_all<C, ACT>(v, acc, sx, sw, bias);
            T *yp = (T *)a.y + first * a.ldy + nn;
#pragma unroll
            for (int j = 0; j < C; j += 2, yp += 2 * a.ldy) {
                uint32_t out;
                if constexpr (RES) {
                    const float other = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[j + 1], 1);
                    const float2 rr = unpack2<T>(r[j / 2]);
                    out = pack2<T>(__fadd_rn(odd ? other : v[j], rr.x),
                                   __fadd_rn(odd ? v[j + 1] : other, rr.y));
                } else {
                    // already at its last rounding: exchange the packed pair
                    // (token j in the low half), then take one half of each
                    const uint32_t own = pack2<T>(v[j], v[j + 1]);
                    const uint32_t other = __shfl_xor_sync(0xffffffffu, own, 1);
                    out = __byte_perm(own, other, odd ? 0x3276 : 0x5410);
                }
                if (!EDGE || j + odd < tokens) *reinterpret_cast<uint32_t *>(yp) = out;
            }
            return;
        }
    }
    const int mine = EDGE && n >= a.N ? 0 : tokens;
    T r[RES ? C : 1];
    if constexpr (RES) {
        const T *rp = (const T *)a.res + (long long)t0 * a.ldres + n;
#pragma unroll
        for (int j = 0; j < C; j++, rp += a.ldres) {
            r[j] = from_float<T>(0.0f);
            if (!EDGE || j < mine) r[j] = *rp;
        }
    }
    finish_all<C, ACT>(v, acc, sx, sw, bias);
    T *yp = (T *)a.y + (long long)t0 * a.ldy + n;
#pragma unroll
    for (int j = 0; j < C; j++, yp += a.ldy) {
        const T out = from_float<T>(RES ? __fadd_rn(v[j], to_float(r[RES ? j : 0])) : v[j]);
        if (!EDGE || j < mine) *yp = out;
    }
}

template <typename T, int C, bool RES, bool EDGE>
__device__ __forceinline__ void epilogue_act(const Args &a, const uint32_t (&acc)[C], int t0, int n,
                                             float sw, float bias, const float *sx, int lane) {
    switch (a.act) {
        case ACT_RELU:
            return epilogue_chunk<T, C, ACT_RELU, RES, EDGE>(a, acc, t0, n, sw, bias, sx, lane);
        case ACT_SILU:
            return epilogue_chunk<T, C, ACT_SILU, RES, EDGE>(a, acc, t0, n, sw, bias, sx, lane);
        case ACT_GELU:
            return epilogue_chunk<T, C, ACT_GELU, RES, EDGE>(a, acc, t0, n, sw, bias, sx, lane);
        default:
            return epilogue_chunk<T, C, ACT_NONE, RES, EDGE>(a, acc, t0, n, sw, bias, sx, lane);
    }
}

// A chunk of a tile that has scales out of the ordinary, one value after
// another and out of line: in the epilogue itself these cases cost every tile
// (2400 x 256 -> 1024 FP32 6.4 us, so 6.2).
template <typename T>
__device__ __noinline__ void epilogue_slow(const Args &a, const uint32_t *acc, int tokens, int t0,
                                           int n, float sw, float bias, const float *sx) {
    if (n >= a.N) return;
    for (int j = 0; j < tokens && t0 + j < a.M; j++) {
        float v = act_keep_nan(scaled((float)(int)acc[j], sx[j], sw, bias), a.act);
        if (a.res)
            v = __fadd_rn(v, to_float(((const T *)a.res)[(long long)(t0 + j) * a.ldres + n]));
        ((T *)a.y)[(long long)(t0 + j) * a.ldy + n] = from_float<T>(v);
    }
}

template <typename T, int C>
__device__ __forceinline__ void epilogue_any(const Args &a, const uint32_t (&acc)[C], int t0, int n,
                                             float sw, float bias, const float *sx, bool ordinary,
                                             int lane) {
    if (!ordinary) {
        uint32_t copy[C];
#pragma unroll
        for (int j = 0; j < C; j++) copy[j] = acc[j];
        epilogue_slow<T>(a, copy, C, t0, n, sw, bias, sx);
        return;
    }
    const bool edge = t0 + C > a.M || n - lane + 32 > a.N;
    if (a.res) {
        if (edge) epilogue_act<T, C, true, true>(a, acc, t0, n, sw, bias, sx, lane);
        else epilogue_act<T, C, true, false>(a, acc, t0, n, sw, bias, sx, lane);
    } else {
        if (edge) epilogue_act<T, C, false, true>(a, acc, t0, n, sw, bias, sx, lane);
        else epilogue_act<T, C, false, false>(a, acc, t0, n, sw, bias, sx, lane);
    }
}

// The calling 8 warps quantise k-blocks kb0 .. kb0 + kbn - 1 of the a.M <= BT
// rows of a.x into `to` ([k-block][BT rows of 128 bytes], 128-byte swizzle:
// 16-byte chunk c of row r at chunk c ^ (r & 7)) and the rows' scales into
// `scale`; amax is scratch for BT words.  Rows past M are left as they are:
// no output depends on them.
template <typename X, int BT>
__device__ __forceinline__ void quantize_slice(const Args &a, int kb0, int kbn, uint8_t *to,
                                               float *scale, unsigned *amax) {
    constexpr int kThreads = 256, kBar = 1;
    const int tid = threadIdx.x - 32 * kWarpEpi;
    auto sync = [] { asm volatile("bar.sync %0, %1;" ::"n"(kBar), "n"(kThreads) : "memory"); };
    const X *x = (const X *)a.x;
    constexpr int V = 16 / (int)sizeof(X);
    const bool vec = ((uintptr_t)x & 15) == 0 && a.K % V == 0 && (a.M == 1 || a.ldx % V == 0);
    // a unit: sixteen neighbouring values of a row; the thread's first unit is
    // loaded before the rows' largest values are known
    const int per_row = kbn * 8, units = a.M * per_row;
    X v[16];
    auto load = [&](int u) {
        const int r = u / per_row, k = kb0 * kBK + (u - r * per_row) * 16;
        const X *row = x + (long long)r * a.ldx + k;
        if (vec && k + 16 <= a.K) {
#pragma unroll
            for (int i = 0; i < 16 / V; i++)
                reinterpret_cast<uint4 *>(v)[i] = reinterpret_cast<const uint4 *>(row)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                v[i] = from_float<X>(0.0f);
                if (k + i < a.K) v[i] = row[i];
            }
        }
    };
    if (tid < units) load(tid);
    if (tid < BT) amax[tid] = 0;
    sync();
    for (int r = 0; r < a.M; r++) {
        const X *row = x + (long long)r * a.ldx;
        unsigned m = 0;
        if (vec) {
            for (int c = tid * V; c < a.K; c += kThreads * V) {
                const uint4 w = *reinterpret_cast<const uint4 *>(row + c);
                const X *e = reinterpret_cast<const X *>(&w);
#pragma unroll
                for (int i = 0; i < V; i++) m = max(m, __float_as_uint(fabsf(to_float(e[i]))));
            }
        } else {
            for (int c = tid; c < a.K; c += kThreads)
                m = max(m, __float_as_uint(fabsf(to_float(row[c]))));
        }
        m = __reduce_max_sync(0xffffffffu, m);
        if ((tid & 31) == 0) atomicMax(&amax[r], m);
    }
    sync();
    for (int u = tid; u < units; u += kThreads) {
        if (u != tid) load(u);
        const int r = u / per_row, at = u - r * per_row, kb = at / 8, c = at % 8;
        const Divisor d(amax[r]);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            w[i] = 0;
#pragma unroll
            for (int e = 0; e < 4; e++)
                w[i] |= (uint32_t)(d(to_float(v[4 * i + e])) & 255) << (8 * e);
        }
        *reinterpret_cast<uint4 *>(to + kb * (BT * kBK) + r * kBK + ((c ^ (r & 7)) * 16)) =
            make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (tid < a.M) scale[tid] = Divisor(amax[tid]).s;
}

// X: int8_t, or the type of the rows that the split form quantises itself.
template <typename T, int BT, int FORM, typename X = int8_t>
__global__ void __launch_bounds__(threads(BT, FORM), FORM == SPLIT ? 2 : 1)
linear_i8_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmQ,
                 const __grid_constant__ Args a) {
    constexpr int S = stages(BT, FORM), kAcc = FORM == SPLIT ? 1 : 2;
    constexpr int kEpiWarps = epi_warps(BT, FORM), kLoadT = load_tokens(BT, FORM);
    constexpr int kTileF = FORM == PAIR ? 2 * kFeat : kFeat;  // channels per tile
    constexpr bool FUSE = sizeof(X) > 1;
    static_assert(!FUSE || FORM == SPLIT, "only the split form quantises");
    constexpr uint32_t kStage = FUSE ? kABytes : stage_bytes(BT, FORM), kCols = tmem_cols(BT, FORM);
    extern __shared__ uint8_t smem_raw[];
    const uint32_t ctrl = smem_u32(smem_raw);
    // full[s]: a stage's bytes landed (pair: both CTAs', in the leader);
    // empty[s]: its MMAs completed; tfull[i]: accumulator i complete;
    // tempty[i]: read by the epilogue (pair: both CTAs', in the leader);
    // sfull[i] / sempty[i]: a tile's scales written / read
    const uint32_t bar_full = ctrl, bar_empty = ctrl + 64, bar_tfull = ctrl + 128,
                   bar_tempty = ctrl + 144, bar_done = ctrl + 160, bar_sfull = ctrl + 168,
                   bar_sempty = ctrl + 184;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem_raw + 200);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem_raw + kAbortAt);
    float *scales = reinterpret_cast<float *>(smem_raw + 256);
    const uint32_t stage0 = (ctrl + kCtrlBytes + 1023) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; s++) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(bar_tfull + 8 * i, 1);
            mbar_init(bar_tempty + 8 * i, FORM == PAIR ? 2 * kEpiWarps : kEpiWarps);
            if (!FUSE) mbar_init(bar_sfull + 8 * i, 1);
            mbar_init(bar_sempty + 8 * i, kEpiWarps);
        }
        mbar_init(bar_done, 1);
        if (FUSE) mbar_init(bar_sfull, kEpiWarps);  // the tokens are quantised
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kWarpMma) {
        if constexpr (FORM == PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             smem_u32(tmem_slot)),
                         "r"(kCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             smem_u32(tmem_slot)),
                         "r"(kCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (FORM == PAIR) cluster_sync();  // the peer's barriers are set up
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    if (warp == kWarpTma && lane == 0) {
        prefetch_tensor_map(&tmW);
        if (!FUSE) prefetch_tensor_map(&tmQ);
    }
    pdl_begin();
    pdl_trigger();

    const uint32_t rank = FORM == WHOLE ? 0 : cluster_rank();
    const uint32_t peers = FORM == WHOLE ? 1 : FORM == PAIR ? 2 : cluster_size();
    const int first = (int)(blockIdx.x / peers);
    const int step = FORM == SPLIT ? a.tiles : (int)(gridDim.x / peers);  // split: one tile
    const int kb0 = FORM == SPLIT ? (int)rank * a.kps : 0;
    const int kbn = FORM == SPLIT ? max(0, min(a.kps, a.kblocks - kb0)) : a.kblocks;

    if (warp == kWarpTma) {
        if (lane == 0) {
            Ring rs(S);
            long long it = 0;
            bool ok = true;
            for (int tile = first; tile < a.tiles && ok; tile += step) {
                int ft, tt;
                tile_of(a, tile, ft, tt);
                for (int kb = 0; kb < kbn; kb++, it++, rs.next()) {
                    if (!wait_for(bar_empty + 8 * rs.i, rs.ph ^ 1, abort_flag)) {
                        ok = false;
                        break;
                    }
                    const uint32_t st = stage0 + rs.i * kStage;
                    const int k = (kb0 + kb) * kBK;
                    if constexpr (FORM == PAIR) {
                        const uint32_t fb = peer_addr(bar_full + 8 * rs.i, 0);
                        if (rank == 0) mbar_expect_tx(bar_full + 8 * rs.i, 2 * kStage);
                        tma_load_2d_pair(st, &tmW, fb, k, ft * kTileF + (int)rank * kFeat);
                        tma_load_2d_pair(st + kABytes, &tmQ, fb, k, tt * BT + (int)rank * kLoadT);
                    } else {
                        const uint32_t fb = bar_full + 8 * rs.i;
                        mbar_expect_tx(fb, kStage);
                        tma_load_2d(st, &tmW, fb, k, ft * kTileF);
                        if constexpr (!FUSE) tma_load_2d(st + kABytes, &tmQ, fb, k, tt * BT);
                    }
                }
            }
            // what was issued must land before the CTA may exit (pair: the
            // leader waits for both, the peer at the cluster's last barrier)
            if (FORM != PAIR || rank == 0)
                for (long long j = it > S ? it - S : 0; j < it; j++) {
                    int dummy = 0;
                    wait_for(bar_full + 8 * (int)(j % S), (uint32_t)((j / S) & 1),
                             (volatile int *)&dummy);
                }
            // so must the leader's arrivals at this CTA's barriers (a later
            // grid's CTA may already have this shared memory by then): the
            // stages' last releases, then the end of all MMAs.  What the
            // epilogue's barriers get, the epilogue has waited for.
            if constexpr (FORM == PAIR) {
                for (long long j = it > S ? it - S : 0; j < it && ok; j++)
                    ok = wait_for(bar_empty + 8 * (int)(j % S), (uint32_t)((j / S) & 1),
                                  abort_flag);
                int dummy = 0;
                if (rank != 0) wait_for(bar_done, 0, (volatile int *)&dummy);
            }
        }
    } else if (warp == kWarpMma) {
        if (lane == 0 && (FORM != PAIR || rank == 0)) {
            // S32 accumulators, signed 8-bit A and B, both K-major
            constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) |
                                       ((uint32_t)(BT >> 3) << 17) |
                                       ((uint32_t)(kTileF >> 4) << 24);
            auto commit = [](uint32_t bar) {
                if constexpr (FORM == PAIR) umma_commit_pair(bar);
                else umma_commit(bar);
            };
            Ring rs(S), ra(kAcc);
            bool ok = true;
            for (int tile = first; tile < a.tiles && ok; tile += step, ra.next()) {
                if (!wait_for(bar_tempty + 8 * ra.i, ra.ph ^ 1, abort_flag)) break;
                if (FUSE && !wait_for(bar_sfull, 0, abort_flag)) break;
                tc_fence_after();
                const uint32_t d = tmem + (uint32_t)(ra.i * BT);
                for (int kb = 0; kb < kbn; kb++, rs.next()) {
                    if (!wait_for(bar_full + 8 * rs.i, rs.ph, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t st = stage0 + rs.i * kStage;
                    // a K = 32 step is 32 bytes into the swizzled row: +2 in the
                    // descriptors' start address
                    const uint64_t da = smem_desc(st, 16, 1024, 2);
                    const uint64_t db = smem_desc(
                        FUSE ? stage0 + S * kStage + kb * (BT * kBK) : st + kABytes, 16, 1024, 2);
#pragma unroll
                    for (int k = 0; k < kBK / 32; k++) {
                        if constexpr (FORM == PAIR)
                            umma_i8_pair(d, da + 2 * k, db + 2 * k, idesc, (kb | k) != 0);
                        else
                            umma_i8(d, da + 2 * k, db + 2 * k, idesc, (kb | k) != 0);
                    }
                    commit(bar_empty + 8 * rs.i);
                }
                if (ok) commit(bar_tfull + 8 * ra.i);
            }
            // all issued MMAs must finish before TMEM is released
            commit(bar_done);
            int dummy = 0;
            wait_for(bar_done, 0, (volatile int *)&dummy);
        }
    } else if (FORM != SPLIT && warp == kWarpScale) {
        // the scales of each tile, one ahead of the epilogue: loaded by the
        // epilogue itself they queue behind its stores
        constexpr int kScaleT = (BT + 31) / 32;
        Ring ra(kAcc);
        for (int tile = first; tile < a.tiles; tile += step, ra.next()) {
            int ft, tt;
            tile_of(a, tile, ft, tt);
            const int n0 = ft * kTileF + (FORM == PAIR ? (int)rank * kFeat : 0), m0 = tt * BT;
            float v[2 * kFeat / 32 + kScaleT];
#pragma unroll
            for (int i = 0; i < kFeat / 32; i++) {
                const int n = n0 + 32 * i + lane;
                v[2 * i] = n < a.N ? __ldg(a.w_scale + n) : 0.0f;
                v[2 * i + 1] = a.bias && n < a.N ? __ldg(a.bias + n) : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < kScaleT; i++)
                v[2 * kFeat / 32 + i] =
                    m0 + 32 * i + lane < a.M ? __ldg(a.q_scale + m0 + 32 * i + lane) : 0.0f;
            bool ordinary = true;
#pragma unroll
            for (int i = 0; i < kFeat / 32; i++) ordinary = ordinary && ordinary_scale(v[2 * i]);
#pragma unroll
            for (int i = 0; i < kScaleT; i++)
                ordinary = ordinary && ordinary_scale(v[2 * kFeat / 32 + i]);
            ordinary = __all_sync(0xffffffffu, ordinary);
            bool good = true;
            if (lane == 0) good = wait_for(bar_sempty + 8 * ra.i, ra.ph ^ 1, abort_flag);
            if (!__shfl_sync(0xffffffffu, good ? 1 : 0, 0)) break;
            float *sc = scales + ra.i * kScaleFloats;
#pragma unroll
            for (int i = 0; i < kFeat / 32; i++) {
                sc[32 * i + lane] = v[2 * i];
                sc[kFeat + 32 * i + lane] = v[2 * i + 1];
            }
#pragma unroll
            for (int i = 0; i < kScaleT; i++) sc[2 * kFeat + 32 * i + lane] = v[2 * kFeat / 32 + i];
            if (lane == 0) *reinterpret_cast<int *>(smem_raw + kOrdinaryAt + 4 * ra.i) = ordinary;
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_sfull + 8 * ra.i);
        }
    } else if (warp >= kWarpEpi) {
        constexpr int kPart = BT / (kEpiWarps / 4), C = kPart < 16 ? kPart : 16;
        const int quad = warp & 3, part = (warp - kWarpEpi) >> 2;
        const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
        Ring ra(kAcc);
        if constexpr (FUSE) {
            quantize_slice<X, BT>(a, kb0, kbn, smem_raw + (stage0 - ctrl) + S * kStage, scales,
                                  reinterpret_cast<unsigned *>(scales + BT));
            // written through the generic proxy, read by the MMAs' async one
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_sfull);
        }
        for (int tile = first; tile < a.tiles; tile += step, ra.next()) {
            int ft, tt;
            tile_of(a, tile, ft, tt);
            const int n = ft * kTileF + (FORM == PAIR ? (int)rank * kFeat : 0) + quad * 32 + lane;
            bool good = true;
            if (lane == 0)
                good = (FORM == SPLIT || wait_for(bar_sfull + 8 * ra.i, ra.ph, abort_flag)) &&
                       wait_for(bar_tfull + 8 * ra.i, ra.ph, abort_flag);
            if (!__shfl_sync(0xffffffffu, good ? 1 : 0, 0)) break;
            tc_fence_after();
            const uint32_t col = tmem + lane_base + (uint32_t)(ra.i * BT + part * kPart);
            const float *sc = scales + ra.i * kScaleFloats;
            const float sw = FORM == SPLIT ? 0.0f : sc[quad * 32 + lane];
            const float bias = FORM == SPLIT ? 0.0f : sc[kFeat + quad * 32 + lane];
            const float *sx = sc + 2 * kFeat + part * kPart;
            const bool ordinary =
                FORM == SPLIT || *reinterpret_cast<const int *>(smem_raw + kOrdinaryAt + 4 * ra.i);
#pragma unroll 1
            for (int c = 0; c < kPart; c += C) {
                const int t0 = tt * BT + part * kPart + c;
                uint32_t acc[C];
                tmem_load(col + c, acc);
                if (c + C >= kPart) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if constexpr (FORM == PAIR)
                            mbar_arrive_relaxed_cluster(peer_addr(bar_tempty + 8 * ra.i, 0));
                        else
                            mbar_arrive_relaxed(bar_tempty + 8 * ra.i);
                    }
                }
                if constexpr (FORM == SPLIT) {
                    // partial sums, token-major: [BT][128] in the stages, all of
                    // which the MMAs have read
                    int *part_sum = reinterpret_cast<int *>(smem_raw + (stage0 - ctrl));
#pragma unroll
                    for (int j = 0; j < C; j++)
                        part_sum[(part * kPart + c + j) * kFeat + quad * 32 + lane] =
                            kbn ? (int)acc[j] : 0;
                } else if (t0 < a.M && n - lane < a.N) {
                    epilogue_any<T, C>(a, acc, t0, n, sw, bias, sx + c, ordinary, lane);
                }
            }
            if constexpr (FORM != SPLIT) {
                __syncwarp();
                if (lane == 0) mbar_arrive_relaxed(bar_sempty + 8 * ra.i);
            }
        }
    }
    __syncwarp();

    if constexpr (FORM == SPLIT) {
        cluster_sync();
        // this CTA's share of the tokens: 4 neighbouring channels a thread,
        // a token per warp at a time
        int ft, tt;
        tile_of(a, first, ft, tt);
        const int share = (BT + (int)peers - 1) / (int)peers;
        const int lo = (int)rank * share, hi = min(min(BT, lo + share), a.M - tt * BT);
        int bad = 0;
        for (uint32_t p = 0; p < peers; p++) bad |= peer_load1(peer_addr(ctrl + kAbortAt, p));
        const int n = ft * kFeat + 4 * lane;
        for (int j = lo + warp; j < hi && !bad; j += threads(BT, FORM) / 32) {
            int4 s = make_int4(0, 0, 0, 0);
            for (uint32_t p = 0; p < peers; p++) {
                const int4 v = peer_load(peer_addr(stage0 + (uint32_t)(j * kFeat + 4 * lane) * 4, p));
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
            const int t = tt * BT + j;
            const float sx = FUSE ? scales[j] : __ldg(a.q_scale + t);
            const int sums[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (n + i >= a.N) break;
                float v = scaled((float)sums[i], sx, __ldg(a.w_scale + n + i),
                                 a.bias ? __ldg(a.bias + n + i) : 0.0f);
                v = act_keep_nan(v, a.act);
                if (a.res)
                    v = __fadd_rn(v, to_float(((const T *)a.res)[(long long)t * a.ldres + n + i]));
                ((T *)a.y)[(long long)t * a.ldy + n + i] = from_float<T>(v);
            }
        }
    }
    // split: peers may still be reading this CTA's sums; pair: the leader's
    // MMAs read the peer's shared memory and write its TMEM
    tc_fence_before();
    if constexpr (FORM == WHOLE) __syncthreads();
    else cluster_sync();
    tc_fence_after();
    if (warp == kWarpMma) {
        if constexpr (FORM == PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                         "r"(kCols)
                         : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                         "r"(kCols)
                         : "memory");
    }
}

int sm_count() {
    int dev = 0, n = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n > 0 ? n : 148;
}

template <typename T, int BT, int FORM, typename X = int8_t>
Status launch(const LinearI8Args &p, Args a, int splits, cudaStream_t st) {
    CUtensorMap tmW, tmQ;
    if (!tma_encode_bytes(&tmW, p.w, p.K, p.N, p.ldw, kBK, kFeat) ||
        !(sizeof(X) > 1 ||
          tma_encode_bytes(&tmQ, p.q, p.K, p.M, p.ldq, kBK, load_tokens(BT, FORM))))
        return ERR_SHAPE;
    if (sizeof(X) > 1) tmQ = tmW;  // not read
    auto kernel = linear_i8_kernel<T, BT, FORM, X>;
    constexpr int smem = sizeof(X) > 1 ? fuse_smem(BT) : smem_bytes(BT, FORM);
    if (!smem_attr_once((const void *)kernel, smem)) {
        cudaGetLastError();
        return ERR_CUDA;
    }
    a.f_tiles = cdiv(p.N, FORM == PAIR ? 2 * kFeat : kFeat);
    a.t_tiles = cdiv(p.M, BT);
    if ((long long)a.f_tiles * a.t_tiles > 0x0fffffff || a.f_tiles > 0x0fffffff) return ERR_SHAPE;
    a.tiles = a.f_tiles * a.t_tiles;
    a.group = FastDiv((uint32_t)(kGroup * a.f_tiles));
    a.kps = cdiv(a.kblocks, splits);
    // CTAs of a cluster, and clusters: one for each tile (split) or as many
    // as the SMs hold
    const int cluster = FORM == PAIR ? 2 : FORM == SPLIT ? splits : 1;
    const int most = FORM == SPLIT ? a.tiles : sm_count() / cluster;
    const int clusters = a.tiles < most ? a.tiles : most;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(clusters * cluster));
    cfg.blockDim = dim3(threads(BT, FORM));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, tmW, tmQ, a);
    return cuda_status();
}

// Which form and token tile.  A model of the time in us, from timings of all
// forms over 26 sizes (M 1..13125, N and K 128..16384, 148 SMs), which it
// meets to about 10 %: a launch with its set-up and last epilogue takes 2.9;
// a k-block takes `step`, or what its CTAs' loads take from L2 (9 TB/s
// together) when that is more; `tail` is what a tile's epilogue adds; a split
// adds the cluster's exchange.  Some of the sizes, with the best form of each
// kind (us; K x N = 4096 x 4096 where nothing else is said):
//   M 1: split 16 by 4 8.0, by 8 8.6, whole 16 12.6;  M 64: split 64 by 4 9.3,
//   whole 64 13.3;  M 256: whole 64 13.7, split 64 by 2 13.8;  M 1024: whole
//   256 18.2, 128 26.8;  M 300, 256 x 256: whole 32 3.5, split 16 by 2 4.8;
//   M 2400, 256 x 1024: whole 64 5.7, 128 6.4, 256 6.7.
// Pairs against single CTAs at 256 tokens: 16384 x 1024 -> 4096 64.0 / 67.0,
// 8192 cubed 410 / 422, 52500 x 256 -> 1536 66.6 / 65.8, 1024 x 4096 -> 4096
// 21.0 / 18.4: pairs halve the token tile's traffic from L2, and pay where
// the main loop is long and every SM has several tiles.
struct Choice {
    int form, bt, splits;
};
Choice choose(int M, int N, int kblocks) {
    constexpr int kTokens[5] = {16, 32, 64, 128, 256};
    constexpr float kStep[5] = {0.27f, 0.30f, 0.31f, 0.355f, 0.42f};
    constexpr float kTail[5] = {0.1f, 0.28f, 0.34f, 1.03f, 2.9f};
    const int sms = sm_count();
    Choice best = {WHOLE, 256, 1};
    float least = 1e30f;
    for (int i = 0; i < 5; i++) {
        const float tiles = (float)cdiv(N, kFeat) * (float)cdiv(M, kTokens[i]);
        const float load = (float)stage_bytes(kTokens[i], WHOLE) / 9e6f;
        for (int splits = 1; splits <= 8; splits *= 2) {
            if (splits > 1 && (kTokens[i] > 64 || splits > kblocks)) break;
            const float kb = (float)cdiv(kblocks, splits);
            const float room = (float)(splits > 1 ? 2 * sms : sms);
            const float ctas = tiles * (float)splits, at_once = fminf(ctas, room);
            const float waves = ceilf(ctas / room);
            const float t = 2.9f + (splits > 1 ? 1.2f + 0.15f * (float)splits : 0.0f) +
                            waves * (kb * fmaxf(kStep[i], at_once * load) + kTail[i]);
            if (t < least) {
                least = t;
                best = {splits > 1 ? SPLIT : WHOLE, kTokens[i], splits};
            }
        }
    }
    if (best.form == SPLIT)  // whole k-blocks, none of the CTAs left without one
        best.splits = cdiv(kblocks, cdiv(kblocks, best.splits));
    if (best.form == WHOLE && best.bt == 256 && kblocks >= 8 &&
        (long long)cdiv(N, 2 * kFeat) * cdiv(M, 256) > sms / 2)
        best.form = PAIR;
    return best;
}

}  // namespace

namespace {

// tile origins stay below 2^31
bool sizes_ok(const LinearI8Args &p) {
    constexpr int kMost = 0x7fffffff - 512;
    return p.M > 0 && p.M <= kMost && p.N > 0 && p.N <= kMost && p.K > 0;
}

// p as the kernels take it; q and its scales apart
Args kernel_args(const LinearI8Args &p) {
    Args a = {};
    a.M = p.M; a.N = p.N; a.kblocks = cdiv(p.K, kBK);
    a.act = p.act;
    a.q_scale = p.q_scale; a.w_scale = p.w_scale; a.bias = p.bias;
    a.res = p.res.p; a.ldres = p.res.ld;
    a.y = (void *)p.y.p; a.ldy = p.y.ld;
    a.pairs = p.type != T_F32 && ((uintptr_t)a.y & 3) == 0 && (p.M == 1 || a.ldy % 2 == 0) &&
              (!a.res || (((uintptr_t)a.res & 3) == 0 && (p.M == 1 || a.ldres % 2 == 0)));
    return a;
}

}  // namespace

Status launch_linear_i8(const LinearI8Args &p, cudaStream_t st) {
    if (p.M == 0) return OK;
    if (!sizes_ok(p)) return ERR_SHAPE;
    const Args a = kernel_args(p);
    const Choice c = choose(p.M, p.N, a.kblocks);
    return with_type(p.type, [&](auto t) {
        using T = decltype(t);
        switch (c.form * 1024 + c.bt) {
            case PAIR * 1024 + 256: return launch<T, 256, PAIR>(p, a, 1, st);
            case SPLIT * 1024 + 16: return launch<T, 16, SPLIT>(p, a, c.splits, st);
            case SPLIT * 1024 + 32: return launch<T, 32, SPLIT>(p, a, c.splits, st);
            case SPLIT * 1024 + 64: return launch<T, 64, SPLIT>(p, a, c.splits, st);
            case WHOLE * 1024 + 16: return launch<T, 16, WHOLE>(p, a, 1, st);
            case WHOLE * 1024 + 32: return launch<T, 32, WHOLE>(p, a, 1, st);
            case WHOLE * 1024 + 64: return launch<T, 64, WHOLE>(p, a, 1, st);
            case WHOLE * 1024 + 128: return launch<T, 128, WHOLE>(p, a, 1, st);
            default: return launch<T, 256, WHOLE>(p, a, 1, st);
        }
    });
}

bool launch_linear_i8_few(const Rows &x, int x_type, const LinearI8Args &p, cudaStream_t st,
                          Status *status) {
    // every CTA reads all rows for their largest values, one after another.
    // K = N = 4096, BF16, against the two kernels: 1 row 8.9 / 9.5 us, 2 rows
    // 9.4 / 9.4, 4 rows 10.5 / 9.7, 16 rows 26 / 10; and a launch less, 2.5 us
    // of the host's time
    if (!sizes_ok(p) || p.M > 2 || (long long)p.M * p.K > 65536) return false;
    Args a = kernel_args(p);
    a.x = x.p; a.ldx = x.ld; a.K = p.K;
    const Choice c = choose(p.M, p.N, a.kblocks);
    // (the whole-K form of 16 tokens as a split in one)
    if (c.bt != 16 || cdiv(a.kblocks, c.splits) > kFuseBlocks ||
        (c.form != SPLIT && cdiv(p.N, kFeat) > 2 * sm_count()))
        return false;
    *status = with_type(p.type, [&](auto t) {
        using T = decltype(t);
        return with_type(x_type, [&](auto xt) {
            return launch<T, 16, SPLIT, decltype(xt)>(p, a, c.splits, st);
        });
    });
    return true;
}

int linear_error_fetch_and_clear() {
    int h = 0, zero = 0;
    cudaMemcpyFromSymbol(&h, g_linear_error, sizeof(int));
    if (h) cudaMemcpyToSymbol(g_linear_error, &zero, sizeof(int));
    return h;
}

}  // namespace ppdl
