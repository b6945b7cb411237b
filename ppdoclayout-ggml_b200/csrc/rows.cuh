// rows.cuh — rows of a matrix held in registers by a group of threads, and
// sums over such a group: the common part of the row kernels (layernorm.cu,
// quantize.cu).
#pragma once

#include <type_traits>

#include "block.cuh"
#include "tc_ptx.cuh"

namespace ppdl {

// a compile-time number as a value (tile sizes for generic lambdas)
template <int V>
using Int = std::integral_constant<int, V>;

// TPR threads hold one row of at most TPR * NE values, NE each, value by
// value (any alignment): consecutive lanes hold consecutive values.
template <typename T, int TPR, int NE>
struct RowTile {
    struct Raw {
        T v[NE];
    };

    static __device__ __forceinline__ int column(int j, int lane) { return j * TPR + lane; }
    static __device__ __forceinline__ void load(Raw &r, const T *row, int D, int lane) {
#pragma unroll
        for (int j = 0; j < NE; j++) {
            r.v[j] = from_float<T>(0.0f);
            if (inside(j, D, lane)) r.v[j] = row[column(j, lane)];
        }
    }
    static __device__ __forceinline__ void store(T *row, const Raw &r, int D, int lane) {
#pragma unroll
        for (int j = 0; j < NE; j++)
            if (inside(j, D, lane)) row[column(j, lane)] = r.v[j];
    }
    // true for value j of the tile inside the row
    static __device__ __forceinline__ bool inside(int j, int D, int lane) {
        return column(j, lane) < D;
    }
    // parameters (weights) at the tile's columns, `none` where w is null
    template <typename WT>
    static __device__ __forceinline__ void load_params(float (&p)[NE], const WT *w, float none,
                                                       int D, int lane) {
#pragma unroll
        for (int j = 0; j < NE; j++) {
            p[j] = none;
            if (w && inside(j, D, lane)) p[j] = to_float(w[column(j, lane)]);
        }
    }
};

// Sums of N values over the TPR threads of each row, known to all of them, in
// an order of their own.  TPR <= 32: shuffles within the row's lanes.  Wider:
// the row's threads are a team with a named barrier (1 + team) of its own;
// the warps' sums go through sh[warps of the block][N], 16-byte aligned.  A
// team that sums again gives another sh (or has a barrier in between).
template <int TPR, int N>
__device__ __forceinline__ void team_sums(float (&v)[N], float *sh, int team) {
    constexpr int kWidth = TPR < 32 ? TPR : 32;
#pragma unroll
    for (int o = kWidth / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if constexpr (TPR > 32) {
        constexpr int kWarps = TPR / 32;
        static_assert(kWarps * N % 2 == 0, "whole pairs");
        sh += team * (kWarps * N);
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int i = 0; i < N; i++) sh[threadIdx.x % TPR / 32 * N + i] = v[i];
        asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(TPR) : "memory");
        // read as vectors; added in the warps' order
        constexpr int kV = kWarps * N % 4 == 0 ? 4 : 2;
        float all[kWarps * N];
#pragma unroll
        for (int i = 0; i < kWarps * N; i += kV) {
            if constexpr (kV == 4) {
                const float4 f = *reinterpret_cast<const float4 *>(sh + i);
                all[i] = f.x; all[i + 1] = f.y; all[i + 2] = f.z; all[i + 3] = f.w;
            } else {
                const float2 f = *reinterpret_cast<const float2 *>(sh + i);
                all[i] = f.x; all[i + 1] = f.y;
            }
        }
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = all[i];
#pragma unroll
        for (int w = 1; w < kWarps; w++)
#pragma unroll
            for (int i = 0; i < N; i++) v[i] += all[w * N + i];
    }
}

// Sixteen-byte vectors of a row held by TPR threads as pairs of FP32 values,
// NE values a thread: vectors lane, lane + TPR, ...
template <typename T, int TPR, int NE>
struct PairTile {
    static constexpr int kVec = 16 / (int)sizeof(T), kVecs = NE / kVec, kPairs = NE / 2;
    static_assert(NE % kVec == 0, "whole vectors");

    struct Raw {
        uint4 u[kVecs];
    };
    static __device__ __forceinline__ int column(int i, int lane) { return (i * TPR + lane) * kVec; }
    // column of pair j's first value
    static __device__ __forceinline__ int pair_column(int j, int lane) {
        return column(j / (kVec / 2), lane) + j % (kVec / 2) * 2;
    }
    // what lies past D is zero
    static __device__ __forceinline__ void load(Raw &r, const T *row, int D, int lane) {
#pragma unroll
        for (int i = 0; i < kVecs; i++) {
            r.u[i] = make_uint4(0, 0, 0, 0);
            if (column(i, lane) < D) r.u[i] = *reinterpret_cast<const uint4 *>(row + column(i, lane));
        }
    }
    static __device__ __forceinline__ void store(T *row, const Raw &r, int D, int lane) {
#pragma unroll
        for (int i = 0; i < kVecs; i++)
            if (column(i, lane) < D) *reinterpret_cast<uint4 *>(row + column(i, lane)) = r.u[i];
    }
    static __device__ __forceinline__ uint32_t word(const Raw &r, int k) {
        const uint4 u = r.u[k / 4];
        return k % 4 == 0 ? u.x : k % 4 == 1 ? u.y : k % 4 == 2 ? u.z : u.w;
    }
    static __device__ __forceinline__ void set_word(Raw &r, int k, uint32_t v) {
        uint4 &u = r.u[k / 4];
        if (k % 4 == 0) u.x = v;
        else if (k % 4 == 1) u.y = v;
        else if (k % 4 == 2) u.z = v;
        else u.w = v;
    }
    static __device__ __forceinline__ float2 pair(const Raw &r, int j) {
        if constexpr (sizeof(T) == 2)
            return unpack2<T>(word(r, j));
        else
            return make_float2(__uint_as_float(word(r, 2 * j)), __uint_as_float(word(r, 2 * j + 1)));
    }
    static __device__ __forceinline__ void set_pair(Raw &r, int j, float2 v) {
        if constexpr (sizeof(T) == 2) {
            set_word(r, j, pack2<T>(v.x, v.y));
        } else {
            set_word(r, 2 * j, __float_as_uint(v.x));
            set_word(r, 2 * j + 1, __float_as_uint(v.y));
        }
    }
    // the parameters (weights) of vector i, `none` where w is null; `wide`: w
    // is 16-byte aligned and a vector of it is at least as long
    template <typename WT>
    static __device__ __forceinline__ void vector_params(float2 (&p)[kVec / 2], const WT *w,
                                                         float none, int i, int D, int lane,
                                                         bool wide) {
        const int c = column(i, lane);
#pragma unroll
        for (int k = 0; k < kVec / 2; k++) p[k] = make_float2(none, none);
        if (!w || c >= D) return;
        constexpr int kBytes = kVec * (int)sizeof(WT);
        if constexpr (kBytes >= 16) {
            if (wide) {
#pragma unroll
                for (int h = 0; h < kBytes / 16; h++) {
                    const uint4 u = reinterpret_cast<const uint4 *>(w + c)[h];
                    if constexpr (sizeof(WT) == 2) {
                        p[4 * h] = unpack2<WT>(u.x);
                        p[4 * h + 1] = unpack2<WT>(u.y);
                        p[4 * h + 2] = unpack2<WT>(u.z);
                        p[4 * h + 3] = unpack2<WT>(u.w);
                    } else {
                        p[2 * h] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
                        p[2 * h + 1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
                    }
                }
                return;
            }
        }
#pragma unroll
        for (int k = 0; k < kVec / 2; k++)
            p[k] = make_float2(to_float(w[c + 2 * k]), to_float(w[c + 2 * k + 1]));
    }
    // parameters (weights) at the tile's columns, `none` where w is null
    template <typename WT>
    static __device__ __forceinline__ void load_params(float2 (&p)[kPairs], const WT *w, float none,
                                                       int D, int lane) {
#pragma unroll
        for (int j = 0; j < kPairs; j++) {
            const int c = pair_column(j, lane);
            p[j] = make_float2(none, none);
            if (w && c < D) p[j] = make_float2(to_float(w[c]), to_float(w[c + 1]));
        }
    }
};

// After a wait that gave up: what is still on its way into a ring (`fills`
// stages in turn, all of them issued) lands before the block may exit.
__device__ __forceinline__ void ring_drain(uint32_t full, int stages, int fills, int *error) {
    for (int s = 0; s < stages && s < fills; s++) {
        int none = 0;
        mbar_wait_bounded(full + 8 * s, (uint32_t)((fills - 1 - s) / stages & 1), &none, error);
    }
}

// Rows (of whole 16-byte vectors) through rings of buffers in shared memory,
// several rows ahead, by bulk copies.  With one row ahead in registers an
// iteration takes a memory latency, and the rows that two or three blocks
// have in flight are not enough to hide it.
//
// A team (the TPR threads of a row, or a warp with its 32 / TPR rows) has a
// ring of its own; a stage holds N matrices' rows.  A stage is refilled
// behind a barrier of the team, by one of its warps in turn, so that the
// copies' issue is neither on one warp's path nor repeated by all (with a
// slice of the row for every warp the backward pass of 16384 x 4096 BF16 took
// 95 us, so 87).  Every wait is bounded; a thread that gave up goes on
// through its rows (barriers stay matched), stores nothing and drains the
// ring.
constexpr int kRingStages = 8;  // at most

template <typename T, int TPR, int NE, int THREADS, int N>
struct RowRing {
    using Tile = PairTile<T, TPR, NE>;
    static constexpr int kTeam = TPR < 32 ? 32 : TPR, kTeams = THREADS / kTeam;
    static constexpr int kPer = kTeam / TPR;     // rows a team has at a time
    static constexpr int kRows = THREADS / TPR;  // rows a block has at a time
    struct Shared {
        uint64_t full[kTeams][kRingStages];
        int abort_word;
    };
    // Pointers and counts advance by additions: an instruction here is one for
    // 32 * NE values only.
    const T *next[N];            // what the lane copies next (lanes < kPer)
    long long advance[N], step;  // from one stage to the next: in elements, in rows
    long long first;             // the calling thread's first row
    uint32_t row_bytes, stage_bytes, full, ring;
    const uint8_t *ptr;
    int n, stages, lane, iters, fills, last_count, mine;
    Ring at{1};
    int *abort_flag, *error;
    bool good = true;

    // bytes of a stage of a block
    static constexpr long long block_stage(int matrices, int D) {
        return (long long)kRows * matrices * D * (int)sizeof(T);
    }

    // src[i] null: no such matrix (the last one only).  smem: stages *
    // block_stage() bytes, 16-byte aligned.  Ends in a barrier of the block.
    __device__ __forceinline__ void setup(const T *const (&src)[N], const long long (&ld)[N],
                                          uint8_t *smem, Shared *shared, int *err, long long rows,
                                          int D, int stages_) {
        const int team = threadIdx.x / kTeam;
        lane = threadIdx.x % 32;
        n = src[N - 1] ? N : N - 1;
        stages = stages_;
        row_bytes = (uint32_t)D * sizeof(T);
        stage_bytes = (uint32_t)(n * kPer) * row_bytes;
        const uint32_t at_byte = (uint32_t)(team * stages) * stage_bytes;
        ptr = smem + at_byte;
        ring = smem_u32(smem) + at_byte;
        full = smem_u32(shared->full[team]);
        abort_flag = &shared->abort_word;
        error = err;
        step = (long long)gridDim.x * kRows;
        const long long team_first = (long long)blockIdx.x * kRows + team * kPer;
        // rows of the team, and of the calling thread among them
        iters = team_first < rows ? (int)((rows - 1 - team_first) / step) + 1 : 0;
        last_count = (int)min((long long)kPer, rows - team_first - (iters - 1) * step);
        first = team_first + (TPR < 32 ? lane / TPR : 0);
        mine = first < rows ? (int)((rows - 1 - first) / step) + 1 : 0;
        fills = 0;
#pragma unroll
        for (int i = 0; i < N; i++) {
            next[i] = src[i] + (team_first + (lane < kPer ? lane : 0)) * ld[i];
            advance[i] = step * ld[i];
        }
        at = Ring(stages);
        if (threadIdx.x % kTeam == 0) {
            for (int s = 0; s < stages; s++) mbar_init(full + 8 * s, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        if (threadIdx.x == 0) shared->abort_word = 0;
        __syncthreads();
    }
    // stage s takes the team's next rows, as far as there are any
    __device__ __forceinline__ void fill(int s) {
        if (fills >= iters) return;
        if (TPR <= 32 || fills % (kTeam / 32) == (int)threadIdx.x % kTeam / 32) {
            const uint32_t bar = full + 8 * s, dst = ring + (uint32_t)s * stage_bytes;
            const int count = kPer == 1 ? 1 : fills == iters - 1 ? last_count : kPer;
            if (lane == 0) mbar_expect_tx(bar, (uint32_t)(n * count) * row_bytes);
            if (kPer > 1) __syncwarp();
            if (lane < count) {
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (i < n)
                        bulk_load(dst + (uint32_t)(i * kPer + lane) * row_bytes, next[i], row_bytes,
                                  bar);
            }
        }
#pragma unroll
        for (int i = 0; i < N; i++) next[i] += advance[i];
        fills++;
    }
    __device__ __forceinline__ void start() {
        for (int s = 0; s < stages; s++) fill(s);
    }
    __device__ __forceinline__ void wait() {
        good &= mbar_wait_bounded(full + 8 * at.i, at.ph, abort_flag, error);
    }
    // the calling thread's row of matrix i in the present stage
    __device__ __forceinline__ const T *row(int i) const {
        return reinterpret_cast<const T *>(ptr + (uint32_t)at.i * stage_bytes +
                                           (uint32_t)(i * kPer + (TPR < 32 ? lane / TPR : 0)) *
                                               row_bytes);
    }
    // behind a barrier of the team after its last read of the present stage
    __device__ __forceinline__ void refill() {
        if (TPR <= 32) __syncwarp();
        fill(at.i);
    }
    // behind the last row
    __device__ __forceinline__ void finish() {
        if (!good) ring_drain(full, stages, iters, error);
    }
};

// Values of a row in shared memory at any alignment held by TPR threads as NP
// pairs each.  16-bit values are read and written as the memory's 32-bit
// words lane, lane + TPR, ...: a row that starts in the middle of a word
// (shift 1) holds column c in half (c + 1) % 2 of word (c + 1) / 2, and the
// words it shares with its neighbours are touched by halves.  FP32 values:
// columns lane + 2 j TPR and TPR behind it.  The caller promises D >= 2 TPR
// (NP / 2), so that pairs 1 .. NP / 2 - 1 need no check.
template <typename T, int TPR, int NP>
struct WordTile {
    static constexpr bool kWords = sizeof(T) == 2;
    struct Raw {
        uint32_t u[kWords ? NP : 2 * NP];
    };
    int lane, shift;
    uint32_t in[2];  // bit j: the pair's first, second value lies in the row

    __device__ __forceinline__ WordTile(int lane_, int shift_, int D)
        : lane(lane_), shift(kWords ? shift_ : 0), in{0, 0} {
#pragma unroll
        for (int j = 0; j < NP; j++)
#pragma unroll
            for (int h = 0; h < 2; h++)
                if ((unsigned)column(j, h) < (unsigned)D) in[h] |= 1u << j;
    }
    __device__ __forceinline__ int column(int j, int h) const {
        return kWords ? 2 * (lane + j * TPR) + h - shift : lane + (2 * j + h) * TPR;
    }
    __device__ __forceinline__ bool inside(int j, int h) const {
        return (j >= 1 && j < NP / 2) || (in[h] >> j & 1);
    }
    // 1 for the pair's values inside the row, 0 for those outside
    __device__ __forceinline__ float2 ones(int j) const {
        return make_float2(inside(j, 0) ? 1.0f : 0.0f, inside(j, 1) ? 1.0f : 0.0f);
    }
    // what lies outside is zero
    __device__ __forceinline__ void load(Raw &r, const T *row) const {
        if constexpr (kWords) {
            const uint16_t *v = reinterpret_cast<const uint16_t *>(row) + 2 * lane - shift;
#pragma unroll
            for (int j = 0; j < NP; j++, v += 2 * TPR) {
                r.u[j] = 0;
                if (inside(j, 0) && inside(j, 1)) r.u[j] = *reinterpret_cast<const uint32_t *>(v);
                else if (inside(j, 0)) r.u[j] = v[0];
                else if (inside(j, 1)) r.u[j] = (uint32_t)v[1] << 16;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 2 * NP; j++) {
                r.u[j] = 0;
                if (inside(j / 2, j % 2)) r.u[j] = __float_as_uint(row[lane + j * TPR]);
            }
        }
    }
    __device__ __forceinline__ void store(T *row, const Raw &r) const {
        if constexpr (kWords) {
            uint16_t *v = reinterpret_cast<uint16_t *>(row) + 2 * lane - shift;
#pragma unroll
            for (int j = 0; j < NP; j++, v += 2 * TPR) {
                if (inside(j, 0) && inside(j, 1)) *reinterpret_cast<uint32_t *>(v) = r.u[j];
                else if (inside(j, 0)) v[0] = (uint16_t)r.u[j];
                else if (inside(j, 1)) v[1] = (uint16_t)(r.u[j] >> 16);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 2 * NP; j++)
                if (inside(j / 2, j % 2)) row[lane + j * TPR] = __uint_as_float(r.u[j]);
        }
    }
    static __device__ __forceinline__ float2 pair(const Raw &r, int j) {
        if constexpr (kWords) return unpack2<T>(r.u[j]);
        else return make_float2(__uint_as_float(r.u[2 * j]), __uint_as_float(r.u[2 * j + 1]));
    }
    static __device__ __forceinline__ void set_pair(Raw &r, int j, float2 v) {
        if constexpr (kWords) {
            r.u[j] = pack2<T>(v.x, v.y);
        } else {
            r.u[2 * j] = __float_as_uint(v.x);
            r.u[2 * j + 1] = __float_as_uint(v.y);
        }
    }
    template <typename WT>
    __device__ __forceinline__ void load_params(float2 (&p)[NP], const WT *w, float none) const {
#pragma unroll
        for (int j = 0; j < NP; j++) {
            p[j] = both(none);
            if (w && inside(j, 0)) p[j].x = to_float(w[column(j, 0)]);
            if (w && inside(j, 1)) p[j].y = to_float(w[column(j, 1)]);
        }
    }
    // where column c of a row with this shift lies in [NP][TPR][2]
    static __device__ __forceinline__ int place(int c, int shift) {
        if constexpr (kWords) return c + shift;
        else return (c / (2 * TPR) * TPR + c % TPR) * 2 + c / TPR % 2;
    }
};

// Dense matrices whose rows are no whole 16-byte vectors (an odd number of
// 16-bit values, say), a group of rows at a time: `rows_at` rows, so many
// that a group is whole vectors and starts on one.  Groups come through a
// ring by bulk copies and results, written over what they came from, leave
// by bulk copies; between the two the rows are read and written in shared
// memory by WordTile, where neither alignment nor the width of an access
// costs memory transactions.  The bytes of the last group past its last whole vector
// are moved by plain loads and stores.  Every wait is bounded; a block that
// gave up goes on and stores nothing.
template <typename T, int N>
struct GroupRing {
    struct Shared {
        uint64_t full[kRingStages];
        int abort_word;
    };
    const T *src[N];  // null: no such matrix (the last one only)
    long long rows, group;  // the present group
    uint32_t matrix_bytes, full, ring;
    uint8_t *ptr;
    int n, stages, D, rows_at, iters;
    Ring at{1};
    int *abort_flag, *error;
    bool good = true;

    __device__ __forceinline__ void setup(const T *const (&s)[N], uint8_t *smem, Shared *shared,
                                          int *err, long long rows_, int D_, int rows_at_,
                                          int stages_) {
#pragma unroll
        for (int i = 0; i < N; i++) src[i] = s[i];
        n = src[N - 1] ? N : N - 1;
        rows = rows_;
        D = D_;
        rows_at = rows_at_;
        stages = stages_;
        matrix_bytes = (uint32_t)(rows_at * D) * sizeof(T);
        ptr = smem;
        ring = smem_u32(smem);
        full = smem_u32(shared->full);
        abort_flag = &shared->abort_word;
        error = err;
        group = blockIdx.x;
        const long long groups = (rows + rows_at - 1) / rows_at;
        iters = group < groups ? (int)((groups - 1 - group) / gridDim.x) + 1 : 0;
        at = Ring(stages);
        if (threadIdx.x == 0) {
            for (int i = 0; i < stages; i++) mbar_init(full + 8 * i, 1);
            shared->abort_word = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncthreads();
    }
    __device__ __forceinline__ int count(long long g) const {
        return (int)min((long long)rows_at, rows - g * rows_at);
    }
    __device__ __forceinline__ uint32_t group_bytes(long long g) const {
        return (uint32_t)(count(g) * D) * sizeof(T);
    }
    // thread 0: the block's group `it` into its stage
    __device__ __forceinline__ void fill(int it) {
        if (it >= iters) return;
        const int s = it % stages;
        const long long g = blockIdx.x + (long long)it * gridDim.x;
        const uint32_t whole = group_bytes(g) & ~15u;
        mbar_expect_tx(full + 8 * s, (uint32_t)n * whole);
        if (!whole) return;
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < n)
                bulk_load(ring + (uint32_t)(s * n + i) * matrix_bytes, src[i] + g * rows_at * D,
                          whole, full + 8 * s);
    }
    __device__ __forceinline__ void start() {
        if (threadIdx.x == 0)
            for (int it = 0; it < stages; it++) fill(it);
    }
    __device__ __forceinline__ T *buffer(int i) const {
        return reinterpret_cast<T *>(ptr + (uint32_t)(at.i * n + i) * matrix_bytes);
    }
    // all threads: the present group is in its buffers
    __device__ __forceinline__ void wait() {
        good &= mbar_wait_bounded(full + 8 * at.i, at.ph, abort_flag, error);
        const uint32_t bytes = group_bytes(group);
        if (bytes & 15u) {
            const int first = (int)((bytes & ~15u) / sizeof(T)), last = (int)(bytes / sizeof(T));
            if ((int)threadIdx.x < last - first)
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (i < n)
                        buffer(i)[first + threadIdx.x] =
                            src[i][group * rows_at * D + first + threadIdx.x];
            __syncthreads();
        }
    }
    // all threads, their results written: matrix i of the stage goes to dst,
    // and j (when given one) to dst2; the stage before this one, read out by
    // now, is filled again
    __device__ __forceinline__ void store(int it, int i, T *dst, int j, T *dst2) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        const uint32_t bytes = group_bytes(group), whole = bytes & ~15u;
        const long long at_value = group * rows_at * D;
        if (threadIdx.x == 0) {
            if (*(volatile int *)abort_flag) good = false;
            if (good && whole) {
                bulk_store(dst + at_value, ring + (uint32_t)(at.i * n + i) * matrix_bytes, whole);
                if (dst2)
                    bulk_store(dst2 + at_value, ring + (uint32_t)(at.i * n + j) * matrix_bytes,
                               whole);
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            if (it > 0) {
                asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                fill(it - 1 + stages);
            }
        }
        if ((bytes & 15u) && good) {
            const int first = (int)(whole / sizeof(T)), last = (int)(bytes / sizeof(T));
            if ((int)threadIdx.x < last - first) {
                dst[at_value + first + threadIdx.x] = buffer(i)[first + threadIdx.x];
                if (dst2) dst2[at_value + first + threadIdx.x] = buffer(j)[first + threadIdx.x];
            }
        }
        at.next();
        group += gridDim.x;
    }
    // thread 0 leaves last: its stores have been written
    __device__ __forceinline__ void finish() {
        if (!good) ring_drain(full, stages, iters, error);
        if (threadIdx.x == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
};

// stages of a block's rings in `bytes` of shared memory
inline int ring_stages(long long bytes, long long stage) {
    const long long n = bytes / stage;
    return n > kRingStages ? kRingStages : (int)n;
}

// true when rows at p with this stride can be read as whole 16-byte vectors
inline bool vector_rows(const void *p, long long ld, long long rows, int D, int size) {
    return !p || (((uintptr_t)p & 15) == 0 && (long long)D * size % 16 == 0 &&
                  (rows <= 1 || ld * size % 16 == 0));
}

}  // namespace ppdl
