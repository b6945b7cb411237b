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

// TPR threads hold one row of at most TPR * NE values, NE each.  VEC: rows
// start on 16 bytes and D is a whole number of 16-byte vectors, a thread
// holds vectors lane, lane + TPR, ...; else single elements, grouped by
// GROUP neighbours (1: consecutive lanes read consecutive elements).
template <typename T, int TPR, int NE, bool VEC, int GROUP = 1>
struct RowTile {
    static constexpr int kVec = VEC ? 16 / (int)sizeof(T) : GROUP;
    static constexpr int kVecs = NE / kVec;
    static_assert(NE % kVec == 0, "whole vectors");

    struct Raw {
        T v[NE];
    };

    // column of the first value of vector i
    static __device__ __forceinline__ int column(int i, int lane) {
        return (i * TPR + lane) * kVec;
    }
    static __device__ __forceinline__ void load(Raw &r, const T *row, int D, int lane) {
#pragma unroll
        for (int i = 0; i < kVecs; i++) {
            const int c = column(i, lane);
            if constexpr (VEC) {
                uint4 u = make_uint4(0, 0, 0, 0);
                if (c < D) u = *reinterpret_cast<const uint4 *>(row + c);
                *reinterpret_cast<uint4 *>(&r.v[i * kVec]) = u;
            } else {
#pragma unroll
                for (int e = 0; e < kVec; e++) {
                    r.v[i * kVec + e] = from_float<T>(0.0f);
                    if (c + e < D) r.v[i * kVec + e] = row[c + e];
                }
            }
        }
    }
    static __device__ __forceinline__ void store(T *row, const Raw &r, int D, int lane) {
#pragma unroll
        for (int i = 0; i < kVecs; i++) {
            const int c = column(i, lane);
            if constexpr (VEC) {
                if (c < D)
                    *reinterpret_cast<uint4 *>(row + c) =
                        *reinterpret_cast<const uint4 *>(&r.v[i * kVec]);
            } else {
#pragma unroll
                for (int e = 0; e < kVec; e++)
                    if (c + e < D) row[c + e] = r.v[i * kVec + e];
            }
        }
    }
    // true for value j of the tile inside the row
    static __device__ __forceinline__ bool inside(int j, int D, int lane) {
        return column(j / kVec, lane) + (VEC ? 0 : j % kVec) < D;
    }
    // NE values of a vector of parameters (weights) of type WT at the tile's
    // columns, `none` where w is null; any alignment of w's element type
    template <typename WT>
    static __device__ __forceinline__ void load_params(float (&p)[NE], const WT *w, float none,
                                                       int D, int lane) {
#pragma unroll
        for (int i = 0; i < kVecs; i++) {
            const int c = column(i, lane);
#pragma unroll
            for (int e = 0; e < kVec; e++) p[i * kVec + e] = none;
            if (!w) continue;
            constexpr int kBytes = kVec * (int)sizeof(WT);
            if (VEC && kBytes >= 16 && c < D && ((uintptr_t)w & 15) == 0) {
                WT u[kVec];
#pragma unroll
                for (int b = 0; b < kBytes / 16; b++)
                    reinterpret_cast<uint4 *>(u)[b] = reinterpret_cast<const uint4 *>(w + c)[b];
#pragma unroll
                for (int e = 0; e < kVec; e++) p[i * kVec + e] = to_float(u[e]);
            } else {
#pragma unroll
                for (int e = 0; e < kVec; e++)
                    if (c + e < D) p[i * kVec + e] = to_float(w[c + e]);
            }
        }
    }
};

// Sums of N values over the TPR threads of each row, known to all of them.
// TPR <= 32: shuffles within the row's lanes.  Wider: the warps' sums go
// through sh[warps of the block][N] and one barrier of the whole block; a
// block that sums again gives another sh (or has a barrier in between).
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float *sh) {
    constexpr int kWidth = TPR < 32 ? TPR : 32;
#pragma unroll
    for (int o = kWidth / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if constexpr (TPR > 32) {
        constexpr int kWarps = TPR / 32;
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int i = 0; i < N; i++) sh[warp * N + i] = v[i];
        __syncthreads();
        sh += warp / kWarps * (kWarps * N);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = sh[i];
#pragma unroll
        for (int w = 1; w < kWarps; w++)
#pragma unroll
            for (int i = 0; i < N; i++) v[i] += sh[w * N + i];
    }
}

// The same for a block of several teams of TPR threads (of a warp, when TPR
// <= 32) that run on their own: a team's barrier is the named one 1 + team.
template <int TPR, int N>
__device__ __forceinline__ void team_sums(float (&v)[N], float *sh, int team) {
    constexpr int kWidth = TPR < 32 ? TPR : 32;
#pragma unroll
    for (int o = kWidth / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if constexpr (TPR > 32) {
        constexpr int kWarps = TPR / 32;
        sh += team * (kWarps * N);
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int i = 0; i < N; i++) sh[threadIdx.x % TPR / 32 * N + i] = v[i];
        asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(TPR) : "memory");
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = sh[i];
#pragma unroll
        for (int w = 1; w < kWarps; w++)
#pragma unroll
            for (int i = 0; i < N; i++) v[i] += sh[w * N + i];
    }
}

// Row buffers in shared memory, filled by bulk copies several rows ahead, for
// persistent blocks over rows that are whole 16-byte vectors.  With one row
// ahead in registers an iteration takes a memory latency, and the rows that
// two or three blocks have in flight are not enough to hide it.
//
// A team (the TPR threads of a row, or a warp with its 32 / TPR rows) has a
// ring of its own: stage = N matrices x kPer rows.  Every wait is bounded; a
// team that gave up goes on through its rows (its barriers stay matched)
// and stores nothing.
constexpr int kRingStages = 8;  // at most

template <typename T, int TPR, int THREADS, int N>
struct RowRing {
    static constexpr int kTeam = TPR < 32 ? 32 : TPR;
    static constexpr int kTeams = THREADS / kTeam, kPer = kTeam / TPR;
    static constexpr int kRows = kTeams * kPer;  // rows a block has at a time

    const T *src[N];  // null: no such matrix (the last one only)
    long long ld[N];
    long long rows, first, step;  // the team's first row, and from one of its stages to the next
    uint32_t row_bytes, stage_bytes, ring, bar0;
    const uint8_t *ptr;
    int n, stages, in_team;
    Ring at{1};
    volatile int *abort_flag;
    int *error;
    bool good = true;

    // bars: [kTeams][kRingStages]; smem: kTeams * stages * stage bytes,
    // 16-byte aligned.  Ends in a barrier of the block.
    __device__ __forceinline__ void setup(uint8_t *smem, uint64_t *bars, int *abort_word, int *err,
                                          long long rows_, int D, int stages_) {
        const int team = threadIdx.x / kTeam;
        in_team = threadIdx.x % kTeam;
        n = src[N - 1] ? N : N - 1;
        rows = rows_;
        stages = stages_;
        row_bytes = (uint32_t)D * sizeof(T);
        stage_bytes = (uint32_t)(n * kPer) * row_bytes;
        ring = smem_u32(smem) + (uint32_t)(team * stages) * stage_bytes;
        ptr = smem + (size_t)(team * stages) * stage_bytes;
        bar0 = smem_u32(bars + team * kRingStages);
        first = (long long)blockIdx.x * kRows + team * kPer;
        step = (long long)gridDim.x * kRows;
        at = Ring(stages);
        abort_flag = abort_word;
        error = err;
        if (threadIdx.x == 0) *abort_word = 0;
        if (in_team == 0) {
            for (int s = 0; s < stages; s++) mbar_init(bar0 + 8 * s, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncthreads();
    }
    // stage s takes rows r .. r + kPer - 1, as far as there are any
    __device__ __forceinline__ void fill(int s, long long r) {
        if (in_team >= 32 || r >= rows) return;
        const int count = (int)min((long long)kPer, rows - r);
        const uint32_t bar = bar0 + 8 * s, dst = ring + (uint32_t)s * stage_bytes;
        if (in_team == 0) mbar_expect_tx(bar, (uint32_t)(n * count) * row_bytes);
        __syncwarp();
        if (in_team < count) {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (i < n)
                    bulk_load(dst + (uint32_t)(i * kPer + in_team) * row_bytes,
                              src[i] + (r + in_team) * ld[i], row_bytes, bar);
        }
    }
    __device__ __forceinline__ void start() {
        for (int s = 0; s < stages; s++) fill(s, first + s * step);
    }
    __device__ __forceinline__ void wait() {
        good &= mbar_wait_bounded(bar0 + 8 * at.i, at.ph, abort_flag, error);
    }
    // the calling thread's row of matrix i in the present stage
    __device__ __forceinline__ const T *row(int i) const {
        return reinterpret_cast<const T *>(ptr + (size_t)at.i * stage_bytes +
                                           (size_t)(i * kPer + in_team / TPR) * row_bytes);
    }
    // after a barrier of the team behind its last read of the stage at rows
    // r0: filled again
    __device__ __forceinline__ void refill(long long r0) { fill(at.i, r0 + stages * step); }
};

// stages of a block's ring in `bytes` of shared memory
inline int ring_stages(int bytes, int matrices, int rows, int D, int size) {
    const long long stage = (long long)matrices * rows * D * size;
    const long long n = bytes / stage;
    return n > kRingStages ? kRingStages : (int)n;
}

// true when rows at p with this stride can be read as whole 16-byte vectors
inline bool vector_rows(const void *p, long long ld, long long rows, int D, int size) {
    return !p || (((uintptr_t)p & 15) == 0 && (long long)D * size % 16 == 0 &&
                  (rows <= 1 || ld * size % 16 == 0));
}

}  // namespace ppdl
