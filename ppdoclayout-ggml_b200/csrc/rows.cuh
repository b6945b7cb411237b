// rows.cuh — rows of a matrix held in registers by a group of threads, and
// sums over such a group: the common part of the row kernels (layernorm.cu,
// quantize.cu).
#pragma once

#include <type_traits>

#include "block.cuh"

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

// true when rows at p with this stride can be read as whole 16-byte vectors
inline bool vector_rows(const void *p, long long ld, long long rows, int D, int size) {
    return !p || (((uintptr_t)p & 15) == 0 && (long long)D * size % 16 == 0 &&
                  (rows <= 1 || ld * size % 16 == 0));
}

}  // namespace ppdl
