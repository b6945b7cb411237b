// block.cuh — element types and small device helpers of the transformer-block
// operators (layernorm.cu, linear_i8.cu, rotary.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace ppdl {

// Element types of the block operators (PPDL_F32 / PPDL_BF16 / PPDL_F16).
enum ElemType : int { T_F32 = 0, T_BF16 = 1, T_F16 = 2 };

inline int elem_size(int type) { return type == T_F32 ? 4 : 2; }
inline bool elem_type_ok(int type) { return type >= T_F32 && type <= T_F16; }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

// Round to nearest even, the only rounding of a result to fewer bits.
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Two 16-bit values in a 32-bit word, the first in its low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&p);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&p);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

// Two FP32 values in one register pair: sm_100 multiplies and adds them in
// one instruction, each rounded as its own.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\t"
        "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z, w;\n\t"
        "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\t"
        "fma.rn.f32x2 z, x, y, w;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\t"
        "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "add.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

__device__ __forceinline__ float2 sub2(float2 a, float2 b) {
    return add2(a, make_float2(-b.x, -b.y));
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// act_apply with a ReLU that keeps a NaN: a token that is not finite has to
// stay visible in its output row (fmaxf would return the zero).
__device__ __forceinline__ float act_keep_nan(float v, int act) {
    if (act != ACT_RELU) return act_apply(v, act);
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(0.0f));
    return r;
}

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery,
// "Division by invariant integers using multiplication", PLDI 1994)
struct FastDiv {
    uint32_t d = 1, mul = 1, shift = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t d_) : d(d_) {
        while ((1ull << shift) < d) shift++;
        mul = (uint32_t)((((1ull << shift) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ int div(int n) const {
        return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift);
    }
};

// f(T{}) with the C++ type of an element type
template <typename F>
inline Status with_type(int type, F f) {
    switch (type) {
        case T_F32: return f(float{});
        case T_BF16: return f(__nv_bfloat16{});
        case T_F16: return f(__half{});
        default: return ERR_SHAPE;
    }
}

// Sum of v over the block, known to every thread; sh holds 32 floats.  The
// order of the additions depends on the block size alone.
__device__ __forceinline__ float block_sum(float v, float *sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? sh[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    return v;
}

}  // namespace ppdl
