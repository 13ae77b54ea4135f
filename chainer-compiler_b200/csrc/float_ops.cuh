// Element types of the float operators (linear.cu, layernorm.cu, logprobs.cu): loads and stores that convert to and from 32 bits, and the
// reductions of a warp.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.h"

namespace chxq {

inline bool is_float_type(int dtype) {
    return dtype == CHXQ_FLOAT32 || dtype == CHXQ_FLOAT16 || dtype == CHXQ_BFLOAT16;
}
inline int float_size(int dtype) {
    return dtype == CHXQ_FLOAT32 ? 4 : 2;
}

__device__ __forceinline__ float to_f32(float v) {
    return v;
}
__device__ __forceinline__ float to_f32(__half v) {
    return __half2float(v);
}
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// A parameter array in its own type, chosen at run time (uniform over the grid).
struct FloatArray {
    const void* p;
    int dtype;
};
__device__ __forceinline__ float load_param(const FloatArray& a, int64_t i) {
    if (a.dtype == CHXQ_FLOAT32) return __ldg(static_cast<const float*>(a.p) + i);
    if (a.dtype == CHXQ_FLOAT16) return __half2float(static_cast<const __half*>(a.p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(a.p)[i]);
}
__device__ __forceinline__ void store_param(void* p, int dtype, int64_t i, float v) {
    if (dtype == CHXQ_FLOAT32) static_cast<float*>(p)[i] = v;
    else if (dtype == CHXQ_FLOAT16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Calls f(T{}) with the element type of a dtype code that is_float_type accepts.
template <typename F>
int with_float_type(int dtype, F&& f) {
    if (dtype == CHXQ_FLOAT32) return f(float{});
    if (dtype == CHXQ_FLOAT16) return f(__half{});
    return f(__nv_bfloat16{});
}

}  // namespace chxq
