// Epilogue of the float matrix product: bias, activation and residual on the 32-bit sum, then the one rounding to the output's type.
#pragma once

#include <type_traits>

#include "float_ops.cuh"

namespace chxq {

struct LinearEpilogue {
    const void* bias;  // [O] or null
    int bias_dtype;
    const void* residual;  // [M, ldr] of the output's type, or null
    int64_t ldr;
    int activation;      // CHXQ_ACT_*
    int residual_first;  // the residual joins in front of the activation
    void* y;
    int64_t ldy;
};

// Gelu through erfc, which keeps its relative accuracy where 1 + erf cancels; the tanh form as z / (1 + exp(-2 u)), for the same reason.
// Large negative z: exp overflows to infinity and the quotient is -0, as the limit is.
// FAST: exponential and quotient by the approximate instructions, a few 2^-22 relative and 2^-24 |z| more from the scaled argument: a
// thousandth of a 16-bit output's rounding.
template <int ACT, bool FAST = false>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == CHXQ_ACT_RELU) return z < 0.f ? 0.f : z;  // NaN stays NaN
    if constexpr (ACT == CHXQ_ACT_GELU) return 0.5f * z * erfcf(z * -0.70710678118654752f);
    if constexpr (ACT == CHXQ_ACT_TANH) return tanhf(z);
    if constexpr (ACT == CHXQ_ACT_GELU_TANH || ACT == CHXQ_ACT_SWISH || ACT == CHXQ_ACT_SIGMOID) {
        const float u = ACT == CHXQ_ACT_GELU_TANH ? -1.5957691216057308f * (z + 0.044715f * z * z * z) : -z;
        const float d = 1.f + (FAST ? __expf(u) : expf(u)), n = ACT == CHXQ_ACT_SIGMOID ? 1.f : z;
        return FAST ? __fdividef(n, d) : n / d;
    }
    return z;
}

// Calls f(integral constant) with the activation code as a compile-time value (uniform over the grid).
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
    switch (act) {
        case CHXQ_ACT_RELU: f(std::integral_constant<int, CHXQ_ACT_RELU>{}); break;
        case CHXQ_ACT_GELU: f(std::integral_constant<int, CHXQ_ACT_GELU>{}); break;
        case CHXQ_ACT_GELU_TANH: f(std::integral_constant<int, CHXQ_ACT_GELU_TANH>{}); break;
        case CHXQ_ACT_SWISH: f(std::integral_constant<int, CHXQ_ACT_SWISH>{}); break;
        case CHXQ_ACT_SIGMOID: f(std::integral_constant<int, CHXQ_ACT_SIGMOID>{}); break;
        case CHXQ_ACT_TANH: f(std::integral_constant<int, CHXQ_ACT_TANH>{}); break;
        default: f(std::integral_constant<int, CHXQ_ACT_NONE>{}); break;
    }
}

// Residual and activation on N sums that hold their bias; one dispatch for all (each activation's code is met once: a cold instruction cache costs the
// smallest products more than their arithmetic).
template <int N, bool FAST>
__device__ __forceinline__ void epilogue_apply(const LinearEpilogue& e, float (&v)[N], const float (&res)[N]) {
    const bool first = e.residual_first;
    with_activation(e.activation, [&](auto act) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = activate<decltype(act)::value, FAST>(v[j] + (first ? res[j] : 0.f)) + (first ? 0.f : res[j]);
    });
}

// One output from its sum.
template <typename T>
__device__ __forceinline__ void epilogue_store(const LinearEpilogue& e, int64_t m, int64_t o, float acc) {
    if (e.bias) acc += load_param({e.bias, e.bias_dtype}, o);
    const float r = e.residual ? to_f32(static_cast<const T*>(e.residual)[m * e.ldr + o]) : 0.f;
    if (e.residual && e.residual_first) acc += r;
    with_activation(e.activation, [&](auto act) { acc = activate<decltype(act)::value>(acc); });
    if (e.residual && !e.residual_first) acc += r;
    static_cast<T*>(e.y)[m * e.ldy + o] = from_f32<T>(acc);
}

}  // namespace chxq
