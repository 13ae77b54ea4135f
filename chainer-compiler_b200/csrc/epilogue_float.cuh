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
template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == CHXQ_ACT_RELU) return z < 0.f ? 0.f : z;  // NaN stays NaN
    if constexpr (ACT == CHXQ_ACT_GELU) return 0.5f * z * erfcf(z * -0.70710678118654752f);
    if constexpr (ACT == CHXQ_ACT_GELU_TANH) return z / (1.f + expf(-1.5957691216057308f * (z + 0.044715f * z * z * z)));
    if constexpr (ACT == CHXQ_ACT_SWISH) return z / (1.f + expf(-z));
    if constexpr (ACT == CHXQ_ACT_SIGMOID) return 1.f / (1.f + expf(-z));
    if constexpr (ACT == CHXQ_ACT_TANH) return tanhf(z);
    return z;
}

__device__ __forceinline__ f32x2 ex2_x2(f32x2 a) {  // 2^a, good to 2^-22
    const float2 f = split_x2(a);
    float x, y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x) : "f"(f.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(f.y));
    return make_x2(x, y);
}
__device__ __forceinline__ f32x2 rcp_x2(f32x2 a) {  // 1 / a, good to 2^-23
    const float2 f = split_x2(a);
    float x, y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(x) : "f"(f.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(f.y));
    return make_x2(x, y);
}
__device__ __forceinline__ f32x2 both(float v) {
    return make_x2(v, v);
}

// Two values at a time for 16-bit outputs, with exponential and reciprocal by the approximate instructions: a few 2^-22 relative near zero.  Further out the
// exponent, which is rounded at its own size, adds 2^-24 of its magnitude (base 2): 18 x 2^-22 for Gelu at z = -10, 8 x 2^-22 for Swish at z = -80, still a
// thousandth of bf16's rounding, and fp16 has no such values.  Exponentials and reciprocals below 2^-126 count as zero (Swish and Sigmoid below -87.3).
// Gelu: erfc by the Chebyshev fit of Press et al., Numerical Recipes, 6.2 ("erfcc", fractional error below 1.2e-7 everywhere): for u >= 0
// erfc(u) = t exp(P(t) - u^2), t = 1 / (1 + u / 2); here with P and u^2 times log2 e.  [4096, 1024] x [4096, 1024]^T with Gelu on one B200: 55 us with
// CUDA's erfcf.
template <int ACT>
__device__ __forceinline__ f32x2 activate_fast(f32x2 z) {
    constexpr float L = 1.4426950408889634f;
    if constexpr (ACT == CHXQ_ACT_GELU) {
        const f32x2 u = mul2(z & 0x7fffffff7fffffffull, both(0.70710678118654752f));
        const f32x2 t = rcp_x2(fma2(u, both(0.5f), both(1.f)));
        f32x2 p = fma2(t, both(0.17087277f * L), both(-0.82215223f * L));
        p = fma2(t, p, both(1.48851587f * L));
        p = fma2(t, p, both(-1.13520398f * L));
        p = fma2(t, p, both(0.27886807f * L));
        p = fma2(t, p, both(-0.18628806f * L));
        p = fma2(t, p, both(0.09678418f * L));
        p = fma2(t, p, both(0.37409196f * L));
        p = fma2(t, p, both(1.00002368f * L));
        p = fma2(t, p, both(-1.26551223f * L));
        const f32x2 e = mul2(t, ex2_x2(fma2(mul2(u, both(-L)), u, p)));
        const float2 zf = split_x2(z), ef = split_x2(e);
        return mul2(mul2(z, both(0.5f)), make_x2(zf.x < 0.f ? ef.x : 2.f - ef.x, zf.y < 0.f ? ef.y : 2.f - ef.y));
    } else if constexpr (ACT == CHXQ_ACT_GELU_TANH || ACT == CHXQ_ACT_SWISH || ACT == CHXQ_ACT_SIGMOID) {
        const f32x2 u = ACT == CHXQ_ACT_GELU_TANH ? mul2(z, fma2(mul2(z, z), both(-1.5957691216057308f * 0.044715f * L), both(-1.5957691216057308f * L))) : mul2(z, both(-L));
        const f32x2 r = rcp_x2(add2(ex2_x2(u), both(1.f)));
        return ACT == CHXQ_ACT_SIGMOID ? r : mul2(z, r);
    } else {
        const float2 f = split_x2(z);
        return make_x2(activate<ACT>(f.x), activate<ACT>(f.y));
    }
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
        for (int j = 0; j < N; j += 2) {
            const f32x2 r = make_x2(res[j], res[j + 1]);
            f32x2 z = make_x2(v[j], v[j + 1]);
            if (first) z = add2(z, r);
            if constexpr (FAST) {
                z = activate_fast<decltype(act)::value>(z);
            } else {
                const float2 f = split_x2(z);
                z = make_x2(activate<decltype(act)::value>(f.x), activate<decltype(act)::value>(f.y));
            }
            if (!first) z = add2(z, r);
            const float2 f = split_x2(z);
            v[j] = f.x;
            v[j + 1] = f.y;
        }
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
