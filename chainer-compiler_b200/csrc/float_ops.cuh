// Element types of the float operators (linear.cu, layernorm.cu, logprobs.cu): loads and stores that convert to and from 32 bits, and the
// reductions of a warp.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "common.h"

namespace chxq {

inline bool is_float_type(int dtype) {
    return dtype == CHXQ_FLOAT32 || dtype == CHXQ_FLOAT16 || dtype == CHXQ_BFLOAT16;
}
inline int float_size(int dtype) {
    return dtype == CHXQ_FLOAT32 ? 4 : 2;
}

// Whether addresses are multiples of the size of the values there: an access elsewhere faults.
template <typename... P>
inline bool on_values_of(int size, const P*... p) {
    return (((uintptr_t)0 | ... | reinterpret_cast<uintptr_t>(p)) & (uintptr_t)(size - 1)) == 0;
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

// Two 32-bit values per instruction.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 make_x2(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 split_x2(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// N consecutive values as one load or store of N * sizeof(T) bytes (2, 4 or 16): the address is a multiple of that.
template <typename T, int N>
struct Pack {
    static constexpr int kBytes = N * (int)sizeof(T), kWords = kBytes >= 4 ? kBytes / 4 : 1;
    static_assert(kBytes == 2 || kBytes == 4 || kBytes == 16, "no such access");
    uint32_t w[kWords];

    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kBytes == 16) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else if constexpr (kBytes == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        static_assert(kBytes == 16, "a 16-byte access");
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0u;
    }
    __device__ __forceinline__ void put(int i, T v) {  // into a zero
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v);
        else w[i >> 1] |= (uint32_t)*reinterpret_cast<const uint16_t*>(&v) << (i & 1 ? 16 : 0);
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        const uint32_t v = w[i >> 1];
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(i & 1 ? v & 0xffff0000u : v << 16);
        const uint16_t h = (uint16_t)(i & 1 ? v >> 16 : v);
        return __half2float(*reinterpret_cast<const __half*>(&h));
    }
    __device__ __forceinline__ f32x2 pair(int i) const {  // values 2 i and 2 i + 1
        if constexpr (sizeof(T) == 4) {
            return make_x2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        } else if constexpr (std::is_same<T, __half>::value) {
            const uint32_t v = w[i];
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
            return make_x2(f.x, f.y);
        } else {
            return make_x2(get(2 * i), get(2 * i + 1));
        }
    }
    __device__ __forceinline__ void set_pair(int i, f32x2 v) {
        const float2 f = split_x2(v);
        if constexpr (sizeof(T) == 4) {
            w[2 * i] = __float_as_uint(f.x);
            w[2 * i + 1] = __float_as_uint(f.y);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __half2 h = __floats2half2_rn(f.x, f.y);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    __device__ __forceinline__ float max_value() const {  // NaN if there is one; N > 1
        if constexpr (sizeof(T) == 4) {
            float m = __uint_as_float(w[0]);
#pragma unroll
            for (int i = 1; i < kWords; ++i) asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(m), "f"(__uint_as_float(w[i])));
            return m;
        } else {
            uint32_t m = w[0];
#pragma unroll
            for (int i = 1; i < kWords; ++i) {
                if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(w[i]));
                else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(w[i]));
            }
            Pack<T, 2> p;
            p.w[0] = m;
            float r;
            asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(p.get(0)), "f"(p.get(1)));
            return r;
        }
    }
    // Bit i: value i is not below `bound` (NaN is not), which is a value of T itself.
    __device__ __forceinline__ uint32_t not_below(float bound) const {
        uint32_t r = 0;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) r |= !(__uint_as_float(w[i]) < bound) ? 1u << i : 0u;
        } else {
            const T h = from_f32<T>(bound);
            const uint32_t b = *reinterpret_cast<const uint16_t*>(&h) * 0x00010001u;
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                uint32_t m;  // per half: all ones where it is not below
                const uint32_t v = w[i];
                if constexpr (std::is_same<T, __half>::value) m = __hgeu2_mask(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&b));
                else m = __hgeu2_mask(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&b));
                r |= ((m & 1u) | (m >> 30 & 2u)) << (2 * i);
            }
        }
        return r;
    }
    __device__ __forceinline__ float pick(int i) const {  // value i, where i is not known at compile time
        static_assert(kWords == 4, "a 16-byte access");
        const int k = sizeof(T) == 4 ? i : i >> 1;
        const uint32_t a = k & 1 ? w[1] : w[0], b = k & 1 ? w[3] : w[2], v = k & 2 ? b : a;
        if constexpr (sizeof(T) == 4) return __uint_as_float(v);
        const uint16_t h = (uint16_t)(v >> (16 * (i & 1)));
        return to_f32(*reinterpret_cast<const T*>(&h));
    }
    __device__ __forceinline__ T value(int i) const {  // as it is stored
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[i]);
        } else {
            const uint16_t h = (uint16_t)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1]);
            return *reinterpret_cast<const T*>(&h);
        }
    }
};

// N consecutive values of a parameter array for a row's 16-byte piece: N = 8 beside a 16-bit type, or 4 beside float32, whose parameters are float32 too.  The
// array starts on a 16-byte boundary.
template <int N>
__device__ __forceinline__ void load_params(const FloatArray& a, int64_t i, float (&f)[N]) {
    static_assert(N == 4 || N == 8, "a 16-byte piece");
    if (N == 4 || a.dtype == CHXQ_FLOAT32) {
        const float* p = static_cast<const float*>(a.p) + i;
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(p + j));
            f[j] = v.x; f[j + 1] = v.y; f[j + 2] = v.z; f[j + 3] = v.w;
        }
    } else if constexpr (N == 8) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.p) + i));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (a.dtype == CHXQ_BFLOAT16) {
                f[2 * j] = __uint_as_float(w[j] << 16);
                f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            } else {
                const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                f[2 * j] = h.x;
                f[2 * j + 1] = h.y;
            }
        }
    }
}

// The same from any place: N loads, of T or of 32 bits.
template <typename T, int N>
__device__ __forceinline__ void load_params_any(const FloatArray& a, int64_t i, float (&f)[N]) {
    if (a.dtype == CHXQ_FLOAT32) {
        const float* p = static_cast<const float*>(a.p) + i;
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = __ldg(p + j);
    } else {
        const T* p = static_cast<const T*>(a.p) + i;
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = to_f32(p[j]);
    }
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
