// LayerNormalization over the last `D` values of each row, and its gradient.
//   m = mean(x), s = 1 / sqrt(mean((x - m)^2) + epsilon), xh = (x - m) s, y = xh scale + bias
//   dx = s (scale dy - mean(scale dy) - xh mean(scale dy xh)),  dscale = sum over rows of dy xh,  dbias = sum over rows of dy
// Sums and statistics are held in 32 bits; the variance is that of the deviations, which does not cancel.
#include "float_ops.cuh"

namespace chxq {
namespace {

constexpr int kThreads = 256;

// Sum over the block, the same for every thread; red: one float per warp.
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.f;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) s += red[i];
    return s;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) layernorm_kernel(const T* __restrict__ x, int64_t ldx, FloatArray scale, FloatArray bias, int64_t rows, int64_t D,
                                                             float eps, T* __restrict__ y, float* __restrict__ mean, float* __restrict__ inv) {
    __shared__ float red[kThreads / 32];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * ldx;
        float s = 0.f;
        for (int64_t i = threadIdx.x; i < D; i += kThreads) s += to_f32(xr[i]);
        const float m = block_sum(s, red) / (float)D;
        s = 0.f;
        for (int64_t i = threadIdx.x; i < D; i += kThreads) {
            const float d = to_f32(xr[i]) - m;
            s = fmaf(d, d, s);
        }
        const float is = 1.f / sqrtf(block_sum(s, red) / (float)D + eps);
        for (int64_t i = threadIdx.x; i < D; i += kThreads) {
            const float h = (to_f32(xr[i]) - m) * is;
            y[r * D + i] = from_f32<T>(fmaf(h, load_param(scale, i), bias.p ? load_param(bias, i) : 0.f));
        }
        if (threadIdx.x == 0) {
            if (mean) mean[r] = m;
            if (inv) inv[r] = is;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) layernorm_dx_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, FloatArray scale,
                                                                const float* __restrict__ mean, const float* __restrict__ inv, int64_t rows, int64_t D,
                                                                T* __restrict__ dx) {
    __shared__ float red[kThreads / 32];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float m = mean[r], is = inv[r];
        float a = 0.f, b = 0.f;
        for (int64_t i = threadIdx.x; i < D; i += kThreads) {
            const float g = to_f32(dy[r * lddy + i]) * load_param(scale, i);
            a += g;
            b = fmaf(g, (to_f32(x[r * ldx + i]) - m) * is, b);
        }
        a = block_sum(a, red) / (float)D;
        b = block_sum(b, red) / (float)D;
        for (int64_t i = threadIdx.x; i < D; i += kThreads) {
            const float g = to_f32(dy[r * lddy + i]) * load_param(scale, i);
            dx[r * D + i] = from_f32<T>((g - a - (to_f32(x[r * ldx + i]) - m) * is * b) * is);
        }
    }
}

// part [shares][2][D]: the sums of a share of the rows.
template <typename T>
__global__ void __launch_bounds__(kThreads) layernorm_dparam_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                                                    const float* __restrict__ mean, const float* __restrict__ inv, int64_t rows, int64_t D,
                                                                    float* __restrict__ part) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= D) return;
    float a = 0.f, b = 0.f;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const float d = to_f32(dy[r * lddy + i]);
        a = fmaf(d, (to_f32(x[r * ldx + i]) - mean[r]) * inv[r], a);
        b += d;
    }
    part[(2 * (int64_t)blockIdx.y) * D + i] = a;
    part[(2 * (int64_t)blockIdx.y + 1) * D + i] = b;
}

__global__ void __launch_bounds__(kThreads) layernorm_dparam_join_kernel(const float* __restrict__ part, int shares, int64_t D, int dtype, void* dscale, void* dbias) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= D) return;
    float a = 0.f, b = 0.f;
    for (int s = 0; s < shares; ++s) {
        a += part[(2 * (int64_t)s) * D + i];
        b += part[(2 * (int64_t)s + 1) * D + i];
    }
    store_param(dscale, dtype, i, a);
    if (dbias) store_param(dbias, dtype, i, b);
}

int shares_of(int64_t rows) {
    return (int)(rows < 148 ? (rows < 1 ? 1 : rows) : 148);
}

}  // namespace
}  // namespace chxq

using namespace chxq;

static int check_norm(const char* op, int dtype, int affine_dtype, int64_t rows, int64_t D) {
    CHXQ_CHECK_ARG(is_float_type(dtype), "%s: x must be float32, float16 or bfloat16", op);
    CHXQ_CHECK_ARG(affine_dtype == dtype || affine_dtype == CHXQ_FLOAT32, "%s: scale and bias must be float32 or have x's type", op);
    CHXQ_CHECK_ARG(rows >= 0 && D >= 1 && D < (1ll << 31), "%s: bad extents", op);
    return CHXQ_OK;
}

extern "C" int chxq_layernorm(const void* x, int64_t ldx, int32_t dtype, const void* scale, const void* bias, int32_t affine_dtype, int64_t rows, int64_t D,
                              float epsilon, void* y, float* mean, float* inv_std_dev, void* stream) {
    const int rc = check_norm("LayerNormalization", dtype, affine_dtype, rows, D);
    if (rc != CHXQ_OK) return rc;
    if (rows == 0) return CHXQ_OK;
    CHXQ_CHECK_ARG(x && scale && y && (rows == 1 || ldx >= D), "LayerNormalization: bad arguments");
    const unsigned grid = (unsigned)(rows < 148 * 8 ? rows : 148 * 8);
    return with_float_type(dtype, [&](auto t) {
        using T = decltype(t);
        layernorm_kernel<T><<<grid, kThreads, 0, as_stream(stream)>>>(static_cast<const T*>(x), ldx, FloatArray{scale, affine_dtype}, FloatArray{bias, affine_dtype},
                                                                      rows, D, epsilon, static_cast<T*>(y), mean, inv_std_dev);
        CHXQ_LAUNCH_CHECK();
        return CHXQ_OK;
    });
}

extern "C" size_t chxq_layernorm_grad_workspace(int64_t rows, int64_t D) {
    return rows < 0 || D < 1 ? 0 : (size_t)shares_of(rows) * 2 * (size_t)D * sizeof(float);
}

extern "C" int chxq_layernorm_grad(const void* dy, int64_t lddy, const void* x, int64_t ldx, int32_t dtype, const void* scale, int32_t affine_dtype,
                                   const float* mean, const float* inv_std_dev, int64_t rows, int64_t D, void* dx, void* dscale, void* dbias, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    const int rc = check_norm("LayerNormalizationGrad", dtype, affine_dtype, rows, D);
    if (rc != CHXQ_OK) return rc;
    CHXQ_CHECK_ARG(dscale && scale && (rows == 0 || (dy && x && mean && inv_std_dev && dx)) && (rows <= 1 || (ldx >= D && lddy >= D)), "LayerNormalizationGrad: bad arguments");
    const size_t need = chxq_layernorm_grad_workspace(rows, D);
    if (!workspace || workspace_bytes < need) return set_error(CHXQ_ERR_WORKSPACE, "LayerNormalizationGrad: needs %zu bytes of workspace", need);
    const int shares = shares_of(rows);
    const unsigned cols = (unsigned)((D + kThreads - 1) / kThreads);
    float* part = static_cast<float*>(workspace);
    cudaStream_t s = as_stream(stream);
    return with_float_type(dtype, [&](auto t) {
        using T = decltype(t);
        const T *g = static_cast<const T*>(dy), *v = static_cast<const T*>(x);
        if (rows > 0) {
            layernorm_dx_kernel<T><<<(unsigned)(rows < 148 * 8 ? rows : 148 * 8), kThreads, 0, s>>>(g, lddy, v, ldx, FloatArray{scale, affine_dtype}, mean, inv_std_dev,
                                                                                                    rows, D, static_cast<T*>(dx));
            CHXQ_LAUNCH_CHECK();
        }
        layernorm_dparam_kernel<T><<<dim3(cols, shares), kThreads, 0, s>>>(g, lddy, v, ldx, mean, inv_std_dev, rows, D, part);
        CHXQ_LAUNCH_CHECK();
        layernorm_dparam_join_kernel<<<cols, kThreads, 0, s>>>(part, shares, D, affine_dtype, dscale, dbias);
        CHXQ_LAUNCH_CHECK();
        return CHXQ_OK;
    });
}
