// LayerNormalization over the last `D` values of each row, and its gradient.
//   m = mean(x), s = 1 / sqrt(mean((x - m)^2) + epsilon), xh = (x - m) s, y = xh scale + bias
//   dx = s (scale dy - mean(scale dy) - xh mean(scale dy xh)),  dscale = sum over rows of dy xh,  dbias = sum over rows of dy
// Sums and statistics are held in 32 bits; the variance is that of the deviations, which does not cancel.
//
// Both directions are bound by HBM: x (and dy) are read once, y (dx) is written once.  So a row stays in registers between its passes.  Accesses
// are 16 bytes wide where rows allow it, else 4, else one value (VEC values each).
#include <algorithm>

#include "float_ops.cuh"
#include "pdl.cuh"

namespace chxq {
namespace {

__device__ __forceinline__ void group_barrier(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// ---- forward --------------------------------------------------------------------------------------------------------------

// A row per block (BLOCK) or per warp; a thread holds NV accesses of it, `stride` = threads per row apart.
template <typename T, int VEC, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) layernorm_kernel(const T* __restrict__ x, int64_t ldx, FloatArray scale, FloatArray bias, int64_t rows, int D,
                                                                       float eps, T* __restrict__ y, float* __restrict__ mean, float* __restrict__ inv) {
    __shared__ float red[2][32];
    pdl_launch_dependents();
    pdl_dependency_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t r = BLOCK ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 8 + warp;
    if (r >= rows) return;  // whole warps, and none of a BLOCK
    const int tid = BLOCK ? (int)threadIdx.x : lane, stride = BLOCK ? (int)blockDim.x : 32;
    auto sum = [&](float v, int which) {
        v = warp_sum(v);
        if constexpr (BLOCK) {
            if (lane == 0) red[which][warp] = v;
            __syncthreads();
            v = warp_sum(lane < (int)(blockDim.x >> 5) ? red[which][lane] : 0.f);
        }
        return v;
    };
    const T* xr = x + r * ldx;
    Pack<T, VEC> v[NV];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (tid + i * stride) * VEC;
        if (c < D) v[i].load(xr + c);
        else v[i].zero();
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += v[i].get(j);
    const float m = sum(s, 0) / (float)D;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if ((tid + i * stride) * VEC < D)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = v[i].get(j) - m;
                s = fmaf(d, d, s);
            }
    const float is = 1.f / sqrtf(sum(s, 1) / (float)D + eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (tid + i * stride) * VEC;
        if (c >= D) continue;
        float g[VEC], b[VEC] = {};
        load_params<VEC>(scale, c, g);
        if (bias.p) load_params<VEC>(bias, c, b);
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[j] = fmaf((v[i].get(j) - m) * is, g[j], b[j]);
        v[i].set(g);
        v[i].store(y + r * D + c);
    }
    if (tid == 0) {
        if (mean) mean[r] = m;
        if (inv) inv[r] = is;
    }
}

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

// Rows that registers do not hold: the passes read them again.
template <typename T>
__global__ void __launch_bounds__(kThreads) layernorm_long_kernel(const T* __restrict__ x, int64_t ldx, FloatArray scale, FloatArray bias, int64_t rows, int64_t D,
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

// ---- gradient -------------------------------------------------------------------------------------------------------------

// p[0 .. N) = (fresh ? 0 : p) + v, in shared memory; p on a 16-byte boundary where N is a multiple of four.
template <int N>
__device__ __forceinline__ void add_to(float* p, const float (&v)[N], bool fresh) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            float4 q = fresh ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<float4*>(p + j);
            q.x += v[j]; q.y += v[j + 1]; q.z += v[j + 2]; q.w += v[j + 3];
            *reinterpret_cast<float4*>(p + j) = q;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) p[j] = (fresh ? 0.f : p[j]) + v[j];
    }
}

// Persistent blocks of `groups` groups of G threads; a group takes every (groups * blocks)-th row, and a thread the same columns of each: NV
// accesses, G apart.  The next row is fetched before the sums of the current one meet.  The columns' sums over the rows stay in registers, or in shared
// memory (SMEM, one group; rows too long for the registers of 512 threads), and leave as one partial sum [2][D] per block.
template <typename T, int VEC, int NV, bool SMEM>
__global__ void __launch_bounds__(SMEM ? 1024 : 512) layernorm_grad_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, FloatArray scale,
                                                                           const float* __restrict__ mean, const float* __restrict__ inv, int64_t rows, int D, int G,
                                                                           int groups, T* __restrict__ dx, float* __restrict__ part) {
    extern __shared__ __align__(16) float sums[];  // [2][D] columns' sums: of the block at the end, or all along (SMEM)
    __shared__ float red[2][32][2];  // by the parity of the row
    pdl_launch_dependents();
    pdl_dependency_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = (int)threadIdx.x / G, t = (int)threadIdx.x - group * G;  // warps belong to one group: G is a multiple of 32
    const int warps = G >> 5, warp0 = group * warps;
    float ag[SMEM ? 1 : NV][VEC] = {}, ab[SMEM ? 1 : NV][VEC] = {};
    if (SMEM)
        for (int i = threadIdx.x; i < 2 * D; i += blockDim.x) sums[i] = 0.f;  // (read by the same thread or behind the first row's barrier)
    if (SMEM) __syncthreads();
    float g[SMEM ? 1 : NV][VEC] = {};  // (SMEM: read again for each row, from the L1)
    if constexpr (!SMEM)
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if ((t + i * G) * VEC < D) load_params<VEC>(scale, (t + i * G) * VEC, g[i]);
    Pack<T, VEC> vx[NV], vd[NV], nx[SMEM ? 1 : NV], nd[SMEM ? 1 : NV];
    float m = 0.f, is = 0.f, nm = 0.f, ns = 0.f;
    auto fetch = [&](int64_t r, Pack<T, VEC>* px, Pack<T, VEC>* pd, float& pm, float& ps) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * G) * VEC;
            if (r < rows && c < D) {
                px[i].load(x + r * ldx + c);
                pd[i].load(dy + r * lddy + c);
            } else {
                px[i].zero();
                pd[i].zero();
            }
        }
        if (r < rows) {
            pm = mean[r];
            ps = inv[r];
        }
    };
    const int64_t step = (int64_t)gridDim.x * groups;
    int64_t r = (int64_t)blockIdx.x * groups + group;
    if (group < groups) fetch(r, vx, vd, m, is);
    const float rd = 1.f / (float)D;
    for (int par = 0; group < groups && r < rows; r += step, par ^= 1) {
        if constexpr (!SMEM) fetch(r + step, nx, nd, nm, ns);
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * G) * VEC;
            float q[2][VEC], gs[VEC] = {};
            if (SMEM && c < D) load_params<VEC>(scale, c, gs);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = vd[i].get(j), xh = (vx[i].get(j) - m) * is, gd = d * (SMEM ? gs[j] : g[SMEM ? 0 : i][j]);
                a += gd;
                b = fmaf(gd, xh, b);
                if constexpr (SMEM) {
                    q[0][j] = d * xh;
                    q[1][j] = d;
                } else {
                    ag[i][j] = fmaf(d, xh, ag[i][j]);
                    ab[i][j] += d;
                }
            }
            if (SMEM && c < D) {
                add_to<VEC>(sums + c, q[0], false);
                add_to<VEC>(sums + D + c, q[1], false);
            }
        }
        a = warp_sum(a);
        b = warp_sum(b);
        if (warps > 1) {
            if (lane == 0) {
                red[par][warp][0] = a;
                red[par][warp][1] = b;
            }
            group_barrier(1 + group, G);
            a = warp_sum(lane < warps ? red[par][warp0 + lane][0] : 0.f);
            b = warp_sum(lane < warps ? red[par][warp0 + lane][1] : 0.f);
        }
        a *= rd;
        b *= rd;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * G) * VEC;
            if (c >= D) continue;
            float q[VEC], gs[VEC];
            if constexpr (SMEM) load_params<VEC>(scale, c, gs);
#pragma unroll
            for (int j = 0; j < VEC; ++j) q[j] = (vd[i].get(j) * (SMEM ? gs[j] : g[SMEM ? 0 : i][j]) - a - (vx[i].get(j) - m) * is * b) * is;
            Pack<T, VEC> o;
            o.set(q);
            o.store(dx + r * D + c);
        }
        if constexpr (SMEM) {
            fetch(r + step, vx, vd, m, is);
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                vx[i] = nx[i];
                vd[i] = nd[i];
            }
            m = nm;
            is = ns;
        }
    }
    // the groups' sums in ascending order
    float* mine = part + 2 * (int64_t)blockIdx.x * D;
    if constexpr (!SMEM) {
        for (int k = 0; k < groups; ++k) {
            if (group == k)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c = (t + i * G) * VEC;
                    if (c < D) {
                        add_to<VEC>(sums + c, ag[i], k == 0);
                        add_to<VEC>(sums + D + c, ab[i], k == 0);
                    }
                }
            __syncthreads();
        }
    } else {
        __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * D; i += blockDim.x) mine[i] = sums[i];
}

// Rows that neither holds: dx with the row read twice, and the parameters' sums in a pass of their own.
template <typename T>
__global__ void __launch_bounds__(kThreads) layernorm_dx_long_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, FloatArray scale,
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

template <typename T>
__global__ void __launch_bounds__(kThreads) layernorm_dparam_long_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
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

// part [shares][2 D] -> the sum of the shares: 32 columns a block, eight threads per column that take every eighth share.
__global__ void __launch_bounds__(kThreads) layernorm_join_kernel(const float* __restrict__ part, int shares, int64_t D, int dtype, void* dscale, void* dbias) {
    __shared__ float acc[8][33];
    pdl_launch_dependents();
    pdl_dependency_wait();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t i = (int64_t)blockIdx.x * 32 + lane;
    float a = 0.f;
    if (i < 2 * D)
        for (int s = w; s < shares; s += 8) a += part[(int64_t)s * 2 * D + i];
    acc[w][lane] = a;
    __syncthreads();
    if (w == 0 && i < 2 * D) {
#pragma unroll
        for (int k = 1; k < 8; ++k) a += acc[k][lane];
        if (i < D) store_param(dscale, dtype, i, a);
        else if (dbias) store_param(dbias, dtype, i - D, a);
    }
}

// How a gradient runs.
struct GradPlan {
    int kind;  // 0: columns' sums in registers, 1: in shared memory, 2: long rows
    int G, groups, blocks;
};

// Values of a row that a thread holds with the columns' sums in registers: 16 in two 16-byte accesses of a 16-bit type -- with the next row's,
// the scale and two sums each they fill the 128 registers that 512 threads have -- and 8 in 32 bits or narrow accesses.
__host__ __device__ constexpr int grad_values(int vec) {
    return vec == 8 ? 16 : 8;
}

GradPlan plan_grad(int64_t rows, int64_t D, int vec) {
    GradPlan p = {2, 0, 1, 0};
    const int e = grad_values(vec);
    if (D <= 512 * e) {
        p.kind = 0;
        p.G = (int)(((D + e - 1) / e + 31) / 32 * 32);
        p.groups = 512 / p.G;
    } else if (D <= 1024 * 16) {
        p.kind = 1;
        p.G = (int)(((D + 15) / 16 + 31) / 32 * 32);
    }
    p.blocks = (int)std::min<int64_t>(std::max<int64_t>((rows + p.groups - 1) / p.groups, 1), 148);
    return p;
}

template <typename T, int VEC>
int launch_grad(const GradPlan& p, const T* dy, int64_t lddy, const T* x, int64_t ldx, FloatArray scale, const float* mean, const float* inv, int64_t rows, int D, T* dx,
                float* part, cudaStream_t s) {
    const size_t smem = (size_t)2 * D * sizeof(float);
    auto go = [&](auto* kernel) {
        if (smem > 48 * 1024) CHXQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        CHXQ_CUDA(launch_pdl(kernel, dim3((unsigned)p.blocks), p.G * p.groups, smem, s, dy, lddy, x, ldx, scale, mean, inv, rows, D, p.G, p.groups, dx, part));
        count_launch(1);
        return CHXQ_OK;
    };
    return p.kind == 0 ? go(layernorm_grad_kernel<T, VEC, grad_values(VEC) / VEC, false>) : go(layernorm_grad_kernel<T, VEC, 16 / VEC, true>);
}

// Values per access: as many as fill 16 bytes, or 4, or one, by what divides the rows and aligns the addresses (of x-like arrays, `bits`; pitches
// in values).  The parameters are read as many at a time.
template <typename T>
int access_width(uintptr_t bits, int64_t D, int64_t pitches, const void* scale, const void* bias) {
    const uintptr_t params = reinterpret_cast<uintptr_t>(scale) | reinterpret_cast<uintptr_t>(bias);
    constexpr int wide = 16 / (int)sizeof(T);
    if (D % wide == 0 && pitches % wide == 0 && (bits & 15u) == 0 && (params & 15u) == 0) return wide;
    if (sizeof(T) == 2 && D % 2 == 0 && pitches % 2 == 0 && (bits & 3u) == 0) return 2;
    return 1;
}

template <typename T, typename F>
int with_width(int width, F&& f) {
    if (width == 16 / (int)sizeof(T)) return f(std::integral_constant<int, 16 / (int)sizeof(T)>{});
    if constexpr (sizeof(T) == 2)
        if (width == 2) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 1>{});
}

}  // namespace
}  // namespace chxq

using namespace chxq;

static int check_norm(const char* op, int dtype, int affine_dtype, int64_t rows, int64_t D) {
    CHXQ_CHECK_ARG(is_float_type(dtype), "%s: x must be float32, float16 or bfloat16", op);
    CHXQ_CHECK_ARG(affine_dtype == dtype || affine_dtype == CHXQ_FLOAT32, "%s: scale and bias must be float32 or have x's type", op);
    CHXQ_CHECK_ARG(rows >= 0 && rows < (1ll << 31) && D >= 1 && D < (1ll << 31), "%s: bad extents", op);
    return CHXQ_OK;
}

extern "C" int chxq_layernorm(const void* x, int64_t ldx, int32_t dtype, const void* scale, const void* bias, int32_t affine_dtype, int64_t rows, int64_t D,
                              float epsilon, void* y, float* mean, float* inv_std_dev, void* stream) {
    const int rc = check_norm("LayerNormalization", dtype, affine_dtype, rows, D);
    if (rc != CHXQ_OK) return rc;
    if (rows == 0) return CHXQ_OK;
    CHXQ_CHECK_ARG(x && scale && y && (rows == 1 || ldx >= D), "LayerNormalization: bad arguments");
    cudaStream_t s = as_stream(stream);
    const FloatArray g = {scale, affine_dtype}, b = {bias, affine_dtype};
    return with_float_type(dtype, [&](auto t) {
        using T = decltype(t);
        const uintptr_t bits = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y);
        return with_width<T>(access_width<T>(bits, D, rows == 1 ? 0 : ldx, scale, bias), [&](auto width) {
            constexpr int VEC = decltype(width)::value;
            const int64_t accesses = (D + VEC - 1) / VEC;
            auto go = [&](auto* kernel, int64_t grid, int threads) {
                CHXQ_CUDA(launch_pdl(kernel, dim3((unsigned)grid), threads, 0, s, static_cast<const T*>(x), ldx, g, b, rows, (int)D, epsilon, static_cast<T*>(y), mean,
                                     inv_std_dev));
                count_launch(1);
                return CHXQ_OK;
            };
            auto threads = [&](int nv) { return (int)(((accesses + nv - 1) / nv + 31) / 32 * 32); };
            if (accesses <= 32) return go(layernorm_kernel<T, VEC, 1, false>, (rows + 7) / 8, 256);
            if (accesses <= 64) return go(layernorm_kernel<T, VEC, 2, false>, (rows + 7) / 8, 256);
            if (accesses <= 128) return go(layernorm_kernel<T, VEC, 4, false>, (rows + 7) / 8, 256);
            if (accesses <= 4 * 1024) return go(layernorm_kernel<T, VEC, 4, true>, rows, threads(4));
            if (accesses <= 16 * 1024 && VEC < 4) return go(layernorm_kernel<T, VEC, VEC < 4 ? 16 : 4, true>, rows, threads(16));
            layernorm_long_kernel<T><<<(unsigned)std::min<int64_t>(rows, 148 * 8), kThreads, 0, s>>>(static_cast<const T*>(x), ldx, g, b, rows, D, epsilon,
                                                                                                     static_cast<T*>(y), mean, inv_std_dev);
            CHXQ_LAUNCH_CHECK();
            return CHXQ_OK;
        });
    });
}

extern "C" size_t chxq_layernorm_grad_workspace(int64_t rows, int64_t D) {
    if (rows < 0 || D < 1) return 0;
    return (size_t)148 * 2 * (size_t)D * sizeof(float);
}

extern "C" int chxq_layernorm_grad(const void* dy, int64_t lddy, const void* x, int64_t ldx, int32_t dtype, const void* scale, int32_t affine_dtype,
                                   const float* mean, const float* inv_std_dev, int64_t rows, int64_t D, void* dx, void* dscale, void* dbias, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    const int rc = check_norm("LayerNormalizationGrad", dtype, affine_dtype, rows, D);
    if (rc != CHXQ_OK) return rc;
    CHXQ_CHECK_ARG(dscale && scale && (rows == 0 || (dy && x && mean && inv_std_dev && dx)) && (rows <= 1 || (ldx >= D && lddy >= D)), "LayerNormalizationGrad: bad arguments");
    const size_t need = chxq_layernorm_grad_workspace(rows, D);
    if (!workspace || workspace_bytes < need) return set_error(CHXQ_ERR_WORKSPACE, "LayerNormalizationGrad: needs %zu bytes of workspace", need);
    float* part = static_cast<float*>(workspace);
    const FloatArray sc = {scale, affine_dtype};
    cudaStream_t s = as_stream(stream);
    int shares = 0;
    const int rc2 = with_float_type(dtype, [&](auto t) {
        using T = decltype(t);
        const T *g = static_cast<const T*>(dy), *v = static_cast<const T*>(x);
        const uintptr_t bits = reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(dx);
        const int64_t pitches = rows <= 1 ? 0 : ldx | lddy;  // as divisible by a power of two as both are
        return with_width<T>(access_width<T>(bits, D, pitches, scale, nullptr), [&](auto width) {
            constexpr int VEC = decltype(width)::value;
            const GradPlan p = plan_grad(rows, D, VEC);
            shares = p.blocks;
            if (p.kind < 2) return launch_grad<T, VEC>(p, g, lddy, v, ldx, sc, mean, inv_std_dev, rows, (int)D, static_cast<T*>(dx), part, s);
            if (rows > 0) {
                layernorm_dx_long_kernel<T><<<(unsigned)std::min<int64_t>(rows, 148 * 8), kThreads, 0, s>>>(g, lddy, v, ldx, sc, mean, inv_std_dev, rows, D, static_cast<T*>(dx));
                CHXQ_LAUNCH_CHECK();
            }
            layernorm_dparam_long_kernel<T><<<dim3((unsigned)((D + kThreads - 1) / kThreads), p.blocks), kThreads, 0, s>>>(g, lddy, v, ldx, mean, inv_std_dev, rows, D, part);
            CHXQ_LAUNCH_CHECK();
            return CHXQ_OK;
        });
    });
    if (rc2 != CHXQ_OK) return rc2;
    CHXQ_CUDA(launch_pdl(layernorm_join_kernel, dim3((unsigned)((2 * D + 31) / 32)), kThreads, 0, s, static_cast<const float*>(part), shares, D, (int)affine_dtype, dscale,
                         dbias));
    count_launch(1);
    return CHXQ_OK;
}
