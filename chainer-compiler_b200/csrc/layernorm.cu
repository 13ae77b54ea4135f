// LayerNormalization over the last `D` values of each row, and its gradient.
//   m = mean(x), s = 1 / sqrt(mean((x - m)^2) + epsilon), xh = (x - m) s, y = xh scale + bias
//   dx = s (scale dy - mean(scale dy) - xh mean(scale dy xh)),  dscale = sum over rows of dy xh,  dbias = sum over rows of dy
// Sums and statistics are held in 32 bits; the variance is that of the deviations, which does not cancel.
//
// Both directions are bound by HBM as far as their instructions allow: x (and dy) are read once, y (dx) is written once, and 16-bit rows leave
// about twenty issue slots per pair of values.  So blocks are persistent, arithmetic goes two values an instruction, a row stays in registers
// between its passes and the next one is fetched into registers meanwhile.
//
// A group of G threads takes a row, and a thread the same columns of every row it sees, so that parameters and columns' sums stay with it.  Rows that
// are no whole number of 16-byte pieces (SHIFT) start at another place of a piece each, but those of a group all at the same: the distance
// between them is a multiple of 16 / sizeof(T) rows.  Pieces that two rows share are read whole and the values of the other row masked.
#include <algorithm>
#include <atomic>

#include "float_ops.cuh"
#include "pdl.cuh"

namespace chxq {
namespace {

__device__ __forceinline__ void group_barrier(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// What a thread is within the block, and the columns it has of the rows of its group.
// FULL: every thread has NV whole pieces.
template <typename T, int NV, bool SHIFT, bool FULL = false>
struct Place {
    static constexpr int VEC = 16 / (int)sizeof(T);
    int G, group, t;  // threads per group (a power of two up to 32, or a multiple of 32), this thread's group and place in it
    int shift;        // columns of the row before in the group's first piece
    int D;

    __device__ __forceinline__ Place(int G_, int D_, int64_t row0, int64_t ld) : G(G_), group((int)threadIdx.x / G_), t((int)threadIdx.x % G_), D(D_) {
        shift = SHIFT ? (int)((row0 * ld) & (VEC - 1)) : 0;
    }
    __device__ __forceinline__ int column(int i) const { return (t + i * G) * VEC - shift; }  // the first of piece i; negative ones belong to the row before
    __device__ __forceinline__ bool any(int i) const { return FULL || column(i) < D; }
    __device__ __forceinline__ bool full(int i) const { return !SHIFT || (column(i) >= 0 && column(i) + VEC <= D); }
    __device__ __forceinline__ bool has(int i, int j) const { return (unsigned)(column(i) + j) < (unsigned)D; }

    // Piece i of the row at `row`; zero where the thread has none.  Rows of whole pieces: the first one is read instead, so that no branch parts the
    // loads ([4096, 12000] fp32: 104 -> 70 us).  SHIFT: the last row's last piece may reach past the buffer and is read value by value.
    __device__ __forceinline__ void load(const T* row, int i, bool last_row, Pack<T, VEC>& v) const {
        if constexpr (!SHIFT) {
            v.load(row + (any(i) ? column(i) : 0));
            if (!any(i)) v.zero();
        } else {
            const bool tail = last_row && column(i) + VEC > D;
            v.zero();
            if (any(i) && !tail) v.load(row + column(i));
            if (tail)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (has(i, j)) v.put(j, row[column(i) + j]);
        }
    }
    // Zeroes the values of piece i that are not the row's.
    __device__ __forceinline__ void mask(int i, f32x2 (&v)[VEC / 2]) const {
        if (full(i)) return;
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
            const float2 f = split_x2(v[j]);
            v[j] = make_x2(has(i, 2 * j) ? f.x : 0.f, has(i, 2 * j + 1) ? f.y : 0.f);
        }
    }
    __device__ __forceinline__ f32x2 param(const FloatArray& a, int i, int j) const {  // columns 2 j, 2 j + 1 of piece i
        return make_x2(a.p && has(i, 2 * j) ? load_param(a, column(i) + 2 * j) : 0.f, a.p && has(i, 2 * j + 1) ? load_param(a, column(i) + 2 * j + 1) : 0.f);
    }
    __device__ __forceinline__ void store(T* row, int i, const Pack<T, VEC>& o) const {
        if (full(i)) {
            o.store(row + column(i));
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (has(i, j)) row[column(i) + j] = o.value(j);
        }
    }
};

// Sum over a group of G threads, the same for all of them; at most sixteen warps.  red: [2][warps of the block] per value, used by turns (par), so
// that one barrier is enough.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], int G, int group, float (*red)[32][N], int par) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float q = __shfl_xor_sync(0xffffffffu, v[k], o);
            if (o < G) v[k] += q;
        }
    if (G <= 32) return;
    const int lane = threadIdx.x & 31, warps = G >> 5;
    if (lane == 0)
#pragma unroll
        for (int k = 0; k < N; ++k) red[par][threadIdx.x >> 5][k] = v[k];
    group_barrier(1 + group, G);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = lane < warps ? red[par][group * warps + lane][k] : 0.f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = __shfl_sync(0xffffffffu, v[k], 0);
}

// ---- forward --------------------------------------------------------------------------------------------------------------

// A row per block (BLOCK) or per group of G <= 32 threads, eight warps a block; blocks come and go, so that some load while others compute and store.
// (Persistent blocks that kept their parameters in registers or shared memory and fetched the next row meanwhile were slower: 74-78 us where this
// form takes 50 for [16384, 4096] bf16.  What a row costs beside its values does not shrink, and fewer warps fit.)
template <typename T, int NV, bool BLOCK, bool SHIFT, bool FULL>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) layernorm_kernel(const T* __restrict__ x, int64_t ldx, FloatArray scale, FloatArray bias, int64_t rows, int D,
                                                                       float eps, int G, T* __restrict__ y, float* __restrict__ mean, float* __restrict__ inv) {
    constexpr int VEC = 16 / (int)sizeof(T);
    __shared__ float red[2][32];
    pdl_launch_dependents();
    pdl_dependency_wait();
    const int lane = threadIdx.x & 31, warps = (int)blockDim.x >> 5;
    const int64_t r = BLOCK ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (256 / G) + (int)threadIdx.x / G;
    const bool live = BLOCK || r < rows;  // (all lanes of a warp take part in its shuffles)
    auto sum = [&](float v, int which) {
        if constexpr (BLOCK) {
            v = warp_sum(v);
            if (lane == 0) red[which][threadIdx.x >> 5] = v;
            __syncthreads();
            v = warp_sum(lane < warps ? red[which][lane] : 0.f);
        } else {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float q = __shfl_xor_sync(0xffffffffu, v, o);
                if (o < G) v += q;
            }
        }
        return v;
    };
    const Place<T, NV, SHIFT, FULL> at(BLOCK ? (int)blockDim.x : G, D, r, ldx);
    const T* xr = x + r * ldx;
    f32x2 v[NV][VEC / 2];
    {
        Pack<T, VEC> q[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (live) at.load(xr, i, r == rows - 1, q[i]);
            else q[i].zero();
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) v[i][j] = q[i].pair(j);
    }
    f32x2 a = 0ull;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if constexpr (SHIFT) at.mask(i, v[i]);
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) a = add2(a, v[i][j]);
    }
    const float rd = 1.f / (float)D;
    float2 f = split_x2(a);
    const float m = sum(f.x + f.y, 0) * rd;
    a = 0ull;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const float nm = at.any(i) ? -m : 0.f;  // pieces that are not there stay zero
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) v[i][j] = add2(v[i][j], make_x2(nm, nm));
        if constexpr (SHIFT) at.mask(i, v[i]);
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) a = fma2(v[i][j], v[i][j], a);
    }
    f = split_x2(a);
    const float var = sum(f.x + f.y, 1) * rd + eps;
    float is = rsqrtf(var);
    is = is * fmaf(-0.5f * var * is, is, 1.5f);  // one Newton step on the approximation, which is good to 2^-22
    if (var == 0.f) is = INFINITY;               // (epsilon 0 and a constant row)
    const f32x2 is2 = make_x2(is, is);
    if (!live) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (!at.any(i)) continue;
        Pack<T, VEC> o;
        float g[VEC], b[VEC] = {};
        if constexpr (!SHIFT) {
            load_params<VEC>(scale, at.column(i), g);
            if (bias.p) load_params<VEC>(bias, at.column(i), b);
        } else if (at.full(i)) {
            load_params_any<T, VEC>(scale, at.column(i), g);
            if (bias.p) load_params_any<T, VEC>(bias, at.column(i), b);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (at.has(i, j)) {
                    const float2 d = split_x2(v[i][j / 2]);
                    y[r * D + at.column(i) + j] = from_f32<T>(fmaf((j & 1 ? d.y : d.x) * is, load_param(scale, at.column(i) + j), bias.p ? load_param(bias, at.column(i) + j) : 0.f));
                }
            continue;
        }
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) o.set_pair(j, fma2(mul2(v[i][j], is2), make_x2(g[2 * j], g[2 * j + 1]), make_x2(b[2 * j], b[2 * j + 1])));
        o.store(y + r * D + at.column(i));
    }
    if (at.t == 0) {
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

// Floats of the columns' sums of a block: [2][D], and of each of its warps where a warp holds several groups; in whole 16-byte pieces.
__host__ __device__ constexpr int grad_sum_floats(int D, int G, int threads) {
    return (2 * D * (G < 32 ? threads / 32 : 1) + 3) / 4 * 4;
}

// As the forward pass, with two rows of operands.  The columns' sums over the rows stay in registers, or in shared memory (SMEM, one group: rows too
// long for the registers of 512 threads), and leave as one partial sum [2][D] per block.
template <typename T, int NV, bool SHIFT, bool SMEM>
__global__ void __launch_bounds__(512) layernorm_grad_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, FloatArray scale,
                                                             const float* __restrict__ mean, const float* __restrict__ inv, int64_t rows, int D, int G,
                                                             T* __restrict__ dx, float* __restrict__ part) {
    constexpr int VEC = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) float sums[];
    __shared__ float red[2][32][2];
    pdl_launch_dependents();
    pdl_dependency_wait();
    const int groups = (int)blockDim.x / G, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t step = (int64_t)gridDim.x * groups;
    int64_t r = (int64_t)blockIdx.x * groups + (int)threadIdx.x / G;
    const Place<T, NV, SHIFT> at(G, D, r, ldx);
    const T *px = x + r * ldx, *pd = dy + r * lddy;
    T* po = dx + r * D;
    const int64_t sx = step * ldx, sd = step * lddy, so = step * D;
    Pack<T, VEC> vx[NV], vd[NV], nx[NV], nd[NV];
    float m = 0.f, is = 0.f, nm = 0.f, ns = 0.f;
    if (r < rows) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            at.load(px, i, r == rows - 1, nx[i]);
            at.load(pd, i, r == rows - 1, nd[i]);
        }
        nm = mean[r];
        ns = inv[r];
    }
    f32x2 g[NV][VEC / 2];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) g[i][j] = at.param(scale, i, j);
    f32x2 ag[SMEM ? 1 : NV][VEC / 2] = {}, ab[SMEM ? 1 : NV][VEC / 2] = {};
    for (int i = threadIdx.x; i < grad_sum_floats(D, G, (int)blockDim.x); i += blockDim.x) sums[i] = 0.f;
    __syncthreads();
    const float rd = 1.f / (float)D;
    int64_t lead = G < 32 ? (int64_t)blockIdx.x * groups + ((int)threadIdx.x & ~31) / G : r;  // as in the forward pass
    for (int par = 0; lead < rows; lead += step, r += step, par ^= 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            vx[i] = nx[i];
            vd[i] = nd[i];
        }
        m = nm;
        is = ns;
        px += sx;
        pd += sd;
        if (r + step < rows) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                at.load(px, i, r + step == rows - 1, nx[i]);
                at.load(pd, i, r + step == rows - 1, nd[i]);
            }
            nm = mean[r + step];
            ns = inv[r + step];
        }
        const f32x2 is2 = make_x2(is, is), nm2 = make_x2(-m, -m);
        f32x2 a = 0ull, b = 0ull;
        if (r < rows) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (!at.any(i)) continue;
                f32x2 d[VEC / 2], h[VEC / 2];
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) {
                    d[j] = vd[i].pair(j);
                    h[j] = mul2(add2(vx[i].pair(j), nm2), is2);
                }
                if constexpr (SHIFT) {
                    at.mask(i, d);
                    at.mask(i, h);
                }
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) {
                    const f32x2 gd = mul2(d[j], g[i][j]);
                    a = add2(a, gd);
                    b = fma2(gd, h[j], b);
                    if constexpr (!SMEM) {
                        ag[i][j] = fma2(d[j], h[j], ag[i][j]);
                        ab[i][j] = add2(ab[i][j], d[j]);
                    }
                }
                if constexpr (SMEM) {
                    float *pg = sums + at.column(i), *pb = pg + D;
#pragma unroll
                    for (int j = 0; j < VEC / 2; j += 2) {
                        if constexpr (!SHIFT) {  // whole 16-byte pieces, of columns and of sums
                            ulonglong2 *qg = reinterpret_cast<ulonglong2*>(pg + 2 * j), *qb = reinterpret_cast<ulonglong2*>(pb + 2 * j), vg = *qg, vb = *qb;
                            vg.x = fma2(d[j], h[j], vg.x);
                            vg.y = fma2(d[j + 1], h[j + 1], vg.y);
                            vb.x = add2(vb.x, d[j]);
                            vb.y = add2(vb.y, d[j + 1]);
                            *qg = vg;
                            *qb = vb;
                        } else {
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if (at.has(i, 2 * j + k)) {
                                    const float2 fd = split_x2(d[j + k / 2]), fh = split_x2(h[j + k / 2]);
                                    const float e = k & 1 ? fd.y : fd.x;
                                    pg[2 * j + k] = fmaf(e, k & 1 ? fh.y : fh.x, pg[2 * j + k]);
                                    pb[2 * j + k] += e;
                                }
                        }
                    }
                }
            }
        }
        const float2 fa = split_x2(a), fb = split_x2(b);
        float s[2] = {fa.x + fa.y, fb.x + fb.y};
        group_sum<2>(s, G, at.group, red, par);
        const f32x2 na = make_x2(-s[0] * rd, -s[0] * rd), nb = make_x2(-s[1] * rd, -s[1] * rd);
        if (r < rows)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (!at.any(i)) continue;
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j)
                    vx[i].set_pair(j, mul2(fma2(vd[i].pair(j), g[i][j], fma2(mul2(add2(vx[i].pair(j), nm2), is2), nb, na)), is2));
                at.store(po, i, vx[i]);
            }
        po += so;
    }
    __syncthreads();
    if constexpr (!SMEM) {
        // In ascending order: groups of whole warps one after the other; smaller ones within their warp, each warp into sums of its own, which are
        // then added.
        const int warps = (int)blockDim.x >> 5;
        for (int k = 0; k < (G < 32 ? 32 / G : groups); ++k) {
            float* to = sums + (G < 32 ? 2 * D * warp : 0);
            if ((G < 32 ? lane / G : at.group) == k)
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        if (at.has(i, j)) {
                            const float2 fg = split_x2(ag[i][j / 2]), fb = split_x2(ab[i][j / 2]);
                            to[at.column(i) + j] += j & 1 ? fg.y : fg.x;
                            to[D + at.column(i) + j] += j & 1 ? fb.y : fb.x;
                        }
            if (G < 32) __syncwarp();
            else __syncthreads();
        }
        if (G < 32) {
            __syncthreads();
            for (int i = threadIdx.x; i < 2 * D; i += blockDim.x)
                for (int w = 1; w < warps; ++w) sums[i] += sums[2 * D * w + i];
        }
    }
    float* mine = part + 2 * (int64_t)blockIdx.x * D;
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

// How the register kernels run: threads per group, groups per block and blocks.
struct Plan {
    int G, groups, blocks;
};

// Groups for `pieces` pieces of a row, nv each to a thread, in blocks of about `threads` threads, `per_sm` of them on an SM.  G is a power of two
// within a warp, and whole warps above.  Where a row starts at another place of a 16-byte piece than the one before (shift), the number of
// groups is a multiple of vec.
Plan plan_rows(int64_t pieces, int nv, int64_t rows, int threads, int per_sm, bool shift, int vec) {
    Plan p;
    const int64_t t = (pieces + nv - 1) / nv;
    p.G = 1;
    while (p.G < t && p.G < 32) p.G *= 2;
    if (t > 32) p.G = (int)((t + 31) / 32 * 32);
    const int least = std::max(1, 32 / p.G);  // whole warps
    p.groups = std::max(least, threads / p.G);
    while (p.groups > least && (int64_t)p.groups * 148 > 2 * rows) p.groups = std::max(least, p.groups / 2);  // few rows: on more SMs
    int64_t blocks = std::min<int64_t>((rows + p.groups - 1) / p.groups, (int64_t)148 * per_sm);
    if (shift) {
        int unit = vec;  // blocks a multiple of it, and so the groups of vec
        while (unit > 1 && p.groups * (unit / 2) % vec == 0) unit /= 2;
        blocks = blocks > unit ? blocks / unit * unit : unit;  // not more than fit the SMs at a time
    }
    p.blocks = (int)blocks;
    return p;
}

// Pieces of 16 bytes that a row of D values touches wherever it starts.
int64_t pieces_of(int64_t D, int vec, bool shift) {
    return shift ? (D + 2 * vec - 2) / vec : (D + vec - 1) / vec;
}

// Whether arrays that start at the addresses `bits` were made of, with rows `ld` and `other` values apart, keep to the plan of the register kernels: on
// 16-byte boundaries, and every row of one at the same place of a 16-byte piece as that of the others.
bool same_places(uintptr_t bits, int64_t rows, int64_t ld, int64_t other, int vec) {
    return (bits & 15u) == 0 && (rows == 1 || (ld - other) % vec == 0);
}

template <typename F, typename... Args>
int launch_rows(F* kernel, const Plan& p, size_t smem, cudaStream_t s, Args... args) {
    if (smem > 40 * 1024) CHXQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    CHXQ_CUDA(launch_pdl(kernel, dim3((unsigned)p.blocks), p.G * p.groups, smem, s, args...));
    count_launch(1);
    return CHXQ_OK;
}

constexpr int kMaxBlocks = 148;  // of the gradient: one per SM

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
        constexpr int VEC = 16 / (int)sizeof(T);
        const uintptr_t bits = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y);
        const bool shift = D % VEC != 0;
        const int64_t pieces = pieces_of(D, VEC, shift);
        const bool aligned = ((reinterpret_cast<uintptr_t>(scale) | reinterpret_cast<uintptr_t>(bias)) & 15u) == 0;
        if (same_places(bits, rows, ldx, D, VEC) && (shift || aligned)) {
            int64_t grid = rows;
            int threads = 256, G = 0;
            auto go = [&](auto* kernel) {
                CHXQ_CUDA(launch_pdl(kernel, dim3((unsigned)grid), threads, 0, s, static_cast<const T*>(x), ldx, g, b, rows, (int)D, epsilon, G, static_cast<T*>(y), mean,
                                     inv_std_dev));
                count_launch(1);
                return CHXQ_OK;
            };
            if (pieces <= 128) {  // a group of up to a warp per row, up to four pieces a thread
                G = 1;
                while (G * 4 < pieces) G *= 2;
                grid = (rows + 256 / G - 1) / (256 / G);
                if (shift) return go(layernorm_kernel<T, 4, false, true, false>);
                return pieces == 4 * G ? go(layernorm_kernel<T, 4, false, false, true>) : go(layernorm_kernel<T, 4, false, false, false>);
            }
            if (pieces <= 4 * 1024) {
                threads = (int)((pieces + 127) / 128 * 32);
                if (shift) return go(layernorm_kernel<T, 4, true, true, false>);
                return pieces == 4 * threads ? go(layernorm_kernel<T, 4, true, false, true>) : go(layernorm_kernel<T, 4, true, false, false>);
            }
        }
        layernorm_long_kernel<T><<<(unsigned)std::min<int64_t>(rows, 148 * 8), kThreads, 0, s>>>(static_cast<const T*>(x), ldx, g, b, rows, D, epsilon,
                                                                                                 static_cast<T*>(y), mean, inv_std_dev);
        CHXQ_LAUNCH_CHECK();
        return CHXQ_OK;
    });
}

extern "C" size_t chxq_layernorm_grad_workspace(int64_t rows, int64_t D) {
    if (rows < 0 || D < 1) return 0;
    return (size_t)kMaxBlocks * 2 * (size_t)D * sizeof(float);
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
    if (rows > 0) {
        const int rc2 = with_float_type(dtype, [&](auto t) {
            using T = decltype(t);
            constexpr int VEC = 16 / (int)sizeof(T);
            const T *g = static_cast<const T*>(dy), *v = static_cast<const T*>(x);
            const uintptr_t bits = reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(dx);
            const bool shift = D % VEC != 0;
            const int64_t pieces = pieces_of(D, VEC, shift);
            const int nv = pieces <= 2 * 512 ? 2 : (pieces <= 4 * 512 ? 4 : 8);  // from four on with the columns' sums in shared memory
            if (same_places(bits, rows, ldx, D, VEC) && same_places(bits, rows, lddy, D, VEC) && pieces <= nv * 512 && D <= 16 * 1024) {
                const Plan p = plan_rows(pieces, nv, rows, 512, 1, shift, VEC);
                shares = p.blocks;
                auto go = [&](auto* kernel) {
                    return launch_rows(kernel, p, (size_t)grad_sum_floats((int)D, p.G, p.G * p.groups) * 4, s, g, lddy, v, ldx, sc, mean, inv_std_dev, rows, (int)D, p.G,
                                       static_cast<T*>(dx), part);
                };
                if (nv == 2) return shift ? go(layernorm_grad_kernel<T, 2, true, false>) : go(layernorm_grad_kernel<T, 2, false, false>);
                if (nv == 4) return shift ? go(layernorm_grad_kernel<T, 4, true, true>) : go(layernorm_grad_kernel<T, 4, false, true>);
                if constexpr (VEC == 4) return shift ? go(layernorm_grad_kernel<T, 8, true, true>) : go(layernorm_grad_kernel<T, 8, false, true>);
            }
            layernorm_dx_long_kernel<T><<<(unsigned)std::min<int64_t>(rows, 148 * 8), kThreads, 0, s>>>(g, lddy, v, ldx, sc, mean, inv_std_dev, rows, D, static_cast<T*>(dx));
            CHXQ_LAUNCH_CHECK();
            shares = (int)std::min<int64_t>(rows, 148);
            layernorm_dparam_long_kernel<T><<<dim3((unsigned)((D + kThreads - 1) / kThreads), shares), kThreads, 0, s>>>(g, lddy, v, ldx, mean, inv_std_dev, rows, D, part);
            CHXQ_LAUNCH_CHECK();
            return CHXQ_OK;
        });
        if (rc2 != CHXQ_OK) return rc2;
    }
    CHXQ_CUDA(launch_pdl(layernorm_join_kernel, dim3((unsigned)((2 * D + 31) / 32)), kThreads, 0, s, static_cast<const float*>(part), shares, D, (int)affine_dtype, dscale,
                         dbias));
    count_launch(1);
    return CHXQ_OK;
}
