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
#include "tc_kernel.cuh"  // barriers with bounded waits

namespace chxq {
namespace {

// `bytes` (a multiple of sixteen, both addresses on 16-byte boundaries) to shared memory; the barrier counts them.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

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
    int D;            // end of this block's columns: the row's, or the end of its share of the pieces
    int p0;           // first piece of that share

    __device__ __forceinline__ Place(int G_, int D_, int64_t row0, int64_t ld, int p0_ = 0, int share = 0)
        : G(G_), group((int)threadIdx.x / G_), t((int)threadIdx.x % G_), D(D_), p0(p0_) {
        shift = SHIFT ? (int)((row0 * ld) & (VEC - 1)) : 0;
        if (share) D = min(D, (p0 + share) * VEC - shift);
    }
    __device__ __forceinline__ int column(int i) const { return (p0 + t + i * G) * VEC - shift; }  // the first of piece i; negative ones belong to the row before
    __device__ __forceinline__ bool any(int i) const { return FULL || column(i) < D; }
    __device__ __forceinline__ bool full(int i) const { return !SHIFT || (column(i) >= 0 && column(i) + VEC <= D); }
    __device__ __forceinline__ bool has(int i, int j) const { return (unsigned)(column(i) + j) < (unsigned)D; }

    // Piece i of the row at `row`; zero where the thread has none.  Rows of whole pieces: the first one is read instead, so that no branch parts the
    // loads ([4096, 12000] fp32: 104 -> 70 us).  SHIFT: at the end of the buffer a row's last piece may reach past it and is read value by value.
    __device__ __forceinline__ void load(const T* row, int i, bool end, Pack<T, VEC>& v) const {
        if constexpr (!SHIFT) {
            v.load(row + (any(i) ? column(i) : 0));
            if (!any(i)) v.zero();
        } else {
            const bool tail = end && column(i) + VEC > D;
            v.zero();
            if (any(i) && !tail) v.load(row + column(i));
            if (tail)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (has(i, j)) v.put(j, row[column(i) + j]);
        }
    }
    // The same for a row that is not looked at yet: nothing here waits for the load, so a piece that the thread does not have is left as it is.
    __device__ __forceinline__ void load_ahead(const T* row, int i, bool end, Pack<T, VEC>& v) const {
        const bool tail = SHIFT && end && column(i) + VEC > D;
        if (any(i) && !tail) v.load(row + column(i));
        if (tail) {
            v.zero();
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
    // The columns' values of a parameter array; zero outside the row.  (The loads of a whole piece are in flight together; asked for one by one, each behind
    // its own test, they took longer than the rest of a small gradient.)
    __device__ __forceinline__ void params(const FloatArray& a, f32x2 (&f)[NV][VEC / 2]) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float v[VEC] = {};
            if (any(i)) {
                if (full(i)) {
                    load_params_any<T, VEC>(a, column(i), v);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        if (has(i, j)) v[j] = load_param(a, column(i) + j);
                }
            }
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) f[i][j] = make_x2(v[2 * j], v[2 * j + 1]);
        }
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

// Whether pieces of row r may reach past the end of the buffer: the last row's, and of rows shorter than a piece any of the last ones'.
template <int VEC>
__device__ __forceinline__ bool at_end(int64_t r, int64_t rows, int D) {
    return r >= rows - (D < VEC ? VEC : 1);
}

// Sums over a group of G <= 32 threads, the same for all of them.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], int G) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float q = __shfl_xor_sync(0xffffffffu, v[k], o);
            if (o < G) v[k] += q;
        }
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
            if (live) at.load(xr, i, at_end<VEC>(r, rows, D), q[i]);
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
    const float rd = 1.f / (float)D;  // (its rounding, 2^-24, is far below that of a sum of D terms)
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
    if (var == INFINITY) is = 0.f;               // (squares past the range of 32 bits; the step would make NaN of it)
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

// Floats of the columns' sums of a block: [2][D] of each of its warps.
__host__ __device__ constexpr int grad_sum_floats(int D, int threads) {
    return 2 * D * (threads / 32);
}

// First row and distance of the rows of a group.  With SHIFT the groups of a block start at the same place of a piece: gridDim.x is a multiple of VEC.
template <bool SHIFT, int VEC>
__device__ __forceinline__ int64_t first_row(int block, int groups, int group) {
    return SHIFT ? block % VEC + VEC * ((int64_t)(block / VEC) * groups + group) : (int64_t)block * groups + group;
}

// Short rows, in groups of up to a warp: every warp goes its own way, no barrier.  The next row is fetched into registers.  The columns' sums leave as one
// partial sum [2][D] per block.
template <typename T, int NV, bool SHIFT>
__global__ void __launch_bounds__(512) layernorm_grad_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, FloatArray scale,
                                                             const float* __restrict__ mean, const float* __restrict__ inv, int64_t rows, int D, int G,
                                                             T* __restrict__ dx, float* __restrict__ part) {
    constexpr int VEC = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) float sums[];
    pdl_launch_dependents();
    pdl_dependency_wait();
    const int groups = (int)blockDim.x / G, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t step = (int64_t)gridDim.x * groups;
    int64_t r = first_row<SHIFT, VEC>((int)blockIdx.x, groups, (int)threadIdx.x / G);
    const Place<T, NV, SHIFT> at(G, D, r, ldx);
    const T *px = x + r * ldx, *pd = dy + r * lddy;
    T* po = dx + r * D;
    const int64_t sx = step * ldx, sd = step * lddy, so = step * D;
    Pack<T, VEC> vx[NV], vd[NV], nx[NV], nd[NV];
    float m = 0.f, is = 0.f, nm = 0.f, ns = 0.f;
    if (r < rows) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            at.load_ahead(px, i, at_end<VEC>(r, rows, D), nx[i]);
            at.load_ahead(pd, i, at_end<VEC>(r, rows, D), nd[i]);
        }
        nm = mean[r];
        ns = inv[r];
    }
    f32x2 g[NV][VEC / 2];
    at.params(scale, g);
    f32x2 ag[NV][VEC / 2] = {}, ab[NV][VEC / 2] = {};
    for (int i = threadIdx.x; i < grad_sum_floats(D, (int)blockDim.x); i += blockDim.x) sums[i] = 0.f;
    __syncthreads();
    const float rd = 1.f / (float)D;
    // Groups below 32 threads share warps, whose shuffles they all take part in: such a warp goes on until its first group, which has the most rows, is
    // done.
    int64_t lead = r - (int64_t)(lane / G) * (SHIFT ? VEC : 1);
    for (; lead < rows; lead += step, r += step) {
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
                at.load_ahead(px, i, at_end<VEC>(r + step, rows, D), nx[i]);
                at.load_ahead(pd, i, at_end<VEC>(r + step, rows, D), nd[i]);
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
                    ag[i][j] = fma2(d[j], h[j], ag[i][j]);
                    ab[i][j] = add2(ab[i][j], d[j]);
                }
            }
        }
        const float2 fa = split_x2(a), fb = split_x2(b);
        float s[2] = {fa.x + fa.y, fb.x + fb.y};
        group_sum<2>(s, G);
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
    // the groups of a warp, which have the same columns, by shuffles; the warps each in a place of their own, and then in ascending order
    for (int o = G; o < 32; o <<= 1)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
                ag[i][j] = add2(ag[i][j], __shfl_down_sync(0xffffffffu, ag[i][j], o));
                ab[i][j] = add2(ab[i][j], __shfl_down_sync(0xffffffffu, ab[i][j], o));
            }
    if (lane < G)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (at.has(i, j)) {
                    const float2 fg = split_x2(ag[i][j / 2]), fb = split_x2(ab[i][j / 2]);
                    sums[2 * D * warp + at.column(i) + j] = j & 1 ? fg.y : fg.x;
                    sums[2 * D * warp + D + at.column(i) + j] = j & 1 ? fb.y : fb.x;
                }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += blockDim.x)
        for (int w = 1; w < (int)blockDim.x >> 5; ++w) sums[i] += sums[2 * D * w + i];
    float* mine = part + 2 * (int64_t)blockIdx.x * D;
    for (int i = threadIdx.x; i < 2 * D; i += blockDim.x) mine[i] = sums[i];
}

// Rows in between, the common ones.  A group of G threads, whole warps, takes ROWS rows at a time: two, or one where the ring has no more than
// three stages.  They come through a ring in shared memory, a row of x and one of dy per stage by one bulk copy each, as far ahead as there is
// room: with the next row in registers 32 KB are in flight per SM, a third less than the latency of the memory asks for.  Two rows share the barrier
// and hide each other's latencies; the second pass reads shared memory again instead of holding both rows.  The columns' sums stay in registers.
// Rows too long for the registers of 512 threads: the CL blocks of a cluster take a share of the columns each (one group per block), and the rows'
// sums meet across them; one block with its sums in shared memory took 153 us for [4096, 16384] bf16 and 280 for [4096, 12345].
// (A wait that expires raises the status word; the loop then runs on to its end over whatever is there, so that no barrier is missed.
// test_skip: the row of a group whose copies are left out, chxq_tc_test_hooks.)
// [8192, 8192] bf16: 86 us, 73% of a copy's rate (the instructions of two passes over 16-bit values bound it); [16384, 4096] fp32 122 us, the
// memory's; [8192, 8192] fp32 140 us (89%); [4096, 16384] bf16 102 us, [4096, 12345] bf16 103 us, [4096, 14001] fp32 137 us.
constexpr int kMaxStages = 8;
template <typename T, int NV, bool SHIFT, int CL, int ROWS>
__global__ void __launch_bounds__(512) layernorm_grad_ring_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, FloatArray scale,
                                                                  const float* __restrict__ mean, const float* __restrict__ inv, int64_t rows, int D, int G, int stages,
                                                                  int row_bytes, T* __restrict__ dx, float* __restrict__ part, int* status, uint64_t wait_limit_ns,
                                                                  int test_skip) {
    // (row_bytes: of a block's share of a row)
    constexpr int VEC = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) uint8_t ring[];  // [groups][stages][x, dy][row_bytes]; the block's sums [2][D] in the end
    __shared__ __align__(16) float red[2][16 * CL][4];
    __shared__ uint64_t bars[16 / 2 * kMaxStages];
    __shared__ int abort_flag;
    const int groups = (int)blockDim.x / G, group = (int)threadIdx.x / G, lane = threadIdx.x & 31;
    auto bar = [&](int s) { return tc::smem_u32(&bars[group * kMaxStages + s]); };
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < groups * kMaxStages; ++i) tc::mbar_init(tc::smem_u32(&bars[i]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    if constexpr (CL > 1) tc::cluster_sync_all();  // the blocks write into one another's shared memory: all have started
    pdl_launch_dependents();
    pdl_dependency_wait();
    const int rank = CL > 1 ? (int)tc::cluster_ctarank() : 0, share = row_bytes / 16;
    const int64_t step = (int64_t)(gridDim.x / CL) * groups, first = first_row<SHIFT, VEC>((int)blockIdx.x / CL, groups, group);
    const Place<T, NV, SHIFT> at(G, D, first, ldx, rank * share, CL > 1 ? share : 0);
    const int64_t start = rank * share * VEC - at.shift;  // the first piece's column
    const int n = first < rows ? (int)((rows - first + step - 1) / step) : 0;
    uint8_t* mine = ring + (size_t)group * stages * 2 * row_bytes;
    // (one thread) Row k of the group into its stage.  The last row's last piece may reach past the buffer: it is copied value by value.
    auto fetch = [&](int k, int stage) {
        const int64_t r = first + k * step;
        uint8_t* st = mine + (size_t)stage * 2 * row_bytes;
        const int used = max(0, at.D - (int)start);  // values from the first piece's start to the end of the share
        int bytes = (used + VEC - 1) / VEC * 16;
        if constexpr (SHIFT) {
            if (r == rows - 1 && used % VEC != 0) {
                bytes -= 16;
                for (int c = bytes / (int)sizeof(T); c < used; ++c) {
                    reinterpret_cast<T*>(st)[c] = x[r * ldx + start + c];
                    reinterpret_cast<T*>(st + row_bytes)[c] = dy[r * lddy + start + c];
                }
            }
        }
        tc::mbar_expect_tx(bar(stage), 2u * (uint32_t)bytes);
        if (bytes > 0 && k != test_skip) {
            bulk_load(tc::smem_u32(st), x + r * ldx + start, (uint32_t)bytes, bar(stage));
            bulk_load(tc::smem_u32(st + row_bytes), dy + r * lddy + start, (uint32_t)bytes, bar(stage));
        }
    };
    if (at.t == 0)
        for (int k = 0; k < stages && k < n; ++k) fetch(k, k);
    f32x2 g[NV][VEC / 2], ag[NV][VEC / 2] = {}, ab[NV][VEC / 2] = {};
    at.params(scale, g);
    const float rd = 1.f / (float)D;
    auto read = [&](int stage, int which, int i, f32x2 (&v)[VEC / 2]) {
        Pack<T, VEC> q;
        q.load(reinterpret_cast<const T*>(mine + (stage * 2 + which) * row_bytes) + (at.t + i * G) * VEC);
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) v[j] = q.pair(j);
    };
    float m[ROWS] = {}, is[ROWS] = {}, nm[ROWS] = {}, ns[ROWS] = {};
    auto stats = [&](int k) {
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
            if (k + u < n) {
                nm[u] = mean[first + (k + u) * step];
                ns[u] = inv[first + (k + u) * step];
            }
    };
    stats(0);
    int stage[ROWS], phase[ROWS] = {}, old[ROWS] = {};  // of these rows, and the stages of those before
#pragma unroll
    for (int u = 0; u < ROWS; ++u) stage[u] = u;
    for (int k = 0; k < n; k += ROWS) {
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            m[u] = nm[u];
            is[u] = ns[u];
        }
        stats(k + ROWS);
        float s[4] = {};
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            if (k + u >= n) break;
            tc::mbar_wait(bar(stage[u]), (uint32_t)phase[u], &abort_flag, status, 71, 0, wait_limit_ns);
            const f32x2 is2 = make_x2(is[u], is[u]), nm2 = make_x2(-m[u], -m[u]);
            f32x2 a = 0ull, b = 0ull;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (!at.any(i)) continue;
                f32x2 d[VEC / 2], h[VEC / 2];
                read(stage[u], 0, i, h);
                read(stage[u], 1, i, d);
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) h[j] = mul2(add2(h[j], nm2), is2);
                if constexpr (SHIFT) {
                    at.mask(i, d);
                    at.mask(i, h);
                }
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) {
                    const f32x2 gd = mul2(d[j], g[i][j]);
                    a = add2(a, gd);
                    b = fma2(gd, h[j], b);
                    ag[i][j] = fma2(d[j], h[j], ag[i][j]);
                    ab[i][j] = add2(ab[i][j], d[j]);
                }
            }
            const float2 fa = split_x2(a), fb = split_x2(b);
            s[2 * u] = fa.x + fa.y;
            s[2 * u + 1] = fb.x + fb.y;
        }
        // the sums of both rows over the group
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int q = 0; q < 2 * ROWS; ++q) s[q] += __shfl_xor_sync(0xffffffffu, s[q], o);
        const int par = (k / ROWS) & 1, warps = G >> 5;
        if constexpr (CL == 1) {
            if (lane == 0) *reinterpret_cast<float4*>(red[par][threadIdx.x >> 5]) = make_float4(s[0], s[1], s[2], s[3]);
            group_barrier(1 + group, G);
        } else {
            if (lane < CL)  // to every block of the cluster
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(tc::map_to_cta(tc::smem_u32(red[par][rank * warps + (int)(threadIdx.x >> 5)]), (uint32_t)lane)),
                             "f"(s[0]), "f"(s[1]), "f"(s[2]), "f"(s[3])
                             : "memory");
            __syncwarp();
            tc::cluster_sync_all();
        }
        // every thread has left the rows before these: theirs are the stages to refill (but none behind an expired wait: its barrier is still in the phase that
        // a refill has arrived at)
        if (at.t == 0 && k >= ROWS && !*static_cast<volatile int*>(&abort_flag))
#pragma unroll
            for (int u = 0; u < ROWS; ++u)
                if (k - ROWS + u + stages < n) fetch(k - ROWS + u + stages, old[u]);
        s[0] = s[1] = s[2] = s[3] = 0.f;
        for (int e = lane & 15; e < CL * warps; e += 16) {
            const float4 q = *reinterpret_cast<const float4*>(red[par][(CL == 1 ? group * warps : 0) + e]);
            s[0] += q.x; s[1] += q.y; s[2] += q.z; s[3] += q.w;
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
#pragma unroll
            for (int q = 0; q < 2 * ROWS; ++q) s[q] += __shfl_xor_sync(0xffffffffu, s[q], o);
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            if (k + u >= n) break;
            const f32x2 is2 = make_x2(is[u], is[u]), nm2 = make_x2(-m[u], -m[u]), na = make_x2(-s[2 * u] * rd, -s[2 * u] * rd), nb = make_x2(-s[2 * u + 1] * rd, -s[2 * u + 1] * rd);
            T* out = dx + (first + (k + u) * step) * D;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (!at.any(i)) continue;
                f32x2 d[VEC / 2], h[VEC / 2];
                read(stage[u], 0, i, h);
                read(stage[u], 1, i, d);
                Pack<T, VEC> o;
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) o.set_pair(j, mul2(fma2(d[j], g[i][j], fma2(mul2(add2(h[j], nm2), is2), nb, na)), is2));
                at.store(out, i, o);
            }
        }
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            old[u] = stage[u];
            stage[u] += ROWS;
            if (stage[u] >= stages) {
                stage[u] -= stages;
                phase[u] ^= 1;
            }
        }
    }
    __syncthreads();
    if (abort_flag) {  // copies in flight get the time to land
        const uint64_t t0 = tc::global_timer_ns();
        while (tc::global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
        __syncthreads();
    }
    if constexpr (CL > 1) tc::cluster_sync_all();  // the others may still be writing into this block's `red`
    // the groups' sums in ascending order, in the order of the pieces
    float* sums = reinterpret_cast<float*>(ring);
    const int cols = share * VEC;
    for (int k = 0; k < groups; ++k) {
        if (group == k)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (!at.any(i)) continue;
                // (whole pieces: what a thread has of the rows beside its own is zero)
                ulonglong2 *pg = reinterpret_cast<ulonglong2*>(sums + (at.t + i * G) * VEC), *pb = reinterpret_cast<ulonglong2*>(sums + cols + (at.t + i * G) * VEC);
#pragma unroll
                for (int j = 0; j < VEC / 4; ++j) {
                    ulonglong2 vg = make_ulonglong2(ag[i][2 * j], ag[i][2 * j + 1]), vb = make_ulonglong2(ab[i][2 * j], ab[i][2 * j + 1]);
                    if (k) {
                        const ulonglong2 og = pg[j], ob = pb[j];
                        vg = make_ulonglong2(add2(og.x, vg.x), add2(og.y, vg.y));
                        vb = make_ulonglong2(add2(ob.x, vb.x), add2(ob.y, vb.y));
                    }
                    pg[j] = vg;
                    pb[j] = vb;
                }
            }
        __syncthreads();
    }
    float* to = part + 2 * (int64_t)(blockIdx.x / CL) * D;
    for (int i = threadIdx.x; i < cols; i += blockDim.x) {
        const int c = (int)start + i;
        if (c >= 0 && c < at.D) {
            to[c] = sums[i];
            to[D + c] = sums[cols + i];
        }
    }
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

// part [shares][2 D] -> the sum of the shares: 32 columns a block; warps that take every eighth share (up to 40 shares) or every 32nd, at most five each,
// loaded together.
constexpr int kMaxBlocks = 148;  // of the gradient, which the workspace has room for: one per SM of a B200
__global__ void __launch_bounds__(1024) layernorm_join_kernel(const float* __restrict__ part, int shares, int64_t D, int dtype, void* dscale, void* dbias) {
    __shared__ float acc[32][33];
    pdl_launch_dependents();
    pdl_dependency_wait();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = (int)blockDim.x >> 5;
    const int64_t i = (int64_t)blockIdx.x * 32 + lane;
    constexpr int kEach = 5;
    static_assert(kEach * 32 >= kMaxBlocks, "shares per warp");
    float v[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) v[k] = i < 2 * D && w + warps * k < shares ? part[(int64_t)(w + warps * k) * 2 * D + i] : 0.f;
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < kEach; ++k) a += v[k];
    acc[w][lane] = a;
    __syncthreads();
    if (w == 0 && i < 2 * D) {
        a = 0.f;
        for (int k = 0; k < warps; k += 8) {
#pragma unroll
            for (int q = 0; q < 8; ++q) a += acc[k + q][lane];
        }
        if (i < D) store_param(dscale, dtype, i, a);
        else if (dbias) store_param(dbias, dtype, i - D, a);
    }
}

// How the register kernels run: threads per group, groups per block and blocks.
struct Plan {
    int G, groups, blocks;
};

// Groups for `pieces` pieces of a row, nv each to a thread, in blocks of about `threads` threads, one on an SM.  G is a power of two
// within a warp, and whole warps above.  Where a row starts at another place of a 16-byte piece than the one before (shift), the number of
// blocks is a multiple of vec.
Plan plan_rows(int64_t pieces, int nv, int64_t rows, int threads, bool shift, int vec) {
    Plan p;
    const int64_t t = (pieces + nv - 1) / nv;
    p.G = 1;
    while (p.G < t && p.G < 32) p.G *= 2;
    if (t > 32) p.G = (int)((t + 31) / 32 * 32);
    const int least = std::max(1, 32 / p.G);  // whole warps
    p.groups = std::max(least, threads / p.G);
    const int64_t sms = std::min(tc::sm_count(), kMaxBlocks);
    while (p.groups > least && p.groups * sms > 2 * rows) p.groups = std::max(least, p.groups / 2);  // few rows: on more SMs
    int64_t blocks = std::min<int64_t>((rows + p.groups - 1) / p.groups, sms);
    if (shift) blocks = blocks > vec ? blocks / vec * vec : vec;  // not more than fit the SMs at a time
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
    // (always the same limit, that of the longest rows: another thread may be between this and its launch)
    if (smem > 48 * 1024) CHXQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024));
    CHXQ_CUDA(launch_pdl(kernel, dim3((unsigned)p.blocks), p.G * p.groups, smem, s, args...));
    count_launch(1);
    return CHXQ_OK;
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
    CHXQ_CHECK_ARG(on_values_of(float_size(dtype), x, y) && on_values_of(float_size(affine_dtype), scale, bias) && on_values_of(4, mean, inv_std_dev),
                   "LayerNormalization: an address is no multiple of its values' size");
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
        layernorm_long_kernel<T><<<(unsigned)std::min<int64_t>(rows, tc::sm_count() * 8), kThreads, 0, s>>>(static_cast<const T*>(x), ldx, g, b, rows, D, epsilon,
                                                                                                 static_cast<T*>(y), mean, inv_std_dev);
        CHXQ_LAUNCH_CHECK();
        return CHXQ_OK;
    });
}

// Shares of the parameters' sums: one per block, and fewer of rows that are longer than blocks take, 39 MB in all.
static int grad_shares(int64_t D) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(kMaxBlocks, (int64_t)kMaxBlocks * 32768 / D));
}

extern "C" size_t chxq_layernorm_grad_workspace(int64_t rows, int64_t D) {
    if (rows < 0 || D < 1) return 0;
    return (size_t)grad_shares(D) * 2 * (size_t)D * sizeof(float);
}

extern "C" int chxq_layernorm_grad(const void* dy, int64_t lddy, const void* x, int64_t ldx, int32_t dtype, const void* scale, int32_t affine_dtype,
                                   const float* mean, const float* inv_std_dev, int64_t rows, int64_t D, void* dx, void* dscale, void* dbias, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    const int rc = check_norm("LayerNormalizationGrad", dtype, affine_dtype, rows, D);
    if (rc != CHXQ_OK) return rc;
    CHXQ_CHECK_ARG(dscale && scale && (rows == 0 || (dy && x && mean && inv_std_dev && dx)) && (rows <= 1 || (ldx >= D && lddy >= D)), "LayerNormalizationGrad: bad arguments");
    CHXQ_CHECK_ARG(on_values_of(float_size(dtype), dy, x, dx) && on_values_of(float_size(affine_dtype), scale, dscale, dbias) &&
                           on_values_of(4, mean, inv_std_dev, workspace),
                   "LayerNormalizationGrad: an address is no multiple of its values' size");
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
            // Columns of a block in the registers of 512 threads, two pieces each, or four of fp32 (sixteen values at most); longer rows shared by the blocks of a
            // cluster.
            const int nv = VEC == 4 && pieces > 1024 ? 4 : 2, cl = pieces <= nv * 512 ? 1 : (pieces <= nv * 1024 ? 2 : 4);
            if (same_places(bits, rows, ldx, D, VEC) && same_places(bits, rows, lddy, D, VEC) && pieces <= (VEC == 4 ? 4 : 2) * (VEC == 4 ? 1024 : 2048)) {
                const int64_t share = (pieces + cl - 1) / cl;
                Plan p = plan_rows(share, nv, rows, 512, shift, VEC);
                if (cl > 1) {
                    const int64_t most = cl == 2 ? 74 : 32;  // clusters that are resident at once (of four: 33)
                    p.blocks = (int)std::min<int64_t>(std::max<int64_t>(rows, 1), most);
                    if (shift) p.blocks = p.blocks > VEC ? p.blocks / VEC * VEC : VEC;
                }
                shares = p.blocks;
                if (p.G > 32) {
                    const int row_bytes = (int)share * 16;
                    constexpr int room = 220 * 1024;  // (the limit is set to it, whatever a call needs: another thread may be between that and its launch)
                    const int stages = std::min(kMaxStages, room / (p.groups * 2 * row_bytes));
                    // the groups' sums are not laid out by row but by piece: also those of pieces that hold no column
                    const size_t smem = std::max((size_t)stages * p.groups * 2 * row_bytes, (size_t)2 * share * VEC * sizeof(float));
                    int* status = device_status_ptr();
                    if (!status) return set_error(CHXQ_ERR_CUDA, "device status word is unavailable");
                    auto go = [&](auto* kernel) {
                        CHXQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, room));
                        CHXQ_CUDA(launch_pdl_cluster(cl, kernel, dim3((unsigned)(p.blocks * cl)), p.G * p.groups, smem, s, g, lddy, v, ldx, sc, mean, inv_std_dev, rows, (int)D,
                                                     p.G, stages, row_bytes, static_cast<T*>(dx), part, status, (uint64_t)tc::wait_limit_ns_value(), tc::test_skip_kb_value()));
                        count_launch(1);
                        return CHXQ_OK;
                    };
                    constexpr int kMost = 16 / VEC;  // pieces of a thread
                    // Two rows at a time need four stages: those of the rows before are refilled while these are worked on.  A share of up to 16 KB (nv == 2)
                    // leaves six or more, one of up to 32 KB three or more.
                    const bool one = stages < 4;
                    if (nv == 2 && cl == 1) return shift ? go(layernorm_grad_ring_kernel<T, 2, true, 1, 2>) : go(layernorm_grad_ring_kernel<T, 2, false, 1, 2>);
                    if constexpr (VEC == 4) {
                        if (one && cl == 1) return shift ? go(layernorm_grad_ring_kernel<T, 4, true, 1, 1>) : go(layernorm_grad_ring_kernel<T, 4, false, 1, 1>);
                        if (one) return shift ? go(layernorm_grad_ring_kernel<T, 4, true, 2, 1>) : go(layernorm_grad_ring_kernel<T, 4, false, 2, 1>);
                        if (cl == 1) return shift ? go(layernorm_grad_ring_kernel<T, 4, true, 1, 2>) : go(layernorm_grad_ring_kernel<T, 4, false, 1, 2>);
                    }
                    if (cl == 2) return shift ? go(layernorm_grad_ring_kernel<T, kMost, true, 2, 2>) : go(layernorm_grad_ring_kernel<T, kMost, false, 2, 2>);
                    if constexpr (VEC == 8) return shift ? go(layernorm_grad_ring_kernel<T, 2, true, 4, 2>) : go(layernorm_grad_ring_kernel<T, 2, false, 4, 2>);
                }
                auto go = [&](auto* kernel) {
                    return launch_rows(kernel, p, (size_t)grad_sum_floats((int)D, p.G * p.groups) * 4, s, g, lddy, v, ldx, sc, mean, inv_std_dev, rows, (int)D, p.G,
                                       static_cast<T*>(dx), part);
                };
                return shift ? go(layernorm_grad_kernel<T, 2, true>) : go(layernorm_grad_kernel<T, 2, false>);
            }
            layernorm_dx_long_kernel<T><<<(unsigned)std::min<int64_t>(rows, tc::sm_count() * 8), kThreads, 0, s>>>(g, lddy, v, ldx, sc, mean, inv_std_dev, rows, D, static_cast<T*>(dx));
            CHXQ_LAUNCH_CHECK();
            shares = (int)std::min<int64_t>(rows, grad_shares(D));
            layernorm_dparam_long_kernel<T><<<dim3((unsigned)((D + kThreads - 1) / kThreads), shares), kThreads, 0, s>>>(g, lddy, v, ldx, mean, inv_std_dev, rows, D, part);
            CHXQ_LAUNCH_CHECK();
            return CHXQ_OK;
        });
        if (rc2 != CHXQ_OK) return rc2;
    }
    CHXQ_CUDA(launch_pdl(layernorm_join_kernel, dim3((unsigned)((2 * D + 31) / 32)), shares <= 40 ? 256 : 1024, 0, s, static_cast<const float*>(part), shares, D, (int)affine_dtype, dscale,
                         dbias));
    count_launch(1);
    return CHXQ_OK;
}
