// Linear for few rows of x, or few outputs: y[m][o] = sum over k of x[m][k] w[o][k], on the fp32 pipes.
//
// The weights are read once and used for up to eight rows, so that they cost more than the products: [1, 4096] x [4096, 4096]^T in fp32 is 67 MB, 10.4 us
// of memory, and 0.5 us of multiplications.  (The tensor cores' kernel, which splits every fp32 weight into two, takes 26 us for it.)  And a block has its first
// products a memory round trip after its start, where a tile sets up barriers and tensor memory: 2 us against 4.6 for the smallest products.
// A block takes R rows of w and all K: its threads read them side by side, UNROLL pieces of each row of w and of x before the first product, so that R *
// UNROLL loads per thread are in flight; x comes out of L2 once per R outputs, which is what bounds it at eight rows.  Each value's partial sums meet in
// the warp by halving (N values in N - 1 + log2(32 / N) exchanges), then over the warps in ascending order: no order depends on timing.
// One B200, [M, 4096] x [4096, 4096]^T from M = 1: 9.3 us (out of L2, in part), 2: 10.2, 4: 12.8, 8: 15.7; [8, 2048] x [1000, 2048]^T 4.5; [8, 8192] x [8192,
// 8192]^T 61 (68% of a copy's rate).  [1, 1024] x [4096, 1024]^T bf16 3.8.
#pragma once
#include "epilogue_float.cuh"
#include "float_ops.cuh"

namespace chxq {
namespace lin {

// Sums N values over the warp; lane l has value l / (32 / N).
template <int N>
__device__ __forceinline__ float warp_sums(float (&v)[N], int lane) {
    static_assert(N <= 32 && (N & (N - 1)) == 0, "");
    int o = 16;
#pragma unroll
    for (int h = N / 2; h > 0; h /= 2, o /= 2) {
        const bool up = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < h; ++i) v[i] = (up ? v[i + h] : v[i]) + __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + h], o);
    }
    for (; o > 0; o /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    return v[0];
}

// MR: rows of x in a block; blockIdx.y: which of them.  VEC: 16 bytes of values where all rows start on 16-byte boundaries, else 1.
template <typename T, int MR, int R, int VEC, int UNROLL>
__global__ void __launch_bounds__(512) linear_rows_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw, int M, int O, int K, LinearEpilogue e) {
    constexpr int N = MR * R;
    __shared__ float red[16][N];
    pdl_launch_dependents();
    pdl_dependency_wait();
    const int o0 = (int)blockIdx.x * R, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
    const T *wr[R], *xr[MR];
#pragma unroll
    for (int r = 0; r < R; ++r) wr[r] = w + (int64_t)min(o0 + r, O - 1) * ldw;
#pragma unroll
    for (int m = 0; m < MR; ++m) xr[m] = x + (int64_t)min((int)blockIdx.y * MR + m, M - 1) * ldx;
    // the output of this thread, and what else it is made of
    const int om = (int)blockIdx.y * MR + tid / R, oc = o0 + tid % R;
    const bool mine = tid < N && om < M && oc < O;
    const float bias = mine && e.bias ? load_param({e.bias, e.bias_dtype}, oc) : 0.f;
    const float res = mine && e.residual ? to_f32(static_cast<const T*>(e.residual)[om * e.ldr + oc]) : 0.f;
    float acc[N] = {};  // [m][r]
    const uint32_t pieces = (uint32_t)(K / VEC);
    for (uint32_t p = tid; p < pieces; p += UNROLL * threads) {
        Pack<T, VEC> a[UNROLL][R], b[UNROLL][MR];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const uint32_t q = p + u * threads;
            if (q < pieces) {
#pragma unroll
                for (int r = 0; r < R; ++r) a[u][r].load(wr[r] + (int64_t)q * VEC);
#pragma unroll
                for (int m = 0; m < MR; ++m) b[u][m].load(xr[m] + (int64_t)q * VEC);
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (p + u * threads < pieces) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    float av[R];
#pragma unroll
                    for (int r = 0; r < R; ++r) av[r] = a[u][r].get(j);
#pragma unroll
                    for (int m = 0; m < MR; ++m) {
                        const float bv = b[u][m].get(j);
#pragma unroll
                        for (int r = 0; r < R; ++r) acc[m * R + r] = fmaf(av[r], bv, acc[m * R + r]);
                    }
                }
            }
    }
    if (VEC > 1 && tid < K % VEC) {  // what no whole piece holds
        const int64_t k = (int64_t)pieces * VEC + tid;
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int r = 0; r < R; ++r) acc[m * R + r] = fmaf(to_f32(wr[r][k]), to_f32(xr[m][k]), acc[m * R + r]);
    }
    const float s = warp_sums<N>(acc, lane);
    if (lane % (32 / N) == 0) red[warp][lane / (32 / N)] = s;
    __syncthreads();
    if (!mine) return;
    float z = 0.f;
    for (int i = 0; i < threads / 32; ++i) z += red[i][tid];
    z += bias;
    if (e.residual_first) z += res;
    with_activation(e.activation, [&](auto act) { z = activate<decltype(act)::value>(z); });
    if (!e.residual_first && e.residual) z += res;
    static_cast<T*>(e.y)[om * e.ldy + oc] = from_f32<T>(z);
}

}  // namespace lin
}  // namespace chxq
