// Linear in fp32, one k-ascending chain of fused multiply-adds per output (the same bits as the other kernels of this form), for large products.
//
// A block of 256 threads takes 16 TM x 16 TN outputs, a thread TM x TN of them (rows of x by rows of w): per k it reads TM + TN values from shared
// memory for TM TN multiply-adds, two an instruction (one by one: 452 us where this takes 401 for 2048^3, for want of registers).  Both operands lie in
// shared memory by k, so that a thread's values are neighbours; the next sixteen k travel through registers meanwhile.
// Bound: the fp32 pipes, busy 65% of the time for [2048, 2048] x [2048, 2048]^T (401 us, 43 TFLOP/s): 256 blocks are not two for each of 148 SMs.
#pragma once
#include "float_ops.cuh"

namespace chxq {

constexpr int kChainK = 16;  // k of a slice

// VEC: 4 where all rows start on 16-byte boundaries (K a multiple of four), else 1.
template <int TM, int TN, int VEC>
__global__ void __launch_bounds__(256, TM * TN > 32 ? 2 : 3) linear_chain_kernel(const float* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b, int N,
                                                                                 int K, int O, float* __restrict__ y) {
    constexpr int BM = 16 * TM, BN = 16 * TN, kPitchM = BM + 4, kPitchN = BN + 4;
    static_assert(TM % 4 == 0 && TN % 4 == 0, "");
    __shared__ __align__(16) float xs[2][kChainK][kPitchM], ws[2][kChainK][kPitchN];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    // a warp's threads: four along x by eight along w, so that a warp reads 16 and 32 neighbouring values
    const int tm = (warp >> 1) * 4 + (lane >> 3), tn = (warp & 1) * 8 + (lane & 7);
    const int n0 = blockIdx.y * BM, o0 = blockIdx.x * BN;
    // staging: thread t moves pieces of VEC values of k at (t % (16 / VEC)) VEC, of rows t / (16 / VEC) + a multiple of R
    constexpr int kPer = kChainK / VEC, R = 256 / kPer, kX = BM / R, kW = BN / R;
    const int sk = (t % kPer) * VEC, sr = t / kPer;
    Pack<float, VEC> px[kX], pw[kW];
    auto fetch = [&](int k0) {
        const bool in = k0 + sk < K;
#pragma unroll
        for (int i = 0; i < kX; ++i) {
            px[i].zero();
            if (in) px[i].load(x + (int64_t)min(n0 + sr + i * R, N - 1) * K + k0 + sk);
        }
#pragma unroll
        for (int i = 0; i < kW; ++i) {
            pw[i].zero();
            if (in) pw[i].load(w + (int64_t)min(o0 + sr + i * R, O - 1) * K + k0 + sk);
        }
    };
    f32x2 acc[TM][TN / 2] = {};
    fetch(0);
    int buf = 0;
    for (int k0 = 0; k0 < K; k0 += kChainK, buf ^= 1) {
#pragma unroll
        for (int i = 0; i < kX; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) xs[buf][sk + j][sr + i * R] = px[i].get(j);
#pragma unroll
        for (int i = 0; i < kW; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) ws[buf][sk + j][sr + i * R] = pw[i].get(j);
        __syncthreads();
        if (k0 + kChainK < K) fetch(k0 + kChainK);
        // Past K both operands are zero: fma(0, 0, acc) leaves acc as it is.
#pragma unroll
        for (int k = 0; k < kChainK; ++k) {
            float a[TM];
            f32x2 c[TN / 2];
#pragma unroll
            for (int i = 0; i < TM / 4; ++i) {
                const float4 v = *reinterpret_cast<const float4*>(&xs[buf][k][i * 64 + tm * 4]);
                a[4 * i] = v.x; a[4 * i + 1] = v.y; a[4 * i + 2] = v.z; a[4 * i + 3] = v.w;
            }
#pragma unroll
            for (int j = 0; j < TN / 4; ++j) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&ws[buf][k][j * 64 + tn * 4]);
                c[2 * j] = v.x; c[2 * j + 1] = v.y;
            }
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN / 2; ++j) acc[i][j] = fma2(make_x2(a[i], a[i]), c[j], acc[i][j]);
        }
        // (the other buffer is written next; its readers have passed this iteration's barrier)
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int n = n0 + (i / 4) * 64 + tm * 4 + i % 4;
        if (n >= N) continue;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int o = o0 + (j / 4) * 64 + tn * 4 + j % 4;
            const float2 v = split_x2(acc[i][j / 2]);
            if (o < O) y[(int64_t)n * O + o] = __fadd_rn(j % 2 ? v.y : v.x, b ? b[o] : 0.f);
        }
    }
}

}  // namespace chxq
