// Float matrix product, one tile per cluster: 128 rows of w times BN rows of x, the K blocks shared by the S CTAs of a cluster.
//
// For products with few rows of x, which are bound by the read of w: with w as the instruction's 128-row operand, sixteen rows of x cost a
// sixteen-column instruction instead of a 128-row tile that is mostly padding, and sharing K keeps every SM streaming.  Also for products
// in between, with too few 256 x 256 blocks for the CTA pairs.
//
// A CTA (256 threads): warp 0 loads w, warp 2 loads x (one lane each, TMA, 128-byte swizzle, STAGES stages), warp 1 owns the TMEM and issues
// the MMAs (one lane).  The sums then go from TMEM to shared memory as [row of x][row of w] in 32 bits; behind a cluster barrier each CTA takes
// BN / S rows of x, adds the S shares in ascending order (the same bits on every run) through distributed shared memory and runs the epilogue.
// Waits are bounded as in tc_kernel.cuh; a CTA that gives up still comes to both cluster barriers.
#pragma once

#include "linear_tc.cuh"

namespace chxq {
namespace lin {

template <int BN, int STAGES>
struct TileConfig {
    static constexpr int kTileW = 128 * 128, kTileX = BN * 128, kStage = kTileW + kTileX;
    static constexpr int kSums = BN * 128 * 4;
    static constexpr int kData = STAGES * kStage > kSums ? STAGES * kStage : kSums;
    static constexpr int kBarOffset = kData;
    static constexpr int kSmem = 1024 + kBarOffset + (2 * STAGES + 1) * 8 + 16;
    static constexpr int kTmemCols = BN < 32 ? 32 : BN;
    static_assert(kSmem <= 227 * 1024, "shared memory over the per-CTA limit");
};

// From the shares of a tile, [BN][128] sums in the shared memory of each CTA of the cluster, to the outputs of this CTA's rows of x: the shares added in
// ascending order (the same bits on every run), then bias, activation and residual.  `warp`: this one of WARPS.
// VEC: four neighbouring values per lane and access; else rows of y off 16-byte boundaries, lanes 32 values apart.  A few rows at a time, so that their loads
// are in flight together ([509, 1283] x [2999, 1283]^T with a residual: 46 us one by one).
template <typename T, int BN, int WARPS, bool VEC>
__device__ __forceinline__ void tile_epilogue_rows(const TcArgs& p, const float* sums, int x0, int w0, int rank, int split, int warp, int lane) {
    constexpr bool kFast = sizeof(T) == 2;
    constexpr int kRows = BN * 8 / WARPS >= 128 ? 4 : (BN >= 64 ? 2 : 1);
    const int cols = (BN + split - 1) / split;  // rows of x of this CTA
    const int c1 = min(min((rank + 1) * cols, BN), p.M - x0);
    auto feature = [&](int j) { return w0 + (VEC ? 4 * lane + j : lane + 32 * j); };
    bool in[4];
    float bias[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        in[j] = feature(j) < p.O;
        bias[j] = p.e.bias && in[j] ? load_param({p.e.bias, p.e.bias_dtype}, feature(j)) : 0.f;
    }
    const uint32_t mine = smem_u32(sums) + (VEC ? 16u : 4u) * (uint32_t)lane;
    for (int c0 = rank * cols + warp; c0 < c1; c0 += WARPS * kRows) {
        float v[kRows * 4], res[kRows * 4] = {};
#pragma unroll
        for (int i = 0; i < kRows * 4; ++i) v[i] = bias[i % 4];
        auto row = [&](int k) { return c0 + k * WARPS; };
        auto have = [&](int k) { return kRows == 1 || row(k) < c1; };  // (reading another row in its place would double the traffic between the CTAs)
        if (p.e.residual) {
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                if (!have(k)) break;
                const T* pr = static_cast<const T*>(p.e.residual) + (int64_t)(x0 + row(k)) * p.e.ldr;
                if constexpr (!VEC) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (in[j]) res[4 * k + j] = to_f32(pr[feature(j)]);
                } else if (in[0]) {
                    if constexpr (sizeof(T) == 4) {
                        const float4 q = *reinterpret_cast<const float4*>(pr + feature(0));
                        res[4 * k] = q.x; res[4 * k + 1] = q.y; res[4 * k + 2] = q.z; res[4 * k + 3] = q.w;
                    } else {
                        const uint2 q = *reinterpret_cast<const uint2*>(pr + feature(0));
                        const float2 lo = unpack16<T>(q.x), hi = unpack16<T>(q.y);
                        res[4 * k] = lo.x; res[4 * k + 1] = lo.y; res[4 * k + 2] = hi.x; res[4 * k + 3] = hi.y;
                    }
                }
            }
        }
        // four shares at a time, their loads in flight together
        for (int s0 = 0; s0 < split; s0 += 4) {
            float q[4][kRows * 4] = {};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if (s0 + s >= split) break;
                const uint32_t from = split > 1 ? map_to_cta(mine, s0 + s) : mine;
#pragma unroll
                for (int k = 0; k < kRows; ++k) {
                    if (!have(k)) break;
                    const uint32_t at = from + (uint32_t)(row(k) * 512);
                    if constexpr (VEC)
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(q[s][4 * k]), "=f"(q[s][4 * k + 1]), "=f"(q[s][4 * k + 2]), "=f"(q[s][4 * k + 3])
                                     : "r"(at));
                    else
#pragma unroll
                        for (int j = 0; j < 4; ++j) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(q[s][4 * k + j]) : "r"(at + 128u * j));
                }
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
                if (s0 + s < split)
#pragma unroll
                    for (int i = 0; i < kRows * 4; ++i) v[i] += q[s][i];
        }
        epilogue_apply<kRows * 4, kFast>(p.e, v, res);
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            if (!have(k)) break;
            T* py = static_cast<T*>(p.e.y) + (int64_t)(x0 + c0 + k * WARPS) * p.e.ldy;
            if constexpr (!VEC) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (in[j]) py[feature(j)] = from_f32<T>(v[4 * k + j]);
            } else if (in[0]) {
                if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(py + feature(0)) = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                else *reinterpret_cast<uint2*>(py + feature(0)) = make_uint2(pack16<T>(v[4 * k], v[4 * k + 1]), pack16<T>(v[4 * k + 2], v[4 * k + 3]));
            }
        }
    }
}
template <typename T, int BN, int WARPS>
__device__ __forceinline__ void tile_epilogue(const TcArgs& p, const float* sums, int x0, int w0, int rank, int split, int warp, int lane) {
    if (p.vec) tile_epilogue_rows<T, BN, WARPS, true>(p, sums, x0, w0, rank, split, warp, lane);
    else tile_epilogue_rows<T, BN, WARPS, false>(p, sums, x0, w0, rank, split, warp, lane);
}

template <typename T, int BN, int STAGES>
__global__ void __launch_bounds__(256) linear_tile_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const TcArgs p, int split,
                                                          int x_tiles) {
    using Cfg = TileConfig<BN, STAGES>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kBarOffset);
    uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (STAGES + s); };
    const uint32_t done = bar0 + 8u * (2 * STAGES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full(s), 2);  // one arrival per producer
            mbar_init(empty(s), 1);
        }
        mbar_init(done, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_ptr), Cfg::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_ptr;
    pdl_launch_dependents();
    pdl_dependency_wait();

    const int rank = split > 1 ? (int)cluster_ctarank() : 0;
    const int tile = (int)blockIdx.x / split;
    const int x0 = (tile % x_tiles) * BN, w0 = (tile / x_tiles) * 128;  // neighbours share their rows of w
    const int kb0 = (int)((int64_t)p.k_blocks * rank / split), kb1 = (int)((int64_t)p.k_blocks * (rank + 1) / split);  // split <= k_blocks: never empty

    if (lane == 0 && (warp == 0 || warp == 2)) {
        const bool is_w = warp == 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            const int s = (kb - kb0) % STAGES;
            if (!mbar_wait(empty(s), ((uint32_t)((kb - kb0) / STAGES) & 1u) ^ 1u, abort_flag, p.status, 41, 0, p.wait_limit_ns)) break;
            uint8_t* st = smem + s * Cfg::kStage;
            mbar_expect_tx(full(s), is_w ? Cfg::kTileW : Cfg::kTileX);
            if (is_w) {
                if (kb != p.test_skip_kb) tma_load_2d(smem_u32(st), &tmW, full(s), kb * 128, w0);
            } else tma_load_2d(smem_u32(st + Cfg::kTileW), &tmX, full(s), kb * 128, x0);
        }
    } else if (lane == 0 && warp == 1) {
        bool ok = true;
        const uint32_t hi = kmajor_desc_hi<128>(), idesc = p.idesc | idesc_extents(128, BN);
        for (int kb = kb0; kb < kb1; ++kb) {
            const int s = (kb - kb0) % STAGES;
            if (!mbar_wait(full(s), (uint32_t)((kb - kb0) / STAGES) & 1u, abort_flag, p.status, 42, 0, p.wait_limit_ns)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t a = kmajor_desc_lo(smem_u32(smem + s * Cfg::kStage)), b = kmajor_desc_lo(smem_u32(smem + s * Cfg::kStage + Cfg::kTileW));
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_f16<false>(tmem, a + 2u * k, b + 2u * k, hi, idesc, kb > kb0 || k > 0 ? 1u : 0u);
            umma_commit(empty(s));
        }
        if (ok) umma_commit(done);
    }
    __syncwarp();
    const bool got = __all_sync(0xffffffffu, mbar_wait(done, 0, abort_flag, p.status, 43, 32, p.wait_limit_ns));
    tc_fence_after();
    float* sums = reinterpret_cast<float*>(smem);  // [BN][128]; every stage has been read by now
    if (got) {
        // warps w and w + 4 read the TMEM lanes 32 (w mod 4) .. +31 (rows of w), each half of the columns (rows of x)
        const int f = (warp & 3) * 32 + lane, half = warp >> 2;
#pragma unroll
        for (int c = 0; c < BN / 16; ++c) {
            if (BN > 16 && (c & 1) != half) continue;
            if (BN == 16 && half) continue;
            uint32_t r[16];
            tmem_ld_32x32b_x16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(c * 16), r);
            tmem_ld_wait16(r);
#pragma unroll
            for (int j = 0; j < 16; ++j) sums[(c * 16 + j) * 128 + f] = __uint_as_float(r[j]);
        }
    }
    tc_fence_before();
    if (split > 1) cluster_sync_all();
    else __syncthreads();
    if (got) tile_epilogue<T, BN, 8>(p, sums, x0, w0, rank, split, warp, lane);
    __syncthreads();
    if (*abort_flag) {  // copies in flight get the time to land
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
        __syncthreads();
    }
    if (split > 1) cluster_sync_all();  // the others may still be reading this CTA's sums
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, Cfg::kTmemCols);
    }
}

// ---- fp32 operands ---------------------------------------------------------------------------------------------------------
//
// The tensor cores multiply tf32, eleven significant bits.  A value is split as a = h + l with h = tf32(a) and l = tf32(a - h), rounded to nearest, 22 bits in
// all, and the product taken as h h' + h l' + l h': what is left out is below 2^-21 |a a'|, the rounding of an fp32 product in a sum of a few.  (Sums of fewer
// than 32 terms are therefore further off than a chain of fp32 products, 9.8e-8 against 4.2e-8 for K = 4.)
// The sums: h h' goes through TMEM in chains of kChain K blocks (at most 16 instructions, whose additions the tensor core may truncate), each then
// added in registers; the two small products have an accumulator of their own, 2^-11 in size, for the whole of K.  [2048, 2048] x [2048, 2048]^T:
// 3.5e-7 off the sums in 64 bits (root mean square, relative); chains of eight 6.4e-7 for 2% less time, of two 2.2e-7 for 5% more; an fp32
// product 8.1e-7.
// The operands: w is split into tensor memory, two stages of h and l, x in place in shared memory with l beside it.  (Both in shared memory: 192 KB of
// traffic a K block instead of 112, 140 us for 2048^3 where this takes 112.)  h and l of x are neighbours, so that one instruction of 2 BN columns
// takes h of w times both: h h' into the chain's accumulator and h l' into the small products'.  Those lie between the accumulators of even and of odd
// chains, and x's halves change places with the chain.  Since the instruction adds to both or to none, a chain starts from zeros that are written.
// Roles as above, with 640 threads: warps 0 and 2 load, warp 1 issues, warps 4-19 split, in two groups that take the K blocks by turns, drain the chains and
// run the epilogue.
// Bound: a K block of 128 x 128 takes 0.8 us where the tensor pipe needs 0.41: the splitting (some twenty instructions per sixteen bytes) and the
// issuing thread (eight products and a commit of 75 to 90 cycles each beside busy warps).
template <int BN, int STAGES>
struct TileF32Config {
    static constexpr int kTileW = 128 * 128, kTileX = BN * 128, kStage = kTileW + 2 * kTileX;
    static constexpr int kSums = BN * 128 * 4;
    static constexpr int kData = STAGES * kStage > kSums ? STAGES * kStage : kSums;
    static constexpr int kNumBars = 3 * STAGES + 5;
    static constexpr int kSmem = 1024 + kData + kNumBars * 8 + 16;
    static constexpr int kChain = 4;  // K blocks of 32 values
    static constexpr int kTmemW = 3 * BN;  // first column of two stages of w, 32 columns of h and 32 of l each
    static constexpr int kTmemCols = kTmemW + 128 <= 256 ? 256 : 512;
    static_assert(kSmem <= 227 * 1024, "shared memory over the per-CTA limit");
};

// v = l / kLowScale - n + a rest below 2^-22 |v|: the high part negated, so that the subtraction needs no negation (both operands' are: h h' has its sign, and the
// small products, negative, are subtracted); by integer rounding (the conversion instruction runs at a sixteenth of the rate: 279 us where this took 140 for
// 2048^3).
// The low part is held kLowScale times as large, so that it is not lost below the smallest normal value: unscaled, values of 2^-118 had 2^-20 of error and
// those of 2^-125 kept eleven bits.  (With 2^12 the low part of what is cut off below would overflow.)  Of the bits behind its eleven the tensor core
// takes no notice.
// What rounds to infinity, infinities and NaN: the sum of the differences is not finite there, and those four values are done again.
constexpr float kLowScale = 2048.f;
__device__ __forceinline__ void split_tf32_special(uint32_t v, uint32_t& n, uint32_t& l) {
    const uint32_t a = v & 0x7fffffffu;
    if (a < 0x7f7ff000u) return;
    n = a > 0x7f800000u ? 0x7fffffffu : (v & 0xffffe000u) ^ 0x80000000u;  // NaN; infinity, or cut off instead of rounded
    l = a >= 0x7f800000u ? 0u : __float_as_uint((__uint_as_float(v) + __uint_as_float(n)) * kLowScale);
}
__device__ __forceinline__ void split_tf32(const uint4& v, uint32_t* n, uint32_t* l) {
    const uint32_t in[4] = {v.x, v.y, v.z, v.w};
    f32x2 d[2];
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
        n[j] = ((in[j] + 0x1000u) & 0xffffe000u) ^ 0x80000000u;
        n[j + 1] = ((in[j + 1] + 0x1000u) & 0xffffe000u) ^ 0x80000000u;
        d[j / 2] = add2(make_x2(__uint_as_float(in[j]), __uint_as_float(in[j + 1])), make_x2(__uint_as_float(n[j]), __uint_as_float(n[j + 1])));
        const float2 f = split_x2(mul2(d[j / 2], both(kLowScale)));
        l[j] = __float_as_uint(f.x) + 0x1000u;
        l[j + 1] = __float_as_uint(f.y) + 0x1000u;
    }
    const float2 z = split_x2(add2(d[0], d[1]));
    if (!(fabsf(z.x + z.y) < INFINITY)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) split_tf32_special(in[j], n[j], l[j]);
    }
}

template <int BN, int STAGES>
__global__ void __launch_bounds__(640) linear_tile_f32_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const TcArgs p, int split,
                                                              int x_tiles) {
    using Cfg = TileF32Config<BN, STAGES>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kData);
    uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(bars + Cfg::kNumBars);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto ready = [&](int s) { return bar0 + 8u * (STAGES + s); };  // split into h and l, w in tensor memory
    auto empty = [&](int s) { return bar0 + 8u * (2 * STAGES + s); };
    auto cfull = [&](int b) { return bar0 + 8u * (3 * STAGES + b); };       // a chain is complete in its accumulator
    auto cempty = [&](int b) { return bar0 + 8u * (3 * STAGES + 2 + b); };  // ... and has been drained and cleared
    const uint32_t done = bar0 + 8u * (3 * STAGES + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full(s), 2);
            mbar_init(ready(s), 8);  // one arrival per splitting warp
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(cfull(b), 1);
            mbar_init(cempty(b), 16);
        }
        mbar_init(done, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_ptr), Cfg::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_ptr;  // accumulators: even chains, the small products, odd chains; then w
    pdl_launch_dependents();
    pdl_dependency_wait();

    const int rank = split > 1 ? (int)cluster_ctarank() : 0;
    const int tile = (int)blockIdx.x / split;
    const int x0 = (tile % x_tiles) * BN, w0 = (tile / x_tiles) * 128;
    const int kb0 = (int)((int64_t)p.k_blocks * rank / split), blocks = (int)((int64_t)p.k_blocks * (rank + 1) / split) - kb0;  // at least one
    const int chains = (blocks + Cfg::kChain - 1) / Cfg::kChain;
    float* sums = reinterpret_cast<float*>(smem);
    bool got = false;
    // Where x goes in its stage, h in place and l beside it: h first in even chains, last in odd ones.
    auto x_high = [](int kb) { return Cfg::kTileW + (kb / Cfg::kChain & 1) * Cfg::kTileX; };
    auto x_low = [](int kb) { return Cfg::kTileW + (~(kb / Cfg::kChain) & 1) * Cfg::kTileX; };

    if (warp < 4) {
        if (lane == 0 && (warp == 0 || warp == 2)) {
            const bool is_w = warp == 0;
            for (int kb = 0; kb < blocks; ++kb) {
                const int s = kb % STAGES;
                if (!mbar_wait(empty(s), ((uint32_t)(kb / STAGES) & 1u) ^ 1u, abort_flag, p.status, 61, 0, p.wait_limit_ns)) break;
                uint8_t* st = smem + s * Cfg::kStage;
                mbar_expect_tx(full(s), is_w ? Cfg::kTileW : Cfg::kTileX);
                if (is_w) {
                    if (kb0 + kb != p.test_skip_kb) tma_load_2d(smem_u32(st), &tmW, full(s), (kb0 + kb) * 128, w0);
                } else tma_load_2d(smem_u32(st + x_high(kb)), &tmX, full(s), (kb0 + kb) * 128, x0);
            }
        } else if (lane == 0 && warp == 1) {
            bool ok = true;
            const uint32_t hi = kmajor_desc_hi<128>(), wide = idesc_tf32() | idesc_extents(128, 2 * BN), narrow = idesc_tf32() | idesc_extents(128, BN);
            for (int kb = 0; kb < blocks; ++kb) {
                const int s = kb % STAGES, c = kb / Cfg::kChain, in = kb % Cfg::kChain;
                if (in == 0 && !mbar_wait(cempty(c & 1), (uint32_t)(c >> 1) & 1u, abort_flag, p.status, 62, 0, p.wait_limit_ns)) {
                    ok = false;
                    break;
                }
                if (!mbar_wait(ready(s), (uint32_t)(kb / STAGES) & 1u, abort_flag, p.status, 63, 0, p.wait_limit_ns)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t both = kmajor_desc_lo(smem_u32(smem + s * Cfg::kStage + Cfg::kTileW)), xh = kmajor_desc_lo(smem_u32(smem + s * Cfg::kStage + x_high(kb)));
                const uint32_t wh = tmem + (uint32_t)(Cfg::kTmemW + (kb & 1) * 64), wl = wh + 32u;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    umma_tf32(tmem + (uint32_t)((c & 1) * BN), wh + 8u * k, both + 2u * k, hi, wide, 1u);
                    umma_tf32(tmem + (uint32_t)BN, wl + 8u * k, xh + 2u * k, hi, narrow, 1u);
                }
                umma_commit(empty(s));
                if (in == Cfg::kChain - 1 || kb == blocks - 1) umma_commit(cfull(c & 1));
            }
            if (ok) umma_commit(done);
        }
        __syncwarp();
    } else {
        // Warps 4-19: one of four per 32 TMEM lanes (rows of w), and up to four for the columns (rows of x), at least sixteen columns each.
        const int e = warp - 4, quarter = (warp & 3) * 32, f = quarter + lane, part = e >> 2;
        constexpr int kParts = BN >= 64 ? 4 : BN / 16, kCols = BN / kParts;
        const bool mine = part < kParts;
        const uint32_t column0 = (uint32_t)(part * kCols), lanes = tmem + ((uint32_t)quarter << 16) + column0;
        float acc[kCols] = {};
        got = true;
        // Adds columns of TMEM: a chain's, or subtracts the small products', which are kLowScale times as large -- these only from sums that are finite: next to an
        // infinity they are NaN (infinity times l = 0).
        auto add = [&](uint32_t at, bool small) {
#pragma unroll
            for (int c = 0; c < kCols / 16; ++c) {
                uint32_t r[16];
                tmem_ld_32x32b_x16(at + (uint32_t)(c * 16), r);
                tmem_ld_wait16(r);
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (!small || fabsf(acc[c * 16 + j]) < INFINITY) acc[c * 16 + j] += __uint_as_float(r[j]) * (small ? -1.f / kLowScale : 1.f);
            }
        };
        // The accumulators start from zeros that are written: an instruction adds to those of a chain and of the small products together.
        auto clear = [&](uint32_t at) {
            const uint32_t z[16] = {};
#pragma unroll
            for (int c = 0; c < kCols / 16; ++c) tmem_st_32x32b_x16(at + (uint32_t)(c * 16), z);
        };
        if (mine) {
            clear(lanes);
            clear(lanes + (uint32_t)BN);
            clear(lanes + 2u * BN);
            tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(cempty(0));
            mbar_arrive(cempty(1));
        }
        auto drain = [&](int c) {  // chain c into the registers; false: gave up
            if (!__all_sync(0xffffffffu, mbar_wait(cfull(c & 1), (uint32_t)(c >> 1) & 1u, abort_flag, p.status, 64, 32, p.wait_limit_ns))) return false;
            tc_fence_after();
            if (mine) {
                add(lanes + (uint32_t)((c & 1) * 2 * BN), false);
                clear(lanes + (uint32_t)((c & 1) * 2 * BN));
                tmem_st_wait();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(cempty(c & 1));
            return true;
        };
        // The warps split in two groups, which take the K blocks by turns: eight warps a block, each 32 rows of w by half of their columns.
        const int group = part & 1, half = part >> 1, tid = half * 128 + f;
        int drained = 0;
        for (int kb = group; kb < blocks && got; kb += 2) {
            const int s = kb % STAGES;
            // Half a chain on, the one before has been multiplied.
            if (kb % Cfg::kChain >= Cfg::kChain / 2 && kb % Cfg::kChain < Cfg::kChain / 2 + 2 && kb >= Cfg::kChain && !(got = drain(drained++))) break;
            got = __all_sync(0xffffffffu, mbar_wait(full(s), (uint32_t)(kb / STAGES) & 1u, abort_flag, p.status, 65, 0, p.wait_limit_ns));
            if (!got) break;
            // w: row f, sixteen of the block's 32 columns, into tensor memory; TMA has swizzled the row's pieces
            const uint4* raw_w = reinterpret_cast<const uint4*>(smem + s * Cfg::kStage) + f * 8;
            uint32_t wh[16], wl[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) split_tf32(raw_w[(4 * half + j) ^ (f & 7)], wh + 4 * j, wl + 4 * j);
            uint4* raw = reinterpret_cast<uint4*>(smem + s * Cfg::kStage + x_high(kb));
            uint4* low = reinterpret_cast<uint4*>(smem + s * Cfg::kStage + x_low(kb));
#pragma unroll
            for (int j = 0; j < (BN * 8 + 255) / 256; ++j) {
                const int i = tid + j * 256;
                if (BN * 8 % 256 == 0 || i < BN * 8) {
                    uint32_t h[4], l[4];
                    split_tf32(raw[i], h, l);
                    raw[i] = make_uint4(h[0], h[1], h[2], h[3]);
                    low[i] = make_uint4(l[0], l[1], l[2], l[3]);
                }
            }
            if (kb >= 2) {  // the block before the last in its place has been multiplied
                got = __all_sync(0xffffffffu, mbar_wait(empty((kb - 2) % STAGES), (uint32_t)((kb - 2) / STAGES) & 1u, abort_flag, p.status, 67, 0, p.wait_limit_ns));
                if (!got) break;
            }
            tc_fence_after();
            const uint32_t to = tmem + ((uint32_t)quarter << 16) + (uint32_t)(Cfg::kTmemW + (kb & 1) * 64 + half * 16);
            tmem_st_32x32b_x16(to, wh);
            tmem_st_32x32b_x16(to + 32u, wl);
            tmem_st_wait();
            tc_fence_before();
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(ready(s));
        }
        while (got && drained < chains) got = drain(drained++);
        if (got) got = __all_sync(0xffffffffu, mbar_wait(done, 0, abort_flag, p.status, 66, 32, p.wait_limit_ns));
        tc_fence_after();
        // Every stage has been read; the warps write the sums together or not at all.
        got = bar_all(1, 512, got);
        if (got && mine) {
            add(lanes + (uint32_t)BN, true);
#pragma unroll
            for (int c = 0; c < kCols; ++c) sums[((int)column0 + c) * 128 + f] = acc[c];
        }
    }
    tc_fence_before();
    if (split > 1) cluster_sync_all();
    else __syncthreads();
    if (got) tile_epilogue<float, BN, 16>(p, sums, x0, w0, rank, split, warp - 4, lane);
    __syncthreads();
    if (*abort_flag) {
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
        __syncthreads();
    }
    if (split > 1) cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, Cfg::kTmemCols);
    }
}

}  // namespace lin
}  // namespace chxq
