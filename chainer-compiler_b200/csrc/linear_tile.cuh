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
            if (is_w) tma_load_2d(smem_u32(st), &tmW, full(s), kb * 128, w0);
            else tma_load_2d(smem_u32(st + Cfg::kTileW), &tmX, full(s), kb * 128, x0);
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
    if (got) {
        const int cols = (BN + split - 1) / split;  // rows of x of this CTA
        const bool vec = p.vec != 0;
        auto feature = [&](int j) { return vec ? 4 * lane + j : lane + 32 * j; };
        float bias[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) bias[j] = p.e.bias && w0 + feature(j) < p.O ? load_param({p.e.bias, p.e.bias_dtype}, w0 + feature(j)) : 0.f;
        const uint32_t sums0 = smem_u32(sums);
        for (int c = rank * cols + warp; c < (rank + 1) * cols && c < BN && x0 + c < p.M; c += 8) {
            const int64_t m = x0 + c;
            float v[4] = {}, res[4] = {};
            if (vec) {
                if (w0 + 4 * lane >= p.O) continue;
                for (int s = 0; s < split; ++s) {
                    float4 q;
                    const uint32_t at = sums0 + (uint32_t)(c * 128 + 4 * lane) * 4u;
                    if (split > 1)
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(q.x), "=f"(q.y), "=f"(q.z), "=f"(q.w) : "r"(map_to_cta(at, s)));
                    else
                        q = *reinterpret_cast<const float4*>(sums + c * 128 + 4 * lane);
                    v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
                }
                if (p.e.residual) {
                    const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const T*>(p.e.residual) + m * p.e.ldr + w0 + 4 * lane);
                    const float2 lo = unpack16<T>(q.x), hi = unpack16<T>(q.y);
                    res[0] = lo.x; res[1] = lo.y; res[2] = hi.x; res[3] = hi.y;
                }
                epilogue_apply<4, true>(p.e, v, bias, res);
                *reinterpret_cast<uint2*>(static_cast<T*>(p.e.y) + m * p.e.ldy + w0 + 4 * lane) = make_uint2(pack16<T>(v[0], v[1]), pack16<T>(v[2], v[3]));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int f = feature(j);
                    for (int s = 0; s < split; ++s) {
                        float q;
                        if (split > 1) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(q) : "r"(map_to_cta(sums0 + (uint32_t)(c * 128 + f) * 4u, s)));
                        else q = sums[c * 128 + f];
                        v[j] += q;
                    }
                    if (p.e.residual && w0 + f < p.O) res[j] = to_f32(static_cast<const T*>(p.e.residual)[m * p.e.ldr + w0 + f]);
                }
                epilogue_apply<4, true>(p.e, v, bias, res);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (w0 + feature(j) < p.O) static_cast<T*>(p.e.y)[m * p.e.ldy + w0 + feature(j)] = from_f32<T>(v[j]);
            }
        }
    }
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

}  // namespace lin
}  // namespace chxq
