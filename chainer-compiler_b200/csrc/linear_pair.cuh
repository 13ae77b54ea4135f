// Float matrix product on CTA pairs: 256 rows of x times 256 rows of w per pair with tcgen05.mma.cta_group::2, persistent over the blocks.
//
// Why pairs: with 256 x 256 blocks split over two SMs each SM stages 128 rows of x and HALF of the 256 rows of w, 64 operand bytes per tensor-pipe
// clock where a lone 128 x 128 tile reads 128, all that the shared memory delivers.
//
// A CTA (352 threads): warp 0 loads x, warp 1 owns the TMEM and (first CTA of the pair) issues the MMAs, warp 2 loads w, warps 3-10 run the
// epilogue.  Accumulators are double-buffered in TMEM, so the epilogue of a block runs under the main loop of the next.  The epilogue warps form two
// groups of four (one warp per 32 TMEM lanes); a group takes every other 64 columns of the block, builds them as one swizzled
// [128 rows][128 bytes] tile in shared memory and sends it with one TMA store (rows of y on 16-byte boundaries) or copies it out row by row.
// What crosses the pair is as in tc_kernel3.cuh; no load is multicast.  Waits are bounded as there.
#pragma once

#include "linear_tc.cuh"

namespace chxq {
namespace lin {

constexpr int kPairStages = 6;
constexpr int kPairThreads = 11 * 32;
struct PairConfig {
    static constexpr int kTile = 128 * 128, kStage = 2 * kTile;  // 128 rows of x and 128 rows of w, 128 bytes each
    static constexpr int kOut = kPairStages * kStage;            // two staged output tiles, one per epilogue group
    static constexpr int kBias = kOut + 2 * kTile;               // [256] floats
    static constexpr int kBars = kBias + 256 * 4;
    static constexpr int kNumBars = 2 * kPairStages + 4;
    static constexpr int kSmem = 1024 + kBars + kNumBars * 8 + 16;
    static_assert(kSmem <= 227 * 1024, "shared memory over the per-CTA limit");
};

struct PairArgs {
    TcArgs t;
    int m_blocks, o_blocks;  // blocks of 256 rows of x and of w
    int tma_out;             // the output leaves through tmY
};

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
linear_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmY, const PairArgs a) {
    using Cfg = PairConfig;
    const TcArgs& p = a.t;
    constexpr int kStages = kPairStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // the same offset in both CTAs of a pair
    float* s_bias = reinterpret_cast<float*>(smem + Cfg::kBias);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kBars);
    uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(bars + Cfg::kNumBars);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (kStages + s); };
    auto tfull = [&](int b) { return bar0 + 8u * (2 * kStages + b); };
    auto tempty = [&](int b) { return bar0 + 8u * (2 * kStages + 2 + b); };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full(s), 1);   // first CTA only: one expect for both CTAs' bytes
            mbar_init(empty(s), 1);  // one commit arrival per CTA
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(tfull(b), 1);
            mbar_init(tempty(b), 16);  // first CTA only: eight epilogue warps of each CTA
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(tmem_ptr), 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = *tmem_ptr;
    pdl_launch_dependents();
    pdl_dependency_wait();

    const int items = a.m_blocks * a.o_blocks, pairs = (int)(gridDim.x >> 1), first = (int)(blockIdx.x >> 1);
    // Eight blocks of w at a time, all blocks of x of those before the next eight: the pairs at work then share few blocks of either operand.
    constexpr int kGroup = 8;
    auto coords = [&](int item, int& mb, int& ob) {
        const int per = kGroup * a.m_blocks, g = item / per, width = min(kGroup, a.o_blocks - g * kGroup), in = item - g * per;
        mb = in / width;
        ob = g * kGroup + in % width;
    };

    if (warp == 0 || warp == 2) {
        if (lane == 0) {
            const bool is_x = warp == 0;
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            const uint32_t lead_full = map_to_cta(full(0), 0);
            for (int item = first; item < items && ok; item += pairs) {
                int mb, ob;
                coords(item, mb, ob);
                const int row = (is_x ? mb : ob) * 256 + (int)rank * 128;
                for (int kb = 0; kb < p.k_blocks; ++kb) {
                    if (!mbar_wait(empty(stage), phase ^ 1u, abort_flag, p.status, 51, 0, p.wait_limit_ns)) {
                        ok = false;
                        break;
                    }
                    const uint32_t fb = lead_full + 8u * stage, dst = smem_u32(smem + stage * Cfg::kStage);
                    if (is_x) {
                        if (rank == 0) mbar_expect_tx(full(stage), 2 * Cfg::kStage);
                        tma_load_2d_pair(dst, &tmX, fb, kb * 128, row);
                    } else {
                        tma_load_2d_pair(dst + Cfg::kTile, &tmW, fb, kb * 128, row);
                    }
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            int stage = 0, it = 0;
            uint32_t phase = 0;
            bool ok = true;
            const uint32_t hi = kmajor_desc_hi<128>(), lo0 = kmajor_desc_lo(smem_u32(smem)), idesc = p.idesc | idesc_extents(256, 256);
            for (int item = first; item < items && ok; item += pairs, ++it) {
                const int buf = it & 1;
                if (!mbar_wait(tempty(buf), ((uint32_t)(it >> 1) & 1u) ^ 1u, abort_flag, p.status, 52, 0, p.wait_limit_ns)) break;
                tc_fence_after();
                const uint32_t d = tmem + (uint32_t)(buf * 256);
                for (int kb = 0; kb < p.k_blocks; ++kb) {
                    if (!mbar_wait(full(stage), phase, abort_flag, p.status, 53, 0, p.wait_limit_ns)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t lo = lo0 + (uint32_t)(stage * (Cfg::kStage >> 4));
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_f16<true>(d, lo + 2u * k, lo + (Cfg::kTile >> 4) + 2u * k, hi, idesc, kb > 0 || k > 0 ? 1u : 0u);
                    umma_commit_pair(empty(stage), 3);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (ok) umma_commit_pair(tfull(buf), 3);
            }
        }
    } else {
        const int e = warp - 3, group = e >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const int tid = (int)threadIdx.x - 96;  // 0 .. 255 over the epilogue
        const bool issuer = (e & 3) == 0 && lane == 0;
        uint8_t* out = smem + Cfg::kOut + group * Cfg::kTile;
        const uint32_t lead_tempty = map_to_cta(tempty(0), 0);
        int it = 0;
        for (int item = first; item < items; item += pairs, ++it) {
            const int buf = it & 1;
            int mb, ob;
            coords(item, mb, ob);
            const int m0 = mb * 256 + (int)rank * 128, o0 = ob * 256;
            const int64_t m = m0 + row;
            bar_sync(1, 256);  // the last block's bias has been read
            s_bias[tid] = p.e.bias && o0 + tid < p.O ? load_param({p.e.bias, p.e.bias_dtype}, o0 + tid) : 0.f;
            // the bias is in place, and the eight warps go on or give up together: a warp that left alone would leave the others at a barrier
            const bool got = mbar_wait(tfull(buf), (uint32_t)(it >> 1) & 1u, abort_flag, p.status, 54, 32, p.wait_limit_ns);
            if (!bar_all(1, 256, got)) break;
            tc_fence_after();
            const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * 256);
#pragma unroll 1
            for (int b = group; b < 4; b += 2) {
                const int col = o0 + b * 64;
                if (issuer) tma_store_wait_read<0>();
                bar_sync(2 + group, 128);  // the staged tile is free
#pragma unroll 1
                for (int h = 0; h < 4; ++h) {
                    uint32_t r[16];
                    tmem_ld_32x32b_x16(taddr + (uint32_t)(b * 64 + h * 16), r);
                    float res[16] = {}, v[16], bs[16];
                    const int c0 = col + h * 16;
                    if (p.e.residual && m < p.M) {
                        const T* src = static_cast<const T*>(p.e.residual) + m * p.e.ldr + c0;
                        if (p.vec && c0 + 16 <= p.O) {
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const uint4 q = reinterpret_cast<const uint4*>(src)[j];
                                const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const float2 f = unpack16<T>(w[i]);
                                    res[8 * j + 2 * i] = f.x;
                                    res[8 * j + 2 * i + 1] = f.y;
                                }
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                if (c0 + j < p.O) res[j] = to_f32(src[j]);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) *reinterpret_cast<float4*>(bs + 4 * j) = *reinterpret_cast<const float4*>(s_bias + b * 64 + h * 16 + 4 * j);
                    tmem_ld_wait16(r);
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]) + bs[j];
                    epilogue_apply<16, true>(p.e, v, res);
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        *reinterpret_cast<uint4*>(out + staged_offset<128>(row, 2 * h + j)) =
                                make_uint4(pack16<T>(v[8 * j], v[8 * j + 1]), pack16<T>(v[8 * j + 2], v[8 * j + 3]), pack16<T>(v[8 * j + 4], v[8 * j + 5]),
                                           pack16<T>(v[8 * j + 6], v[8 * j + 7]));
                }
                if (b + 2 >= 4) {  // this warp's last read of the accumulators
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(lead_tempty + 8u * buf);
                }
                fence_async_smem();
                bar_sync(2 + group, 128);
                if (a.tma_out) {
                    if (issuer && col < p.O && m0 < p.M) {
                        tma_store_2d(&tmY, smem_u32(out), col * (int)sizeof(T), m0);
                        tma_store_commit();
                    }
                } else {
                    // rows off 16-byte boundaries: a warp copies its 32 rows, 64 values each
                    for (int i = 0; i < 32; ++i) {
                        const int rr = (e & 3) * 32 + i;
                        if (m0 + rr >= p.M) break;
                        T* dst = static_cast<T*>(p.e.y) + (int64_t)(m0 + rr) * p.e.ldy + col;
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int c = lane + 32 * j;
                            if (col + c < p.O) dst[c] = *reinterpret_cast<const T*>(out + staged_offset<128>(rr, c >> 3) + (c & 7) * 2);
                        }
                    }
                }
            }
        }
        if (issuer) tma_store_wait_all();
    }

    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
        __syncthreads();
    }
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

}  // namespace lin
}  // namespace chxq
