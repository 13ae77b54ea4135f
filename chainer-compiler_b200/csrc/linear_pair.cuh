// Float matrix product on CTA pairs: 256 rows of x times 256 rows of w per pair with tcgen05.mma.cta_group::2, persistent over the blocks.
//
// Why pairs: with 256 x 256 blocks split over two SMs each SM stages 128 rows of x and HALF of the 256 rows of w, 64 operand bytes per tensor-pipe
// clock where a lone 128 x 128 tile reads 128, all that the shared memory delivers.
//
// A CTA (352 threads): warp 0 loads x, warp 1 owns the TMEM and (first CTA of the pair) issues the MMAs, warp 2 loads w, warps 3-10 run the
// epilogue.  Accumulators are double-buffered in TMEM, so the epilogue of a block runs under the main loop of the next.  The epilogue warps form two
// groups of four (one warp per 32 TMEM lanes); a group takes every other 64 columns of the block, builds them as one swizzled
// [128 rows][128 bytes] tile in shared memory and sends it with one TMA store (rows of y on 16-byte boundaries) or copies it out row by row.  The
// residual comes through TMA into that tile, the first 64 columns' under the main loop, the next ones' from the L2, where they are prefetched to.
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
    static constexpr int kNumBars = 2 * kPairStages + 6;
    static constexpr int kSmem = 1024 + kBars + kNumBars * 8 + 16;
    static_assert(kSmem <= 227 * 1024, "shared memory over the per-CTA limit");
};

struct PairArgs {
    TcArgs t;
    int m_blocks, o_blocks;  // blocks of 256 rows of x and of w
    int tma_out;             // the output leaves through tmY
    int tma_res;             // the residual comes through tmR
};

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
linear_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmY,
                   const __grid_constant__ CUtensorMap tmR, const PairArgs a) {
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
    auto rfull = [&](int g) { return bar0 + 8u * (2 * kStages + 4 + g); };  // residual tile of an epilogue group
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
            mbar_init(rfull(b), 1);
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
                    } else if (kb != p.test_skip_kb) {
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
        uint32_t rphase = 0;
        // (the issuer) 64 columns of the residual into the group's tile, once the store before has read it
        auto fetch_residual = [&](int col, int m0) {
            tma_store_wait_read<0>();
            mbar_expect_tx(rfull(group), Cfg::kTile);
            tma_load_2d(smem_u32(out), &tmR, rfull(group), col * (int)sizeof(T), m0);
        };
        int it = 0;
        bool going = true;
        for (int item = first; item < items && going; item += pairs, ++it) {
            const int buf = it & 1;
            int mb, ob;
            coords(item, mb, ob);
            const int m0 = mb * 256 + (int)rank * 128, o0 = ob * 256;
            if (a.tma_res && issuer) {
                fetch_residual(o0 + group * 64, m0);
                if (o0 + (group + 2) * 64 < p.O)
                    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(&tmR)), "r"((o0 + (group + 2) * 64) * (int)sizeof(T)),
                             "r"(m0)
                             : "memory");
            }
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
                if (a.tma_res) {
                    if (b != group && issuer) fetch_residual(col, m0);
                    const bool here = mbar_wait(rfull(group), rphase, abort_flag, p.status, 55, 32, p.wait_limit_ns);
                    rphase ^= 1u;
                    going = bar_all(1, 256, here);  // the eight warps go on or give up together, as above
                    if (!going) break;
                } else {
                    if (issuer) tma_store_wait_read<0>();
                    bar_sync(2 + group, 128);  // the staged tile is free
                    if (p.e.residual) {
                        // rows off 16-byte boundaries: a warp copies the 32 rows that its own lanes read below and write their outputs to, 64 values each
                        // (no other warp touches them before the group's barrier)
                        const int r0 = quarter * 32, n = min(32, p.M - m0 - r0);
                        const T* src = static_cast<const T*>(p.e.residual) + (int64_t)(m0 + r0) * p.e.ldr + col + lane;
                        const bool in0 = col + lane < p.O, in1 = col + lane + 32 < p.O;
#pragma unroll 8
                        for (int i = 0; i < n; ++i, src += p.e.ldr) {
                            const T v0 = in0 ? src[0] : from_f32<T>(0.f), v1 = in1 ? src[32] : from_f32<T>(0.f);
                            *reinterpret_cast<T*>(out + staged_offset<128>(r0 + i, lane >> 3) + (lane & 7) * 2) = v0;
                            *reinterpret_cast<T*>(out + staged_offset<128>(r0 + i, (lane >> 3) + 4) + (lane & 7) * 2) = v1;
                        }
                        __syncwarp();
                    }
                }
                uint32_t r[2][32];
                tmem_ld_32x32b_x32(taddr + (uint32_t)(b * 64), r[0]);
                tmem_ld_32x32b_x32(taddr + (uint32_t)(b * 64 + 32), r[1]);
                tmem_ld_wait32(r[0]);
                tmem_ld_wait32(r[1]);
                const bool before = p.e.residual_first, res = p.e.residual != nullptr;
                with_activation(p.e.activation, [&](auto act) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        T* cell = reinterpret_cast<T*>(out + staged_offset<128>(row, j));
                        Pack<T, 8> o;
                        if (res) o.load(cell);  // (rows past M hold what was there: their outputs are not stored)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int c = 8 * j + 2 * i;
                            f32x2 z = add2(make_x2(__uint_as_float(r[c / 32][c % 32]), __uint_as_float(r[c / 32][c % 32 + 1])),
                                           *reinterpret_cast<const f32x2*>(s_bias + b * 64 + c));
                            if (res && before) z = add2(z, o.pair(i));
                            z = activate_fast<decltype(act)::value>(z);
                            if (res && !before) z = add2(z, o.pair(i));
                            o.set_pair(i, z);
                        }
                        o.store(cell);
                    }
                });
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
                    const int r0 = (e & 3) * 32, n = min(32, p.M - m0 - r0);
                    T* dst = static_cast<T*>(p.e.y) + (int64_t)(m0 + r0) * p.e.ldy + col + lane;
                    const bool in0 = col + lane < p.O, in1 = col + lane + 32 < p.O;
#pragma unroll 8
                    for (int i = 0; i < n; ++i, dst += p.e.ldy) {
                        const T v0 = *reinterpret_cast<const T*>(out + staged_offset<128>(r0 + i, lane >> 3) + (lane & 7) * 2);
                        const T v1 = *reinterpret_cast<const T*>(out + staged_offset<128>(r0 + i, (lane >> 3) + 4) + (lane & 7) * 2);
                        if (in0) dst[0] = v0;
                        if (in1) dst[32] = v1;
                    }
                    if (a.tma_res) bar_sync(2 + group, 128);  // the next residual is fetched into the tile that was copied from
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
