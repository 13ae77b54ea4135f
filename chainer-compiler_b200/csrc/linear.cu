// Linear with bias, activation and residual in its epilogue: y = act(x w^T + b) + r, or act(x w^T + b + r); bf16, fp16 and fp32 operands,
// sums in 32 bits, one rounding at the end.
//
// Three kernels: CTA pairs with 256 x 256 blocks (linear_pair.cuh) for large 16-bit products, clusters that share a tile's K (linear_tile.cuh) for
// few rows of x, for products in between and for fp32, and threads side by side along K for few rows or outputs (linear_rows.cuh).
#include <algorithm>
#include <atomic>

#include "epilogue_float.cuh"
#include "float_ops.cuh"
#include "linear_pair.cuh"
#include "linear_rows.cuh"
#include "linear_tile.cuh"

namespace chxq {
namespace {

// Products without a K: the epilogue of sums of zero.
template <typename T>
__global__ void __launch_bounds__(256) linear_empty_kernel(int64_t M, int64_t O, LinearEpilogue e) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < M * O; i += (int64_t)gridDim.x * 256) epilogue_store<T>(e, i / O, i % O, 0.f);
}

// ---- the tensor-core kernels ------------------------------------------------------------------------------------------------

// Bytes of a row and rows of an operand for one launch of the tensor-core kernels, half of what TMA's 32-bit coordinates count: a tile past 2^31 is an
// illegal instruction.
constexpr int64_t kMostCoordinate = 1ll << 30;

// TMA reads rows that start on 16-byte boundaries.  Operands whose rows do not are copied into such rows in front of the product.
bool rows16(const void* p, int64_t ld, int64_t rows, int size) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (rows == 1 || ld * size % 16 == 0);
}
// The rows of such a copy start on 128-byte lines: of others a row of a tile takes two ([2656, 5781] x [416, 5781]^T fp16: 43.7 us, and 56.7 with rows on
// 16-byte boundaries).
int64_t line_pitch(int64_t K, int size) {
    const int per = 128 / size;
    return (K + per - 1) / per * per;
}
size_t align256(size_t v) {
    return (v + 255) / 256 * 256;
}

struct CopyJob {
    const void* src;
    int64_t ld, rows;
    void* dst;
};

// Rows of K values into rows of `pitch`, whole 16-byte pieces: a thread gathers one piece.  (The last one's values past K are never read: the tensor map ends
// at K.)  U: uint16_t or uint32_t.
template <typename U>
__global__ void __launch_bounds__(256) align_rows_kernel(CopyJob a, CopyJob b, int64_t K, int64_t pitch) {
    constexpr int kPer = 16 / (int)sizeof(U);
    pdl_launch_dependents();
    pdl_dependency_wait();
    const int64_t per_row = pitch / kPer, total = (a.rows + b.rows) * per_row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        int64_t r = i / per_row;
        const int64_t k = (i - r * per_row) * kPer;
        const bool first = r < a.rows;
        if (!first) r -= a.rows;
        const U* s = (first ? static_cast<const U*>(a.src) + r * a.ld : static_cast<const U*>(b.src) + r * b.ld) + k;
        U v[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[j] = k + j < K ? s[j] : (U)0;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = sizeof(U) == 4 ? (uint32_t)v[j % kPer] : (uint32_t)v[2 * j % kPer] | (uint32_t)v[(2 * j + 1) % kPer] << 16;
        *reinterpret_cast<uint4*>((first ? static_cast<U*>(a.dst) : static_cast<U*>(b.dst)) + r * pitch + k) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// What is known of a kernel on each device: whether its dynamic shared memory is set, and how many of its clusters of 1 .. 8 CTAs are resident at once
// (0: not asked yet).
struct KernelState {
    std::atomic<bool> smem_set[64];
    std::atomic<int> slots[64][9];
};

int current_device(int* dev) {
    CHXQ_CUDA(cudaGetDevice(dev));
    if (*dev < 0 || *dev >= 64) return set_error(CHXQ_ERR_UNSUPPORTED, "Linear: device number %d", *dev);
    return CHXQ_OK;
}

template <typename F>
int set_smem(F* kernel, int bytes, KernelState& st, int dev) {
    if (st.smem_set[dev].load(std::memory_order_acquire)) return CHXQ_OK;
    CHXQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    st.smem_set[dev].store(true, std::memory_order_release);
    return CHXQ_OK;
}

template <typename F>
int cluster_slots(F* kernel, int cluster, int threads, int smem, KernelState& st, int dev) {
    int n = st.slots[dev][cluster].load(std::memory_order_acquire);
    if (n > 0) return n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(cluster * tc::sm_count()));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cluster; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        n = std::max(1, 100 / cluster);
    }
    st.slots[dev][cluster].store(n, std::memory_order_release);
    return n;
}

struct Operands {  // as TMA reads them
    const void* x;
    int64_t ldx;
    const void* w;
    int64_t ldw;
};

// kernel: one of linear_tile.cuh's, for bn rows of x, with `split` CTAs for a tile.
template <typename F>
int launch_tile(F* kernel, int bn, int split, int threads, int smem, KernelState& st, int dev, const chxq_linear_params& q, const Operands& op, const lin::TcArgs& args,
                int size, cudaStream_t s) {
    int rc = set_smem(kernel, smem, st, dev);
    if (rc != CHXQ_OK) return rc;
    alignas(64) CUtensorMap tmW, tmX;
    if ((rc = tc::encode_rows_map(&tmW, op.w, q.K * size, q.O, op.ldw * size, 128)) != CHXQ_OK) return rc;
    if ((rc = tc::encode_rows_map(&tmX, op.x, q.K * size, q.M, op.ldx * size, bn)) != CHXQ_OK) return rc;
    const int64_t x_tiles = (q.M + bn - 1) / bn, tiles = x_tiles * ((q.O + 127) / 128);
    if (tiles * split >= (1ll << 31)) return set_error(CHXQ_ERR_UNSUPPORTED, "Linear: too many tiles");
    CHXQ_CUDA(launch_pdl_cluster(split, kernel, dim3((unsigned)(tiles * split)), threads, smem, s, tmW, tmX, args, split, (int)x_tiles));
    count_launch(1);
    return CHXQ_OK;
}

template <typename T, int BN, int STAGES>
int launch_tile_16(const chxq_linear_params& q, const Operands& op, const lin::TcArgs& args, cudaStream_t s) {
    static KernelState state = {};
    int dev = 0;
    const int rc = current_device(&dev);
    if (rc != CHXQ_OK) return rc;
    // An SM holds two CTAs: the sharing CTAs are doubled as long as there are no more of them than that and each has a K block.  One B200, in us by
    // CTAs per tile: [1, 8192] x [8192, 8192]^T (64 tiles) 37.8, 28.5 with two, 25.2 with four, 30.7 with eight; [32, 4096] x [4096, 4096]^T (32 tiles)
    // 21.0, 13.6, 9.8, 9.2.
    const int64_t tiles = ((q.M + BN - 1) / BN) * ((q.O + 127) / 128);
    int split = 1;
    while (split < 8 && tiles * split * 2 <= 2 * tc::sm_count() && split * 2 <= args.k_blocks) split *= 2;
    return launch_tile(lin::linear_tile_kernel<T, BN, STAGES>, BN, split, 256, lin::TileConfig<BN, STAGES>::kSmem, state, dev, q, op, args, 2, s);
}

// fp32 kernels fill an SM.
template <int BN, int STAGES>
struct TileF32 {
    using Cfg = lin::TileF32Config<BN, STAGES>;
    int dev, split = 1, rc;
    int64_t cost = INT64_MAX;

    static KernelState& state() {
        static KernelState st = {};
        return st;
    }
    // How many CTAs share a tile: what is estimated to take the least time, in 0.01 us from one B200: 85 for a K block of a tile of 128 rows of x and 600
    // for a wave of clusters beside that (launch, first loads, joining the sums), 72 and 400 up to 64 rows.  Clusters that do not all fit at once are
    // worth less than smaller ones that do: [256, 2048] x [1000, 2048]^T has 16 tiles of 128 rows, of which the GPU holds 15 as clusters of eight, and
    // takes 30 us that way and 18 as clusters of four.
    TileF32(const chxq_linear_params& q, const lin::TcArgs& args, int device) : dev(device) {
        rc = set_smem(lin::linear_tile_f32_kernel<BN, STAGES>, Cfg::kSmem, state(), dev);  // (the answers below ask for it)
        if (rc != CHXQ_OK) return;
        const int64_t tiles = ((q.M + BN - 1) / BN) * ((q.O + 127) / 128), block = BN == 128 ? 85 : 72, wave = BN == 128 ? 600 : 400;
        for (int c = 1; c <= 8 && c <= args.k_blocks; ++c) {
            const int64_t slots = cluster_slots(lin::linear_tile_f32_kernel<BN, STAGES>, c, 640, Cfg::kSmem, state(), dev);
            const int64_t of = (tiles + slots - 1) / slots * ((args.k_blocks + c - 1) / c * block + wave);
            if (of < cost) {
                cost = of;
                split = c;
            }
        }
    }
    int launch(const chxq_linear_params& q, const Operands& op, const lin::TcArgs& args, cudaStream_t s) const {
        if (rc != CHXQ_OK) return rc;
        return launch_tile(lin::linear_tile_f32_kernel<BN, STAGES>, BN, split, 640, Cfg::kSmem, state(), dev, q, op, args, 4, s);
    }
};

template <typename T>
int launch_pair(const chxq_linear_params& q, const Operands& op, const lin::TcArgs& args, cudaStream_t s) {
    using Cfg = lin::PairConfig;
    static KernelState state = {};
    auto* kernel = lin::linear_pair_kernel<T>;
    int dev = 0, rc = current_device(&dev);
    if (rc != CHXQ_OK || (rc = set_smem(kernel, Cfg::kSmem, state, dev)) != CHXQ_OK) return rc;
    lin::PairArgs a;
    a.t = args;
    const int64_t mb = (q.M + 255) / 256, ob = (q.O + 255) / 256;
    if (mb * ob >= (1ll << 31)) return set_error(CHXQ_ERR_UNSUPPORTED, "Linear: too many blocks");
    a.m_blocks = (int)mb;
    a.o_blocks = (int)ob;
    a.tma_out = rows16(q.y, q.ldy, q.M, 2);
    a.tma_res = q.residual && rows16(q.residual, q.ldr, q.M, 2);
    alignas(64) CUtensorMap tmX, tmW, tmY, tmR;
    if ((rc = tc::encode_rows_map(&tmX, op.x, q.K * 2, q.M, op.ldx * 2, 128)) != CHXQ_OK) return rc;
    if ((rc = tc::encode_rows_map(&tmW, op.w, q.K * 2, q.O, op.ldw * 2, 128)) != CHXQ_OK) return rc;
    tmY = tmR = tmX;  // not used where the output is copied, and where there is no such residual
    if (a.tma_out && (rc = tc::encode_rows_map(&tmY, q.y, q.O * 2, q.M, q.ldy * 2, 128)) != CHXQ_OK) return rc;
    if (a.tma_res && (rc = tc::encode_rows_map(&tmR, q.residual, q.O * 2, q.M, q.ldr * 2, 128)) != CHXQ_OK) return rc;
    const int pairs = (int)std::min<int64_t>(mb * ob, tc::sm_count() / 2);
    CHXQ_CUDA(launch_pdl(kernel, dim3((unsigned)(2 * pairs)), lin::kPairThreads, Cfg::kSmem, s, tmX, tmW, tmY, tmR, a));
    count_launch(1);
    return CHXQ_OK;
}

int k_blocks_of(const chxq_linear_params& q) {  // of 128 bytes
    return (int)((q.K * float_size(q.dtype) + 127) / 128);
}

// Pairs or single tiles (16-bit operands), in units of 0.01 us from one B200: a K block of a 256 x 256 block takes a pair 0.27 us and a launch 6 beside
// that; a K block of a 128 x 128 tile takes an SM 0.27 us, too, and 0.3 at least where its CTA is alone.  [512, 4096] x [4096, 4096]^T: 25.3 us in
// pairs, 22.5 in tiles; [1024, 4096] x [4096, 4096]^T: 27.0 and 35.7; [8192, 64] x [1024, 64]^T: 10.1 and 18.8.
bool takes_pairs(const chxq_linear_params& q) {
    if (q.M <= 128) return false;
    const int64_t tiles128 = ((q.M + 127) / 128) * ((q.O + 127) / 128);
    const int64_t sms = tc::sm_count(), blocks = ((q.M + 255) / 256) * ((q.O + 255) / 256), kb = k_blocks_of(q);
    const int64_t pairs = (blocks + sms / 2 - 1) / (sms / 2) * kb * 27 + 600;
    const int64_t share = std::min<int64_t>(8, std::max<int64_t>(1, 2 * sms / tiles128));
    const int64_t tiles = std::max(tiles128 * kb * 27 / sms, (kb + share - 1) / share * 30) + 500 + tiles128 / (2 * sms) * 300;
    return pairs <= tiles;
}

template <typename T>
int launch_tc(const chxq_linear_params& q, const Operands& op, const lin::TcArgs& args, cudaStream_t s) {
    if (takes_pairs(q)) return launch_pair<T>(q, op, args, s);
    const int64_t tiles128 = ((q.M + 127) / 128) * ((q.O + 127) / 128);
    if (q.M <= 16) return launch_tile_16<T, 16, 6>(q, op, args, s);
    if (q.M <= 32) return launch_tile_16<T, 32, 5>(q, op, args, s);
    // Narrow tiles also where wide ones are so few that eight CTAs each do not fill the SMs twice: [256, 2048] x [1000, 2048]^T 9.1 against 10.5 us, [128,
    // 4096] x [4096, 4096]^T 12.2 against 13.7.
    if (q.M <= 64 || tiles128 <= 32) return launch_tile_16<T, 64, 4>(q, op, args, s);
    return launch_tile_16<T, 128, 3>(q, op, args, s);
}

template <>
int launch_tc<float>(const chxq_linear_params& q, const Operands& op, const lin::TcArgs& args, cudaStream_t s) {
    int dev = 0;
    const int rc = current_device(&dev);
    if (rc != CHXQ_OK) return rc;
    if (q.M <= 16) return TileF32<16, 6>(q, args, dev).launch(q, op, args, s);
    if (q.M <= 32) return TileF32<32, 6>(q, args, dev).launch(q, op, args, s);
    const TileF32<64, 6> narrow(q, args, dev);
    if (q.M <= 64) return narrow.launch(q, op, args, s);
    // Few K blocks in few tiles: narrow ones, of which a wave is over sooner.  In us with 64 and 128 rows: [200, 200] x [200, 200]^T 7.7 and 9.8, [777, 555] x
    // [1333, 555]^T 22.2 and 26.5, [600, 600] x [600, 600]^T 13.2 and 12.6, [1000, 1000] x [1000, 1000]^T 27.5 and 20.4, [813, 864] x [2662, 864]^T 51 and 34.
    const TileF32<128, 4> wide(q, args, dev);
    return narrow.cost < wide.cost ? narrow.launch(q, op, args, s) : wide.launch(q, op, args, s);
}

// Few rows or outputs.  No alignment is asked for: rows off 16-byte boundaries are read value by value ([1, 2147] x [2999, 2147]^T fp32: 8 us, and 27 with copies
// in front of tiles).
template <typename T, int MR>
int launch_rows(const chxq_linear_params& q, const LinearEpilogue& e, cudaStream_t s) {
    constexpr int R = 4, VEC = 16 / (int)sizeof(T);
    const bool vec = rows16(q.x, q.ldx, q.M, sizeof(T)) && rows16(q.w, q.ldw, q.O, sizeof(T));
    const int64_t blocks = (q.O + R - 1) / R, pieces = vec ? q.K / VEC : q.K;
    const int threads = (int)std::min<int64_t>(blocks <= tc::sm_count() ? 512 : 256, std::max<int64_t>(32, (pieces + 31) / 32 * 32));
    auto* kernel = vec ? lin::linear_rows_kernel<T, MR, R, VEC, MR <= 2 ? 4 : (MR == 4 ? 2 : 1)> : lin::linear_rows_kernel<T, MR, R, 1, MR <= 2 ? 8 : 4>;
    CHXQ_CUDA(launch_pdl(kernel, dim3((unsigned)blocks, (unsigned)((q.M + MR - 1) / MR)), threads, 0, s, static_cast<const T*>(q.x), q.ldx, static_cast<const T*>(q.w), q.ldw,
                         (int)q.M, (int)q.O, (int)q.K, e));
    count_launch(1);
    return CHXQ_OK;
}

// Which products they take.  Up to eight rows of fp32, and more of any type in blocks of eight where those run in two waves (two are on an SM at once).
// 16-bit tiles read the weights as fast and convert none: they are left what takes longer than the start of a tile, about 2 us + (0.32 + 0.047 M) us per
// 2^20 weights here against 4.6 + 0.305.  Rows off 16-byte boundaries, read value by value here, tiles copy first: up to four rows of x gain by that at all
// sizes but those of many short rows, more of them as long as 2^22 weights for every eight rows are read.  In us here and in tiles, x and w off 16-byte
// boundaries, bf16: [4, 2001] x [2048, 2001]^T 8.7 and 10.5, [4, 4001] x [4096, 4001]^T 25.7 and 21.6, [8, 1001] x [4096, 1001]^T 11.8 and 11.9, [8, 4001] x
// [1000, 4001]^T 9.6 and 11.3, [8, 8001] x [1000, 8001]^T 16.9 and 15.9, [16, 1001] x [1000, 1001]^T 6.3 and 7.3, [16, 4001] x [1000, 4001]^T 17.3 and 11.4,
// [64, 8001] x [64, 8001]^T 9.0 and 11.8, [64, 8001] x [256, 8001]^T 34.4 and 13.3.  On them: [1, 1024] x [4096, 1024]^T bf16 3.8 and 6.2, [8, 1024] x [4096,
// 1024]^T 5.4 and 6.3, [8, 4096] x [4096, 4096]^T 13.4 and 8.3, [64, 2000] x [64, 2000]^T fp16 3.1 and 6.8; fp32: [64, 8192] x [64, 8192]^T 5.4 and 27,
// [411, 2000] x [16, 2000]^T 5.4 and 11.8, [64, 2048] x [250, 2048]^T 10.1 and 12.2.
// And rows of more than 2^30 bytes, whatever their number: TMA counts a row's bytes in 32 signed bits.
bool few_rows(const chxq_linear_params& q) {
    if (q.K * float_size(q.dtype) > kMostCoordinate) return true;
    if (q.M > 8 && (q.O + 3) / 4 * ((q.M + 7) / 8) > 4 * tc::sm_count()) return false;
    if (q.dtype == CHXQ_FLOAT32) return true;
    const int64_t values = q.O * q.K;
    if (rows16(q.x, q.ldx, q.M, 2) && rows16(q.w, q.ldw, q.O, 2)) return values * (1 + 3 * q.M) <= 110000000;
    return q.M <= 4 || values * ((q.M + 7) / 8) <= 1ll << 22;
}

}  // namespace
}  // namespace chxq

using namespace chxq;

static int check_linear(const chxq_linear_params* p) {
    CHXQ_CHECK_ARG(p != nullptr, "Linear: no parameters");
    CHXQ_CHECK_ARG(is_float_type(p->dtype), "Linear: operands must be float32, float16 or bfloat16");
    CHXQ_CHECK_ARG(p->M >= 0 && p->O >= 0 && p->K >= 0 && p->M < (1ll << 31) && p->O < (1ll << 31) && p->K < (1ll << 31), "Linear: bad extents");
    if (p->M == 0 || p->O == 0) return CHXQ_OK;
    CHXQ_CHECK_ARG(p->y && (p->K == 0 || (p->x && p->w)), "Linear: null operand");
    CHXQ_CHECK_ARG((p->M == 1 || p->ldx >= p->K) && (p->O == 1 || p->ldw >= p->K) && (p->M == 1 || p->ldy >= p->O) &&
                           (!p->residual || p->M == 1 || p->ldr >= p->O),
                   "Linear: rows overlap");
    CHXQ_CHECK_ARG(!p->bias || p->bias_dtype == p->dtype || p->bias_dtype == CHXQ_FLOAT32, "Linear: the bias must be float32 or have the operands' type");
    CHXQ_CHECK_ARG(on_values_of(float_size(p->dtype), p->x, p->w, p->residual, p->y) && (!p->bias || on_values_of(float_size(p->bias_dtype), p->bias)),
                   "Linear: an address is no multiple of its values' size");
    CHXQ_CHECK_ARG(p->activation >= CHXQ_ACT_NONE && p->activation <= CHXQ_ACT_TANH, "Linear: unknown activation %d", p->activation);
    return CHXQ_OK;
}

extern "C" size_t chxq_linear_workspace(const chxq_linear_params* p) {
    if (!p || !is_float_type(p->dtype) || p->K <= 0 || p->M <= 0 || p->O <= 0 || few_rows(*p)) return 0;
    const int size = float_size(p->dtype);
    size_t n = 0;
    if (!rows16(p->x, p->ldx, p->M, size)) n += align256((size_t)(p->M * line_pitch(p->K, size)) * size);
    if (!rows16(p->w, p->ldw, p->O, size)) n += align256((size_t)(p->O * line_pitch(p->K, size)) * size);
    return n;
}

extern "C" int chxq_linear_kernel(const chxq_linear_params* p, int32_t* kernel) {
    CHXQ_CHECK_ARG(kernel != nullptr, "Linear: null pointer");
    const int rc = check_linear(p);
    if (rc != CHXQ_OK) return rc;
    if (p->M == 0 || p->O == 0 || p->K == 0) *kernel = CHXQ_LINEAR_NO_PRODUCT;
    else if (few_rows(*p)) *kernel = CHXQ_LINEAR_ROWS;
    else if (p->dtype == CHXQ_FLOAT32) *kernel = CHXQ_LINEAR_TILES_F32;
    else *kernel = takes_pairs(*p) ? CHXQ_LINEAR_PAIRS : CHXQ_LINEAR_TILES;
    return CHXQ_OK;
}

extern "C" int chxq_linear(const chxq_linear_params* p, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = check_linear(p);
    if (rc != CHXQ_OK) return rc;
    if (p->M == 0 || p->O == 0) return CHXQ_OK;
    if (p->M > kMostCoordinate || p->O > kMostCoordinate) {  // (one workspace for all: each launch waits for the one before)
        const int64_t size = float_size(p->dtype), bias_size = p->bias ? float_size(p->bias_dtype) : 0;
        auto at = [](const void* base, int64_t bytes) { return base ? static_cast<const uint8_t*>(base) + bytes : nullptr; };
        for (int64_t m = 0; m < p->M; m += kMostCoordinate)
            for (int64_t o = 0; o < p->O; o += kMostCoordinate) {
                chxq_linear_params q = *p;
                q.M = std::min(kMostCoordinate, p->M - m);
                q.O = std::min(kMostCoordinate, p->O - o);
                q.x = at(p->x, m * p->ldx * size);
                q.w = at(p->w, o * p->ldw * size);
                q.bias = at(p->bias, o * bias_size);
                q.residual = at(p->residual, (m * p->ldr + o) * size);
                q.y = const_cast<uint8_t*>(at(p->y, (m * p->ldy + o) * size));
                const int part = chxq_linear(&q, workspace, workspace_bytes, stream);
                if (part != CHXQ_OK) return part;
            }
        return CHXQ_OK;
    }
    const size_t need = chxq_linear_workspace(p);
    if (need && (!workspace || workspace_bytes < need)) return set_error(CHXQ_ERR_WORKSPACE, "Linear: needs %zu bytes of workspace", need);
    CHXQ_CHECK_ARG(need == 0 || (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, "Linear: the workspace must be 256-byte aligned");
    const LinearEpilogue e = {p->bias, p->bias_dtype, p->residual, p->ldr, p->activation, p->residual_first, p->y, p->ldy};
    cudaStream_t s = as_stream(stream);
    if (p->K == 0)
        return with_float_type(p->dtype, [&](auto t) {
            linear_empty_kernel<decltype(t)><<<(unsigned)std::min<int64_t>((p->M * p->O + 255) / 256, tc::sm_count() * 8), 256, 0, s>>>(p->M, p->O, e);
            CHXQ_LAUNCH_CHECK();
            return CHXQ_OK;
        });
    if (few_rows(*p)) {
        return with_float_type(p->dtype, [&](auto t) {
            using T = decltype(t);
            if (p->M == 1) return launch_rows<T, 1>(*p, e, s);
            if (p->M == 2) return launch_rows<T, 2>(*p, e, s);
            return p->M <= 4 ? launch_rows<T, 4>(*p, e, s) : launch_rows<T, 8>(*p, e, s);
        });
    }
    const int size = float_size(p->dtype);
    Operands op = {p->x, p->ldx, p->w, p->ldw};
    if (need) {
        const int64_t pitch = line_pitch(p->K, size);
        CopyJob jx = {p->x, p->ldx, 0, nullptr}, jw = {p->w, p->ldw, 0, nullptr};
        uint8_t* ws = static_cast<uint8_t*>(workspace);
        if (!rows16(p->x, p->ldx, p->M, size)) {
            jx.rows = p->M;
            op.x = jx.dst = ws;
            op.ldx = pitch;
            ws += align256((size_t)(p->M * pitch) * size);
        }
        if (!rows16(p->w, p->ldw, p->O, size)) {
            jw.rows = p->O;
            op.w = jw.dst = ws;
            op.ldw = pitch;
        }
        const int64_t blocks = ((jx.rows + jw.rows) * (pitch * size / 16) + 255) / 256;
        CHXQ_CUDA(launch_pdl(size == 4 ? align_rows_kernel<uint32_t> : align_rows_kernel<uint16_t>, dim3((unsigned)std::min<int64_t>(blocks, tc::sm_count() * 16)), 256, 0, s, jx, jw,
                             p->K, pitch));
        count_launch(1);
    }
    lin::TcArgs a;
    a.M = (int)p->M;
    a.O = (int)p->O;
    a.k_blocks = k_blocks_of(*p);
    a.idesc = lin::idesc_f16(p->dtype == CHXQ_BFLOAT16 ? lin::kBf16 : lin::kF16);  // (fp32 has its own)
    a.e = e;
    a.vec = rows16(p->y, p->ldy, p->M, size) && p->O * size % 16 == 0 && (!p->residual || rows16(p->residual, p->ldr, p->M, size));
    a.status = device_status_ptr();
    if (!a.status) return set_error(CHXQ_ERR_CUDA, "device status word is unavailable");
    a.wait_limit_ns = (unsigned long long)tc::wait_limit_ns_value();
    a.test_skip_kb = tc::test_skip_kb_value();
    return with_float_type(p->dtype, [&](auto t) { return launch_tc<decltype(t)>(*p, op, a, s); });
}
