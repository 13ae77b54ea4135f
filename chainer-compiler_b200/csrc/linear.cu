// Linear with bias, activation and residual in its epilogue: y = act(x w^T + b) + r, or act(x w^T + b + r); bf16, fp16 and fp32 operands,
// sums in 32 bits, one rounding at the end.
//
// Three kernels: CTA pairs with 256 x 256 blocks (linear_pair.cuh) for large 16-bit products, clusters that share a tile's K (linear_tile.cuh) for
// few rows of x and products in between, and a general CUDA-core kernel.
#include <algorithm>
#include <atomic>

#include "epilogue_float.cuh"
#include "float_ops.cuh"
#include "linear_pair.cuh"
#include "linear_tile.cuh"

namespace chxq {
namespace {

// General kernel: 64 x 64 outputs a block, 4 x 4 a thread, operands through shared memory in 32 bits.  Any extent, row pitch and alignment.
constexpr int kTile = 64, kSlice = 16;

template <typename T>
__global__ void __launch_bounds__(256) linear_simt_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw, int64_t M, int64_t O,
                                                          int64_t K, LinearEpilogue e) {
    __shared__ float xs[kSlice][kTile + 1], ws[kSlice][kTile + 1];
    const int tid = threadIdx.x;
    const int64_t m0 = (int64_t)blockIdx.y * kTile, o0 = (int64_t)blockIdx.x * kTile;
    const int tm = tid / 16, to = tid % 16;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < K; k0 += kSlice) {
#pragma unroll
        for (int i = 0; i < kTile * kSlice / 256; ++i) {
            const int f = tid + 256 * i, r = f / kSlice, k = f % kSlice;
            const bool in = k0 + k < K;
            xs[k][r] = in && m0 + r < M ? to_f32(x[(m0 + r) * ldx + k0 + k]) : 0.f;
            ws[k][r] = in && o0 + r < O ? to_f32(w[(o0 + r) * ldw + k0 + k]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSlice; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __fmaf_rn(xs[k][tm * 4 + i], ws[k][to + 16 * j], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + tm * 4 + i, o = o0 + to + 16 * j;
            if (m < M && o < O) epilogue_store<T>(e, m, o, acc[i][j]);
        }
}

// ---- the tensor-core kernels ------------------------------------------------------------------------------------------------

// TMA reads rows that start on 16-byte boundaries.  Operands whose rows do not are copied into such rows in front of the product.
bool rows16(const void* p, int64_t ld, int64_t rows) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (rows == 1 || ld % 8 == 0);
}
int64_t pitch16(int64_t K) {
    return (K + 7) / 8 * 8;
}
size_t align256(size_t v) {
    return (v + 255) / 256 * 256;
}

struct CopyJob {
    const uint16_t* src;
    int64_t ld, rows;
    uint16_t* dst;
};

// Rows of K 16-bit values into rows of `pitch`, a multiple of 8: a thread gathers eight values and writes them as 16 bytes.  (The last
// group's values past K are never read: the tensor map ends at K.)
__global__ void __launch_bounds__(256) align_rows_kernel(CopyJob a, CopyJob b, int64_t K, int64_t pitch) {
    pdl_launch_dependents();
    pdl_dependency_wait();
    const int64_t per_row = pitch / 8, total = (a.rows + b.rows) * per_row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        int64_t r = i / per_row;
        const int64_t k = (i - r * per_row) * 8;
        const bool first = r < a.rows;
        if (!first) r -= a.rows;
        const uint16_t* s = (first ? a.src + r * a.ld : b.src + r * b.ld) + k;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = (k + 2 * j < K ? s[2 * j] : 0u) | ((k + 2 * j + 1 < K ? (uint32_t)s[2 * j + 1] : 0u) << 16);
        *reinterpret_cast<uint4*>((first ? a.dst + r * pitch : b.dst + r * pitch) + k) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Sets a kernel's dynamic shared memory once per device.
template <typename F>
int set_smem(F* kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    CHXQ_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;
    if (done.load(std::memory_order_acquire) & bit) return CHXQ_OK;
    CHXQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_release);
    return CHXQ_OK;
}

struct Operands {  // as TMA reads them
    const void* x;
    int64_t ldx;
    const void* w;
    int64_t ldw;
};

template <typename T, int BN, int STAGES>
int launch_tile(const chxq_linear_params& q, const Operands& op, const lin::TcArgs& args, cudaStream_t s) {
    using Cfg = lin::TileConfig<BN, STAGES>;
    static std::atomic<uint64_t> done{0};
    auto* kernel = lin::linear_tile_kernel<T, BN, STAGES>;
    int rc = set_smem(kernel, Cfg::kSmem, done);
    if (rc != CHXQ_OK) return rc;
    alignas(64) CUtensorMap tmW, tmX;
    if ((rc = tc::encode_rows_map(&tmW, op.w, q.K * 2, q.O, op.ldw * 2, 128)) != CHXQ_OK) return rc;
    if ((rc = tc::encode_rows_map(&tmX, op.x, q.K * 2, q.M, op.ldx * 2, BN)) != CHXQ_OK) return rc;
    const int64_t x_tiles = (q.M + BN - 1) / BN, tiles = x_tiles * ((q.O + 127) / 128);
    int split = 1;
    while (split < 8 && tiles * split * 2 <= 2 * tc::sm_count() && split * 2 <= args.k_blocks) split *= 2;
    if (tiles * split >= (1ll << 31)) return set_error(CHXQ_ERR_UNSUPPORTED, "Linear: too many tiles");
    CHXQ_CUDA(launch_pdl_cluster(split, kernel, dim3((unsigned)(tiles * split)), 256, Cfg::kSmem, s, tmW, tmX, args, split, (int)x_tiles));
    count_launch(1);
    return CHXQ_OK;
}

template <typename T>
int launch_pair(const chxq_linear_params& q, const Operands& op, const lin::TcArgs& args, cudaStream_t s) {
    using Cfg = lin::PairConfig;
    static std::atomic<uint64_t> done{0};
    auto* kernel = lin::linear_pair_kernel<T>;
    int rc = set_smem(kernel, Cfg::kSmem, done);
    if (rc != CHXQ_OK) return rc;
    lin::PairArgs a;
    a.t = args;
    const int64_t mb = (q.M + 255) / 256, ob = (q.O + 255) / 256;
    if (mb * ob >= (1ll << 31)) return set_error(CHXQ_ERR_UNSUPPORTED, "Linear: too many blocks");
    a.m_blocks = (int)mb;
    a.o_blocks = (int)ob;
    a.tma_out = rows16(q.y, q.ldy, q.M);
    alignas(64) CUtensorMap tmX, tmW, tmY;
    if ((rc = tc::encode_rows_map(&tmX, op.x, q.K * 2, q.M, op.ldx * 2, 128)) != CHXQ_OK) return rc;
    if ((rc = tc::encode_rows_map(&tmW, op.w, q.K * 2, q.O, op.ldw * 2, 128)) != CHXQ_OK) return rc;
    tmY = tmX;  // not used where the output is copied
    if (a.tma_out && (rc = tc::encode_rows_map(&tmY, q.y, q.O * 2, q.M, q.ldy * 2, 128)) != CHXQ_OK) return rc;
    const int pairs = (int)std::min<int64_t>(mb * ob, tc::sm_count() / 2);
    CHXQ_CUDA(launch_pdl(kernel, dim3((unsigned)(2 * pairs)), lin::kPairThreads, Cfg::kSmem, s, tmX, tmW, tmY, a));
    count_launch(1);
    return CHXQ_OK;
}

template <typename T>
int launch_tc(const chxq_linear_params& q, const Operands& op, const lin::TcArgs& args, cudaStream_t s) {
    const int64_t blocks = ((q.M + 255) / 256) * ((q.O + 255) / 256);
    if (q.M > 128 && blocks >= tc::sm_count() / 4) return launch_pair<T>(q, op, args, s);
    if (q.M <= 16) return launch_tile<T, 16, 6>(q, op, args, s);
    if (q.M <= 32) return launch_tile<T, 32, 5>(q, op, args, s);
    if (q.M <= 64) return launch_tile<T, 64, 4>(q, op, args, s);
    return launch_tile<T, 128, 3>(q, op, args, s);
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
    CHXQ_CHECK_ARG(p->activation >= CHXQ_ACT_NONE && p->activation <= CHXQ_ACT_TANH, "Linear: unknown activation %d", p->activation);
    return CHXQ_OK;
}

// 16-bit operands with a K go to the tensor cores.
static bool tensor_cores(const chxq_linear_params& p) {
    return p.dtype != CHXQ_FLOAT32 && p.K > 0;
}

extern "C" size_t chxq_linear_workspace(const chxq_linear_params* p) {
    if (!p || !tensor_cores(*p) || p->M <= 0 || p->O <= 0) return 0;
    size_t n = 0;
    if (!rows16(p->x, p->ldx, p->M)) n += align256((size_t)(p->M * pitch16(p->K)) * 2);
    if (!rows16(p->w, p->ldw, p->O)) n += align256((size_t)(p->O * pitch16(p->K)) * 2);
    return n;
}

extern "C" int chxq_linear(const chxq_linear_params* p, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = check_linear(p);
    if (rc != CHXQ_OK) return rc;
    if (p->M == 0 || p->O == 0) return CHXQ_OK;
    const size_t need = chxq_linear_workspace(p);
    if (need && (!workspace || workspace_bytes < need)) return set_error(CHXQ_ERR_WORKSPACE, "Linear: needs %zu bytes of workspace", need);
    CHXQ_CHECK_ARG(need == 0 || (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, "Linear: the workspace must be 256-byte aligned");
    const LinearEpilogue e = {p->bias, p->bias_dtype, p->residual, p->ldr, p->activation, p->residual_first, p->y, p->ldy};
    cudaStream_t s = as_stream(stream);
    if (tensor_cores(*p)) {
        Operands op = {p->x, p->ldx, p->w, p->ldw};
        if (need) {
            const int64_t pitch = pitch16(p->K);
            CopyJob jx = {static_cast<const uint16_t*>(p->x), p->ldx, 0, nullptr}, jw = {static_cast<const uint16_t*>(p->w), p->ldw, 0, nullptr};
            uint8_t* ws = static_cast<uint8_t*>(workspace);
            if (!rows16(p->x, p->ldx, p->M)) {
                jx.rows = p->M;
                jx.dst = reinterpret_cast<uint16_t*>(ws);
                ws += align256((size_t)(p->M * pitch) * 2);
                op.x = jx.dst;
                op.ldx = pitch;
            }
            if (!rows16(p->w, p->ldw, p->O)) {
                jw.rows = p->O;
                jw.dst = reinterpret_cast<uint16_t*>(ws);
                op.w = jw.dst;
                op.ldw = pitch;
            }
            const int64_t blocks = ((jx.rows + jw.rows) * (pitch / 8) + 255) / 256;
            CHXQ_CUDA(launch_pdl(align_rows_kernel, dim3((unsigned)std::min<int64_t>(blocks, 148 * 16)), 256, 0, s, jx, jw, p->K, pitch));
            count_launch(1);
        }
        lin::TcArgs a;
        a.M = (int)p->M;
        a.O = (int)p->O;
        a.k_blocks = (int)((p->K + 63) / 64);
        a.idesc = lin::idesc_f16(p->dtype == CHXQ_BFLOAT16 ? lin::kBf16 : lin::kF16);
        a.e = e;
        a.vec = rows16(p->y, p->ldy, p->M) && p->O % 8 == 0 && (!p->residual || rows16(p->residual, p->ldr, p->M));
        a.status = device_status_ptr();
        if (!a.status) return set_error(CHXQ_ERR_CUDA, "device status word is unavailable");
        a.wait_limit_ns = (unsigned long long)tc::wait_limit_ns_value();
        return p->dtype == CHXQ_BFLOAT16 ? launch_tc<__nv_bfloat16>(*p, op, a, s) : launch_tc<__half>(*p, op, a, s);
    }
    const dim3 grid((unsigned)((p->O + kTile - 1) / kTile), (unsigned)((p->M + kTile - 1) / kTile));
    if (grid.y > 65535) return set_error(CHXQ_ERR_UNSUPPORTED, "Linear: too many rows");
    return with_float_type(p->dtype, [&](auto t) {
        using T = decltype(t);
        linear_simt_kernel<T><<<grid, 256, 0, s>>>(static_cast<const T*>(p->x), p->ldx, static_cast<const T*>(p->w), p->ldw, p->M, p->O, p->K, e);
        CHXQ_LAUNCH_CHECK();
        return CHXQ_OK;
    });
}
