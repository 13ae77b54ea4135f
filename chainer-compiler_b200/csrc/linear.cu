// Linear with bias, activation and residual in its epilogue: y = act(x w^T + b) + r, or act(x w^T + b + r); bf16, fp16 and fp32 operands,
// sums in 32 bits, one rounding at the end.
#include "epilogue_float.cuh"
#include "float_ops.cuh"

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

extern "C" size_t chxq_linear_workspace(const chxq_linear_params*) {
    return 0;
}

extern "C" int chxq_linear(const chxq_linear_params* p, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = check_linear(p);
    if (rc != CHXQ_OK) return rc;
    if (p->M == 0 || p->O == 0) return CHXQ_OK;
    const size_t need = chxq_linear_workspace(p);
    if (need && (!workspace || workspace_bytes < need)) return set_error(CHXQ_ERR_WORKSPACE, "Linear: needs %zu bytes of workspace", need);
    const LinearEpilogue e = {p->bias, p->bias_dtype, p->residual, p->ldr, p->activation, p->residual_first, p->y, p->ldy};
    const dim3 grid((unsigned)((p->O + kTile - 1) / kTile), (unsigned)((p->M + kTile - 1) / kTile));
    if (grid.y > 65535) return set_error(CHXQ_ERR_UNSUPPORTED, "Linear: too many rows");
    return with_float_type(p->dtype, [&](auto t) {
        using T = decltype(t);
        linear_simt_kernel<T><<<grid, 256, 0, as_stream(stream)>>>(static_cast<const T*>(p->x), p->ldx, static_cast<const T*>(p->w), p->ldw, p->M, p->O, p->K, e);
        CHXQ_LAUNCH_CHECK();
        return CHXQ_OK;
    });
}
