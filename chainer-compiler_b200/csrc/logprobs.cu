// TokenLogProbs: log probability of one token per row of logits, the row's entropy, the log of its sum and its best alternatives; and the
// gradient by the logits.
//   lse = log sum exp x,  lp = x[token] - lse,  H = -sum p log p = lse - sum p x
//   dx_j = g (1[j = token] - p_j) - h p_j (log p_j + H)
// A logit of -infinity is a forbidden value: it has probability zero and adds nothing.
#include "float_ops.cuh"

namespace chxq {
namespace {

constexpr int kThreads = 256;

struct Best {
    float v;
    int i;
};
__device__ __forceinline__ bool before(const Best& a, const Best& b) {  // a ranks before b: the larger value, then the lower index
    return a.v > b.v || (a.v == b.v && a.i < b.i);
}
__device__ __forceinline__ float rank_value(float v) {  // NaN ranks with +infinity
    return v != v ? INFINITY : v;
}

__device__ __forceinline__ int64_t load_token(const void* tokens, int dtype, int64_t r) {
    return dtype == CHXQ_INT64 ? static_cast<const int64_t*>(tokens)[r] : (int64_t)static_cast<const int32_t*>(tokens)[r];
}

template <typename F>
__device__ __forceinline__ float block_reduce(float v, float* red, F&& f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = red[0];
    for (int i = 1; i < (int)(blockDim.x >> 5); ++i) s = f(s, red[i]);
    return s;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const T* __restrict__ logits, int64_t ld, const void* __restrict__ tokens, int token_dtype,
                                                                  int64_t rows, int64_t V, int num_top, int has_ignore, int64_t ignore,
                                                                  float* __restrict__ logprob, float* __restrict__ entropy, float* __restrict__ lse_out,
                                                                  float* __restrict__ top_lp, int64_t* __restrict__ top_tok) {
    __shared__ float red[kThreads / 32];
    __shared__ Best bred[kThreads / 32];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* x = logits + r * ld;
        float m = -INFINITY;
        bool nan = false;
        for (int64_t i = threadIdx.x; i < V; i += kThreads) {
            const float v = to_f32(x[i]);
            nan = nan || v != v;
            m = fmaxf(m, v);
        }
        m = block_reduce(nan ? INFINITY : m, red, [](float a, float b) { return fmaxf(a, b); });
        float s = 0.f, t = 0.f;
        if (m > -INFINITY)
            for (int64_t i = threadIdx.x; i < V; i += kThreads) {
                const float a = to_f32(x[i]) - m, e = expf(a);
                s += e;
                t += e == 0.f ? 0.f : e * a;
            }
        s = block_reduce(s, red, [](float a, float b) { return a + b; });
        t = block_reduce(t, red, [](float a, float b) { return a + b; });
        const bool empty = m == -INFINITY;
        const float lse = empty ? -INFINITY : m + logf(s);
        if (threadIdx.x == 0) {
            const int64_t tok = load_token(tokens, token_dtype, r);
            float lp = nanf("");
            if (has_ignore && tok == ignore) lp = 0.f;
            else if (tok >= 0 && tok < V) lp = empty ? -INFINITY : (to_f32(x[tok]) - m) - logf(s);  // not through lse, which rounds where m is large
            logprob[r] = lp;
            entropy[r] = empty ? 0.f : logf(s) - t / s;
            lse_out[r] = lse;
        }
        Best last = {INFINITY, -1};
        for (int k = 0; k < num_top; ++k) {
            Best b = {-INFINITY, 0x7fffffff};
            for (int64_t i = threadIdx.x; i < V; i += kThreads) {
                const Best c = {rank_value(to_f32(x[i])), (int)i};
                if (before(last, c) && before(c, b)) b = c;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const Best c = {__shfl_xor_sync(0xffffffffu, b.v, o), __shfl_xor_sync(0xffffffffu, b.i, o)};
                if (before(c, b)) b = c;
            }
            __syncthreads();
            if ((threadIdx.x & 31) == 0) bred[threadIdx.x >> 5] = b;
            __syncthreads();
            last = bred[0];
            for (int i = 1; i < kThreads / 32; ++i)
                if (before(bred[i], last)) last = bred[i];
            if (threadIdx.x == 0) {
                top_tok[r * num_top + k] = last.i;
                top_lp[r * num_top + k] = empty ? -INFINITY : (to_f32(x[last.i]) - m) - logf(s);
            }
        }
    }
}

// log p = (x - shift) - log_total.  lse is the sum of the two and rounds: from 1024 on by up to 2^-14 and more, and in a row of nothing but the type's
// lowest value it holds no digit of log_total at all.  Such rows, which no ordinary network makes, are summed again.
struct RowScale {
    float shift, log_total;
};
template <typename T>
__device__ RowScale row_scale(const T* __restrict__ x, int64_t V, float lse, float* red) {
    if (!(fabsf(lse) > 1024.f) || fabsf(lse) == INFINITY) return {lse, 0.f};
    float m = -INFINITY, s = 0.f;
    for (int64_t i = threadIdx.x; i < V; i += blockDim.x) m = fmaxf(m, to_f32(x[i]));
    m = block_reduce(m, red, [](float a, float b) { return fmaxf(a, b); });
    for (int64_t i = threadIdx.x; i < V; i += blockDim.x) s += expf(to_f32(x[i]) - m);
    return {m, logf(block_reduce(s, red, [](float a, float b) { return a + b; }))};
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_grad_kernel(const float* __restrict__ dlogprob, const float* __restrict__ dentropy,
                                                                       const T* __restrict__ logits, int64_t ld, const void* __restrict__ tokens, int token_dtype,
                                                                       const float* __restrict__ lse, const float* __restrict__ entropy, int64_t rows, int64_t V,
                                                                       int has_ignore, int64_t ignore, T* __restrict__ dlogits) {
    __shared__ float red[kThreads / 32];
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const int64_t tok = load_token(tokens, token_dtype, r);
        const float g = !dlogprob || (has_ignore && tok == ignore) ? 0.f : (tok < 0 || tok >= V ? nanf("") : dlogprob[r]), h = dentropy ? dentropy[r] : 0.f, l = lse[r];
        const float H = entropy ? entropy[r] : 0.f;
        const RowScale sc = row_scale(logits + r * ld, V, l, red);
        for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < V; i += (int64_t)gridDim.x * kThreads) {
            const float v = to_f32(logits[r * ld + i]);
            const float a = v == -INFINITY ? -INFINITY : (v - sc.shift) - sc.log_total, p = expf(a);
            float d = p == 0.f ? 0.f : -p * (g + h * (a + H));
            if (i == tok) d += g;
            dlogits[r * V + i] = from_f32<T>(d);
        }
    }
}

}  // namespace
}  // namespace chxq

using namespace chxq;

static int check_logprobs(const char* op, int dtype, int token_dtype, int64_t ld, int64_t rows, int64_t V) {
    CHXQ_CHECK_ARG(is_float_type(dtype), "%s: logits must be float32, float16 or bfloat16", op);
    CHXQ_CHECK_ARG(token_dtype == CHXQ_INT32 || token_dtype == CHXQ_INT64, "%s: tokens must be int32 or int64", op);
    CHXQ_CHECK_ARG(rows >= 0 && V >= 1 && V < (1ll << 31) && (rows <= 1 || ld >= V), "%s: bad extents", op);
    return CHXQ_OK;
}

extern "C" int chxq_token_logprobs(const void* logits, int64_t ld, int32_t dtype, const void* tokens, int32_t token_dtype, int64_t rows, int64_t V, int32_t num_top,
                                   int32_t has_ignore, int64_t ignore_index, float* logprob, float* entropy, float* log_sum_exp, float* top_logprobs,
                                   int64_t* top_tokens, void* stream) {
    const int rc = check_logprobs("TokenLogProbs", dtype, token_dtype, ld, rows, V);
    if (rc != CHXQ_OK) return rc;
    CHXQ_CHECK_ARG(num_top >= 0 && num_top <= CHXQ_MAX_TOP && num_top <= V, "TokenLogProbs: num_top must be at most %d and at most the number of logits", CHXQ_MAX_TOP);
    if (rows == 0) return CHXQ_OK;
    CHXQ_CHECK_ARG(logits && tokens && logprob && entropy && log_sum_exp && (num_top == 0 || (top_logprobs && top_tokens)), "TokenLogProbs: null argument");
    return with_float_type(dtype, [&](auto t) {
        using T = decltype(t);
        token_logprobs_kernel<T><<<(unsigned)(rows < 148 * 8 ? rows : 148 * 8), kThreads, 0, as_stream(stream)>>>(
                static_cast<const T*>(logits), ld, tokens, token_dtype, rows, V, num_top, has_ignore, ignore_index, logprob, entropy, log_sum_exp, top_logprobs,
                top_tokens);
        CHXQ_LAUNCH_CHECK();
        return CHXQ_OK;
    });
}

extern "C" int chxq_token_logprobs_grad(const float* dlogprob, const float* dentropy, const void* logits, int64_t ld, int32_t dtype, const void* tokens,
                                        int32_t token_dtype, const float* log_sum_exp, const float* entropy, int64_t rows, int64_t V, int32_t has_ignore,
                                        int64_t ignore_index, void* dlogits, void* stream) {
    const int rc = check_logprobs("TokenLogProbsGrad", dtype, token_dtype, ld, rows, V);
    if (rc != CHXQ_OK) return rc;
    if (rows == 0) return CHXQ_OK;
    CHXQ_CHECK_ARG(logits && tokens && log_sum_exp && dlogits && (!dentropy || entropy), "TokenLogProbsGrad: null argument");
    const dim3 grid((unsigned)((V + 4 * kThreads - 1) / (4 * kThreads)), (unsigned)(rows < 65535 ? rows : 65535));
    return with_float_type(dtype, [&](auto t) {
        using T = decltype(t);
        token_logprobs_grad_kernel<T><<<grid, kThreads, 0, as_stream(stream)>>>(dlogprob, dentropy, static_cast<const T*>(logits), ld, tokens, token_dtype,
                                                                                log_sum_exp, entropy, rows, V, has_ignore, ignore_index, static_cast<T*>(dlogits));
        CHXQ_LAUNCH_CHECK();
        return CHXQ_OK;
    });
}
