// TokenLogProbs: log probability of one token per row of logits, the row's entropy, the log of its sum and its best alternatives; and the
// gradient by the logits.
//   lse = log sum exp x,  lp = x[token] - lse,  H = -sum p log p = lse - sum p x
//   dx_j = g (1[j = token] - p_j) - h p_j (log p_j + H)
// A logit of -infinity is a forbidden value: it has probability zero and adds nothing.
#include <algorithm>

#include "float_ops.cuh"
#include "pdl.cuh"
#include "tc_kernel.cuh"  // cluster helpers

namespace chxq {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ int64_t load_token(const void* tokens, int dtype, int64_t r) {
    return dtype == CHXQ_INT64 ? static_cast<const int64_t*>(tokens)[r] : (int64_t)static_cast<const int32_t*>(tokens)[r];
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp2_approx(float a) {  // good to 2^-22
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
    return r;
}

// ---- sums -----------------------------------------------------------------------------------------------------------------

// A part of a row: its largest logit m, s = sum exp(x - m) and t = sum exp(x - m) (x - m).  Without a logit above -infinity: m = -infinity, s = t = 0.
struct Part {
    float m, s, t;
};
__device__ __forceinline__ void rescale(Part& a, float m) {  // to a larger maximum
    // below -10000 the factor is zero, and its product with the difference has to be: the difference must stay finite
    const float d = max_nan(a.m - m, -1e4f), f = a.m == -INFINITY ? 0.f : __expf(d);
    a.t = a.m == -INFINITY ? 0.f : f * fmaf(a.s, d, a.t);
    a.s *= f;
    a.m = m;
}
__device__ __forceinline__ Part join(Part a, Part b) {
    const float m = max_nan(a.m, b.m);
    if (m == -INFINITY) return a;
    rescale(a, m);
    rescale(b, m);
    return {m, a.s + b.s, a.t + b.t};
}

// ---- the best alternatives ------------------------------------------------------------------------------------------------

// A list of 32 logits in descending order, one per lane; equal ones by ascending index; empty places are (-infinity, kNone), behind everything.
constexpr int kNone = 0x7fffffff;
struct Entry {
    float v;
    int i;
};
__device__ __forceinline__ bool before(float va, int ia, float vb, int ib) {
    return va > vb || (va == vb && ia < ib);
}
__device__ __forceinline__ float rank_value(float v) {  // NaN ranks with +infinity
    return v != v ? INFINITY : v;
}
// The lanes' entries in the order of a list.
__device__ __forceinline__ void sort(Entry& e) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size >> 1; d > 0; d >>= 1) {
            const float v = __shfl_xor_sync(0xffffffffu, e.v, d);
            const int i = __shfl_xor_sync(0xffffffffu, e.i, d);
            const bool first = ((lane & size) == 0) == ((lane & d) == 0);  // this lane takes the entry that ranks first
            if (before(v, i, e.v, e.i) == first) e = {v, i};
        }
}
// The best 32 of two lists: the larger of one and the reversed other is a bitonic sequence of them, which five steps sort.
__device__ __forceinline__ void merge(Entry& e, Entry o) {
    const int lane = threadIdx.x & 31;
    o.v = __shfl_sync(0xffffffffu, o.v, 31 - lane);
    o.i = __shfl_sync(0xffffffffu, o.i, 31 - lane);
    if (before(o.v, o.i, e.v, e.i)) e = o;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, e.v, d);
        const int i = __shfl_xor_sync(0xffffffffu, e.i, d);
        if (before(v, i, e.v, e.i) == ((lane & d) == 0)) e = {v, i};
    }
}
// The lanes' values in descending order.
__device__ __forceinline__ float sort_lanes(float v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size >> 1; d > 0; d >>= 1) {
            const float o = __shfl_xor_sync(0xffffffffu, v, d);
            const bool up = (lane & size) == 0, low = (lane & d) == 0;
            v = (up == low) ? fmaxf(v, o) : fminf(v, o);
        }
    return v;
}
// ---- forward --------------------------------------------------------------------------------------------------------------

struct LogprobArgs {
    const void* tokens;
    int token_dtype, num_top, has_ignore;
    int64_t rows, ignore;
    float *logprob, *entropy, *lse, *top_lp;
    int64_t* top_tok;
};

// One pass over a row: the running maximum and the two sums of a thread are rescaled when the maximum grows.  W warps take a row (one for short rows, else
// the block's eight), or the blocks of a cluster (W = 8) a part of it each; the parts meet in shared memory, and the blocks' in the first block's
// through distributed shared memory.  A thread has kU accesses of sixteen bytes in flight; up to 15 bytes at either end of a row are read one by one.
// Alternatives (TOP): the num_top-th largest of 32 running maxima -- each over the threads of one lane number -- bounds the num_top-th best logit from below.
// It is taken anew after 1, 4, 16, ... rounds of accesses (1, 2, 4, ... for many alternatives), so that a few times num_top logits are above
// it; those go into a buffer of their warp, unsorted, and are sorted at the end (or when the buffer is full: ascending rows), 32 at a time.
// Bound: HBM; per logit one conversion, one maximum, four instructions on pairs, a clamp and an exponential.
template <typename T, int W, bool TOP>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const T* __restrict__ logits, int64_t ld, int V, int split, const LogprobArgs p) {
    constexpr int VEC = 16 / (int)sizeof(T), kU = 4;
    constexpr uint32_t kNegInf = sizeof(T) == 4 ? 0xff800000u : (std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u);
    constexpr int kBuffer = 2 * 32 * VEC;  // twice what an access of the warp's lanes may add
    __shared__ Part parts[kWarps];
    __shared__ Entry lists[TOP ? kWarps : 1][32];
    __shared__ float maxima[TOP ? 2 : 1][TOP ? kWarps : 1][32];
    __shared__ Entry buffers[TOP ? kWarps : 1][TOP ? kBuffer : 1];
    __shared__ int counts[kWarps];
    pdl_launch_dependents();
    pdl_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = W == 1 ? (int64_t)blockIdx.x * kWarps + warp : (int64_t)blockIdx.x / split;
    if (W == 1 && r >= p.rows) return;
    const int rank = W == 1 ? 0 : (int)(blockIdx.x % split);
    const T* x = logits + r * ld;
    const int head = min(V, (int)((16u - (reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / (int)sizeof(T));
    const int pieces = (V - head) / VEC, tail = V - head - pieces * VEC;
    const int p0 = (int)((int64_t)pieces * rank / split), p1 = (int)((int64_t)pieces * (rank + 1) / split);
    const T* body = x + head;
    constexpr int kLanes = W * 32;

    float m = -INFINITY;
    f32x2 s2 = 0ull, t2 = 0ull;
    Entry e = {-INFINITY, kNone};
    float thr_v = -INFINITY, floor_v = -INFINITY;  // the list's num_top-th logit; no logit below floor_v is among the best
    int thr_i = kNone;
    if (TOP && lane == 0) counts[warp] = 0;
    __syncwarp();
    // Sorts the warp's buffer into its list.
    bool listed = false;
    auto settle = [&]() {
        __syncwarp();
        const int n = counts[warp];
        for (int c = 0; c < n; c += 32) {
            Entry o = {-INFINITY, kNone};
            if (c + lane < n) o = buffers[warp][c + lane];
            sort(o);
            if (listed) merge(e, o);
            else e = o;
            listed = true;
        }
        __syncwarp();
        if (lane == 0) counts[warp] = 0;
        __syncwarp();
        thr_v = __shfl_sync(0xffffffffu, e.v, p.num_top - 1);
        thr_i = __shfl_sync(0xffffffffu, e.i, p.num_top - 1);
    };
    // The lane's candidates -- value(j) at index i0 + j for every bit j of `which` -- go to the buffer; all lanes take part.  Once there is a list, equal
    // logits behind its num_top-th are turned away (in a row of one value, all of them).
    auto offer = [&](const auto& value, uint32_t which, int i0) __attribute__((always_inline)) {
        if (listed) {
            for (uint32_t w = which; w; w &= w - 1) {
                const int j = __ffs(w) - 1;
                if (!before(rank_value(value(j)), i0 + j, thr_v, thr_i)) which &= ~(1u << j);
            }
        }
        if (which) {
            int at = atomicAdd(&counts[warp], __popc(which));  // (any order: they are sorted later, and no two are equal)
            for (; which; which &= which - 1) {
                const int j = __ffs(which) - 1;
                buffers[warp][at++] = {rank_value(value(j)), i0 + j};
            }
        }
        __syncwarp();
        const bool many = counts[warp] > kBuffer / 2;
        __syncwarp();  // (all lanes have read it before one of them adds to it again, so that they settle together or not at all)
        if (many) settle();
    };
    auto grow = [&](float to) {  // a larger maximum
        const float d = max_nan(m - to, -1e4f), f = exp2_approx(d * kLog2e);  // (as in rescale; the sums are zero while m is -infinity)
        const f32x2 f2 = make_x2(f, f), d2 = make_x2(d, d);
        t2 = mul2(f2, fma2(s2, d2, t2));
        s2 = mul2(f2, s2);
        m = to;
    };
    auto add_pair = [&](f32x2 v) {
        const float2 d = split_x2(add2(v, make_x2(-m, -m)));
        // a forbidden logit's exponential is zero, and its product with the difference has to be: the difference must not be infinite
        const f32x2 c = make_x2(max_nan(d.x, -1e4f), max_nan(d.y, -1e4f));
        const float2 a = split_x2(mul2(c, make_x2(kLog2e, kLog2e)));
        const f32x2 ex = make_x2(exp2_approx(a.x), exp2_approx(a.y));
        s2 = add2(s2, ex);
        t2 = fma2(ex, c, t2);
    };

    const int rounds = (p1 - p0 + kLanes * kU - 1) / (kLanes * kU);
    int update = 0, par = 0;
    for (int round = 0; round < rounds; ++round) {
        const int base = p0 + round * kLanes * kU + (W == 1 ? 0 : warp * 32);
        float pm[kU], gm = -INFINITY;
        Pack<T, VEC> q[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int k = base + u * kLanes + lane;
#pragma unroll
            for (int j = 0; j < 4; ++j) q[u].w[j] = kNegInf;
            if (k < p1) q[u].load(body + (int64_t)k * VEC);
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            pm[u] = q[u].max_value();
            gm = max_nan(gm, pm[u]);
        }
        if (!(gm <= m)) grow(gm);
        if (TOP && round == update) {
            update = p.num_top > 8 ? 2 * update + 1 : 4 * update + 3;
            float top = rank_value(m);
            if constexpr (W > 1) {
                maxima[par][warp][lane] = top;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < kWarps; ++w) top = fmaxf(top, maxima[par][w][lane]);
                par ^= 1;  // (the maxima of two updates ago have been read by all when these are overwritten)
            }
            floor_v = __shfl_sync(0xffffffffu, sort_lanes(top), p.num_top - 1);
        }
        if (m != -INFINITY)
#pragma unroll
            for (int u = 0; u < kU; ++u)
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) add_pair(q[u].pair(j));
        if (TOP && __any_sync(0xffffffffu, !(gm < floor_v))) {  // (NaN passes, too)
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int k = base + u * kLanes + lane;
                const bool some = k < p1 && !(pm[u] < floor_v);
                if (!__any_sync(0xffffffffu, some)) continue;
                offer([&](int j) { return q[u].pick(j); }, some ? q[u].not_below(floor_v) : 0u, head + k * VEC);
            }
        }
    }
    if (rank == 0 && (W == 1 || warp == 0)) {  // the ends of the row, fewer than 32 logits
        const int i = lane < head ? lane : V - tail + (lane - head);
        const bool have = lane < head + tail;
        const float v = have ? to_f32(x[i]) : -INFINITY;
        if (!(v <= m)) grow(v);
        if (m != -INFINITY) add_pair(make_x2(v, -INFINITY));
        if constexpr (TOP) offer([&](int) { return v; }, have && !(v < floor_v) ? 1u : 0u, i);
    }
    if constexpr (TOP) settle();

    const float2 ss = split_x2(s2), tt = split_x2(t2);
    Part a = {m, ss.x + ss.y, tt.x + tt.y};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        a = join(a, {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.t, o)});
    if constexpr (W > 1) {
        for (int d = kWarps / 2; d > 0; d >>= 1) {  // the upper half of the warps hands its part to the lower
            if (warp >= d && warp < 2 * d) {
                if (lane == 0) parts[warp] = a;
                if constexpr (TOP) lists[warp][lane] = e;
            }
            __syncthreads();
            if (warp < d) {
                a = join(a, parts[warp + d]);
                if constexpr (TOP) merge(e, lists[warp + d][lane]);
            }
        }
        if (split > 1) {
            // (every thread comes to both barriers; the second keeps the blocks' shared memory in place until the first block has read it)
            __syncwarp();
            if (warp == 0) {
                if (lane == 0) parts[0] = a;
                if constexpr (TOP) lists[0][lane] = e;
            }
            tc::cluster_sync_all();
            if (rank == 0 && warp == 0)
                for (int c = 1; c < split; ++c) {
                    Part b;
                    const uint32_t at = tc::map_to_cta(tc::smem_u32(&parts[0]), c);
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.m) : "r"(at) : "memory");
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.s) : "r"(at + 4) : "memory");
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.t) : "r"(at + 8) : "memory");
                    a = join(a, b);
                    if constexpr (TOP) {
                        Entry o;
                        const uint32_t le = tc::map_to_cta(tc::smem_u32(&lists[0][lane]), c);
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.v) : "r"(le) : "memory");
                        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(o.i) : "r"(le + 4) : "memory");
                        merge(e, o);
                    }
                }
            tc::cluster_sync_all();
        }
        if (warp != 0 || rank != 0) return;
    }
    const bool empty = a.m == -INFINITY;
    const float log_total = logf(a.s);
    // log probabilities as (x - m) - log_total, not through their rounded sum
    if (TOP && lane < p.num_top) {
        p.top_lp[r * p.num_top + lane] = empty ? -INFINITY : (e.v - a.m) - log_total;
        p.top_tok[r * p.num_top + lane] = e.i;
    }
    if (lane == 0) {
        const int64_t tok = load_token(p.tokens, p.token_dtype, r);
        float lp = nanf("");
        if (p.has_ignore && tok == p.ignore) lp = 0.f;
        else if (tok >= 0 && tok < V) lp = empty ? -INFINITY : (to_f32(x[tok]) - a.m) - log_total;
        p.logprob[r] = lp;
        p.entropy[r] = empty ? 0.f : log_total - a.t / a.s;
        p.lse[r] = empty ? -INFINITY : a.m + log_total;
    }
}

// ---- gradient -------------------------------------------------------------------------------------------------------------

// over the W warps of a row
template <int W, typename F>
__device__ __forceinline__ float row_reduce(float v, float* red, F&& f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    if constexpr (W == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = red[0];
    for (int i = 1; i < W; ++i) s = f(s, red[i]);
    return s;
}

// log p = (x - shift) - log_total.  lse is the sum of the two and rounds: from 1024 on by up to 2^-14 and more, and in a row of nothing but the type's
// lowest value it holds no digit of log_total at all.  Such rows, which no ordinary network makes, are summed again.
struct RowScale {
    float shift, log_total;
};
template <typename T, int W>
__device__ RowScale row_scale(const T* __restrict__ x, int64_t V, float lse, float* red, int t) {
    if (lse == -INFINITY) return {0.f, 0.f};  // nothing but forbidden logits: probabilities of zero
    if (!(fabsf(lse) > 1024.f) || lse == INFINITY) return {lse, 0.f};
    float m = -INFINITY, s = 0.f;
    for (int64_t i = t; i < V; i += W * 32) m = fmaxf(m, to_f32(x[i]));
    m = row_reduce<W>(m, red, [](float a, float b) { return fmaxf(a, b); });
    for (int64_t i = t; i < V; i += W * 32) s += expf(to_f32(x[i]) - m);
    return {m, logf(row_reduce<W>(s, red, [](float a, float b) { return a + b; }))};
}

// W warps take W * 32 * kGradU pieces of sixteen bytes of one row, by where dlogits has them: the block's eight, or one where that covers a row ([6263, 303]
// bf16: 15.6 us with a block for each row, 6.7 with a warp).  The logits are read as pieces too where the row starts at the same place of a piece in both,
// and one by one elsewhere.  What a row has outside of whole pieces, fewer than VEC values at either end, goes to sixteen lanes, a value each.
constexpr int kGradU = 4;
template <typename T, int W>
__global__ void __launch_bounds__(kThreads) token_logprobs_grad_kernel(const float* __restrict__ dlogprob, const float* __restrict__ dentropy,
                                                                       const T* __restrict__ logits, int64_t ld, const void* __restrict__ tokens, int token_dtype,
                                                                       const float* __restrict__ lse, const float* __restrict__ entropy, int64_t rows, int V, int chunks,
                                                                       int has_ignore, int64_t ignore, T* __restrict__ dlogits) {
    constexpr int VEC = 16 / (int)sizeof(T), G = W * 32;
    __shared__ float red[kWarps];
    pdl_launch_dependents();
    pdl_dependency_wait();
    const int64_t r = W == 1 ? (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5) : blockIdx.x / (unsigned)chunks;
    if (W == 1 && r >= rows) return;  // (a whole warp)
    const int chunk = W == 1 ? 0 : (int)(blockIdx.x % (unsigned)chunks), t = (int)threadIdx.x % G;
    const T* x = logits + r * ld;
    T* out = dlogits + r * V;
    const int mis = (int)(reinterpret_cast<uintptr_t>(out) & 15u) / (int)sizeof(T);
    const bool same = (reinterpret_cast<uintptr_t>(out) & 15u) == (reinterpret_cast<uintptr_t>(x) & 15u);
    const int c0 = (chunk * G * kGradU + t) * VEC - mis;  // first column of the thread's first piece
    Pack<T, VEC> q[kGradU];
    auto column = [&](int u) { return c0 + u * G * VEC; };
    auto full = [&](int u) { return column(u) >= 0 && column(u) <= V - VEC; };
#pragma unroll
    for (int u = 0; u < kGradU; ++u) {
        q[u].zero();
        if (full(u) && same) q[u].load(x + column(u));
    }
    // the ends: lanes 0-7 the columns in front of the first whole piece, lanes 8-15 those behind the last
    const int front = min(V, (VEC - mis) % VEC), back = (V - front) % VEC;
    const int edge = chunk == 0 && t < 16 ? ((t & 7) < (t < 8 ? front : back) ? (t < 8 ? t : V - back + (t & 7)) : -1) : -1;
    T at_edge = from_f32<T>(0.f);
    if (edge >= 0) at_edge = x[edge];
    if (!same)
#pragma unroll
        for (int u = 0; u < kGradU; ++u)
            if (full(u))
#pragma unroll
                for (int j = 0; j < VEC; ++j) q[u].put(j, x[column(u) + j]);
    const int64_t tok = load_token(tokens, token_dtype, r);
    const float g = !dlogprob || (has_ignore && tok == ignore) ? 0.f : (tok < 0 || tok >= V ? nanf("") : dlogprob[r]), h = dentropy ? dentropy[r] : 0.f;
    const float H = entropy ? entropy[r] : 0.f;
    const int mine = tok >= 0 && tok < V ? (int)tok : -VEC;  // (never among a thread's columns)
    const RowScale sc = row_scale<T, W>(x, V, lse[r], red, t);
    const f32x2 ns = make_x2(-sc.shift, -sc.shift), nt = make_x2(-sc.log_total, -sc.log_total), k0 = make_x2(-fmaf(h, H, g), -fmaf(h, H, g)), k1 = make_x2(-h, -h);
    // -p (g + h (log p + H)) of two logits; log p is kept finite, since its product with a probability of zero has to be zero
    auto grad = [&](f32x2 v) {
        const float2 a = split_x2(add2(add2(v, ns), nt));
        const f32x2 lp = make_x2(max_nan(a.x, -1e4f), max_nan(a.y, -1e4f));
        const float2 e = split_x2(mul2(lp, make_x2(kLog2e, kLog2e)));
        return mul2(make_x2(exp2_approx(e.x), exp2_approx(e.y)), fma2(lp, k1, k0));
    };
#pragma unroll
    for (int u = 0; u < kGradU; ++u) {
        const int c = column(u);
        if (full(u)) {
            f32x2 d[VEC / 2];
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) d[j] = grad(q[u].pair(j));
            if ((unsigned)(mine - c) < (unsigned)VEC)
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) d[j] = add2(d[j], make_x2(mine == c + 2 * j ? g : 0.f, mine == c + 2 * j + 1 ? g : 0.f));
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) q[u].set_pair(j, d[j]);
            q[u].store(out + c);
        }
    }
    if (edge >= 0) {
        const float d = split_x2(grad(make_x2(to_f32(at_edge), 0.f))).x;
        out[edge] = from_f32<T>(d + (mine == edge ? g : 0.f));
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
    CHXQ_CHECK_ARG(on_values_of(float_size(dtype), logits) && on_values_of(token_dtype == CHXQ_INT64 ? 8 : 4, tokens) &&
                           on_values_of(4, logprob, entropy, log_sum_exp, top_logprobs) && on_values_of(8, top_tokens),
                   "TokenLogProbs: an address is no multiple of its values' size");
    const LogprobArgs a = {tokens, token_dtype, num_top, has_ignore, rows, ignore_index, logprob, entropy, log_sum_exp, top_logprobs, top_tokens};
    cudaStream_t s = as_stream(stream);
    return with_float_type(dtype, [&](auto t) {
        using T = decltype(t);
        // A warp per row where there are rows enough for half of the warps that fit; else a block, or a cluster of them as long as the blocks
        // do not fill the SMs twice and each still has a round of its accesses.
        const int round = kThreads * 4 * 16 / (int)sizeof(T);
        const int64_t sms = tc::sm_count();
        int split = 1;
        while (split < 8 && rows * split < 2 * sms && V >= (int64_t)round * split * 2) split *= 2;
        const bool warps = V <= 16384 && rows >= sms * 8;
        const int64_t grid = warps ? (rows + kWarps - 1) / kWarps : rows * split;
        if (grid >= (1ll << 31)) return set_error(CHXQ_ERR_UNSUPPORTED, "TokenLogProbs: too many rows");
        auto go = [&](auto* kernel) {
            CHXQ_CUDA(launch_pdl_cluster(split, kernel, dim3((unsigned)grid), kThreads, 0, s, static_cast<const T*>(logits), ld, (int)V, split, a));
            count_launch(1);
            return CHXQ_OK;
        };
        if (warps) return num_top ? go(token_logprobs_kernel<T, 1, true>) : go(token_logprobs_kernel<T, 1, false>);
        return num_top ? go(token_logprobs_kernel<T, kWarps, true>) : go(token_logprobs_kernel<T, kWarps, false>);
    });
}

extern "C" int chxq_token_logprobs_grad(const float* dlogprob, const float* dentropy, const void* logits, int64_t ld, int32_t dtype, const void* tokens,
                                        int32_t token_dtype, const float* log_sum_exp, const float* entropy, int64_t rows, int64_t V, int32_t has_ignore,
                                        int64_t ignore_index, void* dlogits, void* stream) {
    const int rc = check_logprobs("TokenLogProbsGrad", dtype, token_dtype, ld, rows, V);
    if (rc != CHXQ_OK) return rc;
    if (rows == 0) return CHXQ_OK;
    CHXQ_CHECK_ARG(logits && tokens && log_sum_exp && dlogits && (!dentropy || entropy), "TokenLogProbsGrad: null argument");
    CHXQ_CHECK_ARG(on_values_of(float_size(dtype), logits, dlogits) && on_values_of(token_dtype == CHXQ_INT64 ? 8 : 4, tokens) &&
                           on_values_of(4, dlogprob, dentropy, log_sum_exp, entropy),
                   "TokenLogProbsGrad: an address is no multiple of its values' size");
    cudaStream_t s = as_stream(stream);
    return with_float_type(dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int VEC = 16 / (int)sizeof(T);
        const int64_t per_warp = 32 * kGradU * VEC, most = V + VEC - 1;  // wherever in a piece a row starts
        const bool warp = most <= per_warp;
        const int64_t chunks = warp ? 1 : (most + kWarps * per_warp - 1) / (kWarps * per_warp), blocks = warp ? (rows + kWarps - 1) / kWarps : chunks * rows;
        if (blocks >= (1ll << 31)) return set_error(CHXQ_ERR_UNSUPPORTED, "TokenLogProbsGrad: too many logits");
        CHXQ_CUDA(launch_pdl(warp ? token_logprobs_grad_kernel<T, 1> : token_logprobs_grad_kernel<T, kWarps>, dim3((unsigned)blocks), kThreads, 0, s, dlogprob, dentropy,
                             static_cast<const T*>(logits), ld, tokens, (int)token_dtype, log_sum_exp, entropy, rows, (int)V, (int)chunks, (int)has_ignore, ignore_index,
                             static_cast<T*>(dlogits)));
        count_launch(1);
        return CHXQ_OK;
    });
}
