// The float matrix product on the tensor cores: what its two kernels (linear_tile.cuh, linear_pair.cuh) share.
#pragma once

#include <cuda.h>

#include "epilogue_float.cuh"
#include "tc_kernel3.cuh"

namespace chxq {
namespace lin {

using namespace tc;

struct TcArgs {
    int M, O;       // rows of x, rows of w
    int k_blocks;   // K in blocks of 128 bytes
    uint32_t idesc;  // instruction descriptor without its extents
    LinearEpilogue e;
    int vec;  // rows of y and of the residual start on 16-byte boundaries and hold whole groups of 16 bytes
    int* status;
    unsigned long long wait_limit_ns;
    int test_skip_kb;  // K block whose rows of w are not loaded (chxq_tc_test_hooks)
};

// Instruction descriptor of tcgen05.mma kind::f16: 32-bit accumulator, both operands K-major and of one type.
constexpr uint32_t kF16 = 0u, kBf16 = 1u;
inline uint32_t idesc_f16(uint32_t type) {
    return (1u << 4) | (type << 7) | (type << 10);
}
__host__ __device__ constexpr uint32_t idesc_extents(int m, int n) {
    return ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// The same of kind::tf32.
__host__ __device__ constexpr uint32_t idesc_tf32() {
    return (1u << 4) | (2u << 7) | (2u << 10);
}
// D[tmem] (+)= A B^T over eight values of K, A in tensor memory: a row a lane, a value a column.
__device__ __forceinline__ void umma_tf32(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            ".reg .b64 db;\n\t"
            "mov.b64 db, {%2, %3};\n\t"
            "setp.ne.b32 p, %5, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], db, %4, p;\n\t"
            "}\n" ::"r"(tmem_d),
            "r"(tmem_a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
            : "memory");
}

// Sixteen columns of the warp's 32 lanes of tensor memory.
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15]), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// D[tmem] (+)= A B^T over 32 bytes of K of each operand, kind::f16, issued by one thread; PAIR: over a CTA pair (M = 256).
// The tensor core holds the sum in 32 bits but cuts it off after each instruction where an addition would round.  A CTA's K stays in one accumulator all the
// same: with K = 8192 and terms of one sign its sums are 3.0e-5 (bf16) and 4.8e-5 (fp16) too small, a hundred-and-thirtieth and a tenth of the type's
// half step; with normal terms 9.6e-6 off where the sums are about 1 (an fp32 product 1.3e-6).  Chains as in the fp32 tiles would cost a pass of the
// accumulators through registers each for what the output's rounding hides: 8192^3 bf16 is 1.66e-3 off the sums in 64 bits, and so is an fp32 product
// rounded once.
template <bool PAIR>
__device__ __forceinline__ void umma_f16(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile(
                "{\n\t"
                ".reg .pred p;\n\t"
                ".reg .b64 da, db;\n\t"
                "mov.b64 da, {%1, %3};\n\t"
                "mov.b64 db, {%2, %3};\n\t"
                "setp.ne.b32 p, %5, 0;\n\t"
                "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %4, p;\n\t"
                "}\n" ::"r"(tmem_d),
                "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
                : "memory");
    else
        asm volatile(
                "{\n\t"
                ".reg .pred p;\n\t"
                ".reg .b64 da, db;\n\t"
                "mov.b64 da, {%1, %3};\n\t"
                "mov.b64 db, {%2, %3};\n\t"
                "setp.ne.b32 p, %5, 0;\n\t"
                "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t"
                "}\n" ::"r"(tmem_d),
                "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
                : "memory");
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src),
                 "r"(c0), "r"(c1)
                 : "memory");
}

__device__ __forceinline__ void bar_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Waits for this thread's outstanding TMEM loads, with their registers passed through as in tmem_ld_wait16.
__device__ __forceinline__ void tmem_ld_wait32(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

// A barrier over `threads` threads that tells each of them whether `ok` held for all.
__device__ __forceinline__ bool bar_all(int id, int threads, bool ok) {
    uint32_t r;
    asm volatile(
            "{\n\t"
            ".reg .pred p, q;\n\t"
            "setp.ne.u32 p, %3, 0;\n\t"
            "bar.red.and.pred q, %1, %2, p;\n\t"
            "selp.u32 %0, 1, 0, q;\n\t"
            "}\n"
            : "=r"(r)
            : "r"(id), "r"(threads), "r"((uint32_t)ok)
            : "memory");
    return r != 0;
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float2 unpack16(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack16<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack16<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

}  // namespace lin
}  // namespace chxq
