// attn_core.cuh -- what the attention kernels share: element types, the
// exponential, argument checks.
//
// For a row with scores s_j = scale * q . k_j the kernels keep, over the tiles
// of keys seen so far, a reference m near max_j s_j, l = sum_j exp(s_j - m) and
// o = sum_j exp(s_j - m) v_j; when m moves, l and o are multiplied by
// exp(m_old - m_new).  Everything is in base 2 (scale * log2 e folded into one
// product per score).  l and o are fp32; only the weights exp(s_j - m) are
// rounded to 16 bits, because the tensor cores multiply them with v in v's type
// (relative error at most 2^-8 per weight for BF16, 2^-11 for F16: what v itself
// carries).  F16 weights are kept 2^6 times larger (l alike, so the factor
// cancels): below 2^-14 F16 loses bits, and a long flat context has many small
// weights.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ane_internal.cuh"
#include "sm100_ptx.cuh"

namespace ane_b200 {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -INFINITY;

template <typename T>
struct Type;
template <>
struct Type<__half> {
    static constexpr float kShift = 6.0f;  // log2 of the weights' factor
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <>
struct Type<__nv_bfloat16> {
    static constexpr float kShift = 0.0f;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// Two adjacent results of a row (columns c, c + 1).
__device__ __forceinline__ void store2(void* row, uint32_t c, uint32_t out_dtype, float a, float b) {
    if (out_dtype == ANE_DTYPE_F32)
        *reinterpret_cast<float2*>(static_cast<float*>(row) + c) = make_float2(a, b);
    else
        *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(row) + c) =
            out_dtype == ANE_DTYPE_F16 ? Type<__half>::pack(a, b) : Type<__nv_bfloat16>::pack(a, b);
}

// ------------------------------------------------------------ argument checks
inline int check_shapes(const char* who, uint32_t dtype, uint32_t out_dtype, uint32_t heads, uint32_t kv_heads,
                        uint32_t dim, float scale) {
    const std::string w = who;
    ANE_ARG_CHECK(dtype == ANE_DTYPE_F16 || dtype == ANE_DTYPE_BF16, w + ": dtype must be F16 or BF16");
    ANE_ARG_CHECK(out_dtype == dtype || out_dtype == ANE_DTYPE_F32, w + ": out_dtype must be the inputs' type or F32");
    ANE_ARG_CHECK(dim >= 8 && dim <= 128 && dim % 8 == 0, w + ": dim must be a multiple of 8, 8 to 128");
    ANE_ARG_CHECK(kv_heads > 0 && kv_heads <= 1024 && heads >= kv_heads && heads % kv_heads == 0 && heads / kv_heads <= 64,
                  w + ": heads must be a multiple of kv_heads, at most 64 times as many");
    ANE_ARG_CHECK(scale > 0.0f && scale <= 1e30f, w + ": scale must be positive");
    return ANE_OK;
}
inline int check_rows(const char* who, const ane_rows* r, size_t elem) {
    ANE_ARG_CHECK(r->data && (uintptr_t)r->data % 16 == 0 && r->token_stride * elem % 16 == 0 &&
                      r->head_stride * elem % 16 == 0,
                  std::string(who) + ": rows must be 16-byte aligned with strides of whole 16 bytes");
    return ANE_OK;
}

}  // namespace attn
}  // namespace ane_b200
