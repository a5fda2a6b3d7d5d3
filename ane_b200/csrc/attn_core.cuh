// attn_core.cuh -- the tile loop of softmax attention on mma.sync, shared by the
// attention kernels: 16 query rows per warp, key/value tiles of 64 tokens.
//
// For a row with scores s_j = scale * q . k_j the kernels keep, over the tiles
// seen so far, m = max_j s_j, l = sum_j exp(s_j - m) and o = sum_j exp(s_j - m)
// v_j; a tile with a larger maximum multiplies l and o by exp(m_old - m_new).
// Everything is in base 2 (scale * log2 e folded into one product per score).
// l and o are fp32; only the weights p_j = exp(s_j - m) are rounded to 16 bits,
// because the tensor cores multiply them with v in v's type (relative error at
// most 2^-8 per weight for BF16, 2^-11 for F16: what v itself carries).  F16
// weights are kept 2^8 times larger than 1-based ones (l alike, so the factor
// cancels): below 2^-14 F16 loses bits, and a long flat context has many small
// weights.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ane_internal.cuh"
#include "sm100_ptx.cuh"

namespace ane_b200 {
namespace attn {

constexpr int kTile = 64;      // tokens per key/value tile
constexpr int kThreads = 128;  // four warps
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -INFINITY;

template <typename T>
struct Type;
template <>
struct Type<__half> {
    static constexpr float kShift = 8.0f;  // log2 of the weights' factor
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
// 16 bytes global -> shared; `bytes` (0 or 16) are read, the rest is zero-filled.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Per-warp state of 16 rows: thread holds rows lane/4 and lane/4 + 8.
template <int DP>
struct Rows {
    uint32_t q[DP / 16][4];
    float o[DP / 8][4];
    float m[2], l[2];
    int vis[2];  // keys that the row sees: token index < vis
};

// Shared-memory tile: 64 rows of DP elements, 16-byte chunks XOR-swizzled by row.
template <int DP>
__device__ __forceinline__ uint32_t tile_off(uint32_t row, uint32_t chunk) {
    return row * (DP * 2) + ((chunk ^ (row & 7)) << 4);
}
template <int DP>
constexpr uint32_t tile_bytes() {
    return kTile * DP * 2;
}

// Query fragments of 16 rows; row pointers NULL for rows that do not exist.
template <int DP>
__device__ __forceinline__ void load_q(Rows<DP>& r, const uint16_t* row0, const uint16_t* row1, uint32_t dim) {
    const uint32_t c = 2 * (threadIdx.x & 3);
#pragma unroll
    for (int kk = 0; kk < DP / 16; kk++) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t e = kk * 16 + half * 8 + c;
            r.q[kk][2 * half] = row0 && e < dim ? *reinterpret_cast<const uint32_t*>(row0 + e) : 0u;
            r.q[kk][2 * half + 1] = row1 && e < dim ? *reinterpret_cast<const uint32_t*>(row1 + e) : 0u;
        }
    }
#pragma unroll
    for (int i = 0; i < DP / 8; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) r.o[i][j] = 0.0f;
    r.m[0] = r.m[1] = kNegInf;
    r.l[0] = r.l[1] = 0.0f;
}

// One warp: tokens tok0 .. tok0 + 8 * NT - 1 of the tile whose first token has
// index j0.
template <typename T, int DP, int NT>
__device__ __forceinline__ void tile_step(Rows<DP>& r, uint32_t ks, uint32_t vs, uint32_t tok0, int j0, float scale2) {
    const uint32_t lane = threadIdx.x & 31, mi = lane >> 3, mr = lane & 7;
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) s[n][j] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; kk++) {
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            uint32_t b[4];
            ldsm4(ks + tile_off<DP>(tok0 + n * 8 + (mi >> 1) * 8 + mr, kk * 2 + (mi & 1)), b);
            Type<T>::mma(s[n], r.q[kk], b[0], b[1]);
            Type<T>::mma(s[n + 1], r.q[kk], b[2], b[3]);
        }
    }
    const int first = j0 + (int)tok0 + 2 * (int)(lane & 3);
    float mx[2] = {kNegInf, kNegInf};
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            // selected, not added: a masked score may be anything, NaN included
            s[n][j] = first + n * 8 + (j & 1) < r.vis[j >> 1] ? s[n][j] * scale2 : kNegInf;
            mx[j >> 1] = fmaxf(mx[j >> 1], s[n][j]);
        }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        const float m = fmaxf(r.m[h], mx[h]);
        const float base = m == kNegInf ? 0.0f : m;  // nothing seen yet: keep exp2(-inf - base) at 0
        const float c = exp2_fast(r.m[h] - base);
        r.m[h] = m;
        r.l[h] *= c;
#pragma unroll
        for (int i = 0; i < DP / 8; i++) {
            r.o[i][2 * h] *= c;
            r.o[i][2 * h + 1] *= c;
        }
        mx[h] = base - Type<T>::kShift;
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            s[n][j] = exp2_fast(s[n][j] - mx[j >> 1]);
            r.l[j >> 1] += s[n][j];
        }
#pragma unroll
    for (int k2 = 0; k2 < NT / 2; k2++) {
        const uint32_t a[4] = {Type<T>::pack(s[2 * k2][0], s[2 * k2][1]), Type<T>::pack(s[2 * k2][2], s[2 * k2][3]),
                               Type<T>::pack(s[2 * k2 + 1][0], s[2 * k2 + 1][1]),
                               Type<T>::pack(s[2 * k2 + 1][2], s[2 * k2 + 1][3])};
#pragma unroll
        for (int n = 0; n < DP / 8; n += 2) {
            uint32_t b[4];
            ldsm4_t(vs + tile_off<DP>(tok0 + k2 * 16 + (mi & 1) * 8 + mr, n + (mi >> 1)), b);
            Type<T>::mma(r.o[n], a, b[0], b[1]);
            Type<T>::mma(r.o[n + 1], a, b[2], b[3]);
        }
    }
}

// Four warps run tiles [t0, t1) of one unit: MW of them along the rows, the
// rest split a tile's tokens.  `row_ptr(token, &k, &v)` gives the addresses of a
// token's rows; tokens at or past `kend` are zero-filled (their weights are 0,
// and 0 * NaN of stale memory would not be).  base: index of tile 0's first
// token.  smem: STAGES stages of a K and a V tile, the block's alone on return.
template <typename T, int DP, int MW, int STAGES, class RowPtr>
__device__ __forceinline__ void run_tiles(Rows<DP>& r, uint8_t* smem, int t0, int t1, int base, int kend, uint32_t dim,
                                          float scale2, RowPtr row_ptr) {
    constexpr int NT = kTile / 8 * MW / 4;
    constexpr int CH = DP / 8;  // 16-byte chunks of a row
    const uint32_t s0 = ptx::smem_u32(smem);
    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t tok0 = (warp / MW) * (NT * 8);
    const uint32_t chunk = threadIdx.x % CH, row0 = threadIdx.x / CH;
    auto load = [&](int t) {
        if (t < t1) {
            const uint32_t st = s0 + (uint32_t)((t - t0) % STAGES) * 2 * tile_bytes<DP>();
#pragma unroll
            for (uint32_t row = row0; row < kTile; row += kThreads / CH) {
                const int j = base + t * kTile + (int)row;
                const uint8_t *k, *v;
                const bool in = j < kend && chunk * 8 < dim;
                row_ptr(in ? j : base, k, v);
                const uint32_t off = tile_off<DP>(row, chunk), bytes = in ? 16u : 0u;
                cp16(st + off, k + (in ? chunk * 16 : 0), bytes);
                cp16(st + tile_bytes<DP>() + off, v + (in ? chunk * 16 : 0), bytes);
            }
        }
        cp_commit();
    };
    for (int t = t0; t < t0 + STAGES - 1; t++) load(t);
    for (int t = t0; t < t1; t++) {
        cp_wait<STAGES - 2>();
        __syncthreads();
        load(t + STAGES - 1);
        const uint32_t st = s0 + (uint32_t)((t - t0) % STAGES) * 2 * tile_bytes<DP>();
        tile_step<T, DP, NT>(r, st, st + tile_bytes<DP>(), tok0, base + t * kTile, scale2);
    }
    cp_wait<0>();
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; h++) {
        r.l[h] += __shfl_xor_sync(0xffffffffu, r.l[h], 1);
        r.l[h] += __shfl_xor_sync(0xffffffffu, r.l[h], 2);
    }
}

// Joins the four warps' states of the same 16 rows (MW == 1) through shared
// memory; afterwards warp 0's Rows hold the whole.
template <int DP>
__device__ __forceinline__ void join_warps(Rows<DP>& r, uint8_t* smem) {
    float* so = reinterpret_cast<float*>(smem);    // [3][16 values... per thread of a warp]
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int W = DP / 2 + 4;  // floats per thread
    if (warp) {
        float* p = so + (warp - 1) * W * 32 + lane;
        p[0] = r.m[0], p[32] = r.m[1], p[64] = r.l[0], p[96] = r.l[1];
#pragma unroll
        for (int i = 0; i < DP / 8; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) p[(4 + i * 4 + j) * 32] = r.o[i][j];
    }
    __syncthreads();
    if (!warp) {
        for (int w = 0; w < 3; w++) {
            const float* p = so + w * W * 32 + lane;
            float ca[2], cb[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float mb = p[32 * h], m = fmaxf(r.m[h], mb), base = m == kNegInf ? 0.0f : m;
                ca[h] = exp2_fast(r.m[h] - base);
                cb[h] = exp2_fast(mb - base);
                r.m[h] = m;
                r.l[h] = r.l[h] * ca[h] + p[32 * (2 + h)] * cb[h];
            }
#pragma unroll
            for (int i = 0; i < DP / 8; i++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    r.o[i][j] = r.o[i][j] * ca[j >> 1] + p[(4 + i * 4 + j) * 32] * cb[j >> 1];
        }
    }
    __syncthreads();
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
