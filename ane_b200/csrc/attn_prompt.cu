// attn_prompt.cu -- causal attention over packed prompts.
#include "attn_core.cuh"

namespace ane_b200 {
namespace {
using namespace attn;

constexpr uint32_t kMaxSeq = 1024;

struct Params {
    uint32_t n_seq, heads, kv_heads, group, dim, total_q, total_k, out_dtype;
    uint32_t tile_tokens;  // query tokens per tile: its rows are (token, head of the group)
    float scale2;
    ane_rows q, k, v, out;
    const int32_t* cu_q;
    const int32_t* cu_k;
    float* lse;
};

// One block: 64 rows (64 / group query tokens x the heads of one key/value head).
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) prompt_kernel(const Params p) {
    constexpr int STAGES = 3;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int where[2];
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    if (threadIdx.x < 32) {  // sequence and tile of this block
        int base = 0, seq = -1, tile = 0;
        for (uint32_t s0 = 0; s0 < p.n_seq && seq < 0; s0 += 32) {
            const uint32_t s = s0 + threadIdx.x;
            const int n = s < p.n_seq ? max(0, p.cu_q[s + 1] - p.cu_q[s]) : 0;
            const int tiles = (n + (int)p.tile_tokens - 1) / (int)p.tile_tokens;
            int sum = tiles;
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, sum, o);
                if ((int)threadIdx.x >= o) sum += t;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, base + sum > (int)blockIdx.x);
            if (hit) {
                const int l = __ffs((int)hit) - 1;
                seq = (int)s0 + l;
                tile = (int)blockIdx.x - (base + __shfl_sync(0xffffffffu, sum - tiles, l));
            }
            base += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (threadIdx.x == 0) where[0] = seq, where[1] = tile;
    }
    __syncthreads();
    const int seq = where[0];
    if (seq < 0) return;
    const int q0 = p.cu_q[seq], k0 = p.cu_k[seq];
    const int lq = min(p.cu_q[seq + 1] - q0, (int)p.total_q - q0);
    const int lk = max(0, min(p.cu_k[seq + 1] - k0, (int)p.total_k - k0));
    if (q0 < 0 || k0 < 0) return;
    const uint32_t h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int first = where[1] * (int)p.tile_tokens;
    Rows<DP> r;
    int tok[2], head[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t row = warp * 16 + lane / 4 + 8 * i;
        tok[i] = first + (int)(row / p.group);
        head[i] = (int)(h * p.group + row % p.group);
        const bool there = row < p.tile_tokens * p.group && tok[i] < lq;
        if (!there) tok[i] = -1;
        r.vis[i] = there ? max(0, min(lk, lk - lq + tok[i] + 1)) : 0;
    }
    auto row_of = [&](int i) {
        return tok[i] < 0 ? nullptr
                          : static_cast<const uint16_t*>(p.q.data) + (size_t)(q0 + tok[i]) * p.q.token_stride +
                                (size_t)head[i] * p.q.head_stride;
    };
    load_q<DP>(r, row_of(0), row_of(1), p.dim);
    const int last = min(first + (int)p.tile_tokens, lq);  // tokens of this tile end here
    const int kend = max(0, min(lk, lk - lq + last));
    const uint8_t* kb = static_cast<const uint8_t*>(p.k.data) + ((size_t)k0 * p.k.token_stride + (size_t)h * p.k.head_stride) * 2;
    const uint8_t* vb = static_cast<const uint8_t*>(p.v.data) + ((size_t)k0 * p.v.token_stride + (size_t)h * p.v.head_stride) * 2;
    const size_t kld = p.k.token_stride * 2, vld = p.v.token_stride * 2;
    run_tiles<T, DP, 4, STAGES>(r, smem, 0, (kend + kTile - 1) / kTile, 0, kend, p.dim, p.scale2,
                                [&](int j, const uint8_t*& k, const uint8_t*& v) {
                                    k = kb + (size_t)j * kld;
                                    v = vb + (size_t)j * vld;
                                });
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if (tok[i] < 0) continue;
        const float inv = r.l[i] > 0.0f ? 1.0f / r.l[i] : (r.l[i] == 0.0f ? 0.0f : r.l[i]);
        uint8_t* row = static_cast<uint8_t*>(p.out.data) +
                       ((size_t)(q0 + tok[i]) * p.out.token_stride + (size_t)head[i] * p.out.head_stride) *
                           (p.out_dtype == ANE_DTYPE_F32 ? 4 : 2);
#pragma unroll
        for (int n = 0; n < DP / 8; n++) {
            const uint32_t c = n * 8 + 2 * (lane & 3);
            if (c < p.dim)
                store2(row, c, p.out_dtype, r.l[i] == 0.0f ? 0.0f : r.o[n][2 * i] * inv,
                       r.l[i] == 0.0f ? 0.0f : r.o[n][2 * i + 1] * inv);
        }
        if (p.lse && (lane & 3) == 0)
            p.lse[(size_t)(q0 + tok[i]) * p.heads + head[i]] =
                r.l[i] == 0.0f ? kNegInf : (r.m[i] + log2f(r.l[i]) - Type<T>::kShift) * kLn2;
    }
}

template <typename T, int DP>
int launch(const Params& p, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    constexpr int smem = 3 * 2 * tile_bytes<DP>();
    int rc = set_max_dynamic_smem(prompt_kernel<T, DP>, smem, done);
    if (rc) return rc;
    const uint32_t tiles = p.total_q / p.tile_tokens + p.n_seq;
    return launch_pdl(prompt_kernel<T, DP>, dim3(tiles, p.kv_heads), dim3(kThreads), smem, s, p);
}

}  // namespace
}  // namespace ane_b200

using namespace ane_b200;

extern "C" int ane_attn_prompt_dev(uint32_t dtype, uint32_t n_seq, uint32_t heads, uint32_t kv_heads, uint32_t dim,
                                   uint32_t total_q, uint32_t total_k, float scale, const ane_rows* q,
                                   const ane_rows* k, const ane_rows* v, const int32_t* cu_q, const int32_t* cu_k,
                                   uint32_t out_dtype, const ane_rows* out, float* lse, void* stream) {
    int rc = attn::check_shapes("attn_prompt", dtype, out_dtype, heads, kv_heads, dim);
    if (rc) return rc;
    ANE_ARG_CHECK(n_seq <= kMaxSeq, "attn_prompt: at most 1024 sequences");
    ANE_ARG_CHECK(total_q <= 0x7fffffffu && total_k <= 0x7fffffffu, "attn_prompt: at most 2^31-1 tokens");
    ANE_ARG_CHECK(q && k && v && out && (n_seq == 0 || cu_q), "attn_prompt: NULL pointer");
    if (n_seq == 0 || total_q == 0) return (rc = require_sm100()) ? rc : ok();
    if ((rc = attn::check_rows("attn_prompt", q, 2)) || (rc = attn::check_rows("attn_prompt", out, out_dtype == ANE_DTYPE_F32 ? 4 : 2)))
        return rc;
    if (total_k && ((rc = attn::check_rows("attn_prompt", k, 2)) || (rc = attn::check_rows("attn_prompt", v, 2)))) return rc;
    if ((rc = require_sm100())) return rc;
    Params p{n_seq, heads, kv_heads, heads / kv_heads, dim, total_q, total_k, out_dtype, 64 / (heads / kv_heads),
             scale * attn::kLog2e, *q, *k, *v, *out, cu_q, cu_k ? cu_k : cu_q, lse};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == ANE_DTYPE_F16)
        rc = dim <= 64 ? launch<__half, 64>(p, s) : launch<__half, 128>(p, s);
    else
        rc = dim <= 64 ? launch<__nv_bfloat16, 64>(p, s) : launch<__nv_bfloat16, 128>(p, s);
    return rc ? rc : ok();
}
