// attn_prompt.cu -- causal attention over packed prompts (the tile loop is
// attn_sm100.cuh).  Items are ordered by the number of key tiles they need, most
// first, and dealt out to the blocks there and back again, so that every block's
// sum of tiles is about the same without a queue in memory.
#include "attn_sm100.cuh"

namespace ane_b200 {
namespace {
using namespace attn;

constexpr uint32_t kMaxSeq = 1024;

struct Params {
    uint32_t n_seq, heads, kv_heads, group, dim, total_q, total_k, out_dtype;
    uint32_t tile_tokens;  // query tokens per tile: 128 / group
    float scale2;
    ane_rows out;
    const int32_t* cu_q;
    const int32_t* cu_k;
    float* lse;
    int* err;
};

struct Seq {
    int q0, k0, lq, lk;
};
// Counts that point outside the buffers are cut to them: nothing is read or
// written out of range whatever cu_q and cu_k hold.
__device__ __forceinline__ Seq sequence(const Params& p, uint32_t s) {
    Seq r{0, 0, 0, 0};
    if (s >= p.n_seq) return r;
    r.q0 = p.cu_q[s];
    r.k0 = p.cu_k[s];
    r.lq = min(p.cu_q[s + 1], (int)p.total_q) - r.q0;
    r.lk = max(0, min(p.cu_k[s + 1], (int)p.total_k) - r.k0);
    if (r.q0 < 0 || r.k0 < 0 || r.lq < 0) r.lq = 0;
    return r;
}
// Items of a sequence (per head) that need at least L key tiles.  Item i ends
// with query token min((i + 1) * w, lq), whose last key is lk - lq + that.
__device__ __forceinline__ int items_from_level(const Seq& s, int L, int w) {
    const int n = (s.lq + w - 1) / w;
    if (n == 0 || L <= 0) return n;
    const int before = kBigKeys * (L - 1);
    if (s.lk <= before) return 0;
    const int x = before - (s.lk - s.lq);
    return n - (x < 0 ? 0 : min(x / w, n - 1));
}

struct PromptJob {
    const Params& p;
    Seq mine;  // of warp 11: sequence `lane`, the first 32 of them kept

    __device__ Seq get(uint32_t s) const { return s < 32 ? mine : sequence(p, s); }
    // Item number `o` in order of falling key tiles.  A whole warp.
    __device__ BigItem find(int o) {
        const int lane = threadIdx.x & 31, w = 2 * (int)p.tile_tokens;
        if (mine.lq < 0) mine = sequence(p, lane);
        auto count = [&](int L) {
            int c = 0;
            for (uint32_t s = lane; s < p.n_seq; s += 32) c += items_from_level(get(s), L, w);
            return (int)__reduce_add_sync(0xffffffffu, c);
        };
        BigItem it{};
        it.head = -1;
        if (count(0) <= o) return it;
        int lo = 0, hi = (int)(p.total_k / kBigKeys) + 2;  // count(lo) > o >= count(hi)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (count(mid) > o) lo = mid; else hi = mid;
        }
        int r = o - count(hi);
        for (uint32_t s0 = 0; s0 < p.n_seq; s0 += 32) {
            const Seq q = get(s0 + lane);
            const int a = items_from_level(q, lo, w), b = items_from_level(q, lo + 1, w);
            int sum = a - b;
            for (int d = 1; d < 32; d <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += t;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, sum > r);
            if (hit) {
                const int l = __ffs((int)hit) - 1;
                const int lq = __shfl_sync(0xffffffffu, q.lq, l), n = (lq + w - 1) / w;
                const int first = (n - __shfl_sync(0xffffffffu, a, l) + r - __shfl_sync(0xffffffffu, sum - (a - b), l)) * w;
                it.q_token = __shfl_sync(0xffffffffu, q.q0, l) + first;
                it.tokens = min(w, lq - first);
                it.k0 = __shfl_sync(0xffffffffu, q.k0, l);
                it.lk = __shfl_sync(0xffffffffu, q.lk, l);
                it.see = it.lk - lq + first;
                it.head = 0;
                for (int t = 0; t < 2; t++) {
                    const int tok = min(it.tokens, (t + 1) * (int)p.tile_tokens);
                    it.end[t] = tok <= t * (int)p.tile_tokens
                                    ? 0
                                    : (max(0, min(it.lk, it.see + tok)) + kBigKeys - 1) / kBigKeys;
                }
                return it;
            }
            r -= __shfl_sync(0xffffffffu, sum, 31);
        }
        return it;
    }
    __device__ BigItem item(int i) {
        const uint64_t w = (uint64_t)i * gridDim.x + (i & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        BigItem it{};
        it.head = -1;
        if (w < 0x7fffffffu) it = find((int)(w / p.kv_heads));
        if (it.head >= 0) it.head = (int)(w % p.kv_heads);
        return it;
    }
    __device__ int box_keys() const { return kBigKeys; }
    __device__ int2 coord(const BigItem& it, int key) const { return make_int2(it.k0 + key, 0); }
    __device__ int visible(const BigItem& it, int token) const { return max(0, min(it.lk, it.see + token + 1)); }

    __device__ void result(const BigItem& it, int row, int token, float m, float l, float shift, uint8_t*& dst,
                           float& factor) const {
        const uint32_t head = it.head * p.group + row % p.group;
        const size_t q = (size_t)it.q_token + token;
        dst = static_cast<uint8_t*>(p.out.data) +
              (q * p.out.token_stride + head * p.out.head_stride) * (p.out_dtype == ANE_DTYPE_F32 ? 4 : 2);
        factor = l == 0.0f ? 0.0f : 1.0f / l;
        if (p.lse) p.lse[q * p.heads + head] = l == 0.0f ? kNegInf : (m + log2f(l) - shift) * kLn2;
    }
    __device__ uint32_t dim() const { return p.dim; }
    __device__ uint32_t out_dtype() const { return p.out_dtype; }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kBigThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const Params p) {
    PromptJob job{p, {0, 0, -1, 0}};
    big_attention<T, DP>(&map_q, &map_k, &map_v, p.group, p.scale2, p.err, job);
}

template <typename T, int DP>
int launch(const CUtensorMap (&map)[3], const Params& p, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    int rc = set_max_dynamic_smem(prompt_kernel<T, DP>, (int)big_smem_bytes<DP>(), done);
    if (rc) return rc;
    // the lengths are on the device: as many items as total_q tokens in n_seq pieces can make
    const uint64_t items = (uint64_t)(p.total_q / (2 * p.tile_tokens) + p.n_seq) * p.kv_heads;
    const uint64_t blocks = items < (uint64_t)num_sms() ? items : (uint64_t)num_sms();
    return launch_pdl(prompt_kernel<T, DP>, dim3((uint32_t)blocks), dim3(kBigThreads), big_smem_bytes<DP>(), s, map[0],
                      map[1], map[2], p);
}

}  // namespace
}  // namespace ane_b200

using namespace ane_b200;

extern "C" int ane_attn_prompt_dev(uint32_t dtype, uint32_t n_seq, uint32_t heads, uint32_t kv_heads, uint32_t dim,
                                   uint32_t total_q, uint32_t total_k, float scale, const ane_rows* q,
                                   const ane_rows* k, const ane_rows* v, const int32_t* cu_q, const int32_t* cu_k,
                                   uint32_t out_dtype, const ane_rows* out, float* lse, void* stream) {
    int rc = attn::check_shapes("attn_prompt", dtype, out_dtype, heads, kv_heads, dim, scale);
    if (rc) return rc;
    ANE_ARG_CHECK(n_seq <= kMaxSeq, "attn_prompt: at most 1024 sequences");
    ANE_ARG_CHECK(total_q <= 0x7fff0000u && total_k <= 0x7fff0000u, "attn_prompt: too many tokens");
    ANE_ARG_CHECK(q && k && v && out && (n_seq == 0 || cu_q), "attn_prompt: NULL pointer");
    if (n_seq == 0 || total_q == 0) return (rc = require_sm100()) ? rc : ok();
    if ((rc = attn::check_rows("attn_prompt", q, 2)) ||
        (rc = attn::check_rows("attn_prompt", out, out_dtype == ANE_DTYPE_F32 ? 4 : 2)))
        return rc;
    if (total_k && ((rc = attn::check_rows("attn_prompt", k, 2)) || (rc = attn::check_rows("attn_prompt", v, 2)))) return rc;
    if ((rc = require_sm100())) return rc;
    const uint32_t group = heads / kv_heads;
    const auto type = dtype == ANE_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    CUtensorMap map[3];
    rc = encode_tensor_map_3d(&map[0], type, q->data, {dim, heads, total_q}, {q->head_stride * 2, q->token_stride * 2},
                              {64, group, 128 / group}, CU_TENSOR_MAP_SWIZZLE_128B);
    // without keys the maps are never used, but have to be of something
    const uint32_t keys = total_k ? total_k : 1;
    const ane_rows *mk = total_k ? k : q, *mv = total_k ? v : q;
    if (!rc)
        rc = encode_tensor_map_4d(&map[1], type, mk->data, {dim, kv_heads, keys, 1},
                                  {mk->head_stride * 2, mk->token_stride * 2, mk->token_stride * 2}, {64, 1, 128, 1},
                                  CU_TENSOR_MAP_SWIZZLE_128B);
    if (!rc)
        rc = encode_tensor_map_4d(&map[2], type, mv->data, {dim, kv_heads, keys, 1},
                                  {mv->head_stride * 2, mv->token_stride * 2, mv->token_stride * 2}, {64, 1, 128, 1},
                                  CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    Params p{n_seq, heads, kv_heads, group, dim, total_q, total_k, out_dtype, 128 / group,
             scale * attn::kLog2e, *out, cu_q, cu_k ? cu_k : cu_q, lse, device_timeout_flag()};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == ANE_DTYPE_F16)
        rc = dim <= 64 ? launch<__half, 64>(map, p, s) : launch<__half, 128>(map, p, s);
    else
        rc = dim <= 64 ? launch<__nv_bfloat16, 64>(map, p, s) : launch<__nv_bfloat16, 128>(map, p, s);
    return rc ? rc : ok();
}
