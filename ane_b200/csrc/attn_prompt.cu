// attn_prompt.cu -- causal attention over packed prompts (the tile loop is
// attn_sm100.cuh).
//
// Many items: they are ordered by the number of key tiles they need, most first,
// and dealt out to the blocks there and back again, so that every block's sum of
// tiles is about the same without a queue in memory.
//
// Few long items for the chip's 148 SMs (a block of a prompt behind a long history):
// all items' key tiles are laid end to end and cut into equal spans,
// one per block.  An item cut by a boundary leaves unnormalised parts (m, l, o),
// which join_kernel adds in the order of the keys.
#include "attn_sm100.cuh"

namespace ane_b200 {
namespace {
using namespace attn;

constexpr uint32_t kMaxSeq = 1024;
constexpr uint32_t kSpanBlocks = 148;

struct Params {
    uint32_t n_seq, heads, kv_heads, group, dim, total_q, total_k, out_dtype;
    uint32_t tile_tokens;  // query tokens per tile: 128 / group
    uint32_t spans;        // blocks that share the keys' line; 0: whole items are dealt out
    float scale2;
    ane_rows out;
    const int32_t* cu_q;
    const int32_t* cu_k;
    float* lse;
    int* err;
    float *po, *pm;        // spans: parts, two per block (one that continues an item, one that begins it)
    struct Cut* cuts;      // spans: per block the item that it begins and does not end
    uint32_t per_magic, per_shift;  // x / w, w = 2 * tile_tokens, is (x * magic >> 32) >> shift for x < 2^31:
                                    // magic = ceil(2^(32 + shift) / w), 2^shift < w <= 2^(shift + 1)
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
__device__ __forceinline__ int items_before(const Params& p, int token) {  // token >= 0
    return (int)(__umulhi((uint32_t)token, p.per_magic) >> p.per_shift);
}
// Items of a sequence (per head) that need at least L key tiles.  Item i ends
// with query token min((i + 1) * w, lq), whose last key is lk - lq + that.
__device__ __forceinline__ int items_from_level(const Params& p, const Seq& s, int L) {
    if (s.lq == 0) return 0;
    const int last = items_before(p, s.lq - 1), before = kBigKeys * (L - 1);
    if (L <= 0) return last + 1;
    if (s.lk <= before) return 0;
    return last + 1 - min(items_before(p, max(before - (s.lk - s.lq), 0)), last);
}

// Room of a sequence's first k items (per head) on the line, in key tokens: what
// the item's last query sees, and kItemCost for its start and end.
constexpr int kItemCost = 384;
__device__ __forceinline__ int64_t room(const Seq& s, int k, int w) {
    const int64_t off = s.lk - s.lq, z = off < 0 ? min((int64_t)k, -off / w) : 0;  // the first z see nothing
    return (int64_t)k * kItemCost + (k - z) * off + w * (((int64_t)k * (k + 1) - z * (z + 1)) / 2);
}

// An item and a position on its part of the line.
struct Place {
    BigItem it;       // whole
    int64_t at, size; // the item begins here; its room
    int tiles;        // key tiles (of the query tile that needs more)
    // the key tile that a position cuts at
    __device__ int cut(int64_t pos) const {
        const int64_t z = pos - at;
        return z <= 0 ? 0 : z >= size ? tiles : (int)(z * tiles / size);
    }
};

struct Cut {
    Place place;
    int64_t span;  // length of a span; 0: no such item
};

struct PromptJob {
    const Params& p;
    Seq mine;  // of a searching warp: sequence `lane`, the first 32 of them kept
    int level, above;        // whole items: `above` of them need at least `level` key tiles, all dealt out
    int64_t pos, end, span;  // spans: what is left of this block's, and their length

    __device__ void start() const {}
    __device__ Seq get(uint32_t s) const { return s < 32 ? mine : sequence(p, s); }
    __device__ void fill(BigItem& it, const Seq& q, int first) const {
        const int tt = (int)p.tile_tokens;
        it.q_token = q.q0 + first;
        it.tokens = min(2 * tt, q.lq - first);
        it.k0 = q.k0;
        it.lk = q.lk;
        it.see = q.lk - q.lq + first;
        it.head = 0;
        for (int t = 0; t < 2; t++) {
            const int tok = min(it.tokens, (t + 1) * tt);
            it.end[t] = tok <= t * tt ? 0 : (max(0, min(it.lk, it.see + tok)) + kBigKeys - 1) / kBigKeys;
        }
    }
    __device__ static Seq broadcast(Seq q, int lane) {
        q.q0 = __shfl_sync(0xffffffffu, q.q0, lane);
        q.k0 = __shfl_sync(0xffffffffu, q.k0, lane);
        q.lq = __shfl_sync(0xffffffffu, q.lq, lane);
        q.lk = __shfl_sync(0xffffffffu, q.lk, lane);
        return q;
    }
    // Item number `o` in order of falling key tiles, `o` not below the last
    // call's: the search goes on from there (from scratch it took 3 to 6 us next to
    // busy warps, longer than a short item).  A whole warp.
    __device__ BigItem find(int o) {
        const int lane = threadIdx.x & 31, w = 2 * (int)p.tile_tokens;
        auto count = [&](int L) {
            int c = 0;
            for (uint32_t s = lane; s < p.n_seq; s += 32) c += items_from_level(p, get(s), L);
            return (int)__reduce_add_sync(0xffffffffu, c);
        };
        BigItem it{};
        it.head = -1;
        // the level that counts more than `o` items, below one that does not
        int hi = level, below = above, lo;
        for (int step = 1;; step *= 2) {
            if (hi <= 0) return it;
            lo = max(hi - step, 0);
            const int c = count(lo);
            if (c > o) break;
            hi = lo;
            below = c;
        }
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1, c = count(mid);
            if (c > o) {
                lo = mid;
            } else {
                hi = mid;
                below = c;
            }
        }
        level = hi;
        above = below;
        int r = o - below;
        for (uint32_t s0 = 0; s0 < p.n_seq; s0 += 32) {
            const Seq q = get(s0 + lane);
            const int a = items_from_level(p, q, lo), b = items_from_level(p, q, hi);
            int sum = a - b;
            for (int d = 1; d < 32; d <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += t;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, sum > r);
            if (hit) {
                const int l = __ffs((int)hit) - 1;
                const Seq one = broadcast(q, l);
                const int last = items_before(p, max(one.lq - 1, 0));
                const int x = last + 1 - __shfl_sync(0xffffffffu, a, l) + r - __shfl_sync(0xffffffffu, sum - (a - b), l);
                fill(it, one, min(max(x, 0), last) * w);  // (sums pass 2^31 only for ranges that overlap)
                return it;
            }
            r -= __shfl_sync(0xffffffffu, sum, 31);
        }
        return it;
    }
    // Length of the line.  A whole warp.
    __device__ int64_t line() const {
        const int lane = threadIdx.x & 31, w = 2 * (int)p.tile_tokens;
        int64_t c = 0;
        for (uint32_t s = lane; s < p.n_seq; s += 32) {
            const Seq q = get(s);
            c += room(q, (q.lq + w - 1) / w, w);
        }
        for (int d = 16; d; d >>= 1) c += __shfl_xor_sync(0xffffffffu, c, d);
        return c * p.kv_heads;
    }
    // The item at a position of the line (below its length).  A whole warp.
    __device__ Place locate(int64_t at) const {
        const int lane = threadIdx.x & 31, w = 2 * (int)p.tile_tokens;
        Place r{};
        r.it.head = -1;
        int64_t base = 0;
        for (uint32_t s0 = 0; s0 < p.n_seq; s0 += 32) {
            const Seq q = get(s0 + lane);
            const int64_t c = room(q, (q.lq + w - 1) / w, w) * p.kv_heads;
            int64_t sum = c;
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t t = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += t;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, base + sum > at);
            if (hit) {
                const int l = __ffs((int)hit) - 1;
                const Seq one = broadcast(q, l);
                base += __shfl_sync(0xffffffffu, sum - c, l);
                int lo = 0, hi = (one.lq + w - 1) / w;  // room(lo) <= x < room(hi)
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (room(one, mid, w) * p.kv_heads <= at - base) lo = mid; else hi = mid;
                }
                const int64_t before = room(one, lo, w);
                r.size = room(one, lo + 1, w) - before;
                fill(r.it, one, lo * w);
                r.it.head = (int)((at - base - before * p.kv_heads) / r.size);
                r.at = base + before * p.kv_heads + r.it.head * r.size;
                r.tiles = max(r.it.end[0], r.it.end[1]);
                return r;
            }
            base += __shfl_sync(0xffffffffu, sum, 31);
        }
        return r;
    }
    __device__ BigItem item(int i) {
        if (i == 0) {
            mine = sequence(p, threadIdx.x & 31);
            if (p.spans) {
                const int64_t all = line();
                span = (all + p.spans - 1) / p.spans;
                pos = min(all, span * blockIdx.x);
                end = min(all, span * (blockIdx.x + 1));
                if ((threadIdx.x & 31) == 0) p.cuts[blockIdx.x].span = 0;
            } else {
                level = above = 0;
                for (uint32_t s = threadIdx.x & 31; s < p.n_seq; s += 32) level = max(level, get(s).lk);
                level = __reduce_max_sync(0xffffffffu, level) / kBigKeys + 2;
            }
        }
        BigItem it{};
        it.head = -1;
        if (!p.spans) {
            const uint64_t w = (uint64_t)i * gridDim.x + (i & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
            if (w < 0x7fffffffu) it = find((int)((uint32_t)w / p.kv_heads));
            if (it.head >= 0) it.head = (int)((uint32_t)w % p.kv_heads);
            it.slot = -1;
            return it;
        }
        while (pos < end) {
            const Place r = locate(pos);
            const int b = r.cut(pos), e = r.cut(end);
            const bool starts = pos == r.at;
            pos = r.at + r.size;
            if (b == e && !(r.tiles == 0 && starts)) continue;
            it = r.it;
            it.begin = b;
            for (int t = 0; t < 2; t++) it.end[t] = min(it.end[t], e);
            it.slot = b == 0 && e == r.tiles ? -1 : 2 * (int)blockIdx.x + (b == 0);
            if (b == 0 && e < r.tiles && (threadIdx.x & 31) == 0) p.cuts[blockIdx.x] = Cut{r, span};
            return it;
        }
        return it;
    }
    __device__ int box_keys() const { return kBigKeys; }
    __device__ int2 coord(const BigItem& it, int key) const { return make_int2(it.k0 + key, 0); }
    __device__ int visible(const BigItem& it, int token) const { return max(0, min(it.lk, it.see + token + 1)); }

    // Where row `row` of an item's tile goes in out, as bytes.
    __device__ uint8_t* out_row(const BigItem& it, int row, int token) const {
        return static_cast<uint8_t*>(p.out.data) +
               (((size_t)it.q_token + token) * p.out.token_stride + (it.head * p.group + row % p.group) * p.out.head_stride) *
                   (p.out_dtype == ANE_DTYPE_F32 ? 4 : 2);
    }
    __device__ void write_lse(const BigItem& it, int row, int token, float m, float l, float shift) const {
        if (p.lse)
            p.lse[((size_t)it.q_token + token) * p.heads + it.head * p.group + row % p.group] =
                l == 0.0f ? kNegInf : (m + log2f(l) - shift) * kLn2;
    }
    __device__ void result(const BigItem& it, int row, int token, float m, float l, float shift, uint8_t*& dst,
                           float& factor) const {
        if (it.slot >= 0) {
            const size_t at = (size_t)it.slot * 2 * kBigRows + (token >= (int)p.tile_tokens ? kBigRows : 0) + row;
            *reinterpret_cast<float2*>(p.pm + at * 2) = make_float2(m, l);
            dst = reinterpret_cast<uint8_t*>(p.po + at * p.dim);
            factor = l == 0.0f ? 0.0f : 1.0f;
            return;
        }
        dst = out_row(it, row, token);
        factor = l == 0.0f ? 0.0f : 1.0f / l;
        write_lse(it, row, token, m, l, shift);
    }
    __device__ uint32_t dim() const { return p.dim; }
    __device__ uint32_t out_dtype(const BigItem& it) const { return it.slot >= 0 ? ANE_DTYPE_F32 : p.out_dtype; }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kBigThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const Params p) {
    PromptJob job{p};
    big_attention<T, DP>(&map_q, &map_k, &map_v, p.group, p.scale2, p.err, job);
}

// Block (c, x): if block c of prompt_kernel began an item without ending it, 32
// of its rows are joined, four per warp.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const Params p) {
    __shared__ BigItem whole;
    __shared__ int parts, slot[kSpanBlocks];
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        const Cut c = p.cuts[blockIdx.x];
        int n = 0;
        if (c.span) {
            whole = c.place.it;
            slot[n++] = 2 * blockIdx.x + 1;
            // the spans after this one that hold a part, to the item's end
            int64_t at = c.span * (blockIdx.x + 1);
            int cut = c.place.cut(at);
            for (uint32_t x = blockIdx.x + 1; cut < c.place.tiles && x < p.spans; x++) {
                at += c.span;
                const int e = c.place.cut(at);
                if (e > cut) slot[n++] = 2 * x;
                cut = e;
            }
        }
        parts = n;
    }
    __syncthreads();
    if (parts == 0) return;
    const bool on = (uint32_t)lane * 4 < p.dim;
    const int flat = blockIdx.y * 32 + warp * 4, t = flat / kBigRows, row = flat % kBigRows;
    float m[4], l[4];
    float4 o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) m[i] = kNegInf, l[i] = 0.0f, o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int x = 0; x < parts; x++) {
        float2 y[4];
        float4 v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {  // rows that do not exist hold anything: their sums are not used
            const size_t at = (size_t)slot[x] * 2 * kBigRows + flat + i;
            y[i] = __ldcg(reinterpret_cast<const float2*>(p.pm + at * 2));
            v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (on) v[i] = __ldcg(reinterpret_cast<const float4*>(p.po + at * p.dim + lane * 4));
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float mn = fmaxf(m[i], y[i].x), base = mn == kNegInf ? 0.0f : mn;
            const float ca = exp2_fast(m[i] - base), cb = exp2_fast(y[i].x - base);
            m[i] = mn;
            l[i] = l[i] * ca + y[i].y * cb;
            o[i].x = o[i].x * ca + v[i].x * cb;
            o[i].y = o[i].y * ca + v[i].y * cb;
            o[i].z = o[i].z * ca + v[i].z * cb;
            o[i].w = o[i].w * ca + v[i].w * cb;
        }
    }
    const PromptJob job{p};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int token = t * (int)p.tile_tokens + (row + i) / (int)p.group;
        if (row + i >= (int)(p.tile_tokens * p.group) || token >= whole.tokens) continue;
        const bool empty = l[i] == 0.0f;
        const float f = empty ? 0.0f : 1.0f / l[i];
        uint8_t* dst = job.out_row(whole, row + i, token);
        if (on) {
            store2(dst, lane * 4, p.out_dtype, empty ? 0.0f : o[i].x * f, empty ? 0.0f : o[i].y * f);
            store2(dst, lane * 4 + 2, p.out_dtype, empty ? 0.0f : o[i].z * f, empty ? 0.0f : o[i].w * f);
        }
        if (lane == 0) job.write_lse(whole, row + i, token, m[i], l[i], Type<T>::kShift);
    }
}

// Spans, or 0 for whole items.  The lengths are on the device; the host knows their
// means.  Where most keys are history, items are alike, and whole ones leave blocks
// idle in their last wave: that has to outweigh the parts and their join (ten key
// tiles a block) and that spans share K and V less (a fifth).  Without such a history
// an item's length is anything up to the longest, and whole ones fill the blocks.
// us whole and as spans, 32/8 heads x 128: 1 block of 1, 200, 500, 1000 tokens behind
// 8000 115 and 49, 117 and 53, 140 and 84, 152 and 152; 4 of 1, 200, 500 behind 8000 127
// and 56, 125 and 137, 232 and 294; 1 of 1, 200 behind 1000 21 and 29, 25 and 34; prompts
// without history: 1 of 1000 tokens 25 and 39, of 2112 41 and 62, 4 of 500 23 and 41.
// Over 926 calls of 1 to 8 sequences the choice costs 0.6 % of the better one's time on
// average, 32 % at most (8/1 heads, 64 tokens behind 3000).
constexpr int64_t kSpanKeys = 10 * kBigKeys;
uint32_t spans_for(uint32_t n_seq, uint32_t group, uint32_t kv_heads, uint32_t total_q, uint32_t total_k) {
    if (n_seq == 0 || total_q == 0) return 0;
    const int64_t queries = ceil_div(total_q, n_seq), keys = total_k / n_seq;
    if (2 * queries > keys) return 0;
    const int64_t items = (int64_t)ceil_div((size_t)queries, 2 * (kBigRows / group)) * n_seq * kv_heads;
    const int64_t waves = (int64_t)ceil_div((size_t)items, kSpanBlocks);
    // times 5 and the number of blocks
    return (waves * 5 * kSpanBlocks - 6 * items) * (keys - queries / 2) > kSpanKeys * 5 * kSpanBlocks ? kSpanBlocks : 0;
}

template <typename T, int DP>
int launch(const CUtensorMap (&map)[3], const Params& p, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    int rc = set_max_dynamic_smem(prompt_kernel<T, DP>, (int)big_smem_bytes<DP>(), done);
    if (rc) return rc;
    uint64_t blocks = p.spans;
    if (!blocks) {
        const uint64_t items = (uint64_t)(p.total_q / (2 * p.tile_tokens) + p.n_seq) * p.kv_heads;
        blocks = items < (uint64_t)num_sms() ? items : (uint64_t)num_sms();
    }
    rc = launch_pdl(prompt_kernel<T, DP>, dim3((uint32_t)blocks), dim3(kBigThreads), big_smem_bytes<DP>(), s, map[0],
                    map[1], map[2], p);
    if (rc || !p.spans) return rc;
    return launch_pdl(join_kernel<T>, dim3(p.spans, 2 * kBigRows / 32), dim3(256), 0, s, p);
}

}  // namespace
}  // namespace ane_b200

using namespace ane_b200;

extern "C" size_t ane_attn_prompt_workspace_size(uint32_t n_seq, uint32_t heads, uint32_t kv_heads, uint32_t dim,
                                                 uint32_t total_q, uint32_t total_k) {
    if (kv_heads == 0 || heads < kv_heads || heads % kv_heads || heads / kv_heads > 64) return 0;
    return round_up((size_t)spans_for(n_seq, heads / kv_heads, kv_heads, total_q, total_k) *
                        (4 * kBigRows * (dim + 2) * 4 + sizeof(Cut)), 256);
}

extern "C" int ane_attn_prompt_dev(uint32_t dtype, uint32_t n_seq, uint32_t heads, uint32_t kv_heads, uint32_t dim,
                                   uint32_t total_q, uint32_t total_k, float scale, const ane_rows* q,
                                   const ane_rows* k, const ane_rows* v, const int32_t* cu_q, const int32_t* cu_k,
                                   uint32_t out_dtype, const ane_rows* out, float* lse, void* workspace,
                                   size_t workspace_bytes, void* stream) {
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
    const uint32_t group = heads / kv_heads;
    const size_t need = ane_attn_prompt_workspace_size(n_seq, heads, kv_heads, dim, total_q, total_k);
    ANE_ARG_CHECK(need == 0 || (workspace && (uintptr_t)workspace % 256 == 0 && workspace_bytes >= need),
                  "attn_prompt: workspace must be 256-byte aligned and of ane_attn_prompt_workspace_size bytes");
    if ((rc = require_sm100())) return rc;
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
             spans_for(n_seq, group, kv_heads, total_q, total_k), scale * attn::kLog2e, *out, cu_q,
             cu_k ? cu_k : cu_q, lse, device_timeout_flag()};
    const uint32_t w = 2 * p.tile_tokens;
    while ((2u << p.per_shift) < w) p.per_shift++;
    p.per_magic = (uint32_t)(((1ull << (32 + p.per_shift)) + w - 1) / w);
    if (p.spans) {
        p.po = static_cast<float*>(workspace);
        p.pm = p.po + (size_t)p.spans * 4 * kBigRows * dim;
        p.cuts = reinterpret_cast<Cut*>(p.pm + (size_t)p.spans * 4 * kBigRows * 2);
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == ANE_DTYPE_F16)
        rc = dim <= 64 ? launch<__half, 64>(map, p, s) : launch<__half, 128>(map, p, s);
    else
        rc = dim <= 64 ? launch<__nv_bfloat16, 64>(map, p, s) : launch<__nv_bfloat16, 128>(map, p, s);
    return rc ? rc : ok();
}
