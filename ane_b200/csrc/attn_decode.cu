// attn_decode.cu -- attention of one new token per sequence over a paged cache
// whose sequences share a prefix.
//
// A key/value head's tokens fall into units: the prefix with all of the batch's
// query rows (batch x heads of the group, in row tiles), and each sequence's own
// tokens with its group of rows.  All units' 64-token tiles are laid end to end
// and cut into equal spans, one per block, so that ragged lengths and a single
// long sequence load the chip alike.  A block leaves per unit it met an
// unnormalised (m, l, o); attn_decode_join_kernel adds them per output row, in
// the order of the tiles, so results do not depend on scheduling.
#include "attn_core.cuh"

namespace ane_b200 {
namespace {
using namespace attn;

constexpr uint32_t kMaxBatch = 1024;
constexpr uint32_t kMaxBlocks = 512;

struct Params {
    uint32_t batch, heads, kv_heads, group, dim, out_dtype;
    uint32_t shared, prefix_tiles, row_tiles, row_tile;  // row_tile: rows per prefix unit (16 or 64)
    uint32_t n_slots, max_pages, pages, page_shift;
    float scale2;
    ane_rows q, out;
    const uint8_t *k, *v;
    size_t page_stride, token_stride, head_stride;  // bytes
    const int32_t *tables, *lens, *slots;
    float* lse;
    int32_t* cum;        // [batch + 2]: tiles of sequences before b (per head); [batch + 1]: tiles per block
    float *po, *pm;      // prefix partials: rows x dim; rows x {m, l}
    float *so, *sm;      // the sequences' own
    uint32_t blocks;
};

__device__ __forceinline__ int slot_of(const Params& p, uint32_t b) {
    const int s = p.slots ? p.slots[b] : (int)b;
    return s >= 0 && (uint32_t)s < p.n_slots ? s : -1;
}
__device__ __forceinline__ int len_of(const Params& p, uint32_t b) {
    const int s = slot_of(p, b);
    if (s < 0) return 0;
    const int64_t cap = (int64_t)p.max_pages << p.page_shift;
    return (int)min((int64_t)max(p.lens[s], 0), min(cap, (int64_t)0x7fffffff));
}
__device__ __forceinline__ int own_tiles(const Params& p, int len) {
    return len > (int)p.shared ? (len - (int)p.shared + kTile - 1) / kTile : 0;
}

template <typename T, int DP, int MW>
__device__ void run_unit(const Params& p, uint8_t* smem, uint32_t h, uint32_t b, uint32_t rt, bool prefix, int t0,
                         int t1, size_t slot) {
    constexpr int STAGES = DP == 128 ? 3 : 4;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Rows<DP> r;
    const uint16_t* qrow[2];
    const int rows = prefix ? (int)(p.batch * p.group) - (int)(rt * p.row_tile) : (int)p.group;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int row = (int)((MW == 1 ? 0 : warp * 16) + lane / 4 + 8 * i);
        qrow[i] = nullptr;
        r.vis[i] = 0;
        if (row < rows) {
            const uint32_t flat = prefix ? rt * p.row_tile + row : (uint32_t)row;
            const uint32_t bb = prefix ? flat / p.group : b, g = flat % p.group;
            qrow[i] = static_cast<const uint16_t*>(p.q.data) + (size_t)bb * p.q.token_stride +
                      (size_t)(h * p.group + g) * p.q.head_stride;
            r.vis[i] = len_of(p, bb);
            if (prefix) r.vis[i] = min(r.vis[i], (int)p.shared);
        }
    }
    load_q<DP>(r, qrow[0], qrow[1], p.dim);
    const int s = slot_of(p, prefix ? 0 : b);
    const int32_t* table = p.tables + (size_t)max(s, 0) * p.max_pages;
    const int kend = prefix ? (int)p.shared : len_of(p, b);
    const int base = prefix ? 0 : (int)p.shared;
    const uint8_t *kh = p.k + (size_t)h * p.head_stride, *vh = p.v + (size_t)h * p.head_stride;
    const uint32_t mask = (1u << p.page_shift) - 1u;
    run_tiles<T, DP, MW, STAGES>(r, smem, t0, t1, base, kend, p.dim, p.scale2,
                                 [&](int j, const uint8_t*& k, const uint8_t*& v) {
                                     const uint32_t e = min((uint32_t)j >> p.page_shift, p.max_pages - 1);
                                     uint32_t page = (uint32_t)table[e];
                                     if (page >= p.pages) page = 0;
                                     const size_t off = (size_t)page * p.page_stride + ((uint32_t)j & mask) * p.token_stride;
                                     k = kh + off;
                                     v = vh + off;
                                 });
    if (MW == 1) join_warps<DP>(r, smem);
    if (MW == 1 && warp) return;
    float* o = prefix ? p.po : p.so;
    float* ml = prefix ? p.pm : p.sm;
    const int limit = min(rows, prefix ? (int)p.row_tile : (int)p.group);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int row = (int)((MW == 1 ? 0 : warp * 16) + lane / 4 + 8 * i);
        if (row >= limit) continue;
        const size_t at = slot * (prefix ? p.row_tile : p.group) + row;
        if ((lane & 3) == 0) *reinterpret_cast<float2*>(ml + at * 2) = make_float2(r.m[i], r.l[i]);
#pragma unroll
        for (int n = 0; n < DP / 8; n++) {
            const uint32_t c = n * 8 + 2 * (lane & 3);
            if (c < p.dim) *reinterpret_cast<float2*>(o + at * p.dim + c) = make_float2(r.o[n][2 * i], r.o[n][2 * i + 1]);
        }
    }
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) decode_kernel(const Params p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int cum[kMaxBatch + 1];
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    for (uint32_t b = threadIdx.x; b < p.batch; b += kThreads) cum[b] = own_tiles(p, len_of(p, b));
    __syncthreads();
    if (threadIdx.x < 32) {
        int base = 0;
        for (uint32_t b0 = 0; b0 < p.batch; b0 += 32) {
            const uint32_t b = b0 + threadIdx.x;
            const int c = b < p.batch ? cum[b] : 0;
            int s = c;
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, s, o);
                if ((int)threadIdx.x >= o) s += t;
            }
            if (b < p.batch) cum[b] = base + s - c;
            base += __shfl_sync(0xffffffffu, s, 31);
        }
        if (threadIdx.x == 0) cum[p.batch] = base;
    }
    __syncthreads();
    const int64_t prefix_all = (int64_t)p.prefix_tiles * p.row_tiles * p.kv_heads;
    const int64_t total = prefix_all + (int64_t)cum[p.batch] * p.kv_heads;
    const int64_t per = (total + gridDim.x - 1) / gridDim.x;
    if (blockIdx.x == 0) {
        for (uint32_t b = threadIdx.x; b <= p.batch; b += kThreads) p.cum[b] = cum[b];
        if (threadIdx.x == 0) p.cum[p.batch + 1] = (int32_t)per;
    }
    int64_t at = (int64_t)blockIdx.x * per;
    const int64_t end = min(at + per, total);
    while (at < end) {
        uint32_t h, b = 0, rt = 0;
        int64_t first;
        int n;
        size_t slot;
        const bool prefix = at < prefix_all;
        if (prefix) {
            const uint32_t u = (uint32_t)(at / p.prefix_tiles);
            h = u / p.row_tiles;
            rt = u % p.row_tiles;
            n = (int)p.prefix_tiles;
            first = (int64_t)u * n;
            slot = blockIdx.x + u;
        } else {
            // cum scaled by kv_heads gives each sequence's first tile; its heads follow one another
            const int64_t x = at - prefix_all;
            uint32_t lo = 0, hi = p.batch - 1;
            while (lo < hi) {
                const uint32_t mid = (lo + hi + 1) >> 1;
                if ((int64_t)cum[mid] * p.kv_heads <= x) lo = mid; else hi = mid - 1;
            }
            b = lo;
            n = cum[b + 1] - cum[b];
            h = (uint32_t)((x - (int64_t)cum[b] * p.kv_heads) / n);
            first = prefix_all + (int64_t)cum[b] * p.kv_heads + (int64_t)h * n;
            slot = blockIdx.x + (size_t)b * p.kv_heads + h;
        }
        const int t0 = (int)(at - first), t1 = (int)min((int64_t)n, end - first);
        if (prefix && p.row_tile == 64)
            run_unit<T, DP, 4>(p, smem, h, b, rt, prefix, t0, t1, slot);
        else if (prefix || p.group <= 16)
            run_unit<T, DP, 1>(p, smem, h, b, rt, prefix, t0, t1, slot);
        else
            run_unit<T, DP, 4>(p, smem, h, b, rt, prefix, t0, t1, slot);
        at = first + t1;
    }
}

// One block per (sequence, key/value head): joins the partials of its rows.
template <typename T>
__global__ void __launch_bounds__(kThreads) decode_join_kernel(const Params p) {
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const uint32_t b = blockIdx.x, h = blockIdx.y;
    const int64_t per = p.cum[p.batch + 1];
    const int64_t prefix_all = (int64_t)p.prefix_tiles * p.row_tiles * p.kv_heads;
    const int n = p.cum[b + 1] - p.cum[b];
    const int64_t first = prefix_all + (int64_t)p.cum[b] * p.kv_heads + (int64_t)h * n;
    for (uint32_t g = threadIdx.x / 32; g < p.group; g += kThreads / 32) {
        const uint32_t flat = b * p.group + g, rt = flat / p.row_tile, lane = threadIdx.x & 31;
        const uint32_t u = h * p.row_tiles + rt;
        // spans of blocks that hold partials of this row
        const int64_t pfirst = (int64_t)u * p.prefix_tiles;
        const int pc0 = p.prefix_tiles ? (int)(pfirst / per) : 0;
        const int pc1 = p.prefix_tiles ? (int)((pfirst + p.prefix_tiles - 1) / per) + 1 : 0;
        const int sc0 = n ? (int)(first / per) : 0, sc1 = n ? (int)((first + n - 1) / per) + 1 : 0;
        const size_t prow = (size_t)u * p.row_tile + flat % p.row_tile, srow = ((size_t)b * p.kv_heads + h) * p.group + g;
        float m = kNegInf, l = 0.0f;
        float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int pass = 0; pass < 2; pass++) {
            const int c1 = pass ? sc1 : pc1;
            const float* ml = pass ? p.sm : p.pm;
            const float* po = pass ? p.so : p.po;
            const size_t rows = pass ? p.group : p.row_tile, row = pass ? srow : prow;
            for (int c = pass ? sc0 : pc0; c < c1; c++) {
                const size_t at = (size_t)c * rows + row;
                const float2 x = *reinterpret_cast<const float2*>(ml + at * 2);
                const float mn = fmaxf(m, x.x), base = mn == kNegInf ? 0.0f : mn;
                const float ca = exp2_fast(m - base), cb = exp2_fast(x.x - base);
                m = mn;
                l = l * ca + x.y * cb;
                if (lane * 4 < p.dim) {
                    const float4 v = *reinterpret_cast<const float4*>(po + at * p.dim + lane * 4);
                    o[0] = o[0] * ca + v.x * cb;
                    o[1] = o[1] * ca + v.y * cb;
                    o[2] = o[2] * ca + v.z * cb;
                    o[3] = o[3] * ca + v.w * cb;
                }
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint8_t* row = static_cast<uint8_t*>(p.out.data) +
                       ((size_t)b * p.out.token_stride + (size_t)(h * p.group + g) * p.out.head_stride) *
                           (p.out_dtype == ANE_DTYPE_F32 ? 4 : 2);
        if (lane * 4 < p.dim) {
            store2(row, lane * 4, p.out_dtype, l == 0.0f ? 0.0f : o[0] * inv, l == 0.0f ? 0.0f : o[1] * inv);
            store2(row, lane * 4 + 2, p.out_dtype, l == 0.0f ? 0.0f : o[2] * inv, l == 0.0f ? 0.0f : o[3] * inv);
        }
        if (p.lse && lane == 0)
            p.lse[(size_t)b * p.heads + h * p.group + g] = l == 0.0f ? kNegInf : (m + log2f(l) - Type<T>::kShift) * kLn2;
    }
}

struct Layout {
    uint32_t row_tile, row_tiles;
    size_t cum, pm, po, sm, so, bytes;
};
Layout layout(uint32_t batch, uint32_t heads, uint32_t kv_heads, uint32_t dim) {
    Layout l;
    const uint32_t group = heads / kv_heads;
    const size_t rows = (size_t)batch * group;
    l.row_tile = rows <= 16 ? 16 : 64;
    l.row_tiles = (uint32_t)ceil_div(rows, l.row_tile);
    const size_t prefix_rows = (kMaxBlocks + (size_t)kv_heads * l.row_tiles) * l.row_tile;
    const size_t own_rows = (kMaxBlocks + (size_t)batch * kv_heads) * group;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    l.cum = take((batch + 2) * 4);
    l.pm = take(prefix_rows * 8);
    l.sm = take(own_rows * 8);
    l.po = take(prefix_rows * dim * 4);
    l.so = take(own_rows * dim * 4);
    l.bytes = at;
    return l;
}

template <typename T, int DP>
int launch(const Params& p, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    constexpr int smem = (DP == 128 ? 3 : 4) * 2 * tile_bytes<DP>();
    int rc = set_max_dynamic_smem(decode_kernel<T, DP>, smem, done);
    if (rc) return rc;
    if ((rc = launch_pdl(decode_kernel<T, DP>, dim3(p.blocks), dim3(kThreads), smem, s, p))) return rc;
    return launch_pdl(decode_join_kernel<T>, dim3(p.batch, p.kv_heads), dim3(kThreads), 0, s, p);
}

}  // namespace
}  // namespace ane_b200

using namespace ane_b200;

extern "C" size_t ane_attn_decode_workspace_size(uint32_t batch, uint32_t heads, uint32_t kv_heads, uint32_t dim) {
    if (kv_heads == 0 || heads < kv_heads || heads % kv_heads || batch > kMaxBatch) return 0;
    return layout(batch, heads, kv_heads, dim).bytes;
}

extern "C" int ane_attn_decode_dev(uint32_t dtype, uint32_t batch, uint32_t heads, uint32_t kv_heads, uint32_t dim,
                                   float scale, const ane_rows* q, const ane_pages* pages, const int32_t* tables,
                                   uint32_t n_slots, uint32_t max_pages, const int32_t* lens, const int32_t* slots,
                                   uint32_t shared, uint32_t out_dtype, const ane_rows* out, float* lse,
                                   void* workspace, size_t workspace_bytes, void* stream) {
    int rc = attn::check_shapes("attn_decode", dtype, out_dtype, heads, kv_heads, dim, scale);
    if (rc) return rc;
    ANE_ARG_CHECK(batch <= kMaxBatch, "attn_decode: at most 1024 sequences");
    ANE_ARG_CHECK(q && pages && tables && lens && out, "attn_decode: NULL pointer");
    ANE_ARG_CHECK(slots || batch <= n_slots, "attn_decode: without slots the batch must not exceed n_slots");
    ANE_ARG_CHECK(n_slots > 0 && max_pages > 0, "attn_decode: empty table");
    if (batch == 0) return (rc = require_sm100()) ? rc : ok();
    if ((rc = attn::check_rows("attn_decode", q, 2)) ||
        (rc = attn::check_rows("attn_decode", out, out_dtype == ANE_DTYPE_F32 ? 4 : 2)))
        return rc;
    const uint32_t pt = pages->page_tokens;
    ANE_ARG_CHECK(pt >= 8 && pt <= 256 && (pt & (pt - 1)) == 0, "attn_decode: page_tokens must be a power of two from 8 to 256");
    ANE_ARG_CHECK(pages->k && pages->v && pages->pages > 0 && (uintptr_t)pages->k % 16 == 0 &&
                      (uintptr_t)pages->v % 16 == 0 && pages->page_stride % 8 == 0 && pages->token_stride % 8 == 0 &&
                      pages->head_stride % 8 == 0,
                  "attn_decode: pages must be 16-byte aligned with strides of whole 16 bytes");
    ANE_ARG_CHECK((uint64_t)max_pages * pt <= 0x7fffff00u, "attn_decode: at most 2^31 tokens per slot");
    ANE_ARG_CHECK(shared <= (uint64_t)max_pages * pt, "attn_decode: shared exceeds max_pages pages");
    const Layout l = layout(batch, heads, kv_heads, dim);
    ANE_ARG_CHECK(workspace && (uintptr_t)workspace % 256 == 0 && workspace_bytes >= l.bytes,
                  "attn_decode: workspace must be 256-byte aligned and of ane_attn_decode_workspace_size bytes");
    if ((rc = require_sm100())) return rc;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    Params p{};
    p.batch = batch, p.heads = heads, p.kv_heads = kv_heads, p.group = heads / kv_heads, p.dim = dim;
    p.out_dtype = out_dtype;
    p.shared = shared, p.prefix_tiles = (uint32_t)ceil_div(shared, attn::kTile);
    p.row_tiles = l.row_tiles, p.row_tile = l.row_tile;
    p.n_slots = n_slots, p.max_pages = max_pages, p.pages = pages->pages;
    while ((1u << p.page_shift) < pt) p.page_shift++;
    p.scale2 = scale * attn::kLog2e;
    p.q = *q, p.out = *out;
    p.k = static_cast<const uint8_t*>(pages->k), p.v = static_cast<const uint8_t*>(pages->v);
    p.page_stride = pages->page_stride * 2, p.token_stride = pages->token_stride * 2, p.head_stride = pages->head_stride * 2;
    p.tables = tables, p.lens = lens, p.slots = slots, p.lse = lse;
    p.cum = reinterpret_cast<int32_t*>(ws + l.cum);
    p.pm = reinterpret_cast<float*>(ws + l.pm), p.po = reinterpret_cast<float*>(ws + l.po);
    p.sm = reinterpret_cast<float*>(ws + l.sm), p.so = reinterpret_cast<float*>(ws + l.so);
    // two blocks per SM fit (96 KB of tiles each)
    p.blocks = (uint32_t)num_sms() * 2 < kMaxBlocks ? (uint32_t)num_sms() * 2 : kMaxBlocks;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == ANE_DTYPE_F16)
        rc = dim <= 64 ? launch<__half, 64>(p, s) : launch<__half, 128>(p, s);
    else
        rc = dim <= 64 ? launch<__nv_bfloat16, 64>(p, s) : launch<__nv_bfloat16, 128>(p, s);
    return rc ? rc : ok();
}
