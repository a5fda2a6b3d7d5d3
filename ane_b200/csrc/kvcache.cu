// kvcache.cu -- pages of a key/value cache: reserve, write, fork, free, copy,
// compact.  No counterpart in the reference (its ggml backend keeps no cache of
// its own).
//
// A cache is two pools of pages (K and V, [layers][pages][page_tokens][heads]
// [dim], 16-bit elements), a count of readers per page (refs; 0 = free), and per
// slot a row of page numbers and a token count.  All of it is device memory and
// every operation runs on a stream without the host, so a decode loop that
// forks, grows and frees sequences stays capturable.  Results do not depend on
// the order in which blocks run: free pages are always taken lowest first, in
// the order of the requests.
//
// Every block plans for itself: it packs refs into a bitmap in shared memory
// (one bit per page, with a running count per word), after which "the r-th free
// page" and "the r-th page in use above x" are a binary search.  A plan costs
// each block pages * 4 bytes of L2 reads and saves a launch and a device-wide
// barrier.  What a plan reads (refs of free pages, lens) is changed only by the
// last block to have planned, which a counter elects.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ane_internal.cuh"
#include "sm100_ptx.cuh"

namespace ane_b200 {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxRequests = 1024;
constexpr uint32_t kMaxPages = 1u << 19;  // their bitmap and counts take 128 KB of shared memory

struct Pool {
    uint8_t* k;
    uint8_t* v;
    uint32_t layers, pages, page_tokens, max_pages, slots;
    uint32_t token_bytes;  // heads * dim * 2, a multiple of 16
    int32_t* refs;
    int32_t* tables;
    int32_t* lens;
    uint32_t* ctl;  // one zeroed word: blocks that have planned
};

// Bitmap of pages in use with the running count of set bits before each word.
struct Bits {
    uint32_t* word;
    uint32_t* before;
    uint32_t words, pages, used;

    // pages in use below page p
    __device__ uint32_t rank(uint32_t p) const {
        return before[p >> 5] + __popc(word[p >> 5] & ((1u << (p & 31)) - 1u));
    }
    // r-th page (from 0) that is in use (set = true) or free; the caller keeps r
    // below the number of such pages
    template <bool set>
    __device__ uint32_t select(uint32_t r) const {
        uint32_t lo = 0, hi = words - 1;
        while (lo < hi) {  // last word whose count before it is <= r
            const uint32_t mid = (lo + hi + 1) >> 1;
            const uint32_t c = set ? before[mid] : mid * 32u - before[mid];
            if (c <= r) lo = mid; else hi = mid - 1;
        }
        uint32_t w = set ? word[lo] : ~word[lo];
        for (uint32_t i = r - (set ? before[lo] : lo * 32u - before[lo]); i > 0; i--) w &= w - 1;
        return lo * 32u + (uint32_t)(__ffs((int)w) - 1);
    }
};

// All threads of the block; smem holds 2 * words + 1 uint32.  Bits past the last
// page read as in use, so they are never handed out.
__device__ Bits pack_refs(const int32_t* refs, uint32_t pages, uint32_t* smem) {
    Bits b;
    b.pages = pages;
    b.words = (pages + 31) >> 5;
    b.word = smem;
    b.before = smem + b.words;
    for (uint32_t p = threadIdx.x; p < b.words * 32u; p += blockDim.x) {
        const uint32_t w = __ballot_sync(0xffffffffu, p >= pages || refs[p] != 0);
        if ((threadIdx.x & 31) == 0) b.word[p >> 5] = w;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        uint32_t base = 0;
        for (uint32_t w0 = 0; w0 < b.words; w0 += 32) {
            const uint32_t w = w0 + threadIdx.x;
            const uint32_t c = w < b.words ? __popc(b.word[w]) : 0;
            uint32_t s = c;
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t t = __shfl_up_sync(0xffffffffu, s, o);
                if ((int)threadIdx.x >= o) s += t;
            }
            if (w < b.words) b.before[w] = base + s - c;
            base += __shfl_sync(0xffffffffu, s, 31);
        }
        if (threadIdx.x == 0) b.before[b.words] = base;
    }
    __syncthreads();
    b.used = b.before[b.words] - (b.words * 32u - pages);
    return b;
}
__host__ __device__ inline size_t bits_bytes(uint32_t pages) { return ((size_t)((pages + 31) / 32) * 2 + 1) * 4; }

// Exclusive sums of v[0..n) in place (one warp's work is enough for n <= 1024);
// returns the total.  All threads.
__device__ uint32_t exclusive_scan(uint32_t* v, uint32_t n, uint32_t* total) {
    __syncthreads();
    if (threadIdx.x < 32) {
        uint32_t base = 0;
        for (uint32_t i0 = 0; i0 < n; i0 += 32) {
            const uint32_t i = i0 + threadIdx.x;
            const uint32_t c = i < n ? v[i] : 0;
            uint32_t s = c;
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t t = __shfl_up_sync(0xffffffffu, s, o);
                if ((int)threadIdx.x >= o) s += t;
            }
            if (i < n) v[i] = base + s - c;
            base += __shfl_sync(0xffffffffu, s, 31);
        }
        if (threadIdx.x == 0) *total = base;
    }
    __syncthreads();
    return *total;
}

// True in the last block whose plan is made: the others' reads of refs and lens
// have all returned.  All threads; leaves the counter at zero for the next call.
__device__ bool last_to_plan(uint32_t* ctl, uint32_t* flag) {
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        const bool last = atomicAdd(ctl, 1u) == gridDim.x - 1;
        if (last) *ctl = 0;
        __threadfence();
        *flag = last;
    }
    __syncthreads();
    return *flag != 0;
}

// Is slot s the first of its kind in list[0..i]?  (A slot named twice counts once.)
__device__ bool first_of(const int32_t* list, uint32_t i, int32_t s) {
    for (uint32_t j = 0; j < i; j++)
        if (list[j] == s) return false;
    return true;
}

// The block copies `bytes` (a multiple of 16); eight loads in flight per thread.
__device__ void copy_block(uint8_t* dst, const uint8_t* src, size_t bytes) {
    const uint4* s = reinterpret_cast<const uint4*>(src);
    uint4* d = reinterpret_cast<uint4*>(dst);
    const size_t n = bytes >> 4;
    size_t i = threadIdx.x;
    for (; i + 7 * kThreads < n; i += 8 * kThreads) {
        uint4 r[8];
#pragma unroll
        for (int u = 0; u < 8; u++) r[u] = s[i + u * kThreads];
#pragma unroll
        for (int u = 0; u < 8; u++) d[i + u * kThreads] = r[u];
    }
    for (; i < n; i += kThreads) d[i] = s[i];
}

// ----------------------------------------------------------------- reserve
// One block.  Request i grows slot s by c tokens: its new pages go to the end of
// its row.  Requests are granted in order while the free pages last.
__global__ void __launch_bounds__(1024) reserve_kernel(Pool p, uint32_t n, const int32_t* slots,
                                                       const int32_t* counts, int32_t* granted) {
    extern __shared__ uint32_t smem[];
    __shared__ uint32_t off[kMaxRequests];
    __shared__ int32_t slot[kMaxRequests];
    __shared__ int32_t have[kMaxRequests];  // pages the row holds; -1: refused
    __shared__ uint32_t total;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const Bits bits = pack_refs(p.refs, p.pages, smem);
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) slot[i] = slots[i];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const int32_t s = slot[i], c = counts[i];
        uint32_t need = 0;
        have[i] = -1;
        if (s >= 0 && (uint32_t)s < p.slots && c >= 0 && first_of(slot, i, s)) {
            const uint32_t len = (uint32_t)p.lens[s];
            const uint64_t want = ((uint64_t)len + (uint32_t)c + p.page_tokens - 1) / p.page_tokens;
            if (want <= p.max_pages && (uint64_t)len + (uint32_t)c <= 0x7fffffffu) {
                have[i] = (int32_t)((len + p.page_tokens - 1) / p.page_tokens);
                need = (uint32_t)want - (uint32_t)have[i];
            }
        }
        off[i] = need;
    }
    const uint32_t all = exclusive_scan(off, n, &total);
    const uint32_t free_pages = p.pages - bits.used;
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const uint32_t end = i + 1 < n ? off[i + 1] : all;
        const bool ok = have[i] >= 0 && (end == off[i] || end <= free_pages);
        granted[i] = ok ? 1 : 0;
        if (ok) p.lens[slot[i]] += counts[i];
    }
    // one thread per new page; a request's pages come one after another
    for (uint32_t r = threadIdx.x; r < min(all, free_pages); r += blockDim.x) {
        uint32_t lo = 0, hi = n - 1;
        while (lo < hi) {  // last request that starts at or before r
            const uint32_t mid = (lo + hi + 1) >> 1;
            if (off[mid] <= r) lo = mid; else hi = mid - 1;
        }
        const uint32_t end = lo + 1 < n ? off[lo + 1] : all;
        if (end > free_pages) continue;
        const uint32_t page = bits.select<false>(r);
        p.refs[page] = 1;
        p.tables[(size_t)slot[lo] * p.max_pages + have[lo] + (r - off[lo])] = (int32_t)page;
    }
}

// ------------------------------------------------------------------- write
template <typename Dst>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// One token per block: its heads * dim values of K and V go to the token's place
// (the last counts[r] tokens of request r's slot), rounded once from fp32 rows.
template <typename Dst>
__global__ void __launch_bounds__(kThreads) write_kernel(Pool p, uint32_t layer, uint32_t n, const int32_t* slots,
                                                         const int32_t* cu, const int32_t* granted, uint32_t src_f32,
                                                         ane_rows k, ane_rows v, uint32_t dim) {
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const int32_t t = (int32_t)blockIdx.x;
    uint32_t lo = cu ? 0 : blockIdx.x, hi = cu ? n - 1 : blockIdx.x;
    if (cu && (t < cu[0] || t >= cu[n])) return;  // rows of no request
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= t) lo = mid; else hi = mid - 1;
    }
    const int32_t s = slots[lo];
    if (!granted) {  // (reserve_kernel grants a slot's first request alone)
        bool again = false;
        for (uint32_t j = threadIdx.x; j < lo; j += kThreads) again |= slots[j] == s;
        if (__syncthreads_or(again)) return;
    }
    if (s < 0 || (uint32_t)s >= p.slots || (granted && !granted[lo])) return;
    const int32_t pos = p.lens[s] - (cu ? cu[lo + 1] - t : 1);
    if (pos < 0 || (uint32_t)pos / p.page_tokens >= p.max_pages) return;
    const int32_t page = p.tables[(size_t)s * p.max_pages + (uint32_t)pos / p.page_tokens];
    if (page < 0 || (uint32_t)page >= p.pages) return;
    const size_t at = (((size_t)layer * p.pages + page) * p.page_tokens + (uint32_t)pos % p.page_tokens) *
                      p.token_bytes;
    const uint32_t chunks = p.token_bytes / 16, per_head = dim / 8;  // 16-byte chunks of 8 elements
    for (uint32_t c = threadIdx.x; c < 2 * chunks; c += kThreads) {
        const bool is_v = c >= chunks;
        const uint32_t cc = is_v ? c - chunks : c;
        const ane_rows& rows = is_v ? v : k;
        const size_t e = (size_t)t * rows.token_stride + (size_t)(cc / per_head) * rows.head_stride +
                         (size_t)(cc % per_head) * 8;
        const uint8_t* src = static_cast<const uint8_t*>(rows.data);
        uint4 out;
        if (src_f32) {
            const float4 a = *reinterpret_cast<const float4*>(src + e * 4);
            const float4 b = *reinterpret_cast<const float4*>(src + e * 4 + 16);
            out = make_uint4(pack2<Dst>(a.x, a.y), pack2<Dst>(a.z, a.w), pack2<Dst>(b.x, b.y), pack2<Dst>(b.z, b.w));
        } else {
            out = *reinterpret_cast<const uint4*>(src + e * 2);
        }
        *reinterpret_cast<uint4*>((is_v ? p.v : p.k) + at + (size_t)cc * 16) = out;
    }
}

// -------------------------------------------------------------------- fork
// Child rows take the parent's whole pages (one more reader each) and a copy of
// its part page.  Work items: per child its table row, then one copy per layer
// and pool; blocks take every gridDim.x-th item.
__global__ void __launch_bounds__(kThreads) fork_kernel(Pool p, uint32_t n, const int32_t* parents,
                                                        const int32_t* children, int32_t* granted) {
    extern __shared__ uint32_t smem[];
    __shared__ int32_t child[kMaxRequests];
    __shared__ int32_t parent[kMaxRequests];
    __shared__ int32_t len[kMaxRequests];   // tokens; -1: refused
    __shared__ uint32_t off[kMaxRequests];  // rank of the request's new page among the free ones
    __shared__ uint32_t total, flag;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const Bits bits = pack_refs(p.refs, p.pages, smem);
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        child[i] = children[i];
        parent[i] = parents[i];
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const int32_t c = child[i], s = parent[i];
        len[i] = -1;
        uint32_t need = 0;
        if (c >= 0 && (uint32_t)c < p.slots && s >= 0 && (uint32_t)s < p.slots && p.lens[c] == 0 &&
            first_of(child, i, c)) {
            const int32_t tokens = p.lens[s];
            if (tokens >= 0 && (uint64_t)tokens <= (uint64_t)p.max_pages * p.page_tokens) {
                len[i] = tokens;
                need = (uint32_t)tokens % p.page_tokens != 0;
            }
        }
        off[i] = need;
    }
    const uint32_t all = exclusive_scan(off, n, &total);
    const uint32_t free_pages = p.pages - bits.used;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const uint32_t end = i + 1 < n ? off[i + 1] : all;
        if (len[i] >= 0 && end > off[i] && end > free_pages) len[i] = -1;
    }
    if (last_to_plan(p.ctl, &flag)) {
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            granted[i] = len[i] >= 0 ? 1 : 0;
            if (len[i] <= 0) continue;
            p.lens[child[i]] = len[i];
            if ((uint32_t)len[i] % p.page_tokens) p.refs[bits.select<false>(off[i])] = 1;
        }
    }
    const uint32_t parts = 1 + 2 * p.layers;
    for (uint32_t item = blockIdx.x; item < n * parts; item += gridDim.x) {
        const uint32_t i = item / parts, part = item % parts;
        if (len[i] <= 0) continue;
        const uint32_t whole = (uint32_t)len[i] / p.page_tokens, rest = (uint32_t)len[i] % p.page_tokens;
        const int32_t* from = p.tables + (size_t)parent[i] * p.max_pages;
        int32_t* to = p.tables + (size_t)child[i] * p.max_pages;
        if (part == 0) {
            for (uint32_t e = threadIdx.x; e < whole; e += kThreads) {
                const int32_t page = from[e];
                to[e] = page;
                if (page >= 0 && (uint32_t)page < p.pages) atomicAdd(&p.refs[page], 1);
            }
            if (threadIdx.x == 0 && rest) to[whole] = (int32_t)bits.select<false>(off[i]);
        } else if (rest) {
            const int32_t old = from[whole];
            if (old < 0 || (uint32_t)old >= p.pages) continue;
            const size_t page_bytes = (size_t)p.page_tokens * p.token_bytes;
            uint8_t* pool = ((part & 1) ? p.k : p.v) + (size_t)((part - 1) >> 1) * p.pages * page_bytes;
            copy_block(pool + bits.select<false>(off[i]) * page_bytes, pool + (size_t)old * page_bytes,
                       (size_t)rest * p.token_bytes);
        }
    }
}

// -------------------------------------------------------------------- free
// One block per slot named; entries of its row stay as they are.
__global__ void __launch_bounds__(kThreads) free_kernel(Pool p, const int32_t* slots) {
    __shared__ uint32_t mine;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const int32_t s = slots[blockIdx.x];
    if (threadIdx.x == 0) mine = 1;
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < blockIdx.x; j += kThreads)
        if (slots[j] == s) mine = 0;  // an earlier block frees it
    __syncthreads();
    if (!mine || s < 0 || (uint32_t)s >= p.slots) return;
    const uint32_t count = min(((uint32_t)p.lens[s] + p.page_tokens - 1) / p.page_tokens, p.max_pages);
    for (uint32_t e = threadIdx.x; e < count; e += kThreads) {
        const int32_t page = p.tables[(size_t)s * p.max_pages + e];
        if (page >= 0 && (uint32_t)page < p.pages) atomicSub(&p.refs[page], 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) p.lens[s] = 0;
}

// -------------------------------------------------------------------- copy
// Page src[i] of one cache to page dst[i] of another of the same shape (or the
// same one).  Items: pair, layer, pool.
__global__ void __launch_bounds__(kThreads) copy_pages_kernel(Pool a, Pool b, uint32_t n, const int32_t* src,
                                                              const int32_t* dst) {
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const size_t page_bytes = (size_t)a.page_tokens * a.token_bytes;
    const uint64_t items = (uint64_t)n * 2 * a.layers;
    for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const uint32_t i = (uint32_t)(item / (2 * a.layers)), part = (uint32_t)(item % (2 * a.layers));
        const int32_t s = src[i], d = dst[i];
        if (s < 0 || (uint32_t)s >= a.pages || d < 0 || (uint32_t)d >= b.pages) continue;
        const size_t l = part >> 1;
        copy_block(((part & 1) ? b.v : b.k) + (l * b.pages + d) * page_bytes,
                   ((part & 1) ? a.v : a.k) + (l * a.pages + s) * page_bytes, page_bytes);
    }
}

// ----------------------------------------------------------------- compact
// With `used` pages in use, the r-th page in use at or above `used` moves to the
// r-th free page below it.  Both counts are equal, sources and targets do not
// overlap, and the sources stay intact.
__global__ void __launch_bounds__(kThreads) compact_kernel(Pool p, int32_t* refs_out, int32_t* tables_out,
                                                           int32_t* remap, int32_t* live) {
    extern __shared__ uint32_t smem[];
    __shared__ uint32_t flag;
    ptx::griddep_launch_dependents();
    ptx::griddep_wait();
    const Bits bits = pack_refs(p.refs, p.pages, smem);
    const uint32_t used = bits.used;
    const uint32_t low = used < p.pages ? bits.rank(used) : used;  // pages in use that stay
    const uint32_t movers = used - low;
    auto target = [&](uint32_t page) {  // of a page in use
        return page < used ? page : bits.select<false>(bits.rank(page) - low);
    };
    // rows first: reading lens and writing tables_out (which may be the table
    // itself) touch nothing that a plan reads
    for (uint32_t s = blockIdx.x; s < p.slots; s += gridDim.x) {
        const uint32_t count = min(((uint32_t)p.lens[s] + p.page_tokens - 1) / p.page_tokens, p.max_pages);
        for (uint32_t e = threadIdx.x; e < p.max_pages; e += kThreads) {
            const int32_t page = p.tables[(size_t)s * p.max_pages + e];
            const bool mine = e < count && page >= 0 && (uint32_t)page < p.pages;
            if (mine || tables_out != p.tables)
                tables_out[(size_t)s * p.max_pages + e] = mine ? (int32_t)target((uint32_t)page) : page;
        }
    }
    if (last_to_plan(p.ctl, &flag)) {
        if (threadIdx.x == 0) *live = (int32_t)used;
        // first what moves and what stays, reading refs of pages in use only ...
        for (uint32_t q = threadIdx.x; q < p.pages; q += kThreads) {
            const bool in_use = (bits.word[q >> 5] >> (q & 31)) & 1;
            remap[q] = in_use ? (int32_t)target(q) : -1;
            if (in_use) refs_out[target(q)] = p.refs[q];
        }
        __syncthreads();
        // ... then the tail, which is free now
        for (uint32_t q = used + threadIdx.x; q < p.pages; q += kThreads) refs_out[q] = 0;
    }
    const size_t page_bytes = (size_t)p.page_tokens * p.token_bytes;
    const uint64_t items = (uint64_t)movers * 2 * p.layers;
    for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const uint32_t r = (uint32_t)(item % movers), part = (uint32_t)(item / movers);
        uint8_t* pool = ((part & 1) ? p.v : p.k) + (size_t)(part >> 1) * p.pages * page_bytes;
        copy_block(pool + bits.select<false>(r) * page_bytes, pool + bits.select<true>(low + r) * page_bytes,
                   page_bytes);
    }
}

// ------------------------------------------------------------------ launch
// Argument checks that every call makes; fills `p`.
int make_pool(const ane_kv_cache* c, Pool* p) {
    ANE_ARG_CHECK(c != nullptr, "kv cache: NULL descriptor");
    ANE_ARG_CHECK(c->dtype == ANE_DTYPE_F16 || c->dtype == ANE_DTYPE_BF16, "kv cache: dtype must be F16 or BF16");
    ANE_ARG_CHECK(c->k && c->v && c->refs && c->tables && c->lens && c->ctl, "kv cache: NULL pointer");
    ANE_ARG_CHECK(c->layers > 0 && c->pages > 0 && c->heads > 0 && c->slots > 0 && c->max_pages > 0,
                  "kv cache: layers, pages, heads, slots and max_pages must be positive");
    ANE_ARG_CHECK(c->pages <= kMaxPages, "kv cache: at most 2^19 pages");
    ANE_ARG_CHECK(c->page_tokens >= 8 && c->page_tokens <= 256 && (c->page_tokens & (c->page_tokens - 1)) == 0,
                  "kv cache: page_tokens must be a power of two from 8 to 256");
    ANE_ARG_CHECK(c->dim >= 8 && c->dim <= 128 && c->dim % 8 == 0, "kv cache: dim must be a multiple of 8, 8 to 128");
    ANE_ARG_CHECK(c->heads <= 1024 && c->layers <= 65536 && c->slots <= (1u << 24) && c->max_pages <= kMaxPages,
                  "kv cache: too many heads, layers, slots or pages per slot");
    ANE_ARG_CHECK(((uintptr_t)c->k % 16) == 0 && ((uintptr_t)c->v % 16) == 0, "kv cache: pools must be 16-byte aligned");
    *p = Pool{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), c->layers, c->pages, c->page_tokens,
              c->max_pages, c->slots, c->heads * c->dim * 2, c->refs, c->tables, c->lens, c->ctl};
    return ANE_OK;
}

// Shared memory for the bitmap of the largest cache, allowed once per device.
template <typename F>
int allow_bits(F* kernel, std::atomic<uint64_t>& done) {
    return set_max_dynamic_smem(kernel, (int)bits_bytes(kMaxPages), done);
}

}  // namespace
}  // namespace ane_b200

using namespace ane_b200;

extern "C" {

int ane_kv_reserve_dev(const ane_kv_cache* cache, uint32_t n, const int32_t* slots, const int32_t* counts,
                       int32_t* granted, void* stream) {
    Pool p;
    ANE_ARG_CHECK(n <= kMaxRequests, "kv_reserve: at most 1024 requests per call");
    ANE_ARG_CHECK(n == 0 || (slots && counts && granted), "kv_reserve: NULL pointer");
    int rc = make_pool(cache, &p);
    if (rc) return rc;
    if ((rc = require_sm100())) return rc;
    if (n == 0) return ok();
    static std::atomic<uint64_t> done{0};
    if ((rc = allow_bits(reserve_kernel, done))) return rc;
    rc = launch_pdl(reserve_kernel, dim3(1), dim3(1024), bits_bytes(p.pages), static_cast<cudaStream_t>(stream), p, n,
                    slots, counts, granted);
    return rc ? rc : ok();
}

int ane_kv_write_dev(const ane_kv_cache* cache, uint32_t layer, uint32_t n, const int32_t* slots, const int32_t* cu,
                     const int32_t* granted, uint32_t tokens, uint32_t src_dtype, const ane_rows* k,
                     const ane_rows* v, void* stream) {
    Pool p;
    ANE_ARG_CHECK(n == 0 || (slots && k && v), "kv_write: NULL pointer");
    ANE_ARG_CHECK(cu || tokens == n, "kv_write: without cu every request has one token");
    ANE_ARG_CHECK(cache && (src_dtype == ANE_DTYPE_F32 || src_dtype == cache->dtype),
                  "kv_write: rows must be F32 or of the cache's dtype");
    const size_t elem = src_dtype == ANE_DTYPE_F32 ? 4 : 2;
    for (const ane_rows* r : {k, v}) {
        if (n == 0 || tokens == 0) break;  // (no rows may have no memory)
        ANE_ARG_CHECK(r->data && (uintptr_t)r->data % 16 == 0 && r->token_stride * elem % 16 == 0 &&
                          r->head_stride * elem % 16 == 0,
                      "kv_write: rows must be 16-byte aligned with strides of whole 16 bytes");
    }
    ANE_ARG_CHECK(layer < cache->layers, "kv_write: no such layer");
    int rc = make_pool(cache, &p);
    if (rc) return rc;
    if ((rc = require_sm100())) return rc;
    if (n == 0 || tokens == 0) return ok();
    auto kernel = cache->dtype == ANE_DTYPE_F16 ? write_kernel<__half> : write_kernel<__nv_bfloat16>;
    rc = launch_pdl(kernel, dim3(tokens), dim3(kThreads), 0, static_cast<cudaStream_t>(stream), p, layer, n, slots, cu,
                    granted, (uint32_t)(src_dtype == ANE_DTYPE_F32), *k, *v, cache->dim);
    return rc ? rc : ok();
}

int ane_kv_fork_dev(const ane_kv_cache* cache, uint32_t n, const int32_t* parents, const int32_t* children,
                    int32_t* granted, void* stream) {
    Pool p;
    ANE_ARG_CHECK(n <= kMaxRequests, "kv_fork: at most 1024 requests per call");
    ANE_ARG_CHECK(n == 0 || (parents && children && granted), "kv_fork: NULL pointer");
    int rc = make_pool(cache, &p);
    if (rc) return rc;
    if ((rc = require_sm100())) return rc;
    if (n == 0) return ok();
    static std::atomic<uint64_t> done{0};
    if ((rc = allow_bits(fork_kernel, done))) return rc;
    // 148 MB of part pages written and 18 read in 44 us with four blocks per SM (two 50,
    // eight 57); a plain fill of those 148 MB takes 41.  Reading a parent's page once for
    // all its children changed nothing.
    const size_t items = (size_t)n * (1 + 2 * p.layers);
    const uint32_t grid = (uint32_t)(items < (size_t)num_sms() * 4 ? items : (size_t)num_sms() * 4);
    rc = launch_pdl(fork_kernel, dim3(grid), dim3(kThreads), bits_bytes(p.pages), static_cast<cudaStream_t>(stream), p,
                    n, parents, children, granted);
    return rc ? rc : ok();
}

int ane_kv_free_dev(const ane_kv_cache* cache, uint32_t n, const int32_t* slots, void* stream) {
    Pool p;
    ANE_ARG_CHECK(n <= kMaxRequests, "kv_free: at most 1024 requests per call");
    ANE_ARG_CHECK(n == 0 || slots, "kv_free: NULL pointer");
    int rc = make_pool(cache, &p);
    if (rc) return rc;
    if ((rc = require_sm100())) return rc;
    if (n == 0) return ok();
    rc = launch_pdl(free_kernel, dim3(n), dim3(kThreads), 0, static_cast<cudaStream_t>(stream), p, slots);
    return rc ? rc : ok();
}

int ane_kv_copy_pages_dev(const ane_kv_cache* from, const ane_kv_cache* to, uint32_t n, const int32_t* src,
                          const int32_t* dst, void* stream) {
    Pool a, b;
    ANE_ARG_CHECK(n == 0 || (src && dst), "kv_copy_pages: NULL pointer");
    int rc = make_pool(from, &a);
    if (rc) return rc;
    rc = make_pool(to, &b);
    if (rc) return rc;
    ANE_ARG_CHECK(from->dtype == to->dtype && a.layers == b.layers && a.page_tokens == b.page_tokens &&
                      from->heads == to->heads && from->dim == to->dim,
                  "kv_copy_pages: the caches differ in dtype, layers, page_tokens, heads or dim");
    if ((rc = require_sm100())) return rc;
    if (n == 0) return ok();
    const uint64_t items = (uint64_t)n * 2 * a.layers;
    const uint32_t grid = (uint32_t)(items < (uint64_t)num_sms() * 4 ? items : (uint64_t)num_sms() * 4);
    rc = launch_pdl(copy_pages_kernel, dim3(grid), dim3(kThreads), 0, static_cast<cudaStream_t>(stream), a, b, n, src,
                    dst);
    return rc ? rc : ok();
}

int ane_kv_compact_dev(const ane_kv_cache* cache, int32_t* refs_out, int32_t* tables_out, int32_t* remap,
                       int32_t* live, void* stream) {
    Pool p;
    ANE_ARG_CHECK(refs_out && tables_out && remap && live, "kv_compact: NULL pointer");
    int rc = make_pool(cache, &p);
    if (rc || (rc = require_sm100())) return rc;
    static std::atomic<uint64_t> done{0};
    if ((rc = allow_bits(compact_kernel, done))) return rc;
    // At most half of the pages move, K and V.  Two blocks per SM keep 64 KB in
    // flight there: 1124 MB read and written in 187 us (four blocks 201, eight 199).
    const uint64_t items = (uint64_t)p.pages * p.layers;
    const uint32_t grid = (uint32_t)(items < (uint64_t)num_sms() * 2 ? items : (uint64_t)num_sms() * 2);
    rc = launch_pdl(compact_kernel, dim3(grid), dim3(kThreads), bits_bytes(p.pages), static_cast<cudaStream_t>(stream),
                    p, refs_out, tables_out, remap, live);
    return rc ? rc : ok();
}

}  // extern "C"
