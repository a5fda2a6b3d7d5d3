// attn_decode.cu -- attention of one new token per sequence over a paged cache
// whose sequences share a prefix.
//
// decode_kernel works on units of at most 16 query rows (as many sequences as
// fit, with the heads that share a key/value head) on mma.sync: a unit's keys are
// the shared prefix, which all of its rows see, and then each of its sequences'
// own tokens, which only that sequence's rows see.  (A sequence that ends inside
// the prefix has all its tokens as its own.)  It is bound by the bytes of K
// and V, so all units' 64-token tiles are laid end to end and cut into equal
// spans, one per block: ragged lengths and a single long sequence load the chip
// alike.  Two producer warps stream a span's tiles through a ring by TMA, across
// unit boundaries (a warp issues its lanes' boxes one by one, about 50 ns each:
// with pages of 16 a tile is 16 boxes), while four warps compute, each a quarter
// of a tile's tokens.
//
// Every unit reads the prefix again.  With many rows prefix_kernel does the prefix
// instead, on tcgen05 (attn_sm100.cuh), 256 rows against every key tile.
//
// Both leave unnormalised partial results (m, l, o); join_kernel adds them per
// output row in a fixed order, so results do not depend on scheduling.  Where
// units are known to be short, a block does a whole one and writes the result.
#include "attn_sm100.cuh"

namespace ane_b200 {
namespace {
using namespace attn;

constexpr uint32_t kMaxBatch = 1024;
constexpr uint32_t kMaxBlocks = 512;   // of decode_kernel
constexpr uint32_t kBigBlocks = 148;   // of prefix_kernel, about
constexpr int kTile = 64;              // tokens per key/value tile
constexpr int kThreads = 192;          // four computing warps, the producers of K and of V
constexpr int kJoinThreads = 128;
// Up to so many sequences join_kernel counts the own tiles itself, which hides behind
// the last blocks of decode_kernel but costs each of its blocks a pass over the batch;
// above, it reads decode_kernel's counts.  32/8 heads, 600 tokens each, us counted and
// read: 24 sequences 20.7 and 22.8, 64 43.2 and 45.2, 96 58 and 58, 128 75 and 72, 256
// 157 and 128, 1024 1208 and 457.
constexpr uint32_t kCountedBatch = 96;
constexpr uint32_t kKept = 256;        // sequences whose slot and length stay in shared memory
constexpr int kPagesAhead = 4;         // tiles whose page numbers are read ahead
constexpr int kUnits = 4;              // units announced ahead
constexpr int kUnitCost = 2;           // a unit's start and end cost about what two tiles do
// Units of at most so many tiles, as far as the width of the tables tells (the host
// does not know the lengths), are not cut: a call then costs the host one launch, 2 us,
// less, and the device goes through a unit's tiles one after another.  2 sequences x 32
// heads, us in a graph, whole and cut: 3 tiles a unit 8.8 and 9.6, 5 10.1 and 10.2, 6
// 10.9 and 10.1, 7 11.5 and 10.4; called from Python with other inputs each time: 7
// tiles 12.4 and 14.4.  From 8 on the device's time shows there too (1 sequence of 510
// in a graph: 11.5 and 10.4).
constexpr uint32_t kWholeTiles = 7;

struct Params {
    uint32_t batch, heads, kv_heads, group, dim, out_dtype;
    uint32_t shared;         // tokens of the prefix
    uint32_t prefix_tiles;   // its tiles in decode_kernel (0: none, or prefix_kernel does them)
    uint32_t per_unit;       // sequences of a unit
    uint32_t groups, subs;   // units per key/value head: groups of sequences x parts of 16 heads
    uint32_t rows;           // rows of a unit's partial result
    uint32_t whole;          // 1: a block per unit, results written
    uint32_t blocks;         // of decode_kernel
    uint32_t big_splits;     // spans of prefix_kernel (0: not used)
    uint32_t n_slots, max_pages, pages, page_shift, box_keys;
    float scale2;
    ane_rows q, out;
    const int32_t *tables, *lens, *slots;
    float* lse;
    int32_t* cum;       // [batch + 1] own tiles of the sequences before b, for join_kernel (NULL: it counts them)
    float *po, *pm;     // prefix_kernel's partials: rows x dim; rows x {m, l}
    float *so, *sm;     // decode_kernel's
    int* err;
};

__device__ __forceinline__ int slot_of(const Params& p, uint32_t b) {
    const int s = p.slots ? __ldcg(p.slots + b) : (int)b;
    return s >= 0 && (uint32_t)s < p.n_slots ? s : -1;
}
// {slot, tokens} of sequence b; no slot: {-1, 0}
__device__ __forceinline__ int2 seq_of(const Params& p, uint32_t b) {
    const int s = slot_of(p, b);
    return make_int2(s, s < 0 ? 0 : min(max(__ldcg(p.lens + s), 0), (int)(p.max_pages << p.page_shift)));
}
__device__ __forceinline__ int len_of(const Params& p, uint32_t b) { return seq_of(p, b).y; }
// Keys of the prefix that a sequence's rows see as such: all or none.  With some
// of them, V of the others would meet a weight of 0 in the products, which does not
// silence an infinity or NaN there.
__device__ __forceinline__ int prefix_seen(const Params& p, int len) { return len < (int)p.shared ? 0 : (int)p.shared; }
// Own tiles start where the box of tokens does that holds the first own one.
__device__ __forceinline__ int own_base(const Params& p, int len) {
    return prefix_seen(p, len) & ~((int)p.box_keys - 1);
}
__device__ __forceinline__ int own_tiles(const Params& p, int len) {
    return len == (int)p.shared ? 0 : (len - own_base(p, len) + kTile - 1) / kTile;
}
// Place on the line where the units of group g begin, counted per head and part.
// cum: own tiles of the sequences before b.
__device__ __forceinline__ int group_start(const Params& p, const int32_t* cum, uint32_t g) {
    return (int)(g * (kUnitCost + p.prefix_tiles)) + cum[min(g * p.per_unit, p.batch)];
}
// Slot through whose pages the prefix is read: the first sequence that reaches its
// end, or the first of those that reach farthest (the others may be idle, and their
// table rows stale).  A whole warp; seq(b): {slot, tokens}.
template <class Seq>
__device__ __forceinline__ int prefix_slot(const Params& p, Seq seq) {
    uint32_t most = 0, at = 0;
    int slot = 0;
    for (uint32_t b = threadIdx.x & 31; b < p.batch; b += 32) {
        const int2 q = seq(b);
        const uint32_t n = min((uint32_t)q.y, p.shared);
        if (n > most) most = n, at = b, slot = q.x;
    }
    const uint32_t first = __reduce_min_sync(0xffffffffu, most == __reduce_max_sync(0xffffffffu, most) ? at : ~0u);
    return __shfl_sync(0xffffffffu, slot, (int)(first & 31));
}
// A unit's row: sequence (of the unit) and head (of its part of 16, or of the
// group); the same for all units.
struct RowPlace {
    uint16_t seq, head;
};
__device__ __forceinline__ RowPlace row_place(const Params& p, uint32_t row) {
    if (p.group > 16) return {0, (uint16_t)row};
    return {(uint16_t)(row / p.group), (uint16_t)(row % p.group)};
}
// Sequence and head of the group; false: no such row.
__device__ __forceinline__ bool row_of(const Params& p, uint32_t grp, uint32_t sub, RowPlace r, uint32_t& b,
                                       uint32_t& g) {
    b = grp * p.per_unit + r.seq;
    g = sub * 16 + r.head;
    return r.seq < p.per_unit && b < p.batch && g < p.group;
}
// {token in page, page} of key j; entries past the row and pages outside the
// pool are never followed.
__device__ __forceinline__ int2 page_of(const Params& p, const int32_t* table, int j) {
    const uint32_t e = min((uint32_t)j >> p.page_shift, p.max_pages - 1);
    const uint32_t page = (uint32_t)__ldcg(table + e);
    return make_int2(j & ((1 << p.page_shift) - 1), page < p.pages ? (int)page : 0);
}

struct Unit {
    int head, grp, sub;  // head -1: no more units
    int t0, t1;          // tiles
    int slot;            // place of the partial result
};
struct Tile {
    int who;             // sequence of the unit, -1: the prefix
    int key, lo, kend;   // its first key; keys lo .. kend - 1 count
};

template <int DP>
struct DecodeSmem {
    static constexpr int kStages = DP == 128 ? 3 : 6;
    static constexpr int kHalf = kTile * 128;        // 64 tokens x 64 elements
    static constexpr int kBytes = kTile * DP * 2;    // a K or a V tile
    uint8_t kv[kStages][2][kBytes];
    uint8_t q[2][16 * DP * 2];       // query rows of this unit and the next
    int vis[2][16];                  // prefix keys that each row sees
    float2 ml[kStages][4][16];       // {m, l} of each warp's rows
    int cum[kMaxBatch + 1];          // own tiles of the sequences before b
    int2 seq[kKept];                 // {slot, len} of the first sequences
    int prefix_slot;
    Unit unit[kUnits];
    Tile tile[kStages];
    RowPlace place[16];
    uint64_t full[kStages], empty[kStages], joined[kStages], unit_full[kUnits], unit_empty[kUnits], q_full[2];
};
template <int DP>
constexpr size_t decode_smem_bytes() {
    return sizeof(DecodeSmem<DP>) + 1024;
}
// two blocks per SM (228 KB, 1 KB of it reserved per block)
static_assert(2 * (decode_smem_bytes<128>() + 1024) <= 233472 && 2 * (decode_smem_bytes<64>() + 1024) <= 233472, "");

// Byte offset of 16-byte chunk c of token row t in a tile as TMA's 128-byte
// swizzle lays it out, 64-element halves one after the other.
__device__ __forceinline__ uint32_t tile_off(uint32_t t, uint32_t c) {
    return (c >> 3) * (kTile * 128) + t * 128 + (((c & 7) ^ (t & 7)) << 4);
}

// Query rows: the same with halves of 16 rows.
__device__ __forceinline__ uint32_t q_off(uint32_t row, uint32_t c) {
    return (c >> 3) * (16 * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {  // bytes < 16: zero-filled
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// A warp's state of a unit's 16 rows: thread holds rows lane / 4 and lane / 4 + 8.
template <int DP>
struct Query {
    uint32_t q[DP / 16][4];
    int vis[2];  // keys of the present tile's part that the row sees, from its lo
};
template <int DP>
struct Sums {
    float o[DP / 8][4];
    float m[2], l[2];
};

// One warp: 16 tokens of a tile (rows tok0 .. of shared memory, keys j0 ..
// counted from the unit's lo).
template <typename T, int DP>
__device__ __forceinline__ void tile_step(const Query<DP>& q, Sums<DP>& r, uint32_t ks, uint32_t vs, uint32_t tok0,
                                          int j0, float scale2) {
    const uint32_t lane = threadIdx.x & 31, mi = lane >> 3, mr = lane & 7;
    float s[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int kk = 0; kk < DP / 16; kk++) {
        uint32_t b[4];
        ldsm4(ks + tile_off(tok0 + (mi >> 1) * 8 + mr, kk * 2 + (mi & 1)), b);
        Type<T>::mma(s[0], q.q[kk], b[0], b[1]);
        Type<T>::mma(s[1], q.q[kk], b[2], b[3]);
    }
    const int first = j0 + 2 * (int)(lane & 3);
    float mx[2] = {kNegInf, kNegInf};
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            // selected, not added: a masked score may be anything, NaN included
            s[n][j] = (uint32_t)(first + n * 8 + (j & 1)) < (uint32_t)q.vis[j >> 1] ? s[n][j] * scale2 : kNegInf;
            mx[j >> 1] = fmaxf(mx[j >> 1], s[n][j]);
        }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
    }
    // most tiles do not move a maximum
    if (__any_sync(0xffffffffu, mx[0] > r.m[0] || mx[1] > r.m[1])) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float m = fmaxf(r.m[h], mx[h]), base = m == kNegInf ? 0.0f : m;
            const float c = exp2_fast(r.m[h] - base);
            r.m[h] = m;
            r.l[h] *= c;
#pragma unroll
            for (int i = 0; i < DP / 8; i++) {
                r.o[i][2 * h] *= c;
                r.o[i][2 * h + 1] *= c;
            }
        }
    }
    const float off[2] = {Type<T>::kShift - (r.m[0] == kNegInf ? 0.0f : r.m[0]),
                          Type<T>::kShift - (r.m[1] == kNegInf ? 0.0f : r.m[1])};
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            s[n][j] = exp2_fast(s[n][j] + off[j >> 1]);
            r.l[j >> 1] += s[n][j];
        }
    const uint32_t a[4] = {Type<T>::pack(s[0][0], s[0][1]), Type<T>::pack(s[0][2], s[0][3]),
                           Type<T>::pack(s[1][0], s[1][1]), Type<T>::pack(s[1][2], s[1][3])};
#pragma unroll
    for (int n = 0; n < DP / 8; n += 2) {
        uint32_t b[4];
        ldsm4_t(vs + tile_off(tok0 + (mi & 1) * 8 + mr, n + (mi >> 1)), b);
        Type<T>::mma(r.o[n], a, b[0], b[1]);
        Type<T>::mma(r.o[n + 1], a, b[2], b[3]);
    }
}

// A unit's rows belong to several sequences, and the product of a weight of 0 with
// an infinity or NaN in another sequence's V would reach them.  So such values of
// a sequence's own V (16 tokens of a tile; nothing is there but in a broken cache)
// go to that sequence's rows by themselves and are cleared before the products.
// One warp; tok0: its first token row, `sees`: whether the thread's rows see it.
template <typename T, int DP>
__device__ __forceinline__ void set_apart(Sums<DP>& r, uint8_t* v, uint32_t tok0, const bool (&sees)[2]) {
    constexpr uint32_t kLimit = sizeof(T) && Type<T>::kShift > 0.0f ? 0x7c00u : 0x7f80u;  // infinity
    const uint32_t lane = threadIdx.x & 31;
    uint32_t most = 0;  // the largest magnitudes, as integers, in the two halves
#pragma unroll
    for (int i = 0; i < DP / 16; i++) {
        const uint32_t e = i * 32 + lane;
        const uint4 x = *reinterpret_cast<const uint4*>(v + tile_off(tok0 + e % 16, e / 16));
        most = __vmaxu2(__vmaxu2(most, x.x & 0x7fff7fffu), x.y & 0x7fff7fffu);
        most = __vmaxu2(__vmaxu2(most, x.z & 0x7fff7fffu), x.w & 0x7fff7fffu);
    }
    if (!__any_sync(0xffffffffu, (most & 0xffffu) >= kLimit || (most >> 16) >= kLimit)) return;
    for (uint32_t t = 0; t < 16; t++) {
#pragma unroll
        for (int x = 0; x < DP / 8; x++) {
            const uint32_t two = *reinterpret_cast<const uint32_t*>(v + tile_off(tok0 + t, x) + 4 * (lane & 3));
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const uint16_t bits = (uint16_t)(two >> (16 * k));
                if ((bits & 0x7fffu) < kLimit) continue;
                const float f = (bits & 0x7fffu) > kLimit ? NAN : (bits >> 15) ? -INFINITY : INFINITY;
                if (sees[0]) r.o[x][k] += f;
                if (sees[1]) r.o[x][2 + k] += f;
            }
        }
    }
    __syncwarp();
    for (int i = 0; i < DP / 16; i++) {
        const uint32_t e = i * 32 + lane;
        uint32_t* x = reinterpret_cast<uint32_t*>(v + tile_off(tok0 + e % 16, e / 16));
        for (int k = 0; k < 4; k++) {
            if ((x[k] & 0x7fffu) >= kLimit) x[k] &= 0xffff0000u;
            if ((x[k] >> 16 & 0x7fffu) >= kLimit) x[k] &= 0x0000ffffu;
        }
    }
    ptx::fence_proxy_async_smem();
    __syncwarp();
}

// Word i of this lane's accumulators in the 16 token rows of a stage that only
// `warp` reads (and has read).  Words 4 x .. 4 x + 3 are column block x of 8.
template <int DP>
__device__ __forceinline__ float* spill(uint8_t (*kv)[kTile * DP * 2], int warp, int i) {
    constexpr int kPerPiece = 16;  // 16 rows x 128 bytes = 16 words per lane
    const int piece = i / kPerPiece, halves = DP / 64;
    uint8_t* base = kv[piece / halves] + (piece % halves) * (kTile * 128) + warp * 16 * 128;
    return reinterpret_cast<float*>(base) + (i % kPerPiece) * 32 + (threadIdx.x & 31);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 2)
    decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const Params p) {
    using S = DecodeSmem<DP>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    S& sm = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x < 16) sm.place[threadIdx.x] = row_place(p, threadIdx.x);
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; s++) {
            ptx::mbar_init(&sm.full[s], 2);
            ptx::mbar_init(&sm.empty[s], 4);
            ptx::mbar_init(&sm.joined[s], 4);
        }
        for (int u = 0; u < kUnits; u++) {
            ptx::mbar_init(&sm.unit_full[u], 1);
            ptx::mbar_init(&sm.unit_empty[u], 4);
        }
        for (int q = 0; q < 2; q++) ptx::mbar_init(&sm.q_full[q], 129);  // all computing threads, and the row limits
        ptx::fence_mbarrier_init();
        ptx::prefetch_tmap(&map_k);
        ptx::prefetch_tmap(&map_v);
    }
    // After prefix_kernel this grid starts when all of that one's blocks have
    // seen the work before them finished, so the inputs are there (read past L1,
    // which may hold what they were before); it waits for prefix_kernel itself
    // only at the end.
    if (p.big_splits == 0) {
        ptx::griddep_wait();  // in this order: join_kernel reads the lengths without waiting
        ptx::griddep_launch_dependents();
    }
    for (uint32_t b = threadIdx.x; b < p.batch; b += kThreads) {
        const int2 q = seq_of(p, b);
        if (b < kKept) sm.seq[b] = q;
        sm.cum[b] = own_tiles(p, q.y);
    }
    auto seq = [&](uint32_t b) { return b < kKept ? sm.seq[b] : seq_of(p, b); };
    __syncthreads();
    if (warp == 0) {
        int base = 0;
        for (uint32_t b0 = 0; b0 < p.batch; b0 += 32) {
            const uint32_t b = b0 + lane;
            const int c = b < p.batch ? sm.cum[b] : 0;
            int s = c;
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += t;
            }
            if (b < p.batch) sm.cum[b] = base + s - c;
            base += __shfl_sync(0xffffffffu, s, 31);
        }
        if (lane == 0) sm.cum[p.batch] = base;
    } else if (warp == 1 && p.shared) {
        const int slot = prefix_slot(p, seq);
        if (lane == 0) sm.prefix_slot = slot;
    }
    __syncthreads();
    const int per_g = (int)(p.kv_heads * p.subs);  // units of a group
    if (p.cum && blockIdx.x == 0)
        for (uint32_t b = threadIdx.x; b <= p.batch; b += kThreads) p.cum[b] = sm.cum[b];
    const int total = group_start(p, sm.cum, p.groups) * per_g;
    const int per = (int)(((unsigned)total + gridDim.x - 1) / gridDim.x);

    if (warp >= 4) {
        // -------------------------------------------------------- producers
        // warp 4 loads K and announces units, warp 5 loads V
        const bool is_v = warp == 5;
        int at = (int)min((int64_t)blockIdx.x * per, (int64_t)total);
        const int end = (int)min((int64_t)(blockIdx.x + 1) * per, (int64_t)total);
        int g_now = 0;
        bool done = false;
        auto next_unit = [&] {  // the unit with the next tile; moves `at` past its part of the span
            Unit u{};
            u.head = -1;
            if (p.whole) {
                if (done) return u;
                done = true;
                u.grp = (int)blockIdx.x / per_g;
                const int id = (int)blockIdx.x % per_g;
                u.head = id / (int)p.subs;
                u.sub = id % (int)p.subs;
                u.t1 = group_start(p, sm.cum, u.grp + 1) - group_start(p, sm.cum, u.grp) - kUnitCost;
                return u;
            }
            while (at < end) {
                const int x = at / per_g;  // start(g) <= x < start(g + 1)
                int hi = (int)p.groups - 1;
                while (g_now < hi) {
                    const int mid = (g_now + hi + 1) >> 1;
                    if (group_start(p, sm.cum, mid) <= x) g_now = mid; else hi = mid - 1;
                }
                const int g0 = group_start(p, sm.cum, g_now), n = group_start(p, sm.cum, g_now + 1) - g0;
                const int id = (at - g0 * per_g) / n, first = g0 * per_g + id * n;
                u.grp = g_now;
                u.head = id / (int)p.subs;
                u.sub = id % (int)p.subs;
                u.slot = (int)blockIdx.x + g_now * per_g + id;
                u.t0 = max(at - first - kUnitCost, 0);
                u.t1 = min(n, end - first) - kUnitCost;
                at = first + min(n, end - first);
                if (u.t1 > u.t0) return u;
            }
            u.head = -1;
            return u;
        };
        uint32_t said = 0, n = 0;
        bool ok = true;
        auto announce = [&](const Unit& u) {
            if (is_v) return;
            const uint32_t e = said % kUnits;
            ok = ok && __all_sync(0xffffffffu, ptx::mbar_wait(&sm.unit_empty[e], ((said / kUnits) & 1) ^ 1, p.err));
            if (ok && lane == 0) {
                sm.unit[e] = u;
                ptx::mbar_arrive(&sm.unit_full[e]);
            }
            said++;
        };
        // one lane per box: 64 elements, box_keys tokens
        constexpr int kHalves = DP / 64;
        const int box_shift = 31 - __clz((int)p.box_keys), key_boxes = kTile >> box_shift, boxes = key_boxes * kHalves;
        const bool lane_on = lane < boxes;
        const int key0 = lane / kHalves * (int)p.box_keys, half = lane % kHalves;
        const CUtensorMap* map = is_v ? &map_v : &map_k;
        // Where tiles come from: a tile, its sequence's table, tiles left of that.
        struct Cursor {
            Tile t;
            const int32_t* table;
            int left;
        };
        auto own = [&](int b) { return sm.cum[b + 1] - sm.cum[b]; };
        auto to_sequence = [&](Cursor& c, const Unit& u, int b, int skip) {
            const int2 q = seq((uint32_t)b);
            const int seen = prefix_seen(p, q.y);
            c.t = Tile{b - u.grp * (int)p.per_unit, own_base(p, q.y) + skip * kTile, seen, q.y};
            c.table = p.tables + (size_t)max(q.y < (int)p.shared ? sm.prefix_slot : q.x, 0) * p.max_pages;
            c.left = own(b) - skip;
        };
        auto seek = [&](const Unit& u) {  // u has tiles
            Cursor c;
            int t = u.t0, b = u.grp * (int)p.per_unit;
            if (t < (int)p.prefix_tiles) {
                c.t = Tile{-1, t * kTile, 0, (int)p.shared};
                c.table = p.tables + (size_t)sm.prefix_slot * p.max_pages;
                c.left = (int)p.prefix_tiles - t;
                return c;
            }
            t -= (int)p.prefix_tiles;
            while (t >= own(b)) t -= own(b++);
            to_sequence(c, u, b, t);
            return c;
        };
        auto advance = [&](Cursor& c, const Unit& u) {  // there is a next tile
            c.t.key += kTile;
            if (--c.left) return;
            int b = u.grp * (int)p.per_unit + c.t.who + 1;
            while (own(b) == 0) b++;
            to_sequence(c, u, b, 0);
        };
        auto entry = [&](const Cursor& c) {  // page number of this lane's box
            const int j = c.t.key + key0;
            return lane_on && j < c.t.kend ? __ldcg(c.table + min((uint32_t)j >> p.page_shift, p.max_pages - 1)) : 0;
        };
        // A unit's cursors (tile to load; tile whose page is read) and the page
        // numbers between them.
        struct Ahead {
            Cursor load, read;
            int page[kPagesAhead];
        };
        auto begin = [&](const Unit& u) {  // u has tiles
            Ahead a;
            a.load = a.read = seek(u);
#pragma unroll
            for (int d = 0; d < kPagesAhead; d++) {
                a.page[d] = 0;
                if (u.t0 + d >= u.t1) continue;
                if (d) advance(a.read, u);
                a.page[d] = entry(a.read);
            }
            return a;
        };
        Unit u = next_unit(), following = u;
        announce(u);
        Ahead a{}, af{};
        if (u.head >= 0 && u.t1 > u.t0) a = begin(u);
        // announces the next unit and reads what it starts with
        auto look_ahead = [&] {
            following = next_unit();
            announce(following);
            if (following.head >= 0) af = begin(following);
        };
        while (ok && u.head >= 0) {
            int t = u.t0, stop = min(u.t0 + S::kStages, u.t1);
            for (;;) {
#pragma unroll
                for (int d = 0; d < kPagesAhead; d++) {  // (page numbers on their way cannot change registers)
                    if (!ok || t >= stop || ((t - u.t0) & (kPagesAhead - 1)) != d) continue;
                    const Tile now = a.load.t;
                    const int page = a.page[d];
                    if (t + 1 < u.t1) advance(a.load, u);
                    const uint32_t st = n % S::kStages;
                    ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.empty[st], ((n / S::kStages) & 1) ^ 1, p.err));
                    if (!ok) continue;
                    // boxes past the last key are left out
                    const int live = min(key_boxes, (now.kend - now.key + (int)p.box_keys - 1) >> box_shift);
                    if (lane == 0) {
                        if (!is_v) sm.tile[st] = now;
                        ptx::mbar_arrive_expect_tx(&sm.full[st], kHalves * 128 * p.box_keys * live);
                    }
                    __syncwarp();
                    const int j = now.key + key0;
                    if (lane_on && j < now.kend)
                        tma_load_4d(sm.kv[st][is_v] + half * S::kHalf + key0 * 128, map, &sm.full[st],
                                    half * 64, u.head, j & ((1 << p.page_shift) - 1), (uint32_t)page < p.pages ? page : 0);
                    if (t + kPagesAhead < u.t1) advance(a.read, u), a.page[d] = entry(a.read);
                    t++;
                    n++;
                }
                if (!ok) break;
                // with the first tiles on their way (in one place: its code is long)
                if (t == min(u.t0 + S::kStages, u.t1)) look_ahead(), stop = u.t1;
                if (t >= u.t1) break;
            }
            u = following;
            a = af;
        }
    } else {
        // -------------------------------------------------------- computing
        uint32_t seen = 0, n = 0, join_phase = 0;
        bool ok = true;
        const RowPlace place[2] = {sm.place[lane / 4], sm.place[lane / 4 + 8]};
        Unit u, un;
        // the next unit, and its query rows on their way to the other place
        auto fetch = [&](Unit& dst) {
            const uint32_t e = seen % kUnits, to = seen & 1;
            ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.unit_full[e], (seen / kUnits) & 1, p.err));
            if (!ok) return;
            seen++;
            dst = sm.unit[e];
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&sm.unit_empty[e]);
            if (dst.head < 0) return;
            constexpr int kChunks = DP / 8;
            uint32_t b, g;
#pragma unroll
            for (int i = 0; i < kChunks / 8; i++) {
                const uint32_t c = threadIdx.x + i * 128, row = c / kChunks, ch = c % kChunks;
                const bool on = row_of(p, dst.grp, dst.sub, sm.place[row], b, g) && ch * 8 < p.dim;
                const uint16_t* src = static_cast<const uint16_t*>(p.q.data) +
                                      (on ? (size_t)b * p.q.token_stride + (size_t)(dst.head * p.group + g) * p.q.head_stride + ch * 8 : 0);
                cp16(ptx::smem_u32(sm.q[to] + q_off(row, ch)), src, on ? 16 : 0);
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(ptx::smem_u32(&sm.q_full[to])) : "memory");
            if (warp == 0) {
                if (lane < 16)
                    sm.vis[to][lane] = row_of(p, dst.grp, dst.sub, sm.place[lane], b, g) ? prefix_seen(p, seq(b).y) : 0;
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&sm.q_full[to]);
            }
        };
        fetch(u);
        for (uint32_t nu = 0; ok && u.head >= 0; nu++, u = un) {
            const uint32_t e = nu & 1;
            ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.q_full[e], (nu >> 1) & 1, p.err));
            if (!ok) break;
            Query<DP> q;
#pragma unroll
            for (int kk = 0; kk < DP / 16; kk++)
                ldsm4(ptx::smem_u32(sm.q[e] + q_off((lane >> 3 & 1) * 8 + (lane & 7), kk * 2 + (lane >> 4))), q.q[kk]);
            const int vis[2] = {sm.vis[e][lane / 4], sm.vis[e][lane / 4 + 8]};
            un.head = -2;  // not looked at yet
            Sums<DP> r;
#pragma unroll
            for (int i = 0; i < DP / 8; i++) r.o[i][0] = r.o[i][1] = r.o[i][2] = r.o[i][3] = 0.0f;
            r.m[0] = r.m[1] = kNegInf;
            r.l[0] = r.l[1] = 0.0f;
            uint32_t st = 0;
            for (int t = u.t0; t < u.t1; t++, n++) {
                st = n % S::kStages;
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.full[st], (n / S::kStages) & 1, p.err));
                if (!ok) break;
                const Tile now = sm.tile[st];
                const int j0 = now.key + warp * 16;
                if (j0 + 16 > now.kend || j0 < now.lo) {
                    // rows of V that do not count: a weight of 0 does not silence a NaN
                    for (int i = lane; i < 16 * DP / 8; i += 32) {
                        const int tok = warp * 16 + i % 16, key = now.key + tok;
                        if (key >= now.kend || key < now.lo)
                            *reinterpret_cast<uint4*>(sm.kv[st][1] + tile_off(tok, i / 16)) = make_uint4(0, 0, 0, 0);
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                }
                if (j0 < now.kend && j0 + 16 > now.lo) {
#pragma unroll
                    for (int h = 0; h < 2; h++) q.vis[h] = now.who < 0 ? vis[h] : (int)place[h].seq == now.who ? now.kend - now.lo : 0;
                    if (now.who >= 0 && p.per_unit > 1 && p.batch > 1)
                        set_apart<T, DP>(r, sm.kv[st][1], warp * 16, {q.vis[0] > 0, q.vis[1] > 0});
                    tile_step<T, DP>(q, r, ptx::smem_u32(sm.kv[st][0]), ptx::smem_u32(sm.kv[st][1]), warp * 16,
                                     j0 - now.lo, p.scale2);
                }
                __syncwarp();
                if (t + 1 < u.t1 && lane == 0) ptx::mbar_arrive(&sm.empty[st]);
                // rows that have seen nothing so far start from 0, whatever the prefix's V made of their weights of 0
                if (t + 1 == (int)p.prefix_tiles || t + 1 == u.t1) {
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int i = 0; i < DP / 8; i++)
                            if (r.m[h] == kNegInf) r.o[i][2 * h] = r.o[i][2 * h + 1] = 0.0f;
                }
                if (t == u.t0) fetch(un);
                if (!ok) break;
            }
            if (!ok) break;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                r.l[h] += __shfl_xor_sync(0xffffffffu, r.l[h], 1);
                r.l[h] += __shfl_xor_sync(0xffffffffu, r.l[h], 2);
            }
            constexpr int kQuarter = DP / 8;  // words per lane
            float m[2] = {kNegInf, kNegInf}, l[2] = {0.0f, 0.0f}, o[kQuarter];
#pragma unroll
            for (int i = 0; i < kQuarter; i++) o[i] = 0.0f;
            if (u.t1 <= u.t0) fetch(un);
            if (!ok) break;
            if (u.t1 > u.t0) {
                // the warps' sums meet in the last tile's stage, which is still theirs;
                // each warp joins a quarter of the columns
                if ((lane & 3) == 0) {
                    sm.ml[st][warp][lane / 4] = make_float2(r.m[0], r.l[0]);
                    sm.ml[st][warp][lane / 4 + 8] = make_float2(r.m[1], r.l[1]);
                }
#pragma unroll
                for (int i = 0; i < DP / 2; i++) *spill<DP>(sm.kv[st], warp, i) = r.o[i >> 2][i & 3];
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&sm.joined[st]);
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.joined[st], (join_phase >> st) & 1, p.err));
                if (!ok) break;
                join_phase ^= 1u << st;
                float2 ml[2][4];
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        ml[h][w] = sm.ml[st][w][lane / 4 + 8 * h];
                        m[h] = fmaxf(m[h], ml[h][w].x);
                    }
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    float f[2];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        f[h] = exp2_fast(ml[h][w].x - (m[h] == kNegInf ? 0.0f : m[h]));
                        l[h] += ml[h][w].y * f[h];
                    }
#pragma unroll
                    for (int i = 0; i < kQuarter; i++) o[i] += *spill<DP>(sm.kv[st], w, warp * kQuarter + i) * f[(i & 3) >> 1];
                }
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&sm.empty[st]);
            }
            // rows of this warp's quarter of the columns
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t row = lane / 4 + 8 * h;
                uint32_t b, g;
                if (!row_of(p, u.grp, u.sub, place[h], b, g)) continue;
                const uint32_t head = u.head * p.group + g;
                const bool empty = l[h] == 0.0f;
                const float f = empty ? 0.0f : 1.0f / l[h];
                const size_t at = (size_t)u.slot * p.rows + row;
                uint8_t* out = static_cast<uint8_t*>(p.out.data) +
                               ((size_t)b * p.out.token_stride + (size_t)head * p.out.head_stride) *
                                   (p.out_dtype == ANE_DTYPE_F32 ? 4 : 2);
                if (warp == 0 && (lane & 3) == 0) {
                    if (!p.whole)
                        *reinterpret_cast<float2*>(p.sm + at * 2) = make_float2(m[h], l[h]);
                    else if (p.lse)
                        p.lse[(size_t)b * p.heads + head] = empty ? kNegInf : (m[h] + log2f(l[h]) - Type<T>::kShift) * kLn2;
                }
#pragma unroll
                for (int x = 0; x < kQuarter / 4; x++) {
                    const uint32_t c = (warp * (kQuarter / 4) + x) * 8 + 2 * (lane & 3);
                    if (c >= p.dim) continue;
                    const float y0 = o[4 * x + 2 * h], y1 = o[4 * x + 2 * h + 1];
                    if (!p.whole)
                        *reinterpret_cast<float2*>(p.so + at * p.dim + c) = make_float2(y0, y1);
                    else
                        store2(out, c, p.out_dtype, empty ? 0.0f : y0 * f, empty ? 0.0f : y1 * f);
                }
            }
        }
    }
    if (p.big_splits != 0) {
        ptx::griddep_launch_dependents();
        ptx::griddep_wait();
    }
}

// ------------------------------------------------------- prefix on tcgen05
struct PrefixJob {
    const Params& p;
    uint32_t pairs;  // items along the rows: two tiles of 128 / group sequences each
    const int32_t* table;

    __device__ void start() {
        table = p.tables + (size_t)prefix_slot(p, [&](uint32_t b) { return seq_of(p, b); }) * p.max_pages;
    }

    __device__ BigItem item(int i) const {
        const uint32_t tt = kBigRows / p.group, w = (uint32_t)i * gridDim.x + blockIdx.x;  // split, head, pair
        const int tiles = (int)((p.shared + kBigKeys - 1) / kBigKeys);
        BigItem it{};
        it.head = -1;
        if (w < p.big_splits * p.kv_heads * pairs) {
            const uint32_t split = w / (p.kv_heads * pairs), pair = w % pairs;
            it.head = (int)(w / pairs % p.kv_heads);
            it.q_token = (int)(pair * 2 * tt);
            it.tokens = (int)min(2 * tt, p.batch - pair * 2 * tt);
            it.lk = (int)p.shared;
            it.begin = (int)((uint64_t)tiles * split / p.big_splits);
            const int end = (int)((uint64_t)tiles * (split + 1) / p.big_splits);
            it.end[0] = end;
            it.end[1] = it.tokens > (int)tt ? end : it.begin;
            it.slot = (int)split;
        }
        return it;
    }
    __device__ int box_keys() const { return (int)p.box_keys; }
    __device__ int2 coord(const BigItem& it, int key) const {
        return page_of(p, table, min(key, (int)p.shared - 1) & ~((int)p.box_keys - 1));
    }
    __device__ int visible(const BigItem& it, int token) const {
        return prefix_seen(p, len_of(p, (uint32_t)(it.q_token + token)));
    }
    __device__ void result(const BigItem& it, int row, int token, float m, float l, float shift, uint8_t*& dst,
                           float& factor) const {
        const size_t rows = (size_t)p.batch * p.group;
        const size_t at = ((size_t)it.slot * p.kv_heads + it.head) * rows + (size_t)(it.q_token + token) * p.group + row % p.group;
        *reinterpret_cast<float2*>(p.pm + at * 2) = make_float2(m, l);
        dst = reinterpret_cast<uint8_t*>(p.po + at * p.dim);
        factor = l == 0.0f ? 0.0f : 1.0f;
    }
    __device__ uint32_t dim() const { return p.dim; }
    __device__ uint32_t out_dtype(const BigItem&) const { return ANE_DTYPE_F32; }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kBigThreads, 1)
    prefix_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const Params p, uint32_t pairs) {
    PrefixJob job{p, pairs, nullptr};
    big_attention<T, DP>(&map_q, &map_k, &map_v, p.group, p.scale2, p.err, job);
}

// -------------------------------------------------------------------- join
// One block per output row; its warps take the partial results in turn.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Params p) {
    __shared__ float sm_m[4], sm_l[4];
    __shared__ float4 sm_o[4][32];
    __shared__ int sm_tiles[4][3];
    ptx::griddep_launch_dependents();
    const uint32_t b = blockIdx.x, head = blockIdx.y, h = head / p.group, g = head % p.group;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // spans [pc, pe) of prefix_kernel and [oc, oe) of decode_kernel's blocks hold
    // partials of this row: of span c at row prow + c * pstep, orow + c * p.rows
    const int pc = 0, pe = (int)p.big_splits;
    const size_t all_rows = (size_t)p.batch * p.group;
    const size_t prow = (size_t)h * all_rows + b * p.group + g, pstep = all_rows * p.kv_heads;
    const uint32_t grp = b / p.per_unit, sub = p.group > 16 ? g / 16 : 0;
    const uint32_t row = p.group > 16 ? g % 16 : b % p.per_unit * p.group + g;
    // Where decode_kernel's blocks cut the line: own tiles of the sequences before the
    // row's unit, of the unit and of all.
    int tiles[3] = {0, 0, 0};
    if (p.cum) {
        ptx::griddep_wait();
        tiles[0] = __ldcg(p.cum + grp * p.per_unit);
        tiles[1] = __ldcg(p.cum + min((grp + 1) * p.per_unit, p.batch)) - tiles[0];
        tiles[2] = __ldcg(p.cum + p.batch);
    } else {  // from the lengths, while those blocks end
        for (uint32_t x = threadIdx.x; x < p.batch; x += kJoinThreads) {
            const int own = own_tiles(p, len_of(p, x)), u = (int)(x / p.per_unit) - (int)grp;
            tiles[0] += u < 0 ? own : 0;
            tiles[1] += u == 0 ? own : 0;
            tiles[2] += own;
        }
#pragma unroll
        for (int i = 0; i < 3; i++) {
            tiles[i] = __reduce_add_sync(0xffffffffu, tiles[i]);
            if (lane == 0) sm_tiles[warp][i] = tiles[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 3; i++) tiles[i] = sm_tiles[0][i] + sm_tiles[1][i] + sm_tiles[2][i] + sm_tiles[3][i];
        ptx::griddep_wait();
    }
    const int per_g = (int)(p.kv_heads * p.subs), id = (int)(h * p.subs + sub), c0 = tiles[0];
    const int total = ((int)(p.groups * (kUnitCost + p.prefix_tiles)) + tiles[2]) * per_g;
    const int per = (int)(((unsigned)total + p.blocks - 1) / p.blocks);
    const int n = tiles[1] + (int)p.prefix_tiles;  // tiles of the row's unit
    int oc = 0, oe = 0;
    if (n) {
        const int first = ((int)(grp * (kUnitCost + p.prefix_tiles)) + c0) * per_g + id * (n + kUnitCost) + kUnitCost;
        oc = first / per;
        oe = (first + n - 1) / per + 1;
    }
    const size_t orow = (size_t)((int)grp * per_g + id) * p.rows + row;
    float m = kNegInf, l = 0.0f;
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const bool on = (uint32_t)lane * 4 < p.dim;
    // four partials of each warp on their way at a time
    const int count = (pe - pc) + (oe - oc);
    for (int i0 = warp; i0 < count; i0 += 16) {
        float2 x[4];
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = i0 + 4 * k;
            const bool pre = i < pe - pc;
            const size_t at = pre ? prow + (size_t)(pc + i) * pstep : orow + (size_t)(oc + i - (pe - pc)) * p.rows;
            x[k] = make_float2(kNegInf, 0.0f);
            v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i < count) {
                x[k] = __ldcg(reinterpret_cast<const float2*>((pre ? p.pm : p.sm) + at * 2));
                if (on) v[k] = __ldcg(reinterpret_cast<const float4*>((pre ? p.po : p.so) + at * p.dim + lane * 4));
            }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float mn = fmaxf(m, x[k].x), base = mn == kNegInf ? 0.0f : mn;
            const float ca = exp2_fast(m - base), cb = exp2_fast(x[k].x - base);
            m = mn;
            l = l * ca + x[k].y * cb;
            o[0] = o[0] * ca + v[k].x * cb;
            o[1] = o[1] * ca + v[k].y * cb;
            o[2] = o[2] * ca + v[k].z * cb;
            o[3] = o[3] * ca + v[k].w * cb;
        }
    }
    if (lane == 0) sm_m[warp] = m, sm_l[warp] = l;
    sm_o[warp][lane] = make_float4(o[0], o[1], o[2], o[3]);
    __syncthreads();
    const uint32_t c = threadIdx.x;
    m = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
    const float base = m == kNegInf ? 0.0f : m;
    float sum = 0.0f;
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const float f = exp2_fast(sm_m[w] - base);
        l += sm_l[w] * f;
        sum += reinterpret_cast<const float*>(sm_o[w])[c] * f;
    }
    if (c < p.dim) {
        const float y = l == 0.0f ? 0.0f : sum / l;
        const size_t at = (size_t)b * p.out.token_stride + (size_t)head * p.out.head_stride + c;
        if (p.out_dtype == ANE_DTYPE_F32)
            static_cast<float*>(p.out.data)[at] = y;
        else
            static_cast<uint16_t*>(p.out.data)[at] = (uint16_t)Type<T>::pack(y, 0.0f);
    }
    if (p.lse && c == 0) p.lse[(size_t)b * p.heads + head] = l == 0.0f ? kNegInf : (m + log2f(l) - Type<T>::kShift) * kLn2;
}

// ------------------------------------------------------------------ launch
struct Layout {
    uint32_t per_unit, groups, subs, rows, pairs, big_splits;
    size_t cum, pm, po, sm, so, bytes;
};
Layout layout(uint32_t batch, uint32_t heads, uint32_t kv_heads, uint32_t dim) {
    Layout l;
    const uint32_t group = heads / kv_heads;
    l.per_unit = group > 16 ? 1 : 16 / group;
    l.groups = (uint32_t)ceil_div(batch, l.per_unit);
    l.subs = (uint32_t)ceil_div(group, 16);
    l.rows = group > 16 ? 16 : (l.per_unit < batch ? l.per_unit : batch) * group;
    l.pairs = (uint32_t)ceil_div(batch, 2 * (kBigRows / group));
    l.big_splits = kBigBlocks / (kv_heads * l.pairs);
    if (l.big_splits == 0) l.big_splits = 1;
    const size_t own_rows = (kMaxBlocks + (size_t)kv_heads * l.groups * l.subs) * l.rows;
    const size_t prefix_rows = (size_t)l.big_splits * kv_heads * batch * group;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    l.cum = take((batch + 1) * 4);
    l.pm = take(prefix_rows * 8);
    l.sm = take(own_rows * 8);
    l.po = take(prefix_rows * dim * 4);
    l.so = take(own_rows * dim * 4);
    l.bytes = at;
    return l;
}

template <typename T, int DP>
int launch(const CUtensorMap (&map)[3], const Params& p, uint32_t pairs, cudaStream_t s) {
    static std::atomic<uint64_t> done{0}, done_big{0};
    int rc;
    if (p.big_splits) {
        if ((rc = set_max_dynamic_smem(prefix_kernel<T, DP>, (int)big_smem_bytes<DP>(), done_big))) return rc;
        const uint64_t items = (uint64_t)p.big_splits * p.kv_heads * pairs;
        const uint64_t blocks = items < (uint64_t)num_sms() ? items : (uint64_t)num_sms();
        if ((rc = launch_pdl(prefix_kernel<T, DP>, dim3((uint32_t)blocks), dim3(kBigThreads), big_smem_bytes<DP>(), s,
                             map[0], map[1], map[2], p, pairs)))
            return rc;
    }
    if ((rc = set_max_dynamic_smem(decode_kernel<T, DP>, (int)decode_smem_bytes<DP>(), done))) return rc;
    if ((rc = launch_pdl(decode_kernel<T, DP>, dim3(p.blocks), dim3(kThreads), decode_smem_bytes<DP>(), s, map[1], map[2], p)) ||
        p.whole)
        return rc;
    return launch_pdl(join_kernel<T>, dim3(p.batch, p.heads), dim3(kJoinThreads), 0, s, p);
}

}  // namespace
}  // namespace ane_b200

using namespace ane_b200;

extern "C" size_t ane_attn_decode_workspace_size(uint32_t batch, uint32_t heads, uint32_t kv_heads, uint32_t dim) {
    if (kv_heads == 0 || heads < kv_heads || heads % kv_heads || heads / kv_heads > 64 || batch == 0 || batch > kMaxBatch)
        return 0;
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
    ANE_ARG_CHECK(heads <= 65535, "attn_decode: at most 65535 heads");  // the join's grid
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
    const Layout l = layout(batch, heads, kv_heads, dim);
    const uint64_t most = (uint64_t)max_pages * pt;  // tokens of a slot
    ANE_ARG_CHECK(most <= 0x7fffff00u &&
                      (most / kTile + kUnitCost + 2) * kv_heads * l.subs * ((uint64_t)batch + l.groups) <= 0x7fffffffu,
                  "attn_decode: more than 2^31 tiles of 64 tokens");
    ANE_ARG_CHECK(shared <= most, "attn_decode: shared exceeds max_pages pages");
    ANE_ARG_CHECK(workspace && (uintptr_t)workspace % 256 == 0 && workspace_bytes >= l.bytes,
                  "attn_decode: workspace must be 256-byte aligned and of ane_attn_decode_workspace_size bytes");
    if ((rc = require_sm100())) return rc;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    Params p{};
    p.batch = batch, p.heads = heads, p.kv_heads = kv_heads, p.group = heads / kv_heads, p.dim = dim;
    p.out_dtype = out_dtype;
    p.shared = shared;
    // decode_kernel goes over the prefix once per unit of 16 rows.  The second time costs
    // little (L2), every further one a tile's time: prefix_kernel from where that
    // makes eight tiles a block.  us without and with it: 128 rows x 8 heads behind 2048
    // 23 and 24, behind 4096 29 and 26, behind 16384 64 and 35; 256 rows x 8 heads behind
    // 1000 27 and 29, behind 2048 33 and 31; 64 rows x 32 heads behind 1000 35 and 36,
    // behind 4096 54 and 50; 32 rows x 32 heads behind 16384 72 and 85.  Over 1056 calls
    // of 2 to 256 sequences the choice costs 0.9 % of the better one's time on average.
    const uint32_t units = l.groups * l.subs;
    const uint64_t again = units > 2 ? (uint64_t)(units - 2) * kv_heads * ceil_div(shared, kTile) : 0;
    const bool big = again >= 8 * 2 * (uint64_t)kBigBlocks;
    if (big) {
        const uint32_t tiles = (uint32_t)ceil_div(shared, kBigKeys);
        p.big_splits = l.big_splits < tiles ? l.big_splits : tiles;
    } else {
        p.prefix_tiles = (uint32_t)ceil_div(shared, kTile);
    }
    p.per_unit = l.per_unit, p.groups = l.groups, p.subs = l.subs, p.rows = l.rows;
    p.n_slots = n_slots, p.max_pages = max_pages, p.pages = pages->pages;
    while ((1u << p.page_shift) < pt) p.page_shift++;
    p.scale2 = scale * attn::kLog2e;
    p.q = *q, p.out = *out;
    p.tables = tables, p.lens = lens, p.slots = slots, p.lse = lse;
    if (batch > kCountedBatch) p.cum = reinterpret_cast<int32_t*>(ws + l.cum);
    p.pm = reinterpret_cast<float*>(ws + l.pm), p.po = reinterpret_cast<float*>(ws + l.po);
    p.sm = reinterpret_cast<float*>(ws + l.sm), p.so = reinterpret_cast<float*>(ws + l.so);
    p.err = device_timeout_flag();
    // one box shape for both kernels: a page, or 64 tokens of a larger one
    p.box_keys = pt < (uint32_t)kTile ? pt : (uint32_t)kTile;
    const uint64_t own = ceil_div(most - (shared & ~(p.box_keys - 1)), kTile);  // of a sequence, at most
    p.whole = !big && p.prefix_tiles + (batch < l.per_unit ? batch : l.per_unit) * own <= kWholeTiles;
    const uint32_t spans = (uint32_t)num_sms() * 2;
    p.blocks = p.whole ? kv_heads * l.groups * l.subs : spans < kMaxBlocks ? spans : kMaxBlocks;
    const auto type = dtype == ANE_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    CUtensorMap map[3];
    if (big && (rc = encode_tensor_map_3d(&map[0], type, q->data, {dim, heads, batch},
                                          {q->head_stride * 2, q->token_stride * 2}, {64, p.group, 128 / p.group},
                                          CU_TENSOR_MAP_SWIZZLE_128B)))
        return rc;
    const void* pool[2] = {pages->k, pages->v};
    for (int i = 0; i < 2; i++)
        if ((rc = encode_tensor_map_4d(&map[1 + i], type, pool[i], {dim, kv_heads, pt, pages->pages},
                                       {pages->head_stride * 2, pages->token_stride * 2, pages->page_stride * 2},
                                       {64, 1, p.box_keys, 1}, CU_TENSOR_MAP_SWIZZLE_128B)))
            return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == ANE_DTYPE_F16)
        rc = dim <= 64 ? launch<__half, 64>(map, p, l.pairs, s) : launch<__half, 128>(map, p, l.pairs, s);
    else
        rc = dim <= 64 ? launch<__nv_bfloat16, 64>(map, p, l.pairs, s) : launch<__nv_bfloat16, 128>(map, p, l.pairs, s);
    return rc ? rc : ok();
}
