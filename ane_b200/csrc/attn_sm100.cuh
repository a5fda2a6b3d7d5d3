// attn_sm100.cuh -- softmax attention of 256 query rows against key/value tiles
// on the tensor cores, for prompts (packed keys, causal) and for a batch's
// shared prefix (paged keys, partial results).
//
// A work item is one key/value head, two query tiles of 128 rows and a span of
// key tiles.  A row is (query token, head of the group): the query heads that
// share a key/value head share its tiles.  Per tile of 128 keys:
//   S = Q K^T           tcgen05.mma, operands in shared memory, S in TMEM
//   P = exp2(S - m)     one thread per row: registers, back into TMEM as 16 bit
//   O += P V            tcgen05.mma, P from TMEM, V as an MN-major operand
// While one tile's threads are at their exponentials, the tensor cores work on
// the other tile.  A row's reference m is moved only when its new maximum passes
// it by 2^8: then (rarely) O is rescaled in TMEM, otherwise the larger weights
// stand and cancel against the row sum, which is kept in fp32.  F16 weights are
// stored 2^6 times larger (2^14 at most), as attn_core.cuh explains.
//
// What bounds it: per tile of 128 x 128 scores and head dim 128 the tensor cores
// take 1024 cycles (both products), the 16384 exponentials 1024 cycles of the
// special-function units, and a tile's products wait for its exponentials, the
// next scores for those products.  Measured per pair of tiles: 2800 cycles at head
// dim 64 and 128 alike, 73 % of the tensor cores' time at 128; a tile on its own
// takes as long, so it is that chain (scores ready -> weights 2500 cycles -> last
// products and next scores 960) that is left.  Hence P is handed over in parts and
// the weights do not wait for the tile's maximum.  Tried and slower (16384 tokens,
// 1613 us then): 2, 3, 4 of eight exponentials as a polynomial on the FMA units
// (1791, 1790, 1899); two threads per row (2250); the two warps of a scheduler
// taking turns at their exponentials (1635); with head dim 64, P apart from S so
// that the next scores do not wait for P (174 -> 190 us on a block of 1024).  Over
// seconds the chip's power limit holds the clock at 1.45 GHz.
//
// Warps (384 threads): 0-3 and 4-7 softmax of tile 0 and 1; 8 loads (TMA);
// 9 issues the MMAs and owns TMEM; 10 clears the rows of V that lie past the
// last key (a weight of 0 does not silence a NaN there); 11 finds the items.
// Registers: 384 x 168 at launch; 256 x 208 + 128 x 88 after the split, the same
// 64,512.
#pragma once
#include "attn_core.cuh"

namespace ane_b200 {
namespace attn {

constexpr int kBigThreads = 384;
constexpr int kBigRows = 128;    // rows of a query tile
constexpr int kBigKeys = 128;    // keys of a key/value tile
constexpr float kSlack = 8.0f;   // log2 of how far weights may pass 1
constexpr int kItemRing = 4;     // items announced ahead

struct BigItem {
    int q_token;     // first query token (a row of q); tokens of the item: `tokens`
    int tokens;
    int k0;          // packed keys: row of key 0
    int lk;          // keys of the sequence (or shared tokens)
    int see;         // packed: token i of the item sees keys 0 .. see + i
    int head;        // key/value head; -1: no such item
    int begin;       // first key tile
    int end[2];      // key tiles of query tile 0 and 1 end here (begin or less: none)
    int slot;        // partial results: their place
};

template <int DP>
struct BigSmem {
    static constexpr int kStages = DP == 128 ? 4 : 8;
    static constexpr int kTileBytes = 128 * DP * 2;
    uint8_t q[2][kTileBytes];
    uint8_t kv[kStages][kTileBytes];
    uint8_t out[8][32 * 128];  // per softmax warp: 128 bytes of 32 result rows
    uint64_t q_full, q_empty, kv_full[kStages], kv_empty[kStages], tail_full[kStages];
    uint64_t s_full[2], p_part[3][2], o_full[2];  // P: 64, 32 and 32 keys
    uint64_t item_full[kItemRing], item_empty[kItemRing];
    uint32_t tmem;
    BigItem items[kItemRing];
};
template <int DP>
constexpr size_t big_smem_bytes() {
    return sizeof(BigSmem<DP>) + 1024;
}
static_assert(big_smem_bytes<128>() <= 232448 && big_smem_bytes<64>() <= 232448, "shared memory budget");

__device__ __forceinline__ uint64_t desc_k(uint32_t base, int kk) {  // 16 elements at element 16 kk, K-major
    return ptx::sdesc_kmajor_sw128(base + (kk >> 2) * 16384 + (kk & 3) * 32);
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z,
                                            int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(ptx::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(ptx::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Stores that stay predicated: a branch around each cost more than the store.
__device__ __forceinline__ void store16_if(bool on, void* dst, uint4 v) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %0, 0;\n\t"
        "@p st.global.v4.b32 [%1], {%2, %3, %4, %5};\n\t}" ::"r"((int)on),
        "l"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
        : "memory");
}
// One warp: the DP accumulator columns of its 32 rows (TMEM address `to`), times
// factor, to each row's dst (NULL: no such row), as T or F32.  128 bytes
// of every row at a time go through shared memory, so that a store instruction
// writes four rows' whole lines (a row per lane would touch 32 lines).
// any: false if there is no accumulator (the rows are 0).
template <typename T>
__device__ __forceinline__ uint32_t pack_out(uint32_t a, uint32_t b) {
    return Type<T>::pack(__uint_as_float(a), __uint_as_float(b));
}
template <typename T, int DP>
__device__ __forceinline__ void store_rows(uint8_t* stage, uint8_t* dst, float factor, bool any, uint32_t to,
                                           uint32_t dim, uint32_t out_dtype) {
    const int lane = threadIdx.x & 31;
    const uint32_t row_bytes = dim * (out_dtype == ANE_DTYPE_F32 ? 4 : 2), at0 = (lane & 7) * 16;
    const uint32_t keep = any && factor != 0.0f ? 0xffffffffu : 0u;  // 0 whatever the accumulator holds
    const float2 f2 = make_float2(factor, factor);
    uint4* mine = reinterpret_cast<uint4*>(stage + lane * 128);
    unsigned long long to_row[8];  // of the rows that this lane stores
#pragma unroll
    for (int i = 0; i < 8; i++)
        to_row[i] = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), i * 4 + (lane >> 3));
    auto flush = [&](uint32_t at) {  // the staged 128 bytes go to byte `at` of the rows
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = i * 4 + (lane >> 3);
            const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
            store16_if(to_row[i] && at + at0 < row_bytes, reinterpret_cast<uint8_t*>(to_row[i]) + at + at0, v);
        }
        __syncwarp();
    };
    // one wait for all columns: each costs some 350 cycles next to running MMAs
    // (read even if there is nothing: a branch here made the compiler spill)
    uint32_t o[DP / 32][32];
#pragma unroll
    for (int c = 0; c < DP / 32; c++) ptx::tmem_ld_32x32b_x32(to + c * 32, o[c]);
    ptx::tmem_ld_wait();
#pragma unroll
    for (int c = 0; c < DP / 32; c++) ptx::pin32(o[c]);
#pragma unroll
    for (int c = 0; c < DP / 32; c++)
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const float2 y = ptx::fmul2(make_float2(__uint_as_float(o[c][i]), __uint_as_float(o[c][i + 1])), f2);
            o[c][i] = __float_as_uint(y.x);
            o[c][i + 1] = __float_as_uint(y.y);
        }
    if (out_dtype == ANE_DTYPE_F32) {
#pragma unroll
        for (int c = 0; c < DP / 32; c++) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t* x = &o[c][4 * i];
                mine[i ^ (lane & 7)] = make_uint4(x[0] & keep, x[1] & keep, x[2] & keep, x[3] & keep);
            }
            flush(c * 128);
        }
    } else {
#pragma unroll
        for (int c = 0; c < DP / 32; c += 2) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t* x = &o[c + (i >> 2)][8 * (i & 3)];
                mine[i ^ (lane & 7)] = make_uint4(pack_out<T>(x[0], x[1]) & keep, pack_out<T>(x[2], x[3]) & keep,
                                                  pack_out<T>(x[4], x[5]) & keep, pack_out<T>(x[6], x[7]) & keep);
            }
            flush(c * 64);
        }
    }
}

// The kernel's frame.  Job supplies:
//   start()                     called by the loading warp before coord
//   item(i)                     item i of this block (a whole warp; head -1: no more)
//   box_keys()                  keys per TMA box (a multiple of 8 that divides 128)
//   coord(item, key)            {token, page} coordinates of the box that starts at a key
//   visible(item, token)        keys that query token `token` of the item sees
//   result(item, row, token, m, l, shift, dst, factor)  where a row's result goes, what it is
//                               multiplied by (0: it is 0), its statistics written
//   out_dtype(item), dim()
template <typename T, int DP, class Job>
__device__ __forceinline__ void big_attention(const CUtensorMap* map_q, const CUtensorMap* map_k,
                                              const CUtensorMap* map_v, uint32_t group, float scale2, int* err,
                                              Job& job) {
    using S = BigSmem<DP>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    S& sm = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr int kBoxes = DP / 64;  // 64-element boxes of 128 rows x 128 bytes
    constexpr int kBoxBytes = 128 * 128;
    constexpr float kShift = Type<T>::kShift;  // with kSlack: F16 weights stay below 2^14
    constexpr bool kBf16 = Type<T>::kShift == 0.0f;
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int tile_tokens = kBigRows / (int)group;

    if (threadIdx.x == 0) {
        ptx::mbar_init(&sm.q_full, 1);
        ptx::mbar_init(&sm.q_empty, 1);
        for (int s = 0; s < S::kStages; s++) {
            ptx::mbar_init(&sm.kv_full[s], 1);
            ptx::mbar_init(&sm.kv_empty[s], 1);
            ptx::mbar_init(&sm.tail_full[s], 1);
        }
        for (int t = 0; t < 2; t++) {
            ptx::mbar_init(&sm.s_full[t], 1);
            for (int x = 0; x < 3; x++) ptx::mbar_init(&sm.p_part[x][t], 4);
            ptx::mbar_init(&sm.o_full[t], 1);
        }
        for (int i = 0; i < kItemRing; i++) {
            ptx::mbar_init(&sm.item_full[i], 1);
            ptx::mbar_init(&sm.item_empty[i], 11);  // 8 softmax warps, loads, MMAs, V rows
        }
        ptx::fence_mbarrier_init();
        ptx::prefetch_tmap(map_q);
        ptx::prefetch_tmap(map_k);
        ptx::prefetch_tmap(map_v);
    }
    if (warp == 9) {
        ptx::tmem_alloc(&sm.tmem, 512);
        ptx::tmem_relinquish();
    }
    // in this order: a dependent grid that does not wait may still rely on the
    // work before this one (attn_decode.cu)
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = sm.tmem;  // columns: S0 0, S1 128, O0 256, O1 384
    // item i, for a whole warp; false: no more, or gave up
    auto take = [&](int i, BigItem& it) {
        const int e = i % kItemRing;
        if (!__all_sync(0xffffffffu, ptx::mbar_wait(&sm.item_full[e], (i / kItemRing) & 1, err))) return false;
        it = sm.items[e];
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&sm.item_empty[e]);
        return __all_sync(0xffffffffu, it.head >= 0) != 0;
    };

    if (warp >= 8) {
        ptx::regs_dec<88>();
        if (warp == 8) {
            // ---------------------------------------------------------- loads
            // one lane per box: 64 elements x box_keys keys
            job.start();
            const int box_keys = job.box_keys(), boxes = kBigKeys / box_keys * kBoxes;
            const int key0 = lane / kBoxes * box_keys, x0 = lane % kBoxes * 64;
            const uint32_t dst0 = lane % kBoxes * kBoxBytes + key0 * 128;
            uint32_t n = 0, used = 0;
            bool ok = true;
            BigItem it;
            for (int i = 0; ok && take(i, it); i++) {
                const int end = max(it.end[0], it.end[1]);
                if (end <= it.begin) continue;
                int2 at = lane < boxes ? job.coord(it, it.begin * kBigKeys + key0) : make_int2(0, 0);
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.q_empty, (used & 1) ^ 1, err));
                if (!ok) break;
                used++;
                if (lane == 0) {
                    const uint32_t q_bytes = kBoxes * 128u * group * tile_tokens;
                    ptx::mbar_arrive_expect_tx(&sm.q_full, q_bytes * ((it.end[0] > it.begin) + (it.end[1] > it.begin)));
                    for (int t = 0; t < 2; t++)
                        for (int b = 0; b < kBoxes && it.end[t] > it.begin; b++)
                            ptx::tma_load_3d(sm.q[t] + b * kBoxBytes, map_q, &sm.q_full, b * 64, it.head * (int)group,
                                             it.q_token + t * tile_tokens);
                }
                for (int j = it.begin; j < end && ok; j++) {
                    const int2 next = lane < boxes && j + 1 < end ? job.coord(it, (j + 1) * kBigKeys + key0) : at;
                    for (int kv = 0; kv < 2; kv++, n++) {
                        const int st = n % S::kStages;
                        ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.kv_empty[st], ((n / S::kStages) & 1) ^ 1, err));
                        if (!ok) break;
                        const bool tail = kv && (j + 1) * kBigKeys > it.lk;
                        uint64_t* bar = tail ? &sm.tail_full[st] : &sm.kv_full[st];
                        if (lane == 0) ptx::mbar_arrive_expect_tx(bar, kBoxes * kBoxBytes);
                        __syncwarp();
                        if (lane < boxes) tma_load_4d(sm.kv[st] + dst0, kv ? map_v : map_k, bar, x0, it.head, at.x, at.y);
                    }
                    at = next;
                }
            }
        } else if (warp == 9) {
            // ----------------------------------------------------------- MMAs
            // The whole warp goes through the loop on values that the compiler
            // can see are the same in all lanes, and one elected lane issues:
            // descriptors then stay in uniform registers (a lane on its own
            // moves them there for every MMA, which took longer than the MMA).
            constexpr uint32_t idesc_s = ptx::idesc_f16(kBigRows, kBigKeys, kBf16);
            constexpr uint32_t idesc_o = ptx::idesc_f16(kBigRows, DP, kBf16) | ptx::kIdescBMnMajor;
            const bool lead = ptx::elect_one();
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint32_t q_base = ptx::smem_u32(sm.q[0]), kv_base = ptx::smem_u32(sm.kv[0]);
            uint32_t n = 0, used = 0, pc0 = 0, pc1 = 0;
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity, err));
                if (ok) ptx::tc_fence_after();
                return ok;
            };
            auto full = [&](uint32_t m) { return wait(&sm.kv_full[m % S::kStages], (m / S::kStages) & 1); };
            auto commit = [&](uint64_t* bar) {
                if (lead) ptx::umma_commit(bar);
                __syncwarp();
            };
            auto qk = [&](int t, uint32_t m) {
                const uint32_t a = q_base + t * S::kTileBytes, b = kv_base + (m % S::kStages) * S::kTileBytes;
                if (lead) {
#pragma unroll
                    for (int kk = 0; kk < DP / 16; kk++)
                        ptx::umma_f16(tm + t * 128, desc_k(a, kk), desc_k(b, kk), idesc_s, kk != 0);
                    ptx::umma_commit(&sm.s_full[t]);
                }
                __syncwarp();
            };
            auto pv = [&](int t, uint32_t m, bool add, int first, int last) {  // 16-key steps
                const uint32_t b = kv_base + (m % S::kStages) * S::kTileBytes;
                if (lead) {
#pragma unroll
                    for (int kk = first; kk < last; kk++)
                        ptx::umma_f16_ta(tm + 256 + t * 128, tm + t * 128 + kk * 8,
                                         ptx::sdesc_mn(b + kk * 2048, 128, kBoxBytes), idesc_o, add || kk != 0);
                }
                __syncwarp();
            };
            BigItem it;
            for (int i = 0; ok && take(i, it); i++) {
                const int begin = __shfl_sync(0xffffffffu, it.begin, 0);
                const int end0 = __shfl_sync(0xffffffffu, it.end[0], 0), end1 = __shfl_sync(0xffffffffu, it.end[1], 0);
                const int end = max(end0, end1);
                if (end <= begin) continue;
                if (!wait(&sm.q_full, used & 1) || !full(n)) break;
                used++;
                if (begin < end0) qk(0, n);
                if (begin < end1) qk(1, n);
                commit(&sm.kv_empty[n % S::kStages]);
                n++;
                if (end == begin + 1) commit(&sm.q_empty);
                for (int j = begin; j < end; j++) {
                    const uint32_t nv = n;
                    const bool next = j + 1 < end;
                    if (!full(nv) || (next && !full(nv + 1))) break;
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        const int et = t ? end1 : end0;
                        if (j >= et) continue;
                        uint32_t& pc = t ? pc1 : pc0;
                        if (!wait(&sm.p_part[0][t], pc & 1)) break;
                        pv(t, nv, j > begin, 0, 4);
                        if (!wait(&sm.p_part[1][t], pc & 1)) break;
                        pv(t, nv, true, 4, 6);
                        if (!wait(&sm.p_part[2][t], pc & 1)) break;
                        pc++;
                        pv(t, nv, true, 6, 8);
                        if (j == et - 1) commit(&sm.o_full[t]);
                        else qk(t, nv + 1);
                    }
                    if (!ok) break;
                    commit(&sm.kv_empty[nv % S::kStages]);
                    n = nv + 1;
                    if (next) {
                        commit(&sm.kv_empty[n % S::kStages]);
                        n++;
                        if (j + 2 == end) commit(&sm.q_empty);
                    }
                }
            }
        } else if (warp == 10) {
            // -------------------------------------------- rows of V past the end
            uint32_t n = 0, phase = 0;  // phase: bit per stage
            BigItem it;
            for (int i = 0; take(i, it); i++) {
                const int end = max(it.end[0], it.end[1]);
                if (end <= it.begin) continue;
                n += 2 * (uint32_t)(end - it.begin);  // V of the last tile is number n - 1
                const int keep = it.lk - (end - 1) * kBigKeys;
                if (keep >= kBigKeys) continue;
                const int st = (n - 1) % S::kStages;
                if (!__all_sync(0xffffffffu, ptx::mbar_wait(&sm.tail_full[st], (phase >> st) & 1, err))) break;
                phase ^= 1u << st;
                for (int r = keep * 8 + lane; r < kBigKeys * 8; r += 32)
#pragma unroll
                    for (int b = 0; b < kBoxes; b++)
                        *reinterpret_cast<uint4*>(sm.kv[st] + b * kBoxBytes + r * 16) = make_uint4(0, 0, 0, 0);
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&sm.kv_full[st]);
            }
        } else if (warp == 11) {
            // ---------------------------------------------------------- items
            for (int i = 0;; i++) {
                const BigItem it = job.item(i);
                const int e = i % kItemRing;
                if (!__all_sync(0xffffffffu, ptx::mbar_wait(&sm.item_empty[e], ((i / kItemRing) & 1) ^ 1, err))) break;
                if (lane == 0) {
                    sm.items[e] = it;
                    ptx::mbar_arrive(&sm.item_full[e]);
                }
                if (it.head < 0) break;
            }
        }
    } else {
        // ------------------------------------------------------------- softmax
        ptx::regs_inc<208>();
        const int t = warp >> 2;
        const int row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + t * 128, to = tmem + lanes + 256 + t * 128;
        const int token = t * tile_tokens + row / (int)group;  // of the item
        const bool real = row < tile_tokens * (int)group;
        uint32_t sc = 0, oc = 0;
        bool ok = true;
        for (int i = 0; ok; i++) {
            const int e = i % kItemRing;
            ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.item_full[e], (i / kItemRing) & 1, err));
            const BigItem& it = sm.items[e];  // stays there until this warp is done with it
            if (!ok || it.head < 0) break;
            const int begin = it.begin, end = it.end[t];
            const int vis = real && token < it.tokens ? job.visible(it, token) : 0;
            float m = kNegInf, l = 0.0f;
            for (int j = begin; j < end; j++) {
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.s_full[t], sc & 1, err));
                if (!ok) break;
                sc++;
                ptx::tc_fence_after();
                uint32_t s[4][32], w[16];
                float2 sum[2];
                const float2 sc2 = make_float2(scale2, scale2);
                // weights of keys 32 c .. 32 c + 31 of the tile
                auto weights = [&](int c) {
                    const float off = kShift - (m == kNegInf ? 0.0f : m);
                    const float2 off2 = make_float2(off, off);
#pragma unroll
                    for (int x = 0; x < 16; x++) {
                        float2 e = ptx::ffma2(make_float2(__uint_as_float(s[c][2 * x]), __uint_as_float(s[c][2 * x + 1])), sc2, off2);
                        e.x = exp2_fast(e.x);
                        e.y = exp2_fast(e.y);
                        sum[x & 1] = c == 0 && x < 2 ? e : ptx::fadd2(sum[x & 1], e);
                        w[x] = Type<T>::pack(e.x, e.y);
                    }
                };
                auto largest = [&] {
                    float mx[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        mx[c] = __uint_as_float(s[c][0]);
#pragma unroll
                        for (int x = 1; x < 31; x += 2)
                            mx[c] = max3(mx[c], __uint_as_float(s[c][x]), __uint_as_float(s[c][x + 1]));
                    }
                    mx[0] = max3(mx[0], __uint_as_float(s[0][31]), __uint_as_float(s[1][31]));
                    mx[1] = max3(mx[1], __uint_as_float(s[2][31]), __uint_as_float(s[3][31]));
                    return max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * scale2;
                };
                // moves the rows' references to their maxima so far
                auto raise = [&](float top) {
                    const float mn = fmaxf(m, top), base = mn == kNegInf ? 0.0f : mn;
                    const float c = exp2_fast(m - base);
                    if (j > begin) {
#pragma unroll 1
                        for (int x = 0; x < DP; x += 32) {
                            uint32_t o[32];
                            ptx::tmem_ld_32x32b_x32(to + x, o);
                            ptx::tmem_ld_wait();
                            ptx::pin32(o);
#pragma unroll
                            for (int y = 0; y < 32; y++) o[y] = __float_as_uint(__uint_as_float(o[y]) * c);
                            ptx::tmem_st_32x32b_x32(to + x, o);
                        }
                    }
                    l *= c;
                    m = mn;
                };
                auto arrive = [&](int part) {
                    ptx::tmem_st_wait();
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(&sm.p_part[part][t]);
                };
                const int rest = vis - j * kBigKeys;  // keys of this tile that the row sees
                // P goes out while the next keys' weights are computed
                auto first_three = [&](bool have) {
                    if (!have) weights(0);
                    ptx::tmem_st_32x32b_x16(ts, w);
                    weights(1);
                    ptx::tmem_st_32x32b_x16(ts + 16, w);
                    weights(2);
                };
                if (j > begin && __all_sync(0xffffffffu, rest >= kBigKeys)) {
                    // The reference of the tiles before will do for this one too,
                    // nearly always: the weights do not wait for the tile's maximum,
                    // which is looked at before any of them is handed over.
                    ptx::tmem_ld_32x32b_x32(ts, s[0]);
                    ptx::tmem_ld_wait();
                    ptx::pin32(s[0]);
#pragma unroll
                    for (int c = 1; c < 4; c++) ptx::tmem_ld_32x32b_x32(ts + c * 32, s[c]);
                    weights(0);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int c = 1; c < 4; c++) ptx::pin32(s[c]);
                    first_three(true);
                    const float top = largest();
                    if (__any_sync(0xffffffffu, top > m + kSlack)) {
                        raise(top);
                        first_three(false);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 4; c++) ptx::tmem_ld_32x32b_x32(ts + c * 32, s[c]);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < 4; c++) ptx::pin32(s[c]);
                    // selected, not added: a hidden score may be anything, NaN included
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int x = 0; x < 32; x++) s[c][x] = c * 32 + x < rest ? s[c][x] : 0xff800000u;
                    const float top = largest();
                    if (__any_sync(0xffffffffu, top > m + kSlack)) raise(top);
                    first_three(false);
                }
                arrive(0);
                ptx::tmem_st_32x32b_x16(ts + 32, w);
                weights(3);
                arrive(1);
                ptx::tmem_st_32x32b_x16(ts + 48, w);
                arrive(2);
                l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
            }
            if (!ok) break;
            uint8_t* dst = nullptr;
            float factor = 0.0f;
            if (real && token < it.tokens) job.result(it, row, token, m, l, kShift, dst, factor);
            if (begin < end) {
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.o_full[t], oc & 1, err));
                if (!ok) break;
                oc++;
                ptx::tc_fence_after();
            }
            store_rows<T, DP>(sm.out[warp], dst, factor, begin < end, to, job.dim(), job.out_dtype(it));
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&sm.item_empty[e]);
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    __syncwarp();
    if (warp == 9) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512);
    }
}

}  // namespace attn
}  // namespace ane_b200
