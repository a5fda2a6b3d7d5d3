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
// Warps (384 threads): 0-3 and 4-7 softmax of tile 0 and 1; 8 loads (TMA);
// 9 issues the MMAs and owns TMEM; 10 clears the rows of V that lie past the
// last key (a weight of 0 does not silence a NaN there); 11 idles.
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
constexpr int kMaxItems = 32;    // items per block

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
    static constexpr int kStages = DP == 128 ? 5 : 10;
    static constexpr int kTileBytes = 128 * DP * 2;
    uint8_t q[2][kTileBytes];
    uint8_t kv[kStages][kTileBytes];
    uint64_t q_full, q_empty, kv_full[kStages], kv_empty[kStages], tail_full[kStages];
    uint64_t s_full[2], p_full[2], o_full[2];
    uint32_t tmem;
    BigItem items[kMaxItems];
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

// The kernel's frame.  Job supplies:
//   items(sm.items)             all warps: this block's items, ended by head -1
//   box_keys()                  keys per TMA box (a multiple of 8 that divides 128)
//   coord(item, key)            {token, page} coordinates of the box that starts at a key
//   visible(item, token)        keys that query token `token` of the item sees
//   finish(item, t, token, row, tmem_o, m, l)   one thread per row
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
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
            ptx::mbar_init(&sm.p_full[t], 4);
            ptx::mbar_init(&sm.o_full[t], 1);
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
    job.items(sm.items);
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = sm.tmem;  // columns: S0 0, S1 128, O0 256, O1 384

    if (warp >= 8) {
        ptx::regs_dec<88>();
        if (warp == 8) {
            // ---------------------------------------------------------- loads
            // one lane per box: 64 elements x box_keys keys
            const int box_keys = job.box_keys(), boxes = kBigKeys / box_keys * kBoxes;
            const int key0 = lane / kBoxes * box_keys, x0 = lane % kBoxes * 64;
            const uint32_t dst0 = lane % kBoxes * kBoxBytes + key0 * 128;
            uint32_t n = 0, used = 0;
            bool ok = true;
            for (int i = 0; i < kMaxItems && ok; i++) {
                const BigItem it = sm.items[i];
                if (it.head < 0) break;
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
        } else if (warp == 9 && lane == 0) {
            // ----------------------------------------------------------- MMAs
            constexpr uint32_t idesc_s = ptx::idesc_f16(kBigRows, kBigKeys, kBf16);
            constexpr uint32_t idesc_o = ptx::idesc_f16(kBigRows, DP, kBf16) | ptx::kIdescBMnMajor;
            uint32_t n = 0, used = 0, pc[2] = {0, 0};
            bool ok = true;
            auto full = [&](uint32_t m) {
                ok = ptx::mbar_wait(&sm.kv_full[m % S::kStages], (m / S::kStages) & 1, err);
                if (ok) ptx::tc_fence_after();
                return ok;
            };
            auto qk = [&](int t, uint32_t m) {
                const uint32_t a = ptx::smem_u32(sm.q[t]), b = ptx::smem_u32(sm.kv[m % S::kStages]);
#pragma unroll
                for (int kk = 0; kk < DP / 16; kk++)
                    ptx::umma_f16(tmem + t * 128, desc_k(a, kk), desc_k(b, kk), idesc_s, kk != 0);
                ptx::umma_commit(&sm.s_full[t]);
            };
            auto pv = [&](int t, uint32_t m, bool add) {
                const uint32_t b = ptx::smem_u32(sm.kv[m % S::kStages]);
#pragma unroll
                for (int kk = 0; kk < kBigKeys / 16; kk++)
                    ptx::umma_f16_ta(tmem + 256 + t * 128, tmem + t * 128 + kk * 8,
                                     ptx::sdesc_mn(b + kk * 2048, 128, kBoxBytes), idesc_o, add || kk != 0);
            };
            for (int i = 0; i < kMaxItems && ok; i++) {
                const BigItem it = sm.items[i];
                if (it.head < 0) break;
                const int end = max(it.end[0], it.end[1]);
                if (end <= it.begin) continue;
                if (!ptx::mbar_wait(&sm.q_full, used & 1, err)) break;
                used++;
                if (!full(n)) break;
                for (int t = 0; t < 2; t++)
                    if (it.begin < it.end[t]) qk(t, n);
                ptx::umma_commit(&sm.kv_empty[n % S::kStages]);
                n++;
                if (end == it.begin + 1) ptx::umma_commit(&sm.q_empty);
                for (int j = it.begin; j < end && ok; j++) {
                    const uint32_t nv = n;
                    const bool next = j + 1 < end;
                    if (!full(nv)) break;
                    bool have_k = false;
                    for (int t = 0; t < 2 && ok; t++) {
                        if (j >= it.end[t]) continue;
                        if (!(ok = ptx::mbar_wait(&sm.p_full[t], pc[t] & 1, err))) break;
                        pc[t]++;
                        ptx::tc_fence_after();
                        pv(t, nv, j > it.begin);
                        if (j == it.end[t] - 1) ptx::umma_commit(&sm.o_full[t]);
                        if (j + 1 < it.end[t]) {
                            if (!have_k && !full(nv + 1)) break;
                            have_k = true;
                            qk(t, nv + 1);
                        }
                    }
                    if (!ok) break;
                    ptx::umma_commit(&sm.kv_empty[nv % S::kStages]);
                    n = nv + 1;
                    if (next) {
                        ptx::umma_commit(&sm.kv_empty[n % S::kStages]);
                        n++;
                        if (j + 2 == end) ptx::umma_commit(&sm.q_empty);
                    }
                }
            }
        } else if (warp == 10) {
            // -------------------------------------------- rows of V past the end
            uint32_t n = 0, phase = 0;  // phase: bit per stage
            for (int i = 0; i < kMaxItems; i++) {
                const BigItem it = sm.items[i];
                if (it.head < 0) break;
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
        for (int i = 0; i < kMaxItems && ok; i++) {
            const BigItem it = sm.items[i];
            if (it.head < 0) break;
            const bool mine = real && token < it.tokens;
            const int vis = mine ? job.visible(it, token) : 0;
            float m = kNegInf, l = 0.0f;
            for (int j = it.begin; j < it.end[t]; j++) {
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.s_full[t], sc & 1, err));
                if (!ok) break;
                sc++;
                ptx::tc_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; c++) ptx::tmem_ld_32x32b_x32(ts + c * 32, s[c]);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 4; c++) ptx::pin32(s[c]);
                const int rest = vis - j * kBigKeys;  // keys of this tile that the row sees
                if (__any_sync(0xffffffffu, rest < kBigKeys)) {
                    // selected, not added: a hidden score may be anything, NaN included
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int x = 0; x < 32; x++) s[c][x] = c * 32 + x < rest ? s[c][x] : 0xff800000u;
                }
                float mx[4];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    mx[c] = __uint_as_float(s[c][0]);
#pragma unroll
                    for (int x = 1; x < 32; x++) mx[c] = fmaxf(mx[c], __uint_as_float(s[c][x]));
                }
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2;
                if (__any_sync(0xffffffffu, top > m + kSlack)) {
                    const float mn = fmaxf(m, top), base = mn == kNegInf ? 0.0f : mn;
                    const float c = exp2_fast(m - base);
                    if (j > it.begin) {
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
                }
                const float off = kShift - (m == kNegInf ? 0.0f : m);
                const float2 sc2 = make_float2(scale2, scale2), off2 = make_float2(off, off);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t w[32];
#pragma unroll
                    for (int x = 0; x < 32; x++) {
                        const uint32_t* v = &s[2 * h + (x >> 4)][2 * (x & 15)];
                        float2 e = ptx::ffma2(make_float2(__uint_as_float(v[0]), __uint_as_float(v[1])), sc2, off2);
                        e.x = exp2_fast(e.x);
                        e.y = exp2_fast(e.y);
                        sum[x & 1] = ptx::fadd2(sum[x & 1], e);
                        w[x] = Type<T>::pack(e.x, e.y);
                    }
                    ptx::tmem_st_32x32b_x32(ts + h * 32, w);
                }
                l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
                ptx::tmem_st_wait();
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&sm.p_full[t]);
            }
            if (!ok) break;
            if (it.begin < it.end[t]) {
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.o_full[t], oc & 1, err));
                if (!ok) break;
                oc++;
                ptx::tc_fence_after();
            }
            // rows without a tile skip TMEM; the whole warp takes part in the reads
            job.template finish<DP>(it, t, row, token, mine, it.begin < it.end[t], to, m, l, kShift);
            ptx::tc_fence_before();
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

// Columns c .. c + 31 of a result row (16-byte aligned), times inv.
__device__ __forceinline__ void store32(uint8_t* row, uint32_t c, uint32_t dim, uint32_t out_dtype,
                                        const uint32_t (&o)[32], float inv) {
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
        if (c + i >= dim) continue;
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = __uint_as_float(o[i + j]) * inv;
        if (out_dtype == ANE_DTYPE_F32) {
            float4* d = reinterpret_cast<float4*>(row + (size_t)(c + i) * 4);
            d[0] = make_float4(f[0], f[1], f[2], f[3]);
            d[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else if (out_dtype == ANE_DTYPE_F16) {
            *reinterpret_cast<uint4*>(row + (size_t)(c + i) * 2) =
                make_uint4(Type<__half>::pack(f[0], f[1]), Type<__half>::pack(f[2], f[3]),
                           Type<__half>::pack(f[4], f[5]), Type<__half>::pack(f[6], f[7]));
        } else {
            *reinterpret_cast<uint4*>(row + (size_t)(c + i) * 2) =
                make_uint4(Type<__nv_bfloat16>::pack(f[0], f[1]), Type<__nv_bfloat16>::pack(f[2], f[3]),
                           Type<__nv_bfloat16>::pack(f[4], f[5]), Type<__nv_bfloat16>::pack(f[6], f[7]));
        }
    }
}

}  // namespace attn
}  // namespace ane_b200
