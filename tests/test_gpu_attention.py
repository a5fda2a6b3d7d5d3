"""attn_prompt and attn_decode against attention in 64 bits (tests/attn_util.py
derives the error bound): lengths around the tiles, empty sequences and rows,
grouped heads, strides, garbage next to the sequences, long caches."""
import pytest
import torch

from attn_util import check_rows

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def cu_of(lens, start=0):
    c = [start]
    for n in lens:
        c.append(c[-1] + n)
    return c


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prompt_case(ane, lq, lk, heads, kv_heads, dim, dtype, out_dtype=None, layout="fused", spread=1.5, seed=0,
                want_lse=True):
    """Sequences between rows of NaN (before the first and after the last)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pad = 3
    cq, ck = cu_of(lq, pad), cu_of(lk, pad)
    same = lq == lk
    nan = float("nan")

    def rows(total, h):
        if layout == "heads_first":
            return torch.full((h, total, dim), nan, dtype=dtype, device="cuda").permute(1, 0, 2)
        return torch.full((total, h, dim), nan, dtype=dtype, device="cuda")

    if layout == "fused" and same:
        buf = torch.full((cq[-1] + pad, heads + 2 * kv_heads, dim), nan, dtype=dtype, device="cuda")
        q, k, v = buf[:, :heads], buf[:, heads:heads + kv_heads], buf[:, heads + kv_heads:]
    else:
        q, k, v = rows(cq[-1] + pad, heads), rows(ck[-1] + pad, kv_heads), rows(ck[-1] + pad, kv_heads)
    for t, c, sd in ((q, cq, spread), (k, ck, 1.0), (v, ck, 1.0)):
        n = c[-1] - pad
        t[pad:pad + n] = (torch.randn(n, t.shape[1], dim, device="cuda", generator=g) * sd).to(dtype)
    scale = dim ** -0.5
    out = torch.full((cq[-1] + pad, heads, dim), 7.0, dtype=out_dtype or dtype, device="cuda")
    lse = torch.full((cq[-1] + pad, heads), 7.0, device="cuda") if want_lse else None
    got = ane.attn_prompt(q, k, v, i32(cq), None if same else i32(ck), scale=scale, out=out, lse=lse)
    assert got is out
    group = heads // kv_heads
    for s in range(len(lq)):
        for h in sorted({0, heads - 1, heads // 2}):
            visible = torch.arange(lq[s], device="cuda") + 1 + (lk[s] - lq[s])
            visible = visible.clamp(min=0, max=lk[s])
            check_rows(out[cq[s]:cq[s + 1], h], dtype, q[cq[s]:cq[s + 1], h], k[ck[s]:ck[s + 1], h // group],
                       v[ck[s]:ck[s + 1], h // group], scale, visible,
                       lse[cq[s]:cq[s + 1], h] if want_lse else None)
    # rows of no sequence are not written
    assert (out[:pad] == 7.0).all() and (out[cq[-1]:] == 7.0).all()
    return q, k, v, cq, ck, out


@pytest.mark.parametrize("lens", [[1], [2, 1, 1], [0, 5, 0], [63, 64, 65], [127, 128, 129], [255, 256, 257, 0, 31],
                                  [1000], [513, 77, 300]])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(4, 4, 128, F16), (8, 2, 64, BF16)])
def test_prompt_lengths(ane, lens, heads, kv_heads, dim, dtype):
    prompt_case(ane, lens, lens, heads, kv_heads, dim, dtype)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (5, 1), (6, 2), (16, 2), (64, 1), (33, 1)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_groups(ane, heads, kv_heads, dtype):
    prompt_case(ane, [70, 1, 190], [70, 1, 190], heads, kv_heads, 64, dtype)
    prompt_case(ane, [131], [131], heads, kv_heads, 128, dtype)


@pytest.mark.parametrize("dim", [8, 24, 64, 72, 80, 112, 120, 128])
@pytest.mark.parametrize("layout", ["fused", "heads_first"])
def test_prompt_dims_layouts(ane, dim, layout):
    prompt_case(ane, [140, 9], [140, 9], 4, 2, dim, F16, layout=layout)
    prompt_case(ane, [140, 9], [140, 9], 4, 2, dim, BF16, layout=layout, out_dtype=F32)


@pytest.mark.parametrize("lq,lk", [
    ([5, 100], [700, 100]),       # a block at the end of a longer history
    ([130, 64], [131, 1000]),
    ([300, 40, 7], [10, 0, 8]),   # more queries than keys: the first rows see nothing
    ([256], [255]),
    ([1, 1, 1], [129, 1, 512]),
])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_history_and_empty_rows(ane, lq, lk, dtype):
    prompt_case(ane, lq, lk, 8, 4, 128, dtype)
    prompt_case(ane, lq, lk, 2, 2, 64, dtype, out_dtype=F32)


@pytest.mark.parametrize("lq,lk,heads,kv_heads,dim,dtype", [
    ([1], [5000], 8, 8, 128, F16),               # one token against a long history: every item cut many times
    ([3, 0, 1], [40000, 0, 70], 4, 1, 64, BF16),
    ([100, 513, 64], [2100, 513, 1000], 8, 2, 128, BF16),
    ([2000], [1100], 4, 4, 128, F16),            # the first 900 queries see nothing
    ([1500, 900, 0, 700], [1500, 900, 0, 700], 6, 2, 80, F16),
    ([300] * 7, [1000 + 100 * i for i in range(7)], 16, 2, 64, F16),
    ([260], [8200], 5, 1, 128, BF16),
])
def test_prompt_few_items_cut_along_the_keys(ane, lq, lk, heads, kv_heads, dim, dtype):
    prompt_case(ane, lq, lk, heads, kv_heads, dim, dtype)
    prompt_case(ane, lq, lk, heads, kv_heads, dim, dtype, out_dtype=F32, want_lse=False, seed=1)


def test_prompt_cut_items_repeat(ane):
    """The joined parts do not depend on scheduling, nor on what the workspace holds."""
    q, k, v, cq, ck, out = prompt_case(ane, [200, 90], [6000, 3000], 8, 2, 128, F16)
    ws = torch.empty(ane.lib.ane_attn_prompt_workspace_size(2, 8, 2, 128, q.shape[0], k.shape[0]), dtype=torch.uint8,
                     device="cuda")
    assert ws.numel() > 0
    for _ in range(3):
        ws.random_(0, 255)
        got = ane.attn_prompt(q, k, v, i32(cq), i32(ck), workspace=ws)
        assert torch.equal(got[cq[0]:cq[-1]], out[cq[0]:cq[-1]])


def test_prompt_large_scores(ane):
    """Scores of several hundred: the maximum moves far from tile to tile."""
    prompt_case(ane, [600], [600], 2, 1, 128, F16, spread=60.0)
    prompt_case(ane, [600], [600], 2, 1, 128, BF16, spread=200.0)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_many_small_weights(ane, dtype):
    """One strong key and thousands of weak ones that together outweigh it."""
    n, d = 6000, 64
    k = torch.zeros(n, 1, d, device="cuda", dtype=dtype)
    k[0, 0, 0] = 12.0
    v = torch.ones(n, 1, d, device="cuda", dtype=dtype)
    v[0] = -1.0
    q = torch.zeros(n, 1, d, device="cuda", dtype=dtype)
    q[:, 0, 0] = 6.0
    out = ane.attn_prompt(q, k, v, i32([0, n]), scale=0.125)
    check_rows(out[:, 0], dtype, q[:, 0], k[:, 0], v[:, 0], 0.125, torch.arange(1, n + 1, device="cuda"))


def test_prompt_neighbours_may_hold_anything(ane):
    """NaN, infinities and the type's lowest value in one sequence leave the others' bits alone."""
    lens = [37, 90, 128, 5, 200]
    q, k, v, cq, _, clean = prompt_case(ane, lens, lens, 4, 2, 128, F16, seed=3)
    for bad in (float("nan"), float("inf"), -65504.0):
        q2, k2, v2 = q.clone(), k.clone(), v.clone()
        for t in (q2, k2, v2):
            t[cq[1]:cq[2]] = bad
            t[cq[3]:cq[4]] = bad
        out = ane.attn_prompt(q2, k2, v2, i32(cq), scale=128 ** -0.5)
        for s in (0, 2, 4):
            assert torch.equal(out[cq[s]:cq[s + 1]], clean[cq[s]:cq[s + 1]])


def test_prompt_batch_invariant_and_repeatable(ane):
    """Whole items: a sequence's bits do not depend on what it is packed with, nor on the run."""
    lens = [300, 17, 411]
    q, k, v, cq, _, out = prompt_case(ane, lens, lens, 8, 2, 128, BF16, seed=5)
    again = ane.attn_prompt(q, k, v, i32(cq))
    assert torch.equal(again[cq[0]:cq[-1]], out[cq[0]:cq[-1]])
    for s in range(3):
        a, b = cq[s], cq[s + 1]
        one = ane.attn_prompt(q[a:b], k[a:b], v[a:b], i32([0, b - a]))
        assert torch.equal(one, out[a:b])


def test_prompt_many_sequences(ane):
    lens = [(7 * i) % 40 for i in range(1024)]
    prompt_case(ane, lens[:1024], lens[:1024], 2, 1, 64, F16, want_lse=False)


def test_prompt_side_stream_and_graph(ane):
    lens = [200, 64]
    q, k, v, cq, _, out = prompt_case(ane, lens, lens, 4, 4, 128, F16, seed=9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ane.attn_prompt(q, k, v, i32(cq), stream=side)
    side.synchronize()
    assert torch.equal(got[cq[0]:cq[-1]], out[cq[0]:cq[-1]])
    c, res = i32(cq), torch.zeros_like(out)
    ane.attn_prompt(q, k, v, c, out=res)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ane.attn_prompt(q, k, v, c, out=res)
    res.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(res[cq[0]:cq[-1]], out[cq[0]:cq[-1]])


# --------------------------------------------------------------------- decode
def decode_case(ane, lens, shared, heads, kv_heads, dim, page, dtype, out_dtype=None, layout="tokens", seed=0,
                extra_pages=5, first_page=0, want_lse=True, total_pages=None):
    """lens include the shared tokens.  Everything that belongs to no sequence
    (page tails, other pages, table entries) is NaN or out of range."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    B = len(lens)
    full = shared // page
    prefix = list(range(full))
    rows, at = [], full
    for b, n in enumerate(lens):
        need = -(-max(n, shared if b == 0 else 0) // page)
        mine = max(0, need - full)
        rows.append(prefix[:min(need, full)] + list(range(at, at + mine)))
        at += mine
    perm = torch.randperm(at + extra_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    pages = total_pages or at + extra_pages + first_page
    shape = (pages, kv_heads, page, dim) if layout == "heads" else (pages, page, kv_heads, dim)
    make = (lambda: torch.empty(shape, dtype=dtype, device="cuda")) if total_pages else \
        (lambda: torch.full(shape, float("nan"), dtype=dtype, device="cuda"))
    k, v = make(), make()
    if layout == "heads":
        k, v = k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)
    width = max(1, max(len(r) for r in rows)) + 1
    slots = torch.randperm(B + 2, generator=torch.Generator().manual_seed(seed + 1))[:B].tolist()
    tables = torch.full((B + 2, width), 10 ** 9, dtype=torch.int32)
    lens_t = torch.full((B + 2,), 10 ** 6, dtype=torch.int32)
    pk = torch.randn(shared, kv_heads, dim, device="cuda", generator=g).to(dtype)
    pv = torch.randn(shared, kv_heads, dim, device="cuda", generator=g).to(dtype)
    q = (torch.randn(B, heads, dim, device="cuda", generator=g) * 1.5).to(dtype)
    seqs = []
    for b, n in enumerate(lens):
        ids = [first_page + perm[r] for r in rows[b]]
        tables[slots[b], :len(ids)] = torch.tensor(ids, dtype=torch.int32)
        lens_t[slots[b]] = n
        hold = max(n, shared if b == 0 else 0)
        own = max(0, hold - shared)
        ks = torch.cat([pk, torch.randn(own, kv_heads, dim, device="cuda", generator=g).to(dtype)])[:hold]
        vs = torch.cat([pv, torch.randn(own, kv_heads, dim, device="cuda", generator=g).to(dtype)])[:hold]
        for i, p in enumerate(ids):
            part = min(page, hold - i * page)
            k[p, :part] = ks[i * page:i * page + part]
            v[p, :part] = vs[i * page:i * page + part]
        seqs.append((ks[:n], vs[:n]))
    scale = dim ** -0.5
    lse = torch.full((B, heads), 7.0, device="cuda") if want_lse else None
    out = ane.attn_decode(q, k, v, tables.cuda(), lens_t.cuda(), slots=i32(slots), shared=shared, scale=scale,
                          out_dtype=out_dtype, lse=lse)
    group = heads // kv_heads
    for b in range(B):
        ks, vs = seqs[b]
        visible = torch.full((group,), lens[b], device="cuda")
        for h in range(kv_heads):
            a, e = h * group, (h + 1) * group
            check_rows(out[b, a:e], dtype, q[b, a:e], ks[:, h], vs[:, h], scale, visible,
                       lse[b, a:e] if want_lse else None)
    return q, k, v, tables.cuda(), lens_t.cuda(), i32(slots), out


@pytest.mark.parametrize("lens,shared", [
    ([1], 0), ([1], 1), ([64], 64), ([65, 64, 63], 0), ([65, 64, 70], 64), ([200, 130, 129, 131], 129),
    ([300, 0, 257, 1000], 256),       # an empty slot behind a prefix
    ([50, 20, 0, 64], 64),            # all shorter than the shared tokens, row 0 too
    ([5000], 0), ([4100, 4097], 4096), ([2000] * 9, 1990),
])
@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", [(4, 4, 128, 16, F16), (8, 2, 64, 32, BF16)])
def test_decode_lengths(ane, lens, shared, heads, kv_heads, dim, page, dtype):
    decode_case(ane, lens, shared, heads, kv_heads, dim, page, dtype)


@pytest.mark.parametrize("page", [8, 16, 64, 128, 256])
@pytest.mark.parametrize("layout", ["tokens", "heads"])
def test_decode_pages_layouts(ane, page, layout):
    decode_case(ane, [777, 301, 300, 513], 300, 8, 4, 128, page, F16, layout=layout)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (5, 1), (12, 4), (16, 1), (17, 1), (64, 1), (66, 2)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decode_groups(ane, heads, kv_heads, dtype):
    decode_case(ane, [400, 210, 260], 200, heads, kv_heads, 128, 16, dtype)
    decode_case(ane, [9, 70], 0, heads, kv_heads, 64, 16, dtype)


@pytest.mark.parametrize("batch", [2, 15, 16, 17, 33, 64, 65, 130])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2)])
def test_decode_batches(ane, batch, heads, kv_heads):
    lens = [260 + (37 * b) % 200 for b in range(batch)]
    lens[-1] = 0
    decode_case(ane, lens, 260, heads, kv_heads, 128, 32, BF16)
    decode_case(ane, lens, 256, heads, kv_heads, 64, 32, F16, out_dtype=F32)


@pytest.mark.parametrize("dim", [8, 24, 72, 80, 120])
def test_decode_dims(ane, dim):
    decode_case(ane, [333, 140, 141], 140, 6, 3, dim, 16, F16)
    decode_case(ane, [333, 140, 141], 140, 6, 3, dim, 16, BF16, out_dtype=F32)


def test_decode_shared_equals_unshared(ane):
    """Reading the prefix once or once per sequence differs by rounding only."""
    q, k, v, tables, lens, slots, out = decode_case(ane, [700, 650, 901], 640, 8, 2, 128, 16, F16, out_dtype=F32)
    plain = ane.attn_decode(q, k, v, tables, lens, slots=slots, shared=0, out_dtype=F32)
    assert (plain - out).abs().max() < 2 * 2.0 ** -11 * 4


def test_decode_repeatable_stream_graph(ane):
    q, k, v, tables, lens, slots, out = decode_case(ane, [1500, 0, 1301, 1290], 1290, 8, 2, 128, 64, BF16)
    ws = ane.attn_decode_workspace(4, 8, 2, 128)
    for _ in range(3):
        ws.random_(0, 255)
        assert torch.equal(out, ane.attn_decode(q, k, v, tables, lens, slots=slots, shared=1290, workspace=ws))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ane.attn_decode(q, k, v, tables, lens, slots=slots, shared=1290, stream=side)
    side.synchronize()
    assert torch.equal(out, got)
    res = torch.zeros_like(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ane.attn_decode(q, k, v, tables, lens, slots=slots, shared=1290, workspace=ws, out=res)
    res.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, res)


def test_decode_slot_out_of_range_is_empty(ane):
    q, k, v, tables, lens, slots, out = decode_case(ane, [70, 33, 64], 0, 2, 2, 64, 16, F16)
    bad = slots.clone()
    bad[1], bad[2] = -1, 10 ** 6
    got = ane.attn_decode(q, k, v, tables, lens, slots=bad)
    assert torch.equal(got[0], out[0]) and (got[1:] == 0).all()


def test_decode_long_cache_offsets(ane):
    """Pages past 4 GB and past 2^31 elements of a pool."""
    page, kv_heads, dim = 64, 8, 128
    per_page = page * kv_heads * dim
    total = (2 ** 31 + 2 ** 22) // per_page + 64
    decode_case(ane, [1000, 801], 800, 16, kv_heads, dim, page, F16, total_pages=total, first_page=total - 60)


def test_decode_full_batch(ane):
    decode_case(ane, [100 + b % 40 for b in range(1024)], 96, 2, 1, 64, 16, F16, want_lse=False)


@pytest.mark.parametrize("lens,shared,heads,kv_heads,dim,page,dtype", [
    ([2600 + 13 * b for b in range(33)], 2600, 16, 2, 128, 64, BF16),     # 264 rows: a full pair and a few rows
    ([4100 + b for b in range(70)] + [0, 100, 4096], 4096, 8, 8, 64, 16, F16),
    ([1500 + 50 * (b % 9) for b in range(130)], 1411, 20, 4, 80, 8, F16),  # 5 heads a group: 125 rows per tile
    ([2048] * 64, 2048, 32, 8, 128, 256, BF16),                           # nothing of their own
    # an odd number of row tiles (the last is alone in its pair):
    ([870 + 9 * (b % 50) for b in range(95)] + [500], 870, 32, 8, 128, 32, F16),  # fewer key tiles than spans
    ([9001 + b for b in range(5)], 9001, 64, 1, 128, 64, BF16),
    ([700 + b % 70 for b in range(130)], 700, 128, 64, 64, 8, BF16),       # more items than SMs
    ([4096 + b for b in range(40)], 4096, 8, 8, 128, 128, F16),            # one tile, no last rows of V to clear
])
def test_decode_long_prefix_many_rows(ane, lens, shared, heads, kv_heads, dim, page, dtype):
    decode_case(ane, lens, shared, heads, kv_heads, dim, page, dtype)
    decode_case(ane, lens, shared, heads, kv_heads, dim, page, dtype, out_dtype=F32, want_lse=False, seed=2,
                layout="heads")


@pytest.mark.parametrize("heads,kv_heads,dtype,dim", [(4, 4, F16, 128), (8, 2, BF16, 64)])
@pytest.mark.parametrize("shared", [0, 37])
def test_decode_neighbours_may_hold_anything(ane, heads, kv_heads, dtype, dim, shared):
    """NaN, infinities and the type's lowest value in some sequences' own tokens
    leave the others' bits alone, and show in their own results."""
    lens = [shared + n for n in (70, 3, 129, 64, 1, 200, 17)]
    q, k, v, tables, lens_t, slots, out = decode_case(ane, lens, shared, heads, kv_heads, dim, 16, dtype, seed=4)
    clean = ane.attn_decode(q, k, v, tables, lens_t, slots=slots, shared=shared)
    assert torch.equal(clean, out)
    bad_rows = (1, 3, 5)
    for bad in (float("nan"), float("inf"), -65504.0):
        k2, v2, q2 = k.clone(), v.clone(), q.clone()
        for b in bad_rows:
            s = int(slots[b])
            first = -(-shared // 16)  # pages of its own alone
            pages = tables[s, first:-(-lens[b] // 16)].long()
            if len(pages) == 0:
                pages = tables[s, shared // 16:shared // 16 + 1].long()
            v2[pages, :, :, 3] = bad
            if bad == bad:  # NaN scores would make the whole row NaN: only V here
                continue
            k2[pages, 5:, :, 2] = bad
            q2[b, :, 1] = bad
        got = ane.attn_decode(q2, k2, v2, tables, lens_t, slots=slots, shared=shared)
        for b in range(len(lens)):
            if b not in bad_rows:
                assert torch.equal(got[b], clean[b]), (bad, b)
        if bad == float("inf"):
            for b in bad_rows:
                others = [c for c in range(dim) if c != 3]
                assert not torch.isfinite(got[b, :, 3]).any()
                assert torch.equal(got[b][:, others], clean[b][:, others])


SHORT = [
    # lens, shared, heads, kv_heads, dim, page, dtype
    ([130, 40, 0, 100, 137, 1, 64], 100, 4, 4, 128, 16, F16),     # all rows in one unit
    ([700, 90, 640, 300, 65], 600, 8, 2, 64, 32, BF16),           # tiles that a row sees in part, and not at all
    ([400, 33, 399], 333, 24, 1, 80, 8, F16),                     # units of one sequence
    ([1000, 1], 900, 2, 2, 128, 64, BF16),
    ([4100 + b % 9 for b in range(38)] + [0, 100, 4095, 1, 2048], 4096, 32, 8, 64, 16, F16),  # prefix_kernel
    ([2700 + 13 * b for b in range(31)] + [2600, 2599, 77], 2600, 64, 8, 128, 64, BF16),
]


@pytest.mark.parametrize("lens,shared,heads,kv_heads,dim,page,dtype", SHORT)
def test_decode_short_sequences_do_not_see_the_rest_of_the_prefix(ane, lens, shared, heads, kv_heads, dim, page, dtype):
    """What the shared tokens past a sequence's own length hold leaves its bits
    alone; sequences that see them show it in that column alone."""
    q, k, v, tables, lens_t, slots, out = decode_case(ane, lens, shared, heads, kv_heads, dim, page, dtype, seed=6)
    table = tables[int(slots[0])].tolist()
    for cut in sorted({n for n in lens if 0 < n < shared}):
        for bad in (float("nan"), float("inf"), -torch.finfo(dtype).max):
            for hit_k in (False, True):
                k2, v2 = k.clone(), v.clone()
                for t in {cut, cut + 1, (cut + shared) // 2, shared - 1}:
                    if t < cut or t >= shared:
                        continue
                    v2[table[t // page], t % page, :, 3] = bad
                    if hit_k:
                        k2[table[t // page], t % page, :, 2] = bad
                got = ane.attn_decode(q, k2, v2, tables, lens_t, slots=slots, shared=shared)
                for b, n in enumerate(lens):
                    if n <= cut:
                        assert torch.equal(got[b], out[b]), (cut, bad, hit_k, b)
                    elif not hit_k and n >= shared:
                        others = [c for c in range(dim) if c != 3]
                        assert torch.equal(got[b][:, others], out[b][:, others]), (cut, bad, b)
                        assert bad == bad and abs(bad) < 1e39 or not torch.isfinite(got[b, :, 3]).any()


def check_decode(ane, q, k, v, tables, lens, slots, shared, holder, **kw):
    """attn_decode against the definition; the shared tokens are those of batch row `holder`."""
    B, heads, dim = q.shape
    page, kv_heads = k.shape[1:3]
    group = heads // kv_heads
    lse = torch.full((B, heads), 7.0, device="cuda")
    out = ane.attn_decode(q, k, v, tables, lens, slots=slots, shared=shared, lse=lse, **kw)
    for b, s in enumerate(slots.tolist()):
        n = int(lens[s]) if 0 <= s < len(lens) else 0
        t = torch.arange(n, device="cuda")
        row = torch.where(t < shared, int(slots[holder]), s)
        pages = tables[row, t // page].long()
        ks, vs = k[pages, t % page], v[pages, t % page]
        visible = torch.full((group,), n, device="cuda")
        for h in range(kv_heads):
            a, e = h * group, (h + 1) * group
            check_rows(out[b, a:e], q.dtype, q[b, a:e], ks[:, h], vs[:, h], dim ** -0.5, visible, lse[b, a:e])
    return out


@pytest.mark.parametrize("lens,shared,heads,kv_heads,dim,page,dtype", [
    ([180, 0, 40, 150, 131], 129, 4, 4, 128, 16, F16),
    ([700, 90, 640, 0, 620], 600, 8, 2, 64, 32, BF16),
    ([64, 20, 1, 0], 64, 4, 4, 128, 16, F16),
    ([4100 + b % 9 for b in range(38)] + [0, 100, 4095, 1, 2048], 4096, 32, 8, 64, 16, F16),
    ([2700 + 13 * b for b in range(31)] + [2600, 2599, 0], 2600, 64, 8, 128, 64, BF16),
])
def test_decode_prefix_of_a_row_that_holds_it(ane, lens, shared, heads, kv_heads, dim, page, dtype):
    """Idle and short sequences at the head of the batch (their table rows end, or
    are stale, before the shared tokens do) do not carry the prefix."""
    q, k, v, tables, lens_t, slots, _ = decode_case(ane, lens, shared, heads, kv_heads, dim, page, dtype, seed=8)
    order = sorted(range(len(lens)), key=lambda b: lens[b])  # the idle and the short first
    first = next(i for i, b in enumerate(order) if lens[b] >= shared)
    check_decode(ane, q[order], k, v, tables, lens_t, slots[order], shared, first)
    bad = slots[order].clone()
    bad[0] = -1
    check_decode(ane, q[order], k, v, tables, lens_t, bad, shared, first)
    # none holds all of them: the longest does, as far as it goes
    short = lens_t.clone()
    short[slots] = torch.minimum(short[slots], torch.tensor(shared - 3, device="cuda", dtype=torch.int32))
    top = max(min(n, shared - 3) for n in lens)
    first = next(i for i, b in enumerate(order) if min(lens[b], shared - 3) == top)
    check_decode(ane, q[order], k, v, tables, short, slots[order], shared, first)


def give_up_busy(*sizes):
    """Blocks of the current stream's memory, freed while the work that writes them
    still waits there."""
    held = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes]
    torch.cuda._sleep(100_000_000)  # about 50 ms
    for h in held:
        h.fill_(0xff)


@pytest.mark.parametrize("lq,lk", [([200, 64], [200, 64]), ([100, 60], [3000, 2000])])
def test_prompt_on_a_side_stream_next_to_freed_memory(ane, lq, lk):
    q, k, v, cq, ck, out = prompt_case(ane, lq, lk, 4, 2, 128, F16, seed=9)
    c, d, side = i32(cq), i32(ck), torch.cuda.Stream()
    torch.cuda.synchronize()
    ws = ane.lib.ane_attn_prompt_workspace_size(2, 4, 2, 128, q.shape[0], k.shape[0])
    give_up_busy(q.numel() * 2, max(ws, 1))
    got = ane.attn_prompt(q, k, v, c, d, stream=side)
    side.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(got[cq[0]:cq[-1]], out[cq[0]:cq[-1]])


def test_decode_on_a_side_stream_next_to_freed_memory(ane):
    q, k, v, tables, lens, slots, out = decode_case(ane, [1500, 0, 1301, 1290], 1290, 8, 2, 128, 64, BF16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    give_up_busy(q.numel() * 2, ane.attn_decode_workspace(4, 8, 2, 128).numel())
    got = ane.attn_decode(q, k, v, tables, lens, slots=slots, shared=1290, stream=side)
    side.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(got, out)


@pytest.mark.parametrize("batch", [95, 96, 97, 400])
def test_decode_joins_of_many_sequences(ane, batch):
    """Parts of many sequences, however their tables are wide and whatever the
    workspace holds."""
    lens = [(61 * b) % 190 + 20 for b in range(batch)]
    lens[1] = 1500
    q, k, v, tables, lens_t, slots, out = decode_case(ane, lens, 20, 4, 2, 64, 16, F16, seed=7)
    ws = ane.attn_decode_workspace(batch, 4, 2, 64)
    wide = torch.nn.functional.pad(tables, (0, 3000), value=10 ** 9).contiguous()
    for table in (tables, wide):
        ws.random_(0, 255)
        got = ane.attn_decode(q, k, v, table, lens_t, slots=slots, shared=20, workspace=ws)
        assert torch.equal(got, out)


def test_single_rows_of_any_stride(ane):
    """A dimension of one entry may have any stride (torch calls such a tensor
    contiguous)."""
    g = torch.Generator(device="cuda").manual_seed(1)
    buf = torch.randn(3, 8 * 64, device="cuda", generator=g).half()
    odd = lambda i, h: torch.as_strided(buf[i], (1, h, 64), (8 * 64 + 3, 64, 1))  # noqa: E731
    q, k, v = odd(0, 8), odd(1, 2), odd(2, 2)
    out = ane.attn_prompt(q, k, v, i32([0, 1]))
    assert torch.equal(out[0], v[0].repeat_interleave(4, 0))
    one = lambda i: torch.as_strided(buf[i], (5, 1, 64), (64, 67, 1))  # noqa: E731  (one head)
    check_rows(ane.attn_prompt(one(0), one(1), one(2), i32([0, 5]))[:, 0], F16, one(0)[:, 0], one(1)[:, 0], one(2)[:, 0],
               0.125, torch.arange(1, 6, device="cuda"))
    pool = lambda i: torch.as_strided(buf[i], (1, 8, 1, 64), (515, 64, 67, 1))  # noqa: E731  (one page, one head)
    out = ane.attn_decode(odd(0, 8), pool(1), pool(2).contiguous().view(1, 8, 1, 64), i32([[0]]), i32([7]))
    check_rows(out[0], F16, odd(0, 8)[0], pool(1)[0, :7, 0], pool(2)[0, :7, 0], 0.125, torch.full((8,), 7, device="cuda"))


@pytest.mark.parametrize("lens,shared,heads,kv_heads,dim,page,dtype", [
    ([4100 + b % 9 for b in range(38)] + [0, 100, 4095, 1, 2048], 4096, 32, 8, 64, 16, F16),  # prefix_kernel
    ([1500, 700, 0, 1301, 1290, 1291], 1290, 8, 2, 128, 64, BF16),
    ([70 + b for b in range(150)], 64, 8, 2, 64, 16, F16),
])
def test_decode_among_other_work(ane, lens, shared, heads, kv_heads, dim, page, dtype):
    """The kernels of a call start before the ones in front of them have ended:
    inputs that are written just before, overwritten just after, a workspace that the
    next call takes over, on a side stream and in a graph."""
    q, k, v, tables, lens_t, slots, want = decode_case(ane, lens, shared, heads, kv_heads, dim, page, dtype, seed=11)
    swap = torch.arange(len(lens) - 1, -1, -1, device="cuda")
    args = [(q, slots), (q[swap].contiguous(), slots[swap].contiguous())]
    want = [want, ane.attn_decode(args[1][0], k, v, tables, lens_t, slots=args[1][1], shared=shared)]
    ws = ane.attn_decode_workspace(len(lens), heads, kv_heads, dim)
    qn, sn, ln = torch.empty_like(q), torch.empty_like(slots), torch.empty_like(lens_t)

    def chain(stream=None):
        got = []
        for i in (0, 1, 1, 0):
            qn.copy_(args[i][0])
            sn.copy_(args[i][1])
            ln.copy_(lens_t)
            for t in range(2):
                got.append((i, ane.attn_decode(qn, k, v, tables, ln, slots=sn, shared=shared, workspace=ws, stream=stream)))
            qn.fill_(float("nan"))
            ln.zero_()
            sn.fill_(-1)
        return got

    def check(got):
        torch.cuda.synchronize()
        for i, out in got:
            assert torch.equal(out, want[i])

    ws.random_(0, 255)
    check(chain())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ws.random_(0, 255)
        got = chain(side)
    check(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for _ in range(3):
        for _, out in got:
            out.zero_()
        ws.random_(0, 255)
        graph.replay()
        check(got)


@pytest.mark.parametrize("lq,lk", [([200, 90, 0, 7], [6000, 3000, 0, 7]), ([200, 64, 1], [200, 64, 1])])
def test_prompt_among_other_work(ane, lq, lk):
    """Items cut along the keys and whole ones: inputs that are written just before
    and overwritten just after, a workspace that the next call takes over, in a graph."""
    q, k, v, cq, ck, want = prompt_case(ane, lq, lk, 8, 2, 128, BF16, seed=12)
    n = ane.lib.ane_attn_prompt_workspace_size(len(lq), 8, 2, 128, q.shape[0], k.shape[0])
    assert (n > 0) == (max(lk) > 1000)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    c, d, qn, cn = i32(cq), i32(ck), torch.empty_like(q), i32(cq)

    def chain():
        got = []
        for _ in range(3):
            qn.copy_(q)
            cn.copy_(c)
            got += [ane.attn_prompt(qn, k, v, cn, d, workspace=ws) for _ in range(2)]
            qn.fill_(float("nan"))
            cn.zero_()
        return got

    def check(got):
        torch.cuda.synchronize()
        for out in got:
            assert torch.equal(out[cq[0]:cq[-1]], want[cq[0]:cq[-1]])

    ws.random_(0, 255)
    check(chain())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for _ in range(3):
        for out in got:
            out.zero_()
        ws.random_(0, 255)
        graph.replay()
        check(got)


@pytest.mark.parametrize("lq,lk,heads,kv_heads,dim,dtype", [
    ([100, 513, 64], [9100, 8513, 9000], 8, 2, 128, BF16),
    ([2000, 30], [1100, 19000], 4, 4, 128, F16),       # the first 900 queries see nothing
    ([150, 90, 0, 70], [9150, 8000, 0, 15], 6, 2, 80, F16),
    ([30] * 7, [9000 + 100 * i for i in range(7)], 16, 2, 64, F16),
    ([260], [8200], 5, 1, 128, BF16),
    ([700], [9000], 32, 8, 64, BF16),                  # two items and more a block
])
def test_prompt_long_history_cut_along_the_keys(ane, lq, lk, heads, kv_heads, dim, dtype):
    n = ane.lib.ane_attn_prompt_workspace_size(len(lq), heads, kv_heads, dim, sum(lq) + 6, sum(lk) + 6)
    assert n > 0  # parts
    prompt_case(ane, lq, lk, heads, kv_heads, dim, dtype)
    prompt_case(ane, lq, lk, heads, kv_heads, dim, dtype, out_dtype=F32, want_lse=False, seed=1)
