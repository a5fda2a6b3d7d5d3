"""Measured cases of the key/value-cache operators: prompt attention, decode
attention over a paged cache whose sequences share a prefix, forking and freeing
sequences, and compacting the pool of pages.

Every case is a dict of plain values.  Token counts of the sequences of a batch
are not listed one by one: they follow from the case (`_lengths`), so that
`work` and `prepare` agree on them.  `own` selects what `run` calls: plain torch
operations in 32 bits (False) or the framework's entry points (True).
"""
import math
import random

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
PAGE_CHOICES = (16, 32, 64, 128)


# ------------------------------------------------------------------- the cases
def listed():
    """The repository's decode stack has 32 heads of 128 (QKV rows of 12288);
    the grouped-head cases keep 32 query heads over 8 or 4 key/value heads."""
    return [
        # a chat turn of a few words: one short prompt, nothing to spread over the chip
        dict(name="prompt_17", op="prompt", n=1, lo=17, hi=17, past=0, idle=0, heads=32, kv_heads=32, dim=128,
             dtype="f16"),
        # a serving batch of ragged prompts, read in place from the fused QKV rows
        dict(name="prompt_ragged", op="prompt", n=8, lo=37, hi=1531, past=0, idle=1, heads=32, kv_heads=32, dim=128,
             dtype="f16"),
        # a block of a long prompt whose first 7681 tokens are already cached
        dict(name="prompt_chunk", op="prompt", n=2, lo=509, hi=1024, past=7681, idle=0, heads=32, kv_heads=8, dim=64,
             dtype="bf16"),
        # one long document, grouped heads: bound by the matrix products
        dict(name="prompt_16k", op="prompt", n=1, lo=16384, hi=16384, past=0, idle=0, heads=32, kv_heads=8, dim=128,
             dtype="bf16"),
        # two users on a short system prompt: latency of a single step
        dict(name="decode_2", op="decode", n=2, shared=257, lo=1, hi=19, idle=0, heads=32, kv_heads=32, dim=128,
             page=16, dtype="f16"),
        # the batch of 16 of the decode stack behind one instruction prompt, one slot idle
        dict(name="decode_16", op="decode", n=16, shared=2048, lo=1, hi=700, idle=1, heads=32, kv_heads=32, dim=128,
             page=16, dtype="f16"),
        # one long conversation with nothing to share: the split over a long axis
        dict(name="decode_1_long", op="decode", n=1, shared=0, lo=65537, hi=65537, idle=0, heads=32, kv_heads=8,
             dim=128, page=64, dtype="bf16"),
        # many users over one long document: every prefix page is read once for all of them
        dict(name="decode_96_doc", op="decode", n=96, shared=32768, lo=1, hi=1500, idle=2, heads=32, kv_heads=8,
             dim=128, page=64, dtype="bf16"),
        # four sampled continuations of a short chat, one layer's worth of cache
        dict(name="fork_4", op="fork", layers=2, pages=128, page=16, kv_heads=8, dim=128, parents=1, each=4, lo=203,
             hi=203, dtype="f16"),
        # 32 continuations of four conversations on all layers of a 32-layer cache
        dict(name="fork_32", op="fork", layers=32, pages=1024, page=64, kv_heads=8, dim=128, parents=4, each=8, lo=700,
             hi=2200, dtype="bf16"),
        # a small pool after half of its sequences left
        dict(name="compact_96", op="compact", layers=4, pages=96, page=16, kv_heads=8, dim=64, seqs=12, lo=9, hi=110,
             keep=0.5, dtype="f16"),
        # a 32-layer pool, two thirds of the sequences gone: the rest moves down to give the tail back
        dict(name="compact_1500", op="compact", layers=32, pages=1500, page=32, kv_heads=8, dim=128, seqs=60, lo=20,
             hi=1400, keep=0.34, dtype="bf16"),
    ]


def _loguniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15


def draw(rng):
    """A case of the ranges above: 1 to 64 prompts of 1 to 16384 tokens, 1 to 96
    decoding sequences over 0 to 32768 shared tokens, pools of 64 to 1500 pages."""
    cap = {"prompt": "prompt_16k", "decode": "decode_96_doc", "fork": "fork_32", "compact": "compact_1500"}
    largest = {c["name"]: _cost(c) for c in listed()}
    while True:
        op = rng.choice(["prompt", "prompt", "decode", "decode", "fork", "compact"])
        dtype = rng.choice(["f16", "bf16"])
        heads, kv_heads = rng.choice([(32, 32), (32, 8), (32, 4), (16, 16), (20, 4), (8, 1)])
        dim = rng.choice([64, 80, 112, 128, 128])
        if op == "prompt":
            hi = _loguniform(rng, 1, 16384)
            case = dict(op=op, n=_loguniform(rng, 1, 64), lo=max(1, hi // rng.choice([1, 4, 30])), hi=hi,
                        past=rng.choice([0, 0, _loguniform(rng, 1, 8192)]), idle=0, heads=heads, kv_heads=kv_heads,
                        dim=dim, dtype=dtype)
            case["idle"] = rng.choice([0, 1]) if case["n"] > 2 else 0
        elif op == "decode":
            hi = _loguniform(rng, 1, 2048)
            case = dict(op=op, n=_loguniform(rng, 1, 96), shared=rng.choice([0, _loguniform(rng, 16, 32768)]),
                        lo=max(1, hi // rng.choice([1, 4, 30])), hi=hi, idle=0, heads=heads, kv_heads=kv_heads, dim=dim,
                        page=rng.choice(PAGE_CHOICES), dtype=dtype)
            case["idle"] = rng.choice([0, 1]) if case["n"] > 2 else 0
        elif op == "fork":
            case = dict(op=op, layers=_loguniform(rng, 1, 32), pages=_loguniform(rng, 128, 1024),
                        page=rng.choice(PAGE_CHOICES[:3]), kv_heads=rng.choice([1, 4, 8]), dim=dim,
                        parents=rng.randint(1, 4), each=_loguniform(rng, 1, 16), lo=1, hi=0, dtype=dtype)
            room = (case["pages"] - case["parents"] * (case["each"] + 1)) // case["parents"] * case["page"]
            if room < 1:
                continue
            case["hi"] = _loguniform(rng, 1, room)
            case["lo"] = max(1, case["hi"] // 3)
        else:
            case = dict(op=op, layers=_loguniform(rng, 1, 32), pages=_loguniform(rng, 64, 1500),
                        page=rng.choice(PAGE_CHOICES[:3]), kv_heads=rng.choice([1, 4, 8]), dim=dim,
                        seqs=_loguniform(rng, 2, 60), lo=1, hi=0, keep=rng.choice([0.2, 0.34, 0.5, 0.8]), dtype=dtype)
            case["hi"] = case["pages"] // case["seqs"] * case["page"]
            case["lo"] = max(1, case["hi"] // 20)
            if case["hi"] < 1:
                continue
        if _cost(case) <= largest[cap[op]]:
            return case


def _lengths(case, n):
    """n token counts between lo and hi, spread over their logarithm, the longest
    first; the last `idle` of them are 0 (slots that hold nothing now)."""
    rng = random.Random(n * 1000003 + case["lo"] * 1009 + case["hi"])
    out = [case["hi"]] + [_loguniform(rng, case["lo"], case["hi"]) for _ in range(n - 1)]
    for i in range(case.get("idle", 0)):
        out[n - 1 - i] = 0
    return out


def _pages_of(tokens, page):
    return -(-tokens // page)


def _prompt_lengths(case):
    lq = _lengths(case, case["n"])
    lk = [n + case["past"] if n else 0 for n in lq]
    return lq, lk


def _decode_lengths(case):
    """Tokens of each sequence, the shared ones included (0: an idle slot)."""
    return [case["shared"] + n if n else 0 for n in _lengths(case, case["n"])]


def _pool_layout(case):
    """fork / compact: per sequence its tokens and pages, as a pool in use hands
    them out: admitted one after another, pages interleaved by a fixed shuffle."""
    n = case["parents"] if case["op"] == "fork" else case["seqs"]
    lens = _lengths(case, n)
    rng = random.Random(case["pages"] * 31 + n)
    ids = list(range(case["pages"]))
    if case["op"] == "compact":
        rng.shuffle(ids)
    rows, at = [], 0
    for t in lens:
        need = _pages_of(t, case["page"])
        rows.append(ids[at:at + need])
        at += need
    kept = [True] * n
    if case["op"] == "compact":
        kept = [rng.random() < case["keep"] for _ in range(n)]
        kept[0] = True
    return lens, rows, kept


# ------------------------------------------------------------------- the work
def work(case):
    """Bytes and operations that a pass cannot do without: each input read once,
    each output written once, the visible scores only."""
    if case["op"] == "prompt":
        lq, lk = _prompt_lengths(case)
        d, hq, hk = case["dim"], case["heads"], case["kv_heads"]
        seen = sum(q * (k - q) + q * (q + 1) // 2 for q, k in zip(lq, lk))
        return {"bytes": 2 * d * (2 * hq * sum(lq) + 2 * hk * sum(lk)) + 8 * (len(lq) + 1), "flops": 4 * d * hq * seen}
    if case["op"] == "decode":
        lens = _decode_lengths(case)
        d, hq, hk, sh = case["dim"], case["heads"], case["kv_heads"], case["shared"]
        tokens = sh + sum(max(0, n - sh) for n in lens)
        return {"bytes": 2 * d * (2 * hk * tokens + 2 * hq * len(lens)) + 4 * _pages_of(tokens, case["page"]),
                "flops": 4 * d * hq * sum(lens)}
    token = case["layers"] * 2 * case["kv_heads"] * case["dim"] * 2  # bytes of a token on every layer, K and V
    lens, rows, kept = _pool_layout(case)
    if case["op"] == "fork":
        tail = [n % case["page"] for n in lens]
        meta = sum(4 * 4 * len(r) * case["each"] for r in rows)
        return {"bytes": sum(t * token * (1 + case["each"]) for t in tail) + meta, "flops": 0}
    live = sorted(p for r, keep in zip(rows, kept) if keep for p in r)
    moved = sum(1 for p in live if p >= len(live))
    return {"bytes": 2 * moved * case["page"] * token + 4 * 3 * case["pages"] + 8 * len(live), "flops": 0}


# ------------------------------------------------------------------ the inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype):
    return torch.randn(*shape, device=DEV, generator=g, dtype=torch.float32).to(dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pool(g, shape, dtype):
    """A pool of pages filled with normal values, layer by layer."""
    out = torch.empty(shape, dtype=dtype, device=DEV)
    for layer in range(shape[0]):
        out[layer].normal_(generator=g)
    return out


def prepare(case, seed):
    """Queries spread with a standard deviation of 1.5 around a common direction
    per head, and a first token whose key points that way: scores with the spread
    and the strong first token that trained heads show."""
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    st = {"case": case}
    if case["op"] == "prompt":
        lq, lk = _prompt_lengths(case)
        d, hq, hk = case["dim"], case["heads"], case["kv_heads"]
        u = torch.randn(hk, 1, d, device=DEV, generator=g)
        cu = lambda ns: [sum(ns[:i]) for i in range(len(ns) + 1)]  # noqa: E731
        st.update(lq=lq, lk=lk, cu_q=_i32(cu(lq)), cu_k=_i32(cu(lk)), scale=d ** -0.5)
        tq, tk = sum(lq), sum(lk)
        # views of fused projection rows; with cached tokens K and V are buffers of their own
        rows = torch.empty(tq, hq + (0 if case["past"] else 2 * hk), d, dtype=dt, device=DEV).normal_(generator=g)
        q, k, v = rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]
        if case["past"]:
            k = torch.empty(tk, hk, d, dtype=dt, device=DEV).normal_(generator=g)
            v = torch.empty(tk, hk, d, dtype=dt, device=DEV).normal_(generator=g)
        q.copy_((q.float() * 1.5).view(tq, hk, hq // hk, d).add_(u).view(tq, hq, d))
        first = [s for s, n in zip(cu(lk), lk) if n]
        k[first] = (k[first].float() + 0.5 * u.view(1, hk, d)).to(dt)
        st.update(q=q, k=k, v=v)
        if own:
            import ane_b200 as ane
            st["ane"] = ane
        return st
    if case["op"] == "decode":
        lens = _decode_lengths(case)
        n, page, sh = case["n"], case["page"], case["shared"]
        d, hq, hk = case["dim"], case["heads"], case["kv_heads"]
        full = sh // page  # whole pages of the prefix are shared, its last part is a copy of each
        own_pages = [max(0, _pages_of(t, page) - full) for t in lens]
        total = full + sum(own_pages)
        spare = total // 8 + 1
        rng = random.Random(total)
        ids = list(range(total + spare))
        rng.shuffle(ids)
        k = _pool(g, (1, total + spare, page, hk, d), dt)[0]
        v = _pool(g, (1, total + spare, page, hk, d), dt)[0]
        width = max(1, max(_pages_of(t, page) for t in lens)) + 2
        table = [[0] * width for _ in range(n)]
        at = full
        for b in range(n):
            r = (ids[:full] + ids[at:at + own_pages[b]]) if lens[b] else []
            table[b][:len(r)] = r
            at += own_pages[b]
        table_t = _i32(table)
        if sh % page:  # the copied part of the prefix holds the same tokens in every sequence
            src = table[0][full]
            for b in range(1, n):
                if lens[b]:
                    k[table[b][full], :sh % page] = k[src, :sh % page]
                    v[table[b][full], :sh % page] = v[src, :sh % page]
        u = torch.randn(hk, 1, d, device=DEV, generator=g)
        q = ((torch.randn(n, hk, hq // hk, d, device=DEV, generator=g) * 1.5) + u).view(n, hq, d).to(dt)
        heads_first = [table[b][0] for b in range(n) if lens[b]]
        k[sorted(set(heads_first)), 0] += (0.5 * u.view(1, hk, d)).to(dt)
        # the batch's rows sit in the cache's slots in another order
        slots = list(range(n))
        rng.shuffle(slots)
        by_slot = torch.empty_like(table_t)
        by_slot[slots] = table_t
        lens_by_slot = [0] * n
        for b, s in enumerate(slots):
            lens_by_slot[s] = lens[b]
        st.update(q=q, k=k, v=v, tables=by_slot, lens=_i32(lens_by_slot), slots=_i32(slots), host_lens=lens,
                  host_slots=slots, scale=d ** -0.5, shared=sh)
        if own:
            import ane_b200 as ane
            st["ane"] = ane
            st["ws"] = ane.attn_decode_workspace(n, hq, hk, d, device=DEV)
        return st
    lens, rows, kept = _pool_layout(case)
    n = len(lens)
    shape = (case["layers"], case["pages"], case["page"], case["kv_heads"], case["dim"])
    k, v = _pool(g, shape, dt), _pool(g, shape, dt)
    children = case["parents"] * case["each"] if case["op"] == "fork" else 0
    width = max(len(r) for r in rows) + 1
    tables = [r + [-1] * (width - len(r)) for r in rows] + [[-1] * width for _ in range(children)]
    refs = [0] * case["pages"]
    for r, keep in zip(rows, kept):
        for p in r:
            refs[p] = 1 if keep else 0
    st.update(k=k, v=v, refs=_i32(refs), tables=_i32(tables),
              lens=_i32([t if keep else 0 for t, keep in zip(lens, kept)] + [0] * children))
    if case["op"] == "fork":
        st["parents"] = _i32([p for p in range(n) for _ in range(case["each"])])
        st["children"] = _i32([n + i for i in range(children)])
        st["granted"] = _i32([0] * children)
    else:
        st.update(refs_out=torch.empty_like(st["refs"]), tables_out=torch.empty_like(st["tables"]),
                  remap=torch.empty_like(st["refs"]), live=_i32([0]))
    if own:
        from ane_b200.kvcache import KVCache
        st["cache"] = KVCache(k, v, st["refs"], st["tables"], st["lens"])
    return st


# -------------------------------------------------------------------- one pass
def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    op = st["case"]["op"]
    if op == "prompt":
        return st["ane"].attn_prompt(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], scale=st["scale"])
    if op == "decode":
        return st["ane"].attn_decode(st["q"], st["k"], st["v"], st["tables"], st["lens"], slots=st["slots"],
                                     shared=st["shared"], scale=st["scale"], workspace=st["ws"])
    cache = st["cache"]
    if op == "fork":
        cache.fork(st["parents"], st["children"], granted=st["granted"])
        cache.free(st["children"])
        return {"granted": st["granted"], "tables": cache.tables, "refs": cache.refs, "lens": cache.lens,
                "k": cache.k, "v": cache.v}
    cache.compact(refs_out=st["refs_out"], tables_out=st["tables_out"], remap=st["remap"], live=st["live"])
    return {"live": st["live"], "remap": st["remap"], "refs": st["refs_out"], "tables": st["tables_out"],
            "k": cache.k, "v": cache.v}


def _softmax_rows(s):
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    return p / p.sum(-1, keepdim=True)


def _run_plain(st):
    case = st["case"]
    if case["op"] == "prompt":
        return _plain_prompt(st)
    if case["op"] == "decode":
        return _plain_decode(st)
    if case["op"] == "fork":
        return _plain_fork(st)
    return _plain_compact(st)


def _plain_prompt(st):
    q, k, v = st["q"], st["k"], st["v"]
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    q0 = k0 = 0
    for lq, lk in zip(st["lq"], st["lk"]):
        if lq:
            kk = k[k0:k0 + lk].float().permute(1, 2, 0)  # kv head, dim, key
            vv = v[k0:k0 + lk].float().permute(1, 0, 2)
            for r in range(0, lq, 512):
                e = min(lq, r + 512)
                see = lk - lq + e  # keys that the block's last row sees
                qq = q[q0 + r:q0 + e].float().view(e - r, hk, hq // hk, d).permute(1, 2, 0, 3)
                s = torch.matmul(qq.reshape(hk, -1, d), kk[:, :, :see]) * st["scale"]
                rows = torch.arange(lk - lq + r, lk - lq + e, device=q.device)
                hidden = torch.arange(see, device=q.device)[None, :] > rows[:, None]
                s = s.view(hk, hq // hk, e - r, see).masked_fill_(hidden, float("-inf"))
                o = torch.matmul(_softmax_rows(s).view(hk, -1, see), vv[:, :see])
                out[q0 + r:q0 + e] = o.view(hk, hq // hk, e - r, d).permute(2, 0, 1, 3).reshape(e - r, hq, d).to(q.dtype)
        q0, k0 = q0 + lq, k0 + lk
    return out


def _plain_decode(st):
    q, k, v = st["q"], st["k"], st["v"]
    n, hq, d = q.shape
    hk = k.shape[2]
    out = torch.zeros_like(q)
    for b in range(n):
        t = st["host_lens"][b]
        if t:
            pages = st["tables"][st["host_slots"][b], :_pages_of(t, k.shape[1])].long()
            kk = k[pages].reshape(-1, hk, d)[:t].float().permute(1, 2, 0)
            vv = v[pages].reshape(-1, hk, d)[:t].float().permute(1, 0, 2)
            s = torch.matmul(q[b].float().view(hk, hq // hk, d), kk) * st["scale"]
            out[b] = torch.matmul(_softmax_rows(s), vv).view(hq, d).to(q.dtype)
    return out


def _plain_fork(st):
    """Children take their parent's row; whole pages gain a reader, the part page
    at the end is copied to the lowest free pages in the order of the requests."""
    k, v, refs, tables, lens = st["k"], st["v"], st["refs"], st["tables"], st["lens"]
    parents, children = st["parents"].long(), st["children"].long()
    page, width = k.shape[2], tables.shape[1]
    n = lens[parents]
    whole = n // page
    part = (n % page) != 0
    order = torch.sort((refs != 0).to(torch.int32), stable=True).indices  # free pages first, lowest first
    fresh = order[torch.cumsum(part.to(torch.int64), 0) - 1]
    col = torch.arange(width, device=refs.device)
    row = tables[parents]
    shared = col[None, :] < whole[:, None]
    old = torch.gather(row, 1, whole.clamp(max=width - 1).long()[:, None])[:, 0].clamp(min=0).long()
    row = torch.where(shared, row, torch.where((col[None, :] == whole[:, None]) & part[:, None],
                                               fresh[:, None].to(torch.int32), tables[children]))
    used = shared | ((col[None, :] == whole[:, None]) & part[:, None])
    ones = used.to(torch.int32)
    refs.index_add_(0, row.clamp(min=0).reshape(-1).long(), ones.reshape(-1))
    tables[children] = row
    lens[children] = n
    st["granted"].fill_(1)
    tok = torch.arange(page, device=refs.device)
    for pool in (k, v):
        for layer in range(pool.shape[0]):
            src, dst = pool[layer, old], pool[layer, fresh]
            take = ((tok[None, :] < (n % page)[:, None]) & part[:, None])[:, :, None, None]
            # a request without a part page writes its own page back: aim it at its parent's page
            pool[layer, torch.where(part, fresh, old)] = torch.where(take, src, torch.where(part[:, None, None, None],
                                                                                           dst, src))
    # free them again
    refs.index_add_(0, row.clamp(min=0).reshape(-1).long(), -ones.reshape(-1))
    lens[children] = 0
    return {"granted": st["granted"], "tables": tables, "refs": refs, "lens": lens, "k": k, "v": v}


def _plain_compact(st):
    """Pages in use above the number of pages in use move to the free pages below
    it, lowest to lowest."""
    k, v, refs, tables, lens = st["k"], st["v"], st["refs"], st["tables"], st["lens"]
    n, page = refs.shape[0], k.shape[2]
    used = refs > 0
    live = used.sum()
    idx = torch.arange(n, device=refs.device)
    hole, mover = ~used & (idx < live), used & (idx >= live)
    holes = torch.sort((~hole).to(torch.int32), stable=True).indices  # holes first, lowest first
    rank = torch.cumsum(mover.to(torch.int64), 0) - 1
    remap = torch.where(mover, holes[rank.clamp(min=0)], idx)
    remap = torch.where(used, remap, torch.full_like(idx, -1))
    dst = torch.nonzero(mover)[:, 0]
    src, dst = dst, remap[dst]
    for pool in (k, v):
        for layer in range(pool.shape[0]):
            pool[layer, dst] = pool[layer, src]
    st["remap"].copy_(remap)
    st["live"].copy_(live.view(1))
    st["refs_out"].copy_(torch.where(idx < live, torch.where(hole, refs[_inverse(remap, idx)], refs),
                                     torch.zeros_like(refs)))
    mine = torch.arange(tables.shape[1], device=refs.device)[None, :] < ((lens + page - 1) // page)[:, None]
    st["tables_out"].copy_(torch.where(mine, remap[tables.clamp(min=0).long()].to(torch.int32), tables))
    return {"live": st["live"], "remap": st["remap"], "refs": st["refs_out"], "tables": st["tables_out"],
            "k": k, "v": v}


def _inverse(remap, idx):
    inv = torch.zeros(idx.shape[0] + 1, dtype=torch.int64, device=idx.device)
    inv[torch.where(remap >= 0, remap, torch.full_like(remap, idx.shape[0]))] = idx
    return inv[:-1]


# ------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The definitions, one sequence and one head at a time (pages: one page at a
    time, with Python integers for the tables)."""
    st = prepare(case, seed)
    if case["op"] == "prompt":
        q, k, v = st["q"], st["k"], st["v"]
        group = q.shape[1] // k.shape[1]
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        q0 = k0 = 0
        for lq, lk in zip(st["lq"], st["lk"]):
            for h in range(q.shape[1] if lq else 0):
                kh, vh = k[k0:k0 + lk, h // group].double(), v[k0:k0 + lk, h // group].double()
                for r in range(0, lq, 2048):
                    e = min(lq, r + 2048)
                    s = (q[q0 + r:q0 + e, h].double() @ kh.T) * case["dim"] ** -0.5
                    i = torch.arange(r, e, device=q.device)[:, None] + (lk - lq)
                    s[torch.arange(lk, device=q.device)[None, :] > i] = float("-inf")
                    out[q0 + r:q0 + e, h] = (s - torch.logsumexp(s, 1, keepdim=True)).exp() @ vh
            q0, k0 = q0 + lq, k0 + lk
        return out
    if case["op"] == "decode":
        q, k, v = st["q"], st["k"], st["v"]
        group = q.shape[1] // k.shape[2]
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        tables = st["tables"].cpu().tolist()
        for b in range(q.shape[0]):
            t = st["host_lens"][b]
            if not t:
                continue
            row = tables[st["host_slots"][b]][:_pages_of(t, case["page"])]
            for h in range(k.shape[2]):
                kh = k[row, :, h].double().reshape(-1, q.shape[2])[:t]
                vh = v[row, :, h].double().reshape(-1, q.shape[2])[:t]
                s = (kh @ q[b, h * group:(h + 1) * group].double().T) * case["dim"] ** -0.5  # key, query
                w = (s - torch.logsumexp(s, 0, keepdim=True)).exp()
                out[b, h * group:(h + 1) * group] = w.T @ vh
        return out
    k, v = st["k"], st["v"]
    refs, tables, lens = st["refs"].tolist(), st["tables"].tolist(), st["lens"].tolist()
    page = case["page"]
    if case["op"] == "fork":
        before = list(refs)
        for p, c in zip(st["parents"].tolist(), st["children"].tolist()):
            whole, rest = divmod(lens[p], page)
            tables[c][:whole] = tables[p][:whole]
            if rest:
                new = refs.index(0)
                refs[new] = 1
                tables[c][whole] = new
                for pool in (k, v):
                    pool[:, new, :rest] = pool[:, tables[p][whole], :rest]
        return {"granted": torch.ones(len(st["children"]), dtype=torch.int32), "tables": torch.tensor(tables),
                "refs": torch.tensor(before), "lens": torch.tensor(lens), "k": k, "v": v}
    live = sum(r > 0 for r in refs)
    remap = [p if r > 0 else -1 for p, r in enumerate(refs)]
    new_refs = list(refs)
    low = 0
    for p in range(live, len(refs)):
        if refs[p] > 0:
            while refs[low] > 0:
                low += 1
            remap[p] = low
            new_refs[low], new_refs[p] = refs[p], 0
            for pool in (k, v):
                pool[:, low] = pool[:, p]
            low += 1
    for s, t in enumerate(lens):
        for i in range(_pages_of(t, page)):
            tables[s][i] = remap[tables[s][i]]
    return {"live": torch.tensor([live]), "remap": torch.tensor(remap), "refs": torch.tensor(new_refs),
            "tables": torch.tensor(tables), "k": k, "v": v}
