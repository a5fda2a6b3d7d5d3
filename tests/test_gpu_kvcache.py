"""Pages of a key/value cache against a model in Python integers: exact."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Model:
    """The rules of include/ane_b200.h, one request after another."""

    def __init__(self, c):
        self.page, self.pages, self.max_pages = c.page_tokens, c.pages, c.max_pages
        self.refs = c.refs.tolist()
        self.lens = c.lens.tolist()
        self.tables = c.tables.tolist()
        self.k, self.v = c.k.clone(), c.v.clone()

    def need(self, n):
        return -(-n // self.page)

    def grant(self, wants):
        """wants: pages needed per request (None: refused for itself); in order while pages last."""
        free, total, out = self.refs.count(0), 0, []
        for w in wants:
            if w is None:
                out.append(False)
                continue
            total += w
            out.append(w == 0 or total <= free)
        return out

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def reserve(self, slots, counts):
        seen, wants = set(), []
        for s, c in zip(slots, counts):
            ok = 0 <= s < len(self.lens) and s not in seen and c >= 0 and self.need(self.lens[s] + c) <= self.max_pages
            seen.add(s)
            wants.append(self.need(self.lens[s] + c) - self.need(self.lens[s]) if ok else None)
        got = self.grant(wants)
        for s, c, w, g in zip(slots, counts, wants, got):
            if g:
                have = self.need(self.lens[s])
                for i in range(w):
                    self.tables[s][have + i] = self.take()
                self.lens[s] += c
        return [int(g) for g in got]

    def fork(self, parents, children):
        before = list(self.lens)
        seen, wants = set(), []
        for p, c in zip(parents, children):
            ok = 0 <= c < len(before) and 0 <= p < len(before) and before[c] == 0 and c not in seen
            seen.add(c)
            wants.append(int(before[p] % self.page != 0) if ok else None)
        got = self.grant(wants)
        for p, c, g in zip(parents, children, got):
            if not g:
                continue
            whole, rest = divmod(before[p], self.page)
            if rest:
                new, old = self.take(), self.tables[p][whole]
                for pool in (self.k, self.v):
                    pool[:, new, :rest] = pool[:, old, :rest]
                self.tables[c][whole] = new
            for i in range(whole):
                self.tables[c][i] = self.tables[p][i]
                self.refs[self.tables[p][i]] += 1
            self.lens[c] = before[p]
        return [int(g) for g in got]

    def free(self, slots):
        for s in slots:
            if 0 <= s < len(self.lens):
                for i in range(self.need(self.lens[s])):
                    self.refs[self.tables[s][i]] -= 1
                self.lens[s] = 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        remap = [p if r > 0 else -1 for p, r in enumerate(self.refs)]
        holes = [p for p in range(live) if self.refs[p] == 0]
        movers = [p for p in range(live, self.pages) if self.refs[p] > 0]
        for p, h in zip(movers, holes):
            remap[p] = h
            self.refs[h], self.refs[p] = self.refs[p], 0
            for pool in (self.k, self.v):
                pool[:, h] = pool[:, p]
        for s, n in enumerate(self.lens):
            for i in range(self.need(n)):
                self.tables[s][i] = remap[self.tables[s][i]]
        return live, remap

    def same(self, c):
        assert c.refs.tolist() == self.refs
        assert c.lens.tolist() == self.lens
        for s, n in enumerate(self.lens):
            assert c.tables[s].tolist() == self.tables[s], s
        assert torch.equal(c.k.view(torch.int16), self.k.view(torch.int16))
        assert torch.equal(c.v.view(torch.int16), self.v.view(torch.int16))


def new_cache(layers=2, pages=40, page=16, heads=2, dim=64, slots=8, max_pages=10, dtype=torch.float16, seed=0):
    from ane_b200.kvcache import KVCache

    c = KVCache.empty(layers, pages, page, heads, dim, slots, max_pages, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    c.k.normal_(generator=g)
    c.v.normal_(generator=g)
    return c


@pytest.mark.parametrize("page,heads,dim,pages", [(8, 1, 8, 33), (16, 2, 64, 40), (64, 3, 80, 31), (256, 1, 128, 64)])
@pytest.mark.parametrize("seed", [0, 1])
def test_random_life_of_a_cache(ane, page, heads, dim, pages, seed):
    rng = random.Random(seed * 100 + pages)
    c = new_cache(page=page, heads=heads, dim=dim, pages=pages, slots=8, max_pages=10, seed=seed)
    m = Model(c)
    for step in range(60):
        op = rng.choice(["reserve", "reserve", "fork", "free", "compact", "away"])
        n = rng.randint(1, 5)
        if op == "reserve":
            slots = [rng.randrange(-1, 9) for _ in range(n)]
            counts = [rng.choice([0, 1, page - 1, page, page + 1, 3 * page, -1]) for _ in range(n)]
            assert c.reserve(i32(slots), i32(counts)).tolist() == m.reserve(slots, counts)
        elif op == "fork":
            parents = [rng.randrange(-1, 9) for _ in range(n)]
            children = [rng.randrange(-1, 9) for _ in range(n)]
            assert c.fork(i32(parents), i32(children)).tolist() == m.fork(parents, children)
        elif op == "free":
            slots = [rng.randrange(-1, 9) for _ in range(n)]
            c.free(i32(slots))
            m.free(slots)
        elif op == "compact":
            live, remap = c.compact()
            want = m.compact()
            assert (live.item(), remap.tolist()) == want
        else:  # into other arrays: the cache itself keeps its state, the moved copies are there
            refs, tables = torch.empty_like(c.refs), torch.full_like(c.tables, -7)
            before = (c.refs.clone(), c.tables.clone())
            live, remap = c.compact(refs_out=refs, tables_out=tables)
            assert torch.equal(before[0], c.refs) and torch.equal(before[1], c.tables)
            assert (live.item(), remap.tolist()) == m.compact()
            c.refs.copy_(refs)
            c.tables.copy_(tables)
        m.same(c)
        assert c._ctl.item() == 0


def test_pages_run_out_in_order(ane):
    c = new_cache(pages=5, page=8, max_pages=10, slots=4)
    m = Model(c)
    for slots, counts in (([0, 1, 2], [16, 17, 8]), ([2, 3, 1], [8, 1, 1])):
        got = c.reserve(i32(slots), i32(counts)).tolist()
        assert got == m.reserve(slots, counts)
        m.same(c)
    assert got == [0, 0, 1]  # no page is left, but slot 1's part page has room
    got = c.fork(i32([0, 1]), i32([2, 3])).tolist()
    assert got == m.fork([0, 1], [2, 3]) == [1, 0]
    m.same(c)


@pytest.mark.parametrize("pages", [1, 31, 32, 33, 4097, 70001])
def test_many_pages(ane, pages):
    c = new_cache(layers=1, pages=pages, page=8, heads=1, dim=8, slots=4, max_pages=pages)
    m = Model(c)
    third = max(1, pages // 3)
    assert c.reserve(i32([0, 1]), i32([third * 8 - 3, 5])).tolist() == m.reserve([0, 1], [third * 8 - 3, 5])
    assert c.fork(i32([1, 0]), i32([2, 3])).tolist() == m.fork([1, 0], [2, 3])
    m.same(c)
    c.free(i32([0, 3]))
    m.free([0, 3])
    live, remap = c.compact()
    assert (live.item(), remap.tolist()) == m.compact()
    m.same(c)


def test_many_requests(ane):
    c = new_cache(layers=1, pages=1500, page=8, heads=1, dim=8, slots=1200, max_pages=4)
    m = Model(c)
    slots = list(range(600)) + [3, 5] + list(range(600, 1000))
    counts = [(i * 7) % 12 for i in range(len(slots))]
    assert c.reserve(i32(slots), i32(counts)).tolist() == m.reserve(slots, counts)
    parents, children = [i % 1000 for i in range(400)], [1199 - i % 250 for i in range(400)]
    assert c.fork(i32(parents), i32(children)).tolist() == m.fork(parents, children)
    m.same(c)


@pytest.mark.parametrize("src", [torch.float32, torch.float16])
def test_write_rows(ane, src):
    c = new_cache(layers=3, pages=20, page=16, heads=2, dim=72, slots=4, max_pages=6)
    m = Model(c)
    slots, counts = [2, 0, 3], [5, 33, 40]
    granted = c.reserve(i32(slots), i32(counts))
    m.reserve(slots, counts)
    g = torch.Generator(device="cuda").manual_seed(1)
    cu = [0, 5, 38, 78]
    rows = (torch.randn(78, 6, 72, device="cuda", generator=g) * 3).to(src)  # a fused row: q, k, v of two heads each
    k, v = rows[:, 2:4], rows[:, 4:6]
    c.write(1, i32(slots), k, v, cu=i32(cu), granted=granted)
    for i, s in enumerate(slots):
        for t in range(counts[i]):
            page = m.tables[s][t // 16]
            m.k[1, page, t % 16] = k[cu[i] + t].half()
            m.v[1, page, t % 16] = v[cu[i] + t].half()
    m.same(c)
    # one more token each; slot 3's request is not granted and changes nothing
    granted = c.reserve(i32([0, 3, 2]), i32([1, 1000, 1]))
    assert granted.tolist() == m.reserve([0, 3, 2], [1, 1000, 1]) == [1, 0, 1]
    c.write(2, i32([0, 3, 2]), k[:3], v[:3], granted=granted)
    for s, r in ((0, 0), (2, 2)):
        t = m.lens[s] - 1
        m.k[2, m.tables[s][t // 16], t % 16] = k[r].half()
        m.v[2, m.tables[s][t // 16], t % 16] = v[r].half()
    m.same(c)


def test_write_rounds_to_nearest_bf16(ane):
    c = new_cache(layers=1, pages=2, page=8, heads=1, dim=8, slots=1, max_pages=2, dtype=torch.bfloat16)
    c.reserve(i32([0]), i32([1]))
    k = torch.tensor([[[1.00390625, 1.01171875, -1.00390625, 3e38, float("inf"), float("nan"), 1e-40, 0.1]]], device="cuda")
    c.write(0, i32([0]), k, k)
    got = c.k[0, c.tables[0, 0], 0, 0]
    assert torch.equal(got.float().nan_to_num(nan=5.0), k[0, 0].bfloat16().float().nan_to_num(nan=5.0))


def test_copy_pages_between_caches(ane):
    a, b = new_cache(pages=9, seed=1), new_cache(pages=30, seed=2)
    m = Model(b)
    src, dst = [0, 8, 3, -1, 9, 2], [29, 0, 7, 1, 2, 30]
    a.copy_pages(i32(src), i32(dst), into=b)
    for s, d in zip(src, dst):
        if 0 <= s < 9 and 0 <= d < 30:
            m.k[:, d], m.v[:, d] = a.k[:, s], a.v[:, s]
    m.same(b)
    b.copy_pages(i32([29]), i32([5]))
    m.k[:, 5], m.v[:, 5] = m.k[:, 29], m.v[:, 29]
    m.same(b)


def test_cache_past_four_gigabytes(ane):
    """Offsets of a pool that passes 32 bits: the last pages of the last layer."""
    from ane_b200.kvcache import KVCache

    c = KVCache.empty(5, 1024, 256, 16, 128, 4, 1024)
    assert c.k.numel() > 2 ** 31
    n = 1022 * 256 + 100
    assert c.reserve(i32([0]), i32([n])).tolist() == [1]
    row = torch.randn(1, 16, 128, device="cuda")
    c.write(4, i32([0]), row, row * 2)
    assert c.fork(i32([0]), i32([1])).tolist() == [1]
    assert torch.equal(c.k[4, 1023, 99], row[0].half()) and torch.equal(c.v[4, 1023, 99], (row[0] * 2).half())
    c.free(i32([0]))
    assert c.lens.tolist()[:2] == [0, n] and int((c.refs == 0).sum()) == 1
    live, _ = c.compact()
    assert live.item() == 1023 and torch.equal(c.k[4, 1022, 99], row[0].half())


def test_graph_and_side_stream(ane):
    c = new_cache()
    c.reserve(i32([0]), i32([37]))
    m = Model(c)
    par, chi, granted = i32([0, 0]), i32([1, 2]), i32([5, 5])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    c.fork(par, chi, granted=granted, stream=side)
    c.free(chi, stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.fork(par, chi, granted=granted)
        c.free(chi)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    m.fork([0, 0], [1, 2])
    m.free([1, 2])
    m.same(c)
    assert granted.tolist() == [1, 1]


@pytest.mark.parametrize("src", [torch.float32, torch.float16])
def test_write_leaves_rows_outside_cu_alone(ane, src):
    """Rows before cu[0] and from cu[n] on belong to no request: a slot's older
    tokens, and the pages that a fork reads with it, stay as they are."""
    c = new_cache(layers=2, pages=20, page=16, heads=2, dim=64, slots=4, max_pages=6)
    m = Model(c)
    assert c.reserve(i32([0]), i32([37])).tolist() == m.reserve([0], [37])
    assert c.fork(i32([0]), i32([1])).tolist() == m.fork([0], [1])
    slots, cu = [0, 2], [26, 31, 34]  # as many rows before them as reach the whole pages that slot 1 reads too
    granted = c.reserve(i32(slots), i32([5, 3]))
    assert granted.tolist() == m.reserve(slots, [5, 3])
    rows = torch.randn(40, 4, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(src)
    k, v = rows[:, :2], rows[:, 2:]
    c.write(1, i32(slots), k, v, cu=i32(cu), granted=granted)
    for i, s in enumerate(slots):
        n = cu[i + 1] - cu[i]
        for j in range(n):
            t = m.lens[s] - n + j
            m.k[1, m.tables[s][t // 16], t % 16] = k[cu[i] + j].half()
            m.v[1, m.tables[s][t // 16], t % 16] = v[cu[i] + j].half()
    m.same(c)


def test_attend_after_the_first_sequence_left(ane):
    """Continuations of one prompt, of which the first is freed and its table row
    left behind by a compaction: the others still attend to the prompt."""
    c = new_cache(layers=1, pages=40, page=16, heads=2, dim=64, slots=5, max_pages=8)
    assert c.reserve(i32([4]), i32([70])).tolist() == [1]  # lower pages, to be given up
    assert c.reserve(i32([0]), i32([90])).tolist() == [1]
    children = i32([1, 2, 3])
    assert c.fork(i32([0, 0, 0]), children).tolist() == [1, 1, 1]
    assert c.reserve(children, i32([5, 9, 30])).tolist() == [1, 1, 1]
    c.free(i32([4, 1]))
    c.compact()
    q = torch.randn(3, 4, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).half()
    got = c.attend(0, q, children, shared=90, out_dtype=torch.float32)
    want = c.attend(0, q, children, out_dtype=torch.float32)  # nothing shared: each through its own pages
    assert (got[0] == 0).all()
    # rounding of the weights to F16 in both, values of a few units
    assert (got - want).abs().max() < 2 * 2.0 ** -11 * 4


def test_write_takes_a_slot_once(ane):
    """A slot named twice counts once, the first time, also without granted."""
    c = new_cache(layers=1, pages=20, page=16, heads=2, dim=64, slots=600, max_pages=3)
    m = Model(c)
    assert c.reserve(i32([0, 1, 2]), i32([20, 10, 33])).tolist() == m.reserve([0, 1, 2], [20, 10, 33])
    rows = torch.randn(600, 4, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).half()
    k, v = rows[:, :2], rows[:, 2:]

    def wrote(s, back, r):  # row r is the token `back` before the slot's end
        t = m.lens[s] - back
        m.k[0, m.tables[s][t // 16], t % 16], m.v[0, m.tables[s][t // 16], t % 16] = k[r], v[r]

    slots = [2, 0, 2, -1, 0, 600] + [5] * 594
    slots[590] = 1  # far behind its block's own first look
    slots[599] = 1
    c.write(0, i32(slots), k, v)
    for s, r in ((2, 0), (0, 1), (1, 590)):
        wrote(s, 1, r)
    m.same(c)
    c.write(0, i32([1, 0, 1]), k[10:21], v[10:21], cu=i32([0, 3, 4, 11]))
    for i in range(3):
        wrote(1, 3 - i, 10 + i)
    wrote(0, 1, 13)
    m.same(c)


def test_side_stream_next_to_freed_memory(ane):
    """What the cache's calls return does not lie in memory that work on the current
    stream is still to write."""
    c = new_cache(pages=40)
    m = Model(c)
    one, ten, two = i32([1]), i32([10]), i32([2])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    held = [torch.empty(n, dtype=torch.int32, device="cuda") for n in (1, 1, 1, 40)]
    torch.cuda._sleep(100_000_000)  # about 50 ms
    for h in held:
        h.fill_(-5)
    del held, h
    got = [c.reserve(one, ten, stream=side), c.fork(one, two, stream=side), *c.compact(stream=side)]
    side.synchronize()
    torch.cuda.synchronize()
    want = [m.reserve([1], [10]), m.fork([1], [2])]
    live, remap = m.compact()
    assert [g.tolist() for g in got] == want + [[live], remap]
    m.same(c)


def test_write_of_no_rows(ane):
    """Requests without rows, whose tensors have no memory."""
    c = new_cache()
    assert c.reserve(i32([0, 1]), i32([3, 0])).tolist() == [1, 1]
    m = Model(c)
    none = torch.empty(0, 2, 64, device="cuda")
    c.write(0, i32([0, 1]), none, none, cu=i32([0, 0, 0]))
    c.write(0, i32([]), none, none)
    c.write(0, i32([]), none.half(), none.half(), cu=i32([0]))
    m.same(c)
