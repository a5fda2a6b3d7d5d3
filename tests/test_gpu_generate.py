"""Prompt, fork, decode, free and compact together (ane_b200/generate.py)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def small(kv_heads, dtype, **kw):
    from ane_b200.generate import Generator

    return Generator(2, hidden=512, heads=4, kv_heads=kv_heads, ffn=768, slots=8, pages=64, page_tokens=16, max_pages=12,
                     dtype=dtype, **kw)


@pytest.mark.parametrize("kv_heads,dtype", [(4, torch.float16), (2, torch.bfloat16)])
def test_forked_continuations_match_whole_prompts(ane, kv_heads, dtype):
    """A child's output after t steps is the last row of one prompt made of the
    parent's rows and its own.  Both ways round attention's weights and results
    differently (u of the type, twice per layer), and a rounding can move a Q8_0
    activation by one step of its block's maximum / 127: 2 layers x 4 projections
    of such steps in one element of many stay below 3 % of a row's norm."""
    g = torch.Generator(device="cuda").manual_seed(3)
    P, T, kids = 61, 7, 3
    rows = torch.randn(P, 512, device="cuda", generator=g)
    own = torch.randn(T, kids, 512, device="cuda", generator=g)
    gen = small(kv_heads, dtype)
    out, granted = gen.prompt(rows, i32(0), [P])
    assert granted.tolist() == [1]
    children = i32(5, 2, 7)
    assert gen.fork(0, children).tolist() == [1] * kids
    for t in range(T):
        got, ok = gen.step(own[t], children, shared=P)
        assert ok.tolist() == [1] * kids
    assert gen.cache.lens.tolist() == [P, 0, P + T, 0, 0, P + T, 0, P + T]
    # the parent's whole pages are shared by all, everything else is a child's own
    assert sorted(gen.cache.refs.tolist(), reverse=True)[:3] == [1 + kids] * 3
    whole = small(kv_heads, dtype)
    packed = torch.cat([torch.cat([rows, own[:, c]]) for c in range(kids)])
    want, granted = whole.prompt(packed, i32(1, 3, 4), [P + T] * kids)
    assert granted.tolist() == [1] * kids
    want = want[P + T - 1::P + T]
    assert ((got - want).norm(dim=1) / want.norm(dim=1)).max() < 0.03
    # the prompt itself: the same rows, alone and at the head of the longer ones
    first, _ = small(kv_heads, dtype).prompt(torch.cat([rows, own[:, 0]]), i32(0), [P + T])
    assert ((first[:P] - out).norm(dim=1) / out.norm(dim=1)).max() < 0.03

    # moving the pages changes no result: step again after freeing a child and compacting
    gen.cache.free(i32(5, 0))
    before = gen.cache.tables.clone()
    live, remap = gen.cache.compact()
    assert live.item() == int((gen.cache.refs > 0).sum()) and int((gen.cache.refs[live.item():] != 0).sum()) == 0
    other = small(kv_heads, dtype)
    other.cache.k.copy_(gen.cache.k)
    other.cache.v.copy_(gen.cache.v)
    other.cache.refs.copy_(gen.cache.refs)
    other.cache.lens.copy_(gen.cache.lens)
    other.cache.tables.copy_(gen.cache.tables)
    x = torch.randn(2, 512, device="cuda", generator=g)
    a, _ = gen.step(x, i32(2, 7), shared=P)
    b, _ = other.step(x, i32(2, 7), shared=P)
    assert torch.equal(a, b)
    assert not torch.equal(before, gen.cache.tables)


def test_step_without_pages_is_reported(ane):
    gen = small(4, torch.float16)
    gen.prompt(torch.randn(192, 512, device="cuda"), i32(0), [192])  # max_pages of 16 tokens: full
    out, granted = gen.step(torch.randn(1, 512, device="cuda"), i32(0))
    assert granted.tolist() == [0] and gen.cache.lens[0].item() == 192 and torch.isfinite(out).all()


def test_step_replays_in_a_graph(ane):
    """A captured step, replayed, is the same as calling it: pages are taken on the device."""
    x = torch.randn(2, 512, device="cuda")
    rows = torch.randn(40, 512, device="cuda")
    slots = i32(1, 2)
    gens = [small(2, torch.float16) for _ in range(2)]
    for gen in gens:
        gen.prompt(rows, i32(0), [40])
        gen.fork(0, slots)
        gen.step(x, slots, shared=40)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, granted = gens[0].step(x, slots, shared=40)
    for _ in range(20):
        graph.replay()
        want, _ = gens[1].step(x, slots, shared=40)
        assert torch.equal(out, want) and granted.tolist() == [1, 1]
    assert gens[0].cache.lens.tolist() == gens[1].cache.lens.tolist()
    assert torch.equal(gens[0].cache.refs, gens[1].cache.refs)


def test_command_runs(ane, capsys):
    from ane_b200 import generate

    generate.main(["--layers", "1", "--prompt", "37", "--children", "3", "--steps", "3"])
    assert "3 continuations of 3 steps" in capsys.readouterr().out


def test_command_runs_one_step(ane, capsys):
    from ane_b200 import generate

    generate.main(["--layers", "1", "--prompt", "1", "--children", "1", "--steps", "1"])
    assert "1 continuations of 1 steps" in capsys.readouterr().out
