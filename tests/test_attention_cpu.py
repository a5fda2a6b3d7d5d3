"""Refusals of the attention and cache entry points: argument errors come before
any device work, valid arguments without a GPU fail loudly."""
import ctypes

import pytest
import torch

import ane_b200 as ane

L = ane.lib
INVALID, NO_DEVICE = 1, 5
P = ctypes.byref
A = 1 << 20  # a well-aligned address that is never touched


def rows(data=A, token=512, head=64):
    return ane.Rows(data, token, head)


def prompt(dtype=1, n=1, heads=4, kv_heads=2, dim=64, tq=10, tk=10, q=None, k=None, v=None, cu=A, out_dtype=1, out=None):
    q, k, v, out = (rows() if r is None else r for r in (q, k, v, out))
    return L.ane_attn_prompt_dev(dtype, n, heads, kv_heads, dim, tq, tk, 0.1, P(q), P(k), P(v), cu, None, out_dtype,
                                 P(out), None, None, 0, None)


def decode(dtype=1, batch=2, heads=4, kv_heads=2, dim=64, q=None, pages=None, n_slots=4, max_pages=8, shared=0,
           out_dtype=1, ws=A, ws_bytes=None, tables=A, lens=A, slots=None, out=None):
    q, out = (rows() if r is None else r for r in (q, out))
    pages = ane.Pages(A, A, 16, 16, 2048, 128, 64) if pages is None else pages
    if ws_bytes is None:
        ws_bytes = L.ane_attn_decode_workspace_size(batch, heads, kv_heads, dim)
    return L.ane_attn_decode_dev(dtype, batch, heads, kv_heads, dim, 0.1, P(q), P(pages), tables, n_slots, max_pages, lens,
                                 slots, shared, out_dtype, P(out), None, ws, ws_bytes, None)


@pytest.mark.parametrize("bad", [
    dict(dtype=0), dict(dtype=3), dict(out_dtype=2), dict(out_dtype=9), dict(dim=0), dict(dim=132), dict(dim=136),
    dict(dim=12), dict(kv_heads=0), dict(kv_heads=3), dict(heads=0), dict(heads=130, kv_heads=2), dict(n=1025),
    dict(cu=None), dict(q=rows(A + 8)), dict(k=rows(A, 511)), dict(v=rows(A, 512, 60)), dict(out=rows(0)),
    dict(tq=2 ** 31), dict(out_dtype=0, out=rows(A, 510)),
])
def test_prompt_refusals(bad):
    assert prompt(**bad) == INVALID
    assert ane.last_error() == INVALID


@pytest.mark.parametrize("bad", [
    dict(dtype=0), dict(out_dtype=2), dict(dim=20), dict(heads=5), dict(batch=1025), dict(batch=5), dict(max_pages=0),
    dict(n_slots=0), dict(shared=129), dict(ws=0), dict(ws=A + 16), dict(ws_bytes=100), dict(tables=None),
    dict(lens=None), dict(q=rows(A + 2)),
    dict(pages=ane.Pages(A, A, 16, 12, 2048, 128, 64)), dict(pages=ane.Pages(A, A, 16, 512, 2048, 128, 64)),
    dict(pages=ane.Pages(A, A + 4, 16, 16, 2048, 128, 64)), dict(pages=ane.Pages(A, A, 0, 16, 2048, 128, 64)),
    dict(pages=ane.Pages(A, A, 16, 16, 2044, 128, 64)), dict(pages=ane.Pages(0, A, 16, 16, 2048, 128, 64)),
])
def test_decode_refusals(bad):
    assert decode(**bad) == INVALID
    assert ane.last_error() == INVALID


def cache(**kw):
    from ane_b200.kvcache import _Desc

    f = dict(k=A, v=A, dtype=1, layers=2, pages=8, page_tokens=16, heads=2, dim=64, refs=A, tables=A, lens=A, slots=4,
             max_pages=4, ctl=A)
    f.update(kw)
    return _Desc(*[f[n] for n, _ in _Desc._fields_])


def calls(c, n=1):
    """Every cache entry point on descriptor c."""
    yield L.ane_kv_reserve_dev(P(c), n, A, A, A, None)
    yield L.ane_kv_write_dev(P(c), 0, n, A, None, None, n, 0, P(rows()), P(rows()), None)
    yield L.ane_kv_fork_dev(P(c), n, A, A, A, None)
    yield L.ane_kv_free_dev(P(c), n, A, None)
    yield L.ane_kv_copy_pages_dev(P(c), P(c), n, A, A, None)
    yield L.ane_kv_compact_dev(P(c), A, A, A, A, None)


@pytest.mark.parametrize("bad", [
    dict(k=0), dict(v=A + 8), dict(dtype=0), dict(dtype=3), dict(layers=0), dict(pages=0), dict(pages=2 ** 19 + 1),
    dict(page_tokens=4), dict(page_tokens=48), dict(page_tokens=512), dict(heads=0), dict(dim=0), dict(dim=60),
    dict(dim=136), dict(refs=0), dict(tables=0), dict(lens=0), dict(slots=0), dict(max_pages=0), dict(ctl=0),
])
def test_cache_refusals(bad):
    assert all(rc == INVALID for rc in calls(cache(**bad)))


def test_cache_call_refusals():
    c = cache()
    assert L.ane_kv_reserve_dev(P(c), 1025, A, A, A, None) == INVALID
    assert L.ane_kv_fork_dev(P(c), 1025, A, A, A, None) == INVALID
    assert L.ane_kv_free_dev(P(c), 1025, A, None) == INVALID
    assert L.ane_kv_reserve_dev(P(c), 1, A, A, None, None) == INVALID
    assert L.ane_kv_reserve_dev(None, 1, A, A, A, None) == INVALID
    assert L.ane_kv_write_dev(P(c), 2, 1, A, None, None, 1, 0, P(rows()), P(rows()), None) == INVALID  # no such layer
    assert L.ane_kv_write_dev(P(c), 0, 1, A, None, None, 2, 0, P(rows()), P(rows()), None) == INVALID  # rows != n
    assert L.ane_kv_write_dev(P(c), 0, 1, A, None, None, 1, 2, P(rows()), P(rows()), None) == INVALID  # other 16-bit type
    assert L.ane_kv_write_dev(P(c), 0, 1, A, None, None, 1, 1, P(rows(A + 8)), P(rows()), None) == INVALID
    assert L.ane_kv_copy_pages_dev(P(c), P(cache(dim=128)), 1, A, A, None) == INVALID
    assert L.ane_kv_compact_dev(P(c), None, A, A, A, None) == INVALID


def test_no_gpu_means_loud_failure():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert prompt() == NO_DEVICE and prompt(n=0) == NO_DEVICE and decode() == NO_DEVICE
    assert all(rc == NO_DEVICE for rc in calls(cache()))


@pytest.mark.parametrize("scale", [0.0, -0.5, float("nan"), float("inf")])
def test_scale_refusals(scale):
    r, pages = rows(), ane.Pages(A, A, 16, 16, 2048, 128, 64)
    assert L.ane_attn_prompt_dev(1, 1, 4, 2, 64, 10, 10, scale, P(r), P(r), P(r), A, None, 1, P(r), None, None, 0,
                                 None) == INVALID
    n = L.ane_attn_decode_workspace_size(2, 4, 2, 64)
    assert L.ane_attn_decode_dev(1, 2, 4, 2, 64, scale, P(r), P(pages), A, 4, 8, A, None, 0, 1, P(r), None, A, n,
                                 None) == INVALID


def test_prompt_workspace():
    f = L.ane_attn_prompt_workspace_size
    assert f(1, 32, 32, 128, 17, 17) == 0  # nothing to split
    n = f(1, 32, 8, 128, 512, 8192)
    assert n > 0 and n % 256 == 0
    assert prompt(n=1, heads=32, kv_heads=8, dim=128, tq=512, tk=8192) == INVALID  # no workspace given


def test_workspace_size():
    f = L.ane_attn_decode_workspace_size
    assert f(1, 32, 32, 128) > 0 and f(1, 32, 32, 128) % 256 == 0
    assert f(64, 32, 8, 128) > f(1, 32, 8, 128)
    assert f(1025, 32, 8, 128) == 0 and f(1, 32, 0, 128) == 0 and f(1, 33, 32, 128) == 0


def test_python_refusals():
    """The tensor front end refuses what the C call could not see."""
    q = torch.zeros(4, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        ane.attn_prompt(q, q, q, torch.zeros(2, dtype=torch.int32))  # not CUDA tensors
    with pytest.raises(ValueError):
        ane.attn_prompt(q, q, q[:3], torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        ane.attn_prompt(q, q.bfloat16(), q.bfloat16(), torch.zeros(2, dtype=torch.int32))
    from ane_b200.kvcache import KVCache

    k = torch.zeros(1, 4, 16, 2, 64, dtype=torch.float16)
    ints = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    KVCache(k, k.clone(), ints(4), ints(2, 3), ints(2))
    for args in ((k, k[:, :3], ints(4), ints(2, 3), ints(2)), (k, k, ints(5), ints(2, 3), ints(2)),
                 (k, k, ints(4), ints(2, 3), ints(3)), (k, k, ints(4).long(), ints(2, 3), ints(2)),
                 (k.transpose(1, 2), k.transpose(1, 2), ints(16), ints(2, 3), ints(2))):
        with pytest.raises(ValueError):
            KVCache(*args)
    with pytest.raises(TypeError):
        KVCache(k.float(), k.float(), ints(4), ints(2, 3), ints(2))


class OnDevice:
    """A tensor as the bindings see it, said to be on CUDA device `device` (-1: the host)."""

    def __init__(self, t, device=0):
        self._t, self._device = t, device

    is_cuda = property(lambda self: self._device >= 0)

    def get_device(self):
        return self._device

    def __getattr__(self, name):
        return getattr(self._t, name)


@pytest.fixture
def launches(monkeypatch):
    """The calls that would reach the device; none is made."""
    made = []
    for name in ("ane_attn_prompt_dev", "ane_attn_decode_dev", "ane_kv_reserve_dev", "ane_kv_write_dev", "ane_kv_fork_dev",
                 "ane_kv_free_dev", "ane_kv_copy_pages_dev", "ane_kv_compact_dev"):
        monkeypatch.setattr(L, name, lambda *args, name=name: made.append(name) or 0)
    monkeypatch.setattr(ane, "_stream_of", lambda stream, t: 0)
    return made


WHERE = [-1, 1]  # on the host, on another device


def half(*shape):
    return OnDevice(torch.zeros(shape, dtype=torch.float16))


def ints(*shape):
    return OnDevice(torch.zeros(shape, dtype=torch.int32))


def moved(args, name, device):
    args = dict(args)
    if name:
        args[name] = OnDevice(args[name]._t, device)
    return args


@pytest.mark.parametrize("device", WHERE)
def test_prompt_takes_nothing_from_elsewhere(launches, device):
    """A pointer to host memory, or to another device's, never reaches a kernel."""
    n = ane.lib.ane_attn_prompt_workspace_size(1, 4, 2, 64, 64, 2048)
    args = dict(q=half(64, 4, 64), k=half(2048, 2, 64), v=half(2048, 2, 64), cu_q=ints(2), cu_k=ints(2),
                out=half(64, 4, 64), lse=OnDevice(torch.zeros(64, 4)), workspace=OnDevice(torch.zeros(n, dtype=torch.uint8)))
    assert n > 0
    ane.attn_prompt(**args)
    assert launches == ["ane_attn_prompt_dev"]
    for name in args:
        with pytest.raises(ValueError):
            ane.attn_prompt(**moved(args, name, device))
    with pytest.raises(ValueError):
        ane.attn_prompt(**{**args, "workspace": OnDevice(torch.zeros(2 * n, dtype=torch.uint8)[::2])})
    assert len(launches) == 1


@pytest.mark.parametrize("device", WHERE)
def test_decode_takes_nothing_from_elsewhere(launches, device):
    n = ane.lib.ane_attn_decode_workspace_size(2, 4, 2, 64)
    args = dict(q=half(2, 4, 64), k=half(8, 16, 2, 64), v=half(8, 16, 2, 64), tables=ints(3, 4), lens=ints(3),
                slots=ints(2), out=half(2, 4, 64), lse=OnDevice(torch.zeros(2, 4)),
                workspace=OnDevice(torch.zeros(n, dtype=torch.uint8)))
    ane.attn_decode(**args)
    assert launches == ["ane_attn_decode_dev"]
    for name in args:
        with pytest.raises(ValueError):
            ane.attn_decode(**moved(args, name, device))
    assert len(launches) == 1


@pytest.mark.parametrize("device", WHERE)
def test_cache_takes_nothing_from_elsewhere(launches, device):
    from ane_b200.kvcache import KVCache

    def new(d=0):
        pool = OnDevice(torch.zeros(2, 8, 16, 2, 64, dtype=torch.float16), d)
        return KVCache(pool, pool, ints(8), ints(3, 4), ints(3))

    c = new()
    calls = [
        (c.reserve, dict(slots=ints(1), counts=ints(1), granted=ints(1))),
        (c.write, dict(layer=0, slots=ints(1), k=half(1, 2, 64), v=half(1, 2, 64), cu=ints(2), granted=ints(1))),
        (c.fork, dict(parents=ints(1), children=ints(1), granted=ints(1))),
        (c.free, dict(slots=ints(1))),
        (c.copy_pages, dict(src=ints(2), dst=ints(2))),
        (c.compact, dict(refs_out=ints(8), tables_out=ints(3, 4), remap=ints(8), live=ints(1))),
    ]
    for call, args in calls:
        call(**args)
    made = len(launches)
    assert made == len(calls)
    for call, args in calls:
        for name in args:
            if name != "layer":
                with pytest.raises(ValueError):
                    call(**moved(args, name, device))
    with pytest.raises(ValueError):
        c.copy_pages(ints(1), ints(1), into=new(device))
    host = new(-1)
    with pytest.raises(ValueError):
        host.free(OnDevice(torch.zeros(1, dtype=torch.int32), -1))
    assert len(launches) == made


def test_decode_most_heads():
    """One head more than the join's grid takes is refused before anything is launched."""
    assert decode(heads=65536, kv_heads=1024, q=rows(A, 64 * 65536), out=rows(A, 64 * 65536)) == INVALID
    ok = decode(heads=65472, kv_heads=1023, q=rows(A, 64 * 65472), out=rows(A, 64 * 65472), batch=0)
    assert ok == (0 if torch.cuda.is_available() else NO_DEVICE)


@pytest.mark.parametrize("args", [["--steps", "0"], ["--prompt", "0"], ["--layers", "0"], ["--children", "0"],
                                  ["--children", "16"], ["--steps", "-3"]])
def test_generate_command_refusals(args, capsys):
    from ane_b200 import generate

    with pytest.raises(SystemExit) as e:
        generate.main(args)
    assert e.value.code == 2 and "error" in capsys.readouterr().err


def test_prompt_is_cut_where_a_history_is_long():
    """Prompts without one are dealt out as whole items (cut ones take up to twice as
    long), however few they are; a few blocks behind a long one are cut."""
    f = L.ane_attn_prompt_workspace_size
    for tokens in (17, 500, 1000, 2112, 5000, 16384):
        for n in (1, 4, 9):
            assert f(n, 32, 8, 128, tokens, tokens) == 0 and f(n, 8, 8, 64, tokens, tokens) == 0
    assert f(4, 32, 8, 128, 800, 2000) == 0 and f(1, 32, 8, 128, 200, 1200) == 0
    assert f(1, 32, 8, 128, 1, 8001) > 0 and f(2, 32, 8, 64, 1533, 1533 + 2 * 7681) > 0
    assert f(0, 32, 8, 128, 0, 8000) == 0 and f(5, 32, 8, 128, 0, 8000) == 0
    assert f(1024, 64, 1, 128, 2 ** 31 - 2 ** 17, 2 ** 31 - 2 ** 17) == 0
