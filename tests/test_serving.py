"""The paged cache's operators without a device: the shapes their constructors give and what the HIP backend
refuses before it queues anything."""
import ctypes as C

import pytest

from gl import Graph, gl


def refusal(node):
    why = gl.libs()["hip"].ggml_backend_hip_refusal(node)
    return why.decode() if why else None


def rope_multi(g, a, b, c=None, n_dims=64, sections=(8, 12, 12, 0), mode=gl.ROPE_MROPE, base=1e4):
    return g.rope_multi(a, b, c, n_dims, (C.c_int * 4)(*sections), mode, 0, base, 1.0, 0.0, 1.0, 32.0, 1.0)


def operands(g, D=64, H=3, T=5):
    return g.tensor(gl.F32, D, H, T), g.tensor(gl.I32, 4 * T)


@pytest.mark.parametrize("o", [
    dict(), dict(n_dims=32), dict(mode=gl.ROPE_IMROPE), dict(mode=gl.ROPE_VISION, n_dims=32, sections=(16, 16, 0, 0)),
    dict(sections=(1, 0, 0, 0)), dict(sections=(0, 0, 0, 7)),
])
def test_rope_multi_accepts(o):
    with Graph(mem=1 << 20) as g:
        n = rope_multi(g, *operands(g), **o)
        assert refusal(n) is None
        assert list(n.contents.ne) == [64, 3, 5, 1]


@pytest.mark.parametrize("o, says", [
    (dict(n_dims=63), "n_dims"), (dict(n_dims=0), "n_dims"), (dict(n_dims=66), "n_dims"), (dict(mode=0), "mode"),
    (dict(mode=2), "mode"), (dict(mode=gl.ROPE_VISION), "n_dims"), (dict(sections=(0, 0, 0, 0)), "sections"),
    (dict(sections=(-1, 20, 20, 0)), "section"), (dict(base=0.0), "freq_base"), (dict(base=float("inf")), "freq_base"),
    (dict(base=float("nan")), "freq_base"),
])
def test_rope_multi_refuses(o, says):
    with Graph(mem=1 << 20) as g:
        assert says in refusal(rope_multi(g, *operands(g), **o))


def test_rope_multi_refuses_operands():
    with Graph(mem=1 << 20) as g:
        a, b = operands(g)
        assert refusal(rope_multi(g, g.tensor(gl.F16, 64, 3, 5), b))
        assert refusal(rope_multi(g, a, g.tensor(gl.I32, 5)))
        assert refusal(rope_multi(g, a, g.tensor(gl.F32, 20)))
        assert refusal(rope_multi(g, a, None))
        assert refusal(rope_multi(g, g.permute(g.tensor(gl.F32, 3, 64, 5), 1, 0, 2, 3), b))
        assert refusal(rope_multi(g, a, b, g.tensor(gl.F32, 31)))
        assert refusal(rope_multi(g, a, b, g.tensor(gl.F32, 32))) is None
        assert refusal(rope_multi(g, g.tensor(gl.F32, 264, 3, 5), b, n_dims=264))     # more pairs than a launch holds
        past = g.view_3d(g.tensor(gl.F32, 64 * 15), 64, 3, 5, 256, 800, 0)
        assert refusal(rope_multi(g, past, b))


@pytest.mark.parametrize("t", [gl.F32, gl.F16, gl.BF16, gl.Q8_0, gl.Q4_0])
@pytest.mark.parametrize("it", [gl.I32, gl.I64])
def test_set_rows_accepts(t, it):
    with Graph(mem=1 << 20) as g:
        a = g.tensor(t, 64, 10, 4, 6)
        n = g.set_rows(a, g.tensor(gl.F32, 64, 7, 4, 6), g.tensor(it, 7, 2, 3))
        assert refusal(n) is None
        assert list(n.contents.ne) == [64, 10, 4, 6] and n.contents.type == t


def test_set_rows_refuses():
    with Graph(mem=1 << 20) as g:
        a, b, c = g.tensor(gl.F16, 64, 10), g.tensor(gl.F32, 64, 7), g.tensor(gl.I32, 7)
        assert refusal(g.set_rows(a, b, c)) is None
        assert refusal(g.set_rows(a, g.tensor(gl.F32, 32, 7), c))
        assert refusal(g.set_rows(a, g.tensor(gl.F16, 64, 7), c))
        assert refusal(g.set_rows(a, b, g.tensor(gl.I32, 8)))
        assert refusal(g.set_rows(a, b, g.tensor(gl.F32, 7)))
        assert refusal(g.set_rows(a, b, None))
        assert refusal(g.set_rows(g.tensor(gl.Q4_K, 256, 10), g.tensor(gl.F32, 256, 7), c))
        assert refusal(g.set_rows(g.tensor(gl.I32, 64, 10), b, c))
        assert refusal(g.set_rows(g.tensor(gl.F16, 64, 10, 3), g.tensor(gl.F32, 64, 7, 3), g.tensor(gl.I32, 7, 2)))
        assert refusal(g.set_rows(g.transpose(g.tensor(gl.F32, 10, 64)), b, c))
        q = g.tensor(gl.Q4_0, 64, 12)
        assert refusal(g.set_rows(g.view_2d(q, 64, 10, 36, 72), b, c)) is None
        assert refusal(g.set_rows(g.view_2d(q, 64, 5, 108, 0), b, c))         # past the end
        assert refusal(g.set_rows(g.view_2d(q, 64, 4, 18, 0), b, c))          # rows in one another
        assert refusal(g.set_rows(g.view_3d(q, 64, 3, 2, 72, 36, 0), g.tensor(gl.F32, 64, 7, 2), g.tensor(gl.I32, 7, 2))) is None
        assert refusal(g.set_rows(g.view_3d(q, 64, 3, 2, 72, 72, 0), g.tensor(gl.F32, 64, 7, 2), g.tensor(gl.I32, 7, 2)))
        assert refusal(g.set_rows(g.view_2d(q, 64, 10, 36, 9), b, c))         # inside a block
        assert refusal(g.set_rows(g.view_2d(q, 64, 5, 45, 0), g.tensor(gl.F32, 64, 7), c))


def paged(g, T=6, S=2, D=64, H=4, KV=2, P=16, NP=9, most=5, **o):
    x = dict(q=g.tensor(gl.F32, D, H, T), k=g.tensor(gl.Q4_0, D, KV, P, NP), v=g.tensor(gl.Q4_0, D, KV, P, NP),
             pages=g.tensor(gl.I32, most, S), start=g.tensor(gl.I32, S + 1), seen=g.tensor(gl.I32, S))
    x.update(o)
    return g.flash_attn_paged(x["q"], x["k"], x["v"], x["pages"], x["start"], x["seen"], 0.125)


@pytest.mark.parametrize("o", [dict(), dict(D=96), dict(D=128, H=32, KV=8), dict(H=2), dict(P=1), dict(P=100), dict(T=0), dict(S=1), dict(S=0, T=0)])
def test_flash_attn_paged_accepts(o):
    with Graph(mem=1 << 20) as g:
        n = paged(g, **o)
        assert refusal(n) is None
        assert list(n.contents.ne)[:3] == [o.get("D", 64), o.get("H", 4), o.get("T", 6)]


def test_flash_attn_paged_accepts_any_order_of_the_cache():
    with Graph(mem=1 << 20) as g:
        k = g.permute(g.tensor(gl.Q4_0, 64, 16, 2, 9), 0, 2, 1, 3)        # a page's heads one after another
        assert refusal(paged(g, k=k, v=k)) is None


@pytest.mark.parametrize("name, ne, t", [
    ("q", (80, 4, 6), gl.F32), ("q", (64, 3, 6), gl.F32), ("q", (64, 4, 6), gl.F16), ("q", (64, 4, 6, 2), gl.F32),
    ("k", (64, 2, 16, 9), gl.F16), ("k", (64, 2, 16, 9), gl.Q8_0), ("k", (32, 2, 16, 9), gl.Q4_0), ("v", (64, 2, 16, 8), gl.Q4_0),
    ("v", (64, 2, 8, 9), gl.Q4_0), ("pages", (5, 2), gl.F32), ("pages", (5, 3), gl.I32), ("pages", (5, 2, 2), gl.I32),
    ("start", (2,), gl.I32), ("start", (3,), gl.I64), ("seen", (3,), gl.I32), ("seen", (2,), gl.F32), ("seen", (1, 2), gl.I32),
])
def test_flash_attn_paged_refuses(name, ne, t):
    with Graph(mem=1 << 20) as g:
        assert refusal(paged(g, **{name: g.tensor(t, *ne)}))


def test_flash_attn_paged_refuses_a_cache_without_pages_and_tables_of_too_many_positions():
    with Graph(mem=1 << 20) as g:
        assert refusal(paged(g, k=g.tensor(gl.Q4_0, 64, 2, 16, 0), v=g.tensor(gl.Q4_0, 64, 2, 16, 0)))
        t = g.tensor(gl.Q4_0, 64 * 64, 1)
        k = g.view_4d(t, 64, 64, 1, 1, 36, 36 * 64, 36 * 64, 0)                     # 64 heads, a position a page
        q = g.tensor(gl.F32, 64, 64, 6)
        for most, ok in ((1 << 29, True), ((1 << 30) - 32, True), (1 << 30, False)):
            n = paged(g, q=q, k=k, v=k, pages=g.tensor(gl.I32, most, 2))
            assert (refusal(n) is None) == ok
        t = g.tensor(gl.Q4_0, 64 * 1024, 1)
        k = g.view_4d(t, 64, 1024, 1, 1, 36, 36 * 1024, 36 * 1024, 0)
        q = g.tensor(gl.F32, 64, 1024, 6)
        for most, ok in ((1 << 25, True), (1 << 26, False), (1 << 29, False)):
            n = paged(g, q=q, k=k, v=k, pages=g.tensor(gl.I32, most, 2))
            assert (refusal(n) is None) == ok


def test_flash_attn_paged_refuses_missing_operands_and_strides():
    with Graph(mem=1 << 20) as g:
        for name in ("pages", "start", "seen", "k", "v"):
            assert "missing" in refusal(paged(g, **{name: None}))
        k = g.tensor(gl.Q4_0, 64 * 2 * 16 * 9)
        assert refusal(paged(g, k=g.view_4d(k, 64, 2, 16, 9, 36, 72, 1152, 0))) is None
        assert refusal(paged(g, k=g.view_4d(k, 64, 2, 16, 9, 36, 90, 1080, 0))) is None
        assert refusal(paged(g, k=g.view_4d(k, 64, 2, 16, 9, 36, 81, 1080, 0)))
        assert refusal(paged(g, k=g.view_4d(k, 64, 2, 16, 9, 36, 72, 1170, 0)))
        assert refusal(paged(g, S=5000))


def test_verify_refuses_before_a_device():
    """Sequences, numbers and rows are looked at first, the backend after them."""
    import numpy as np

    with Graph(mem=1 << 20) as g:
        p, q = g.tensor(gl.F32, 100, 5), g.tensor(gl.F32, 100, 3)
        n, tok, u = np.array([2, 1], np.int32), np.array([1, 2, 3], np.int32), np.full(5, 0.5)
        for args in ((None, n, tok, u, q), (p, n, tok + 98, u, q), (p, n, tok, u + 0.5, q), (g.tensor(gl.F16, 100, 5), n, tok, u, q),
                     (q, n, tok, u, q), (p, n, tok, u, g.tensor(gl.F32, 99, 3)), (p, n, tok, u, g.tensor(gl.F32, 100, 2)), (p, n, tok, u, q)):
            with pytest.raises(RuntimeError):
                gl.hip_verify(None, *args[:4], draft_probs=args[4])
