"""Verification of drafted tokens on the HIP backend against float64 (serving_ref.verify): whole numbers, equal."""
import numpy as np
import pytest

import serving_ref as ref
from gl import Graph, gl

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    b = gl.hip_backend(0)
    yield b
    gl.libs()["core"].ggml_backend_free(b)


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def draw(rng, drafted, V, with_q=True, near=0.7):
    n, S = int(sum(drafted)), len(drafted)
    logits = 2.5 * rng.standard_normal((n + S, V))
    p = softmax(logits)
    of = np.concatenate([np.arange(k) + sum(drafted[:s]) + s for s, k in enumerate(drafted)]).astype(int)
    q = softmax(logits[of] + near * rng.standard_normal((n, V))) if n else np.zeros((0, V), np.float32)
    tokens = np.array([rng.choice(V, p=r / r.sum(dtype=np.float64)) for r in q.astype(np.float64)], np.int32).reshape(n)
    return dict(p=p, q=q if with_q and n else None, drafted=np.array(drafted, np.int32), tokens=tokens, u=rng.random(n + S))


def tensors(hip, d):
    g = Graph(mem=1 << 20)
    V = d["p"].shape[1]
    p = g.tensor(gl.F32, V, len(d["p"]), data=d["p"])
    q = None if d["q"] is None else g.tensor(gl.F32, V, len(d["q"]), data=d["q"])
    g.compute(hip, [])
    return g, p, q


def check(hip, d):
    g, p, q = tensors(hip, d)
    with g:
        got = gl.hip_verify(hip, p, d["drafted"], d["tokens"], d["u"], draft_probs=q)
        assert all(np.array_equal(a, b) for a, b in zip(got, gl.hip_verify(hip, p, d["drafted"], d["tokens"], d["u"], draft_probs=q)))
    want = ref.verify(d["p"], d["q"], d["drafted"], d["tokens"], d["u"])
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), (got, want)
    return got


@pytest.mark.parametrize("drafted, V", [
    ([0], 1), ([1], 1), ([0], 7), ([3], 100), ([4], 151936), ([2, 0, 5, 1], 2047), ([1, 1, 1], 2048), ([0, 8, 3], 2049),
    ([7] * 40, 5000), ([3, 4, 0, 0, 6, 2, 1, 5], 32064), ([300, 2], 64), ([1] * 300, 33), ([2, 1], 700001),
])
@pytest.mark.parametrize("with_q", [True, False])
def test_verify(hip, drafted, V, with_q):
    rng = np.random.default_rng(len(drafted) + V)
    for _ in range(3 if V < 10000 else 1):
        check(hip, draw(rng, drafted, V, with_q))


def test_verify_many_sequences_and_drafts(hip):
    """More than one launch's numbers hold."""
    check(hip, draw(np.random.default_rng(1), [1024] * 30 + [0, 5], 16))
    check(hip, draw(np.random.default_rng(2), [0, 1] * 2500, 8))
    d = draw(np.random.default_rng(3), [1] * 40, 4100, near=0.0)        # the draft's own distribution: all accepted
    assert (check(hip, d)[0] == 1).all()


def test_verify_draws_at_the_borders(hip):
    """Numbers at 0, just below 1 and at sums of weights; tokens without weight are never drawn."""
    V = 4099
    rng = np.random.default_rng(4)
    w = np.zeros(V, np.float32)
    on = np.sort(rng.permutation(V)[:64])
    w[on] = 2.0 ** -6                                                    # sums of these are exact
    us = [0.0, np.nextafter(1.0, 0.0)] + [k / 64 for k in range(64)] + [np.nextafter(k / 64, 0) for k in range(1, 64)]
    d = dict(p=np.tile(w, (len(us), 1)), q=None, drafted=np.zeros(len(us), np.int32), tokens=np.zeros(0, np.int32), u=np.array(us))
    got = check(hip, d)[1]
    assert np.array_equal(got[2:66], on) and np.array_equal(got[66:], on[:63]) and got[0] == on[0] and got[1] == on[63]


def test_verify_acceptance_at_the_borders(hip):
    """u q(x) equal to p(x) is not accepted, the next number below is; nothing is left where p is nowhere above q."""
    V = 50
    p = np.full((2 * 3, V), 0.0, np.float32)
    p[:, 10], p[:, 20] = 0.25, 0.75
    q = np.zeros((3, V), np.float32)
    q[:, 10], q[:, 20] = 0.5, 0.5
    tokens = np.array([10, 10, 20], np.int32)
    u = np.array([0.5, 0.3, np.nextafter(0.5, 0), 0.3, np.nextafter(1.0, 0), 0.1])
    got = check(hip, dict(p=p, q=q, drafted=np.array([1, 1, 1], np.int32), tokens=tokens, u=u))
    assert list(got[0]) == [0, 1, 1] and list(got[1]) == [20, 20, 10]
    p[0] = q[0] = 0
    p[0, 7], q[0, 7], q[0, 8] = 1.0, 1.0, 0.5
    tokens[0] = 8
    assert list(check(hip, dict(p=p, q=q, drafted=np.array([1, 1, 1], np.int32), tokens=tokens, u=u))[1])[0] == 7


def test_verify_rows_without_a_distribution(hip):
    V = 3000
    d = draw(np.random.default_rng(5), [2, 1, 0, 0, 1], V)
    d["p"][0, 2999] = np.nan
    d["u"][0] = 0.999999                                                # a draw from the row with the NaN
    d["p"][0, d["tokens"][0]] = 0
    d["p"][5] = 0
    d["p"][6, 5] = np.inf
    d["p"][7, d["tokens"][3]] = 0
    d["q"][3, 1] = np.nan
    got = check(hip, d)
    assert got[1][0] == got[1][2] == got[1][3] == got[1][4] == -1 and got[1][1] >= 0


def test_verify_follows_a_graph(hip):
    """Probabilities as a graph's soft_max leaves them, rows of a wider result; the call waits for it."""
    core = gl.libs()["core"]
    rng = np.random.default_rng(6)
    V, rows = 1000, 9
    x = rng.standard_normal((rows, V)).astype(np.float32)
    with Graph(mem=1 << 20) as g:
        p = g.soft_max_ext(g.tensor(gl.F32, V, rows, data=x), None, 2.0, 0.0)
        q = g.soft_max_ext(g.tensor(gl.F32, V, rows, data=x[::-1]), None, 1.0, 0.0)
        pv, qv = g.view_2d(p, 900, 7, V * 4, (V + 60) * 4), g.view_2d(q, 900, 5, V * 4, 2 * V * 4)
        gf = core.ggml_new_graph(g.ctx)
        for t in (pv, qv):
            core.ggml_set_output(t)
            core.ggml_build_forward_expand(gf, t)
        g.buf = core.ggml_backend_alloc_ctx_tensors(g.ctx, hip)
        for t, a in g.inputs:
            core.ggml_backend_tensor_set(t, a.ctypes.data, 0, a.nbytes)
        assert core.ggml_backend_graph_compute_async(hip, gf) == 0
        drafted, tokens, u = np.array([3, 2]), rng.integers(0, 900, 5), rng.random(7)
        got = gl.hip_verify(hip, pv, drafted, tokens, u, draft_probs=qv)
        pn, qn = g.read(p).reshape(rows, V)[1:8, 60:960], g.read(q).reshape(rows, V)[2:7, :900]
    want = ref.verify(pn, qn, drafted, tokens, u)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("V, off, pitch", [(2052, 0, 2052), (2052, 1, 2053), (2052, 2, 2056), (4096, 4, 4101), (4098, 4, 4104)])
def test_verify_rows_at_any_place(hip, V, off, pitch):
    """Rows at 16 bytes and elsewhere, in planes of two and four extents."""
    rng = np.random.default_rng(V + off)
    d = draw(rng, [3, 0, 2, 1, 2], V)
    with Graph(mem=1 << 20) as g:
        views = []
        for rows, planes in ((d["p"], (13, 1)), (d["q"], (2, 4))):
            wide = np.full((len(rows) * pitch + 8), np.nan, np.float32)
            wide[off:off + len(rows) * pitch].reshape(-1, pitch)[:, :V] = rows
            t = g.tensor(gl.F32, wide.size, data=wide)
            views.append(g.view_3d(t, V, *planes, pitch * 4, planes[0] * pitch * 4, off * 4))
        g.compute(hip, [])
        got = gl.hip_verify(hip, views[0], d["drafted"], d["tokens"], d["u"], draft_probs=views[1])
    want = ref.verify(d["p"], d["q"], d["drafted"], d["tokens"], d["u"])
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_verify_refuses(hip):
    d = draw(np.random.default_rng(7), [2, 1], 100)
    g, p, q = tensors(hip, d)
    with g:
        call = lambda p=p, q=q, **k: gl.hip_verify(hip, p, *(k.get(n, d[n]) for n in ("drafted", "tokens", "u")), draft_probs=q)  # noqa: E731
        call()
        for k in (dict(tokens=np.array([0, 100, 1])), dict(tokens=np.array([0, -1, 1])), dict(u=np.array([0.5, 1.0, 0.1, 0.1, 0.1])),
                  dict(u=np.array([0.5, np.nan, 0.1, 0.1, 0.1])), dict(u=np.array([0.5, -0.1, 0.1, 0.1, 0.1])), dict(p=q), dict(q=g.view_2d(q, 100, 2, 400, 0)),
                  dict(q=g.view_2d(q, 50, 3, 400, 0)), dict(drafted=np.array([2000, 1]), tokens=np.zeros(2001, int), u=np.zeros(2003))):
            with pytest.raises(RuntimeError):
                call(**k)
        for k in (dict(tokens=np.array([0, 1])), dict(u=np.zeros(4)), dict(drafted=np.array([-1, 4])), dict(tokens=np.array([0.5, 1, 1])),
                  dict(tokens=np.array([0, 2 ** 32, 1]))):
            with pytest.raises(ValueError):
                call(**k)
        call(p=p, q=None)
        none = gl.hip_verify(hip, p, np.zeros(0, int), np.zeros(0, int), np.zeros(0))
        assert len(none[0]) == len(none[1]) == 0
