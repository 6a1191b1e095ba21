"""The operators of a paged cache together, as a server's steps use them on the HIP backend: rows of a projection
rotated by positions of several axes, keys and values appended to a 4-bit cache on pages, attention over it,
probabilities, and drafted tokens accepted or replaced."""
import numpy as np
import pytest

import serving_ref as ref
from gl import Graph, dequantize, gl, quantize, ptr
from test_gpu_rows import multi, raw

pytestmark = pytest.mark.gpu

D, H, KV, P, PAGES, V, S, MOST = 64, 6, 2, 8, 24, 50, 3, 9
SECTIONS, W = (8, 12, 12, 0), (H + 2 * KV) * D


@pytest.fixture(scope="module")
def hip():
    b = gl.hip_backend(0)
    yield b
    gl.libs()["core"].ggml_backend_free(b)


class Model:
    """Weights, and a cache in device memory that outlives the steps' graphs."""

    def __init__(self, hip, rng):
        self.hip, self.g = hip, Graph(mem=1 << 20)
        self.table = rng.standard_normal((V, W)).astype(np.float32)
        self.head = (0.15 * rng.standard_normal((V, H * D))).astype(np.float32)
        self.pages = rng.permutation(PAGES)[:S * 8].reshape(S, 8).astype(np.int32)
        empty = np.zeros((PAGES * P, KV * D), np.float32)
        self.t_table, self.t_head = self.g.tensor(gl.F32, W, V, data=self.table), self.g.tensor(gl.F32, H * D, V, data=self.head)
        self.k, self.v = (self.g.tensor(gl.Q4_0, KV * D, PAGES * P, data=quantize(empty, gl.Q4_0)) for _ in "kv")
        self.g.compute(hip, [])

    def cache(self, t):
        return dequantize(raw(self.g, t), gl.Q4_0, PAGES * P * KV * D).reshape(PAGES, P, KV, D)

    def step(self, tokens, new, seen, static, pad=1):
        """Tokens of every sequence behind its `seen` positions; a place behind the last stands idle."""
        T = int(sum(new)) + pad
        where = [(s, seen[s] + i) for s in range(S) for i in range(new[s])]
        pos = np.zeros((4, T), np.int32)
        pos[:3, :len(where)] = [[p // 3 * a + p for _, p in where] for a in range(3)]
        idx = np.full(T, -1, np.int64)
        idx[:len(where)] = [self.pages[s, p // P] * P + p % P for s, p in where]
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        length = np.array([seen[s] + new[s] for s in range(S)], np.int32)
        g = Graph(mem=1 << 20)
        rows = g.get_rows(self.t_table, g.tensor(gl.I32, T, data=np.array(list(tokens) + [0] * pad, np.int32)))
        at = g.tensor(gl.I32, 4 * T, data=pos)
        to = g.tensor(gl.I64, T, data=idx)
        view = lambda n, head: g.view_3d(rows, D, n, T, D * 4, W * 4, head * D * 4)  # noqa: E731
        q, k = (multi(g, view(n, h), at, D, SECTIONS, ref.MROPE) for n, h in ((H, 0), (KV, H)))
        ks = g.set_rows(self.k, g.reshape_2d(k, KV * D, T), to)
        vs = g.set_rows(self.v, g.view_2d(rows, KV * D, T, W * 4, (H + KV) * D * 4), to)
        o = g.flash_attn_paged(q, g.reshape_4d(ks, D, KV, P, PAGES), g.reshape_4d(vs, D, KV, P, PAGES),
                               g.tensor(gl.I32, 8, S, data=self.pages), g.tensor(gl.I32, S + 1, data=start),
                               g.tensor(gl.I32, S, data=length), D ** -0.5)
        probs = g.soft_max_ext(g.mul_mat(self.t_head, g.reshape_2d(o, H * D, T)), None, 1.0, 0.0)
        core, gf = g.core, g.core.ggml_new_graph(g.ctx)
        for t in (q, o, probs):
            core.ggml_set_output(t)
        core.ggml_build_forward_expand(gf, probs)
        g.buf = core.ggml_backend_alloc_ctx_tensors(g.ctx, self.hip)
        for t, a in g.inputs:
            core.ggml_backend_tensor_set(t, ptr(a), 0, a.nbytes)
        run = gl.libs()["hip"].ggml_backend_hip_graph_compute_static if static else core.ggml_backend_graph_compute
        assert run(self.hip, gf) == 0
        d = dict(T=T, q=g.read(q).reshape(T, H, D), o=g.read(o).reshape(T, H, D), pos=pos, idx=idx, start=start, seen=length, x=self.table[tokens])
        return g, probs, d

    def check(self, d):
        n = len(d["x"])
        x = d["x"].reshape(n, H + 2 * KV, D)
        want, bound = ref.rope(x[:, :H], d["pos"][:, :n], D, SECTIONS, ref.MROPE, 1e6)
        assert (np.abs(d["q"][:n] - want) <= bound).all()
        k, v = self.cache(self.k), self.cache(self.v)
        want, _ = ref.rope(x[:, H:H + KV], d["pos"][:, :n], D, SECTIONS, ref.MROPE, 1e6)
        at = d["idx"][:n]
        for got, rows in ((k, want), (v, x[:, H + KV:].astype(np.float64))):
            blocks = rows.reshape(n, KV, D // 32, 32)
            # a code stands for a step of the largest value over 8, the last one for it and what lies beyond it (one step
            # at most): a value is off by a step, and the scale's rounding, 8 codes of 2^-11
            off = np.abs(got.reshape(-1, KV, D // 32, 32)[at] - blocks)
            assert (off <= np.abs(blocks).max(-1, keepdims=True) / 8 * (1 + 8 * 2.0 ** -11) + 1e-6).all()
        want, bound, listed = ref.attention(d["q"], k, v, self.pages, d["start"], d["seen"], D ** -0.5)
        assert (np.abs(d["o"] - want)[listed] <= bound[listed]).all() and listed.sum() == n


def serve(hip, seed, static=False, fusion=True):
    """A prompt each, two steps with drafts, a step of single tokens; what is drafted and refused is written over."""
    rng = np.random.default_rng(seed)
    m = Model(hip, rng)
    gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, fusion)
    seen, last, history = np.zeros(S, int), rng.integers(0, V, S), []
    try:
        for new, drafts in (((19, 1, 6), False), ((4, 1, 3), True), ((2, 6, 4), True), ((1, 1, 1), True)):
            tokens = rng.integers(0, V, sum(new))
            start = np.concatenate([[0], np.cumsum(new)])
            tokens[start[:-1]] = last
            g, probs, d = m.step(tokens, new, seen, static)
            with g:
                m.check(d)
                p = g.read(probs).reshape(d["T"], V)
                if drafts:
                    drafted = np.array(new, np.int32) - 1
                    ids = np.concatenate([tokens[start[s] + 1:start[s + 1]] for s in range(S)]).astype(np.int32)
                    q, u = np.full((max(len(ids), 1), V), 1.0 / V, np.float32), rng.random(sum(new))
                    with Graph(mem=1 << 20) as gq:
                        tq = gq.tensor(gl.F32, V, len(q), data=q)
                        gq.compute(hip, [])
                        accepted, last = gl.hip_verify(hip, probs, drafted, ids, u, draft_probs=tq)
                    want = ref.verify(p, q, drafted, ids, u)
                    assert np.array_equal(accepted, want[0]) and np.array_equal(last, want[1])
                    seen = seen + 1 + accepted
                else:
                    with Graph(mem=1 << 20) as gv:
                        rows = gv.get_rows(probs, gv.tensor(gl.I32, S, data=(start[1:] - 1).astype(np.int32)))
                        gv.compute(hip, rows)
                        u = rng.random(S)
                        accepted, last = gl.hip_verify(hip, rows, np.zeros(S, np.int32), np.zeros(0, np.int32), u)
                    assert np.array_equal(last, ref.verify(p[start[1:] - 1], None, np.zeros(S, int), [], u)[1])
                    seen = seen + np.array(new)
                history += [d["q"][:sum(new)], d["o"][:sum(new)], p[:sum(new)], accepted, last]
        history += [raw(m.g, m.k), raw(m.g, m.v)]
    finally:
        gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, True)
        m.g.close()
    return history


@pytest.mark.parametrize("seed", range(3))
def test_serving_steps(hip, seed):
    """Each step against float64; the same bits without fusion (attention and appends) and from the static scratch."""
    first = serve(hip, seed)
    for again in (serve(hip, seed), serve(hip, seed, static=True), serve(hip, seed, fusion=False)):
        assert all(np.array_equal(a, b) for a, b in zip(first, again))
