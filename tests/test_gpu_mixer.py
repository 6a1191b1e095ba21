"""A small state space model on the HIP backend, as a user runs one: two sequences' prompt, then their
single tokens, states and the convolution's rows kept in caches that every graph updates in place,
scores of the tokens by ggml_backend_hip_logprobs.

Every operator is held to its own bound (ssm_ref, and test_gpu_logprobs.reference) on the inputs that
the run gave it, and every cache to what the run before left there, bit for bit."""
import numpy as np
import pytest

import ssm_ref
from gl import Graph, gl, ptr
from test_gpu_logprobs import U, reference
from test_gpu_ssm import near

pytestmark = pytest.mark.gpu

E, V, K, S, POOL = 64, 600, 4, 2, 3
# heads, channels a head, states, groups, one decay a head or a state's own
LAYERS = [(8, 16, 32, 2, 1), (128, 1, 16, 1, 16)]
IDS = np.array([2, 0], np.int32)


@pytest.fixture(scope="module")
def hip():
    b = gl.hip_backend(0)
    yield b
    gl.libs()["core"].ggml_backend_free(b)


class Model:
    """Weights and caches, in tensors of their own that the graphs share."""

    def __init__(self, backend, seed=1):
        rng = np.random.default_rng(seed)
        r = lambda *n: (rng.standard_normal(n) * 0.3).astype(np.float32)  # noqa: E731
        self.backend, self.g, self.v = backend, Graph(mem=1 << 20), {}
        self.t = {}
        self.put("embed", r(V, E), E, V)
        self.put("head", r(V, E), E, V)
        for i, (H, P, N, G, a0) in enumerate(LAYERS):
            D, W = H * P + 2 * G * N, 2 * H * P + 2 * G * N + H
            self.put(f"in{i}", r(W, E), E, W)
            self.put(f"out{i}", r(E, H * P), H * P, E)
            self.put(f"taps{i}", r(D, K), K, D)
            self.put(f"bias{i}", r(D), D)
            self.put(f"dt{i}", r(H) - 2, H)
            self.put(f"A{i}", -(0.5 + rng.random((H, a0))).astype(np.float32), a0, H)
            self.put(f"D{i}", r(H), 1, H)
            self.put(f"norm{i}", 1 + r(E), E)
            self.put(f"rows{i}", r(S, D, K - 1), K - 1, D, S)
            self.put(f"states{i}", r(POOL, H, P, N), N, P, H, POOL)
        self.put("ids", IDS, S, t=gl.I32)
        self.g.buf = self.g.core.ggml_backend_alloc_ctx_tensors(self.g.ctx, backend)
        for n in self.v:
            self.set(n, self.v[n])

    def put(self, name, value, *ne, t=None):
        self.v[name] = value
        self.t[name] = self.g.tensor(gl.F32 if t is None else t, *ne)

    def set(self, name, value):
        value = np.ascontiguousarray(value)
        self.g.core.ggml_backend_tensor_set(self.t[name], ptr(value), 0, value.nbytes)

    def cache(self, i):
        H, P, N, G, _ = LAYERS[i]
        return (self.g.read(self.t[f"rows{i}"]).reshape(S, -1, K - 1), self.g.read(self.t[f"states{i}"]).reshape(POOL, H, P, N))

    def build(self, g, T, tokens):
        """The graph's outputs: the logits, per layer what went in and came out of its operators, the caches' writes."""
        t, outs, writes = self.t, [], []
        h = g.reshape_3d(g.get_rows(t["embed"], tokens), E, T, S)
        for i, (H, P, N, G, a0) in enumerate(LAYERS):
            X, D = H * P, H * P + 2 * G * N
            W = D + X + H
            row = g.mul_mat(t[f"in{i}"], g.mul(g.rms_norm(h, 1e-5), t[f"norm{i}"]))       # gate, convolved, time steps
            nb = lambda a, n: (row, n, T, S, W * 4, T * W * 4, a * 4)  # noqa: E731
            z, xbc, dt = g.view_3d(*nb(0, X)), g.view_3d(*nb(X, D)), g.view_3d(*nb(X + D, H))
            joined = g.concat(t[f"rows{i}"], g.transpose(xbc), 0)
            jb = joined.contents.nb
            keep = g.cpy(g.view_3d(joined, K - 1, D, S, jb[1], jb[2], T * 4), t[f"rows{i}"])
            y = g.silu(g.add(g.ssm_conv(joined, t[f"taps{i}"]), t[f"bias{i}"]))
            x = g.view_4d(y, P, H, T, S, P * 4, D * 4, T * D * 4, 0)
            B, C = (g.view_4d(y, N, G, T, S, N * 4, D * 4, T * D * 4, a * 4) for a in (X, X + G * N))
            dt = g.add(dt, t[f"dt{i}"])
            scan = g.ssm_scan(t[f"states{i}"], x, dt, t[f"A{i}"], B, C, t["ids"], 1)
            one = N * P * H * 4
            states = []
            for s in range(S):
                new = g.view_3d(scan, N, P, H, N * 4, N * P * 4, X * T * S * 4 + s * one)
                states.append(g.cpy(new, g.view_3d(t[f"states{i}"], N, P, H, N * 4, N * P * 4, int(IDS[s]) * one)))
            out = g.add(g.view_4d(scan, P, H, T, S, P * 4, X * 4, T * X * 4, 0), g.mul(x, t[f"D{i}"]))
            gated = g.mul(g.reshape_3d(out, X, T, S), g.silu(g.cont_3d(z, X, T, S)))
            h = g.add(h, g.mul_mat(t[f"out{i}"], gated))
            outs += [row, y, dt, scan]
            writes += [keep] + states
        return [g.mul_mat(t["head"], h)] + outs, writes

    def check(self, T, before, outs):
        """Each layer's operators on what they were given, and the caches after them."""
        for i, (H, P, N, G, a0) in enumerate(LAYERS):
            X, D = H * P, H * P + 2 * G * N
            row, y, dt, scan = outs[4 * i:4 * i + 4]
            rows, states = before[i]
            new_rows, new_states = self.cache(i)
            xbc = row.reshape(S, T, -1)[:, :, X:X + D]
            joined = np.concatenate([rows, xbc.transpose(0, 2, 1)], 2)
            near(y, *ssm_ref.conv(joined, self.v[f"taps{i}"], self.v[f"bias{i}"], True), ("conv", i))
            assert np.array_equal(new_rows, joined[:, :, T:])
            y = y.reshape(S, T, D)
            part = lambda a, *n: y[:, :, a:a + int(np.prod(n))].reshape(S, T, *n)  # noqa: E731
            wy, wh, ye, he = ssm_ref.scan(states[IDS], part(0, H, P), dt.reshape(S, T, H), self.v[f"A{i}"],
                                          part(X, G, N), part(X + G * N, G, N))
            near(scan[:wy.size], wy, ye, ("scan", i))
            near(scan[wy.size:], wh, he, ("state", i))
            want = states.copy()
            want[IDS] = scan[wy.size:].reshape(wh.shape)
            assert np.array_equal(new_states, want)

    def step(self, tokens, n_top=5):
        """tokens [S, T]: their rows' logits and scores (of the tokens that follow), everything checked."""
        T = tokens.shape[1]
        before = [self.cache(i) for i in range(len(LAYERS))]
        with Graph(mem=4 << 20) as g:
            outs, writes = self.build(g, T, g.tensor(gl.I32, S * T, data=tokens.astype(np.int32).ravel()))
            got = g.compute(self.backend, outs + writes)
            self.check(T, before, got[1:])
            follow = (np.arange(S * T, dtype=np.int32) * 7) % V
            lp, ent, ids, top = gl.hip_logprobs(self.backend, outs[0], follow, n_top=n_top)
        logits = got[0].reshape(S * T, V)
        wlp, went, order = reference(logits)
        bound = (V / 256 + 24 + 4 * np.log(V)) * U
        at = np.arange(S * T)
        size = np.abs(logits).max()
        assert (np.abs(lp - wlp[at, follow]) <= bound * (1 + 2 * size + np.abs(wlp[at, follow]))).all()
        assert (np.abs(ent - went) <= bound * (1 + np.log(V)) * (1 + 2 * size)).all()
        assert np.array_equal(ids, order[:, :n_top])
        return logits.reshape(S, T, V)

    def close(self):
        self.g.close()


@pytest.mark.parametrize("fusion", [True, False])
def test_prompt_then_tokens(hip, fusion):
    tokens = np.random.default_rng(3).integers(0, V, (S, 75 + 3 + 30))
    gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, fusion)
    m = Model(hip)
    try:
        at = 0
        for T in (75, 1, 1, 1, 30):
            m.step(tokens[:, at:at + T])
            at += T
    finally:
        gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, True)
        m.close()


def test_one_graph_over_and_over(hip):
    """A step's graph is built once and run again for every token, through each way to run it: the
    caches advance, the results are those of graphs built anew."""
    tokens = np.random.default_rng(4).integers(0, V, (6, S)).astype(np.int32)
    L = gl.libs()
    runs = {}
    for way in ("anew", "compute", "async", "static"):
        m = Model(hip)
        runs[way] = []
        if way == "anew":
            for t in tokens:
                runs[way].append(m.step(t[:, None]).ravel())
        else:
            with Graph(mem=4 << 20) as g:
                toks = g.tensor(gl.I32, S)
                outs, writes = m.build(g, 1, toks)
                gf = g.core.ggml_new_graph(g.ctx)
                g.core.ggml_set_output(outs[0])
                for o in [outs[0]] + writes:
                    g.core.ggml_build_forward_expand(gf, o)
                g.buf = g.core.ggml_backend_alloc_ctx_tensors(g.ctx, hip)
                for t in tokens:
                    g.core.ggml_backend_tensor_set(toks, ptr(t), 0, t.nbytes)
                    run = {"compute": g.core.ggml_backend_graph_compute, "async": g.core.ggml_backend_graph_compute_async,
                           "static": L["hip"].ggml_backend_hip_graph_compute_static}[way]
                    assert run(hip, gf) == 0
                    lp, ent, ids, top = gl.hip_logprobs(hip, outs[0], t, n_top=3)       # waits for the stream
                    logits = g.read(outs[0])
                    assert np.array_equal(ids, reference(logits.reshape(S, V))[2][:, :3])
                    runs[way].append(logits)
        runs[way] += [a for i in range(len(LAYERS)) for a in m.cache(i)]
        m.close()
    for way in ("compute", "async", "static"):
        for a, b in zip(runs[way], runs["anew"]):
            assert np.array_equal(a, b), way


def test_two_backends(hip):
    """Two backends of one device, each with a model of its own, their graphs in turn."""
    other = gl.hip_backend(0)
    tokens = np.random.default_rng(5).integers(0, V, (S, 80))
    a, b = Model(hip, 1), Model(other, 2)
    try:
        for at, T in ((0, 78), (78, 1), (79, 1)):
            a.step(tokens[:, at:at + T])
            b.step(tokens[::-1, at:at + T])
    finally:
        a.close()
        b.close()
        gl.libs()["core"].ggml_backend_free(other)
