"""Rotations of several axes and rows stored by index, on the HIP backend: against float64 (serving_ref), and the
quantized rows against the oracle's quantizers bit for bit."""
import ctypes as C

import numpy as np
import pytest

import serving_ref as ref
from gl import Graph, gl, quantize

pytestmark = pytest.mark.gpu

NP = {gl.F32: np.float32, gl.F16: np.float16}


@pytest.fixture(scope="module")
def hip():
    b = gl.hip_backend(0)
    yield b
    gl.libs()["core"].ggml_backend_free(b)


def multi(g, x, pos, n_dims, sections, mode, base=1e6, freq_scale=1.0, ext=0.0, attn=1.0, n_ctx_orig=0, ff=None):
    return g.rope_multi(x, pos, ff, n_dims, (C.c_int * 4)(*sections), mode, n_ctx_orig, base, freq_scale, ext, attn, 32.0, 1.0)


def positions(rng, T, most=100000):
    return rng.integers(0, most, (4, T)).astype(np.int32)


def near(got, want, bound):
    off = np.abs(got.reshape(want.shape).astype(np.float64) - want)
    assert (off <= bound).all(), (off - bound).max()


@pytest.mark.parametrize("T, H, D, n_dims, sections, mode", [
    (1, 1, 2, 2, (1, 0, 0, 0), ref.MROPE), (1, 32, 128, 128, (16, 24, 24, 0), ref.MROPE), (7, 3, 64, 64, (8, 12, 12, 0), ref.MROPE),
    (33, 5, 96, 96, (24, 20, 4, 0), ref.MROPE), (40, 2, 128, 64, (8, 12, 6, 6), ref.MROPE), (5, 4, 80, 80, (3, 5, 2, 1), ref.MROPE),
    (17, 4, 80, 40, (20, 20, 0, 0), ref.VISION), (9, 16, 64, 32, (16, 16, 0, 0), ref.VISION), (3, 2, 36, 18, (5, 4, 5, 4), ref.VISION),
    (16, 32, 128, 128, (24, 20, 20, 0), ref.IMROPE), (3, 1, 100, 84, (10, 9, 8, 0), ref.IMROPE), (2, 3, 22, 10, (1, 1, 1, 0), ref.IMROPE),
    (300, 9, 128, 128, (16, 24, 24, 0), ref.MROPE), (2, 40, 256, 256, (40, 44, 44, 0), ref.MROPE), (0, 4, 64, 64, (32, 0, 0, 0), ref.MROPE),
])
def test_rope_multi(hip, T, H, D, n_dims, sections, mode):
    rng = np.random.default_rng(T + 10 * H + D)
    x, pos = rng.standard_normal((T, H, D)).astype(np.float32), positions(rng, T)
    with Graph(mem=1 << 20) as g:
        y = g.compute(hip, multi(g, g.tensor(gl.F32, D, H, T, data=x), g.tensor(gl.I32, 4 * T, data=pos), n_dims, sections, mode))
    near(y, *ref.rope(x, pos, n_dims, sections, mode, 1e6))


def test_rope_multi_far_positions(hip):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((8, 2, 64)).astype(np.float32)
    pos = np.array([[2 ** 31 - 1, 10 ** 9, -5, -10 ** 9, 0, 1, 2 ** 24 + 1, 123456789]] * 4, np.int32)
    with Graph(mem=1 << 20) as g:
        y = g.compute(hip, multi(g, g.tensor(gl.F32, 64, 2, 8, data=x), g.tensor(gl.I32, 32, data=pos), 64, (32, 0, 0, 0), ref.MROPE, base=1e4))
    near(y, *ref.rope(x, pos, 64, (32, 0, 0, 0), ref.MROPE, 1e4))


@pytest.mark.parametrize("kw", [dict(freq_scale=0.25), dict(freq_scale=0.25, ext=1.0, n_ctx_orig=4096), dict(attn=1.5),
                                dict(freq_scale=0.5, ext=0.4, attn=0.8, n_ctx_orig=2048)])
@pytest.mark.parametrize("factors", [False, True])
def test_rope_multi_scaling(hip, kw, factors):
    rng = np.random.default_rng(4)
    T, H, D, sections = 11, 3, 128, (16, 24, 24, 0)
    x, pos = rng.standard_normal((T, H, D)).astype(np.float32), positions(rng, T)
    ff = (1 + 3 * rng.random(64)).astype(np.float32) if factors else None
    with Graph(mem=1 << 20) as g:
        c = g.tensor(gl.F32, 64, data=ff) if factors else None
        y = g.compute(hip, multi(g, g.tensor(gl.F32, D, H, T, data=x), g.tensor(gl.I32, 4 * T, data=pos), D, sections, ref.MROPE,
                                 base=1e4, ff=c, **kw))
    near(y, *ref.rope(x, pos, D, sections, ref.MROPE, 1e4, ff=ff, **kw))


def test_rope_multi_slices_and_batches(hip):
    """Heads of a wider projection, and a fourth extent that shares the positions."""
    rng = np.random.default_rng(5)
    B, T, H, D, W = 3, 6, 2, 64, 64 * 5 + 4
    x, pos = rng.standard_normal((B, T, W)).astype(np.float32), positions(rng, T)
    with Graph(mem=1 << 20) as g:
        t = g.tensor(gl.F32, W, T, B, data=x)
        v = g.view_4d(t, D, H, T, B, D * 4, W * 4, T * W * 4, 68 * 4)
        y = g.compute(hip, multi(g, v, g.tensor(gl.I32, 4 * T, data=pos), D, (8, 12, 12, 0), ref.MROPE)).reshape(B, T, H, D)
    for b in range(B):
        near(y[b], *ref.rope(x[b, :, 68:68 + H * D].reshape(T, H, D), pos, D, (8, 12, 12, 0), ref.MROPE, 1e6))


def stored(x, type):
    if type in NP:
        return x.astype(NP[type])
    if type == gl.BF16:
        u = x.view(np.uint32)
        return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return quantize(x, type).reshape(len(x), -1)


def raw(g, t):
    return g.read(t, np.uint8)


def expected(cache, x, idx, type):
    """cache [rows, bytes]"""
    for r, at in enumerate(idx):
        if 0 <= at < len(cache):
            cache[at] = stored(x[r:r + 1], type).reshape(-1).view(np.uint8)
    return cache


def row_bytes(type, n):
    return gl.libs()["core"].ggml_row_size(type, n)


@pytest.mark.parametrize("type", [gl.F32, gl.F16, gl.BF16, gl.Q8_0, gl.Q4_0])
@pytest.mark.parametrize("n, width, rows, it", [
    (1, 32, 1, np.int32), (1, 1024, 40, np.int64), (5, 64, 9, np.int32), (70, 96, 200, np.int64), (33, 2048, 64, np.int32),
    (300, 160, 500, np.int32), (0, 64, 4, np.int32), (9000, 32, 10000, np.int32),
])
def test_set_rows(hip, type, n, width, rows, it):
    rng = np.random.default_rng(n + width)
    x = (rng.standard_normal((n, width)) * np.exp(rng.standard_normal((n, 1)))).astype(np.float32)
    idx = rng.permutation(rows)[:n].astype(it)
    fill = stored(rng.standard_normal((rows, width)).astype(np.float32), type)
    with Graph(mem=1 << 20) as g:
        a = g.tensor(type, width, rows, data=fill)
        b, c = g.tensor(gl.F32, width, n, data=x), g.tensor(gl.I32 if it == np.int32 else gl.I64, n, data=idx)
        out = g.set_rows(a, b, c)
        g.compute(hip, out)
        got = raw(g, a)
        assert np.array_equal(got, raw(g, out))
    want = expected(np.ascontiguousarray(fill).view(np.uint8).reshape(rows, row_bytes(type, width)).copy(), x, idx, type)
    assert np.array_equal(got, want.ravel())


@pytest.mark.parametrize("width", [1, 3, 5, 33, 1027])
def test_set_rows_odd_widths(hip, width):
    rng = np.random.default_rng(width)
    x, idx = rng.standard_normal((6, width)).astype(np.float32), np.array([4, 0, 9, 2, 7, 5], np.int32)
    for type in (gl.F32, gl.F16):
        with Graph(mem=1 << 20) as g:
            a = g.tensor(type, width, 11, data=np.zeros((11, width), NP[type]))
            g.compute(hip, g.set_rows(a, g.tensor(gl.F32, width, 6, data=x), g.tensor(gl.I32, 6, data=idx)))
            got = g.read(a, NP[type]).reshape(11, width)
        want = np.zeros((11, width), NP[type])
        want[idx] = x
        assert np.array_equal(got, want)


@pytest.mark.parametrize("type", [gl.F16, gl.Q4_0])
@pytest.mark.parametrize("n, width", [(8, 64), (200, 256), (700, 64), (20000, 32)])
def test_set_rows_same_index_and_none(hip, type, n, width):
    """Of rows with one index the last is stored, across passes too; others (a page that is not there) are not."""
    rng = np.random.default_rng(n)
    rows = n // 3 + 2
    x = rng.standard_normal((n, width)).astype(np.float32)
    idx = rng.integers(-2, rows + 2, n).astype(np.int64)
    idx[:2], idx[-1] = (-2 ** 40, 2 ** 40), idx[3]
    fill = stored(rng.standard_normal((rows, width)).astype(np.float32), type)
    with Graph(mem=1 << 20) as g:
        a = g.tensor(type, width, rows, data=fill)
        g.compute(hip, g.set_rows(a, g.tensor(gl.F32, width, n, data=x), g.tensor(gl.I64, n, data=idx)))
        got = raw(g, a)
    want = expected(np.ascontiguousarray(fill).view(np.uint8).reshape(rows, -1).copy(), x, idx, type)
    assert np.array_equal(got, want.ravel())


def test_set_rows_values_at_the_edges(hip):
    """Zeros, ties of magnitude, tiny and huge blocks as the quantizer has them; a NaN makes its block's scale one."""
    x = np.zeros((8, 64), np.float32)
    x[1, :32] = np.where(np.arange(32) % 2, 1, -1)
    x[2] = 1e-42
    x[3] = 3e6
    x[4, 5], x[4, 40] = -7, 7
    x[5] = np.linspace(-1, 1, 64)
    x[6, 33] = np.nan
    for type in (gl.Q4_0, gl.Q8_0):
        with Graph(mem=1 << 20) as g:
            a = g.tensor(type, 64, 8)
            g.compute(hip, g.set_rows(a, g.tensor(gl.F32, 64, 8, data=x), g.tensor(gl.I32, 8, data=np.arange(8, dtype=np.int32))))
            got = raw(g, a).reshape(8, 2, -1)
        want = stored(np.nan_to_num(x), type).reshape(8, 2, -1)
        assert np.array_equal(got[[0, 1, 4, 5, 7]], want[[0, 1, 4, 5, 7]])
        assert np.array_equal(got[[2, 3]][..., :2], want[[2, 3]][..., :2])       # scales of 0 and of infinity
        assert np.array_equal(got[6, 0], want[6, 0])
        assert np.isnan(got[6, 1, :2].copy().view(np.float16)).all()


def test_set_rows_third_and_fourth_extents(hip):
    rng = np.random.default_rng(6)
    n2, n3, n, width, rows = 4, 6, 5, 64, 9
    x = rng.standard_normal((n3, n2, n, width)).astype(np.float32)
    idx = np.stack([rng.permutation(rows)[:n] for _ in range(6)]).reshape(3, 2, n).astype(np.int32)
    for type in (gl.F16, gl.Q4_0):
        bytes_ = row_bytes(type, width)
        with Graph(mem=1 << 20) as g:
            a = g.tensor(type, width, rows, n2, n3, data=np.zeros((n3, n2, rows, bytes_), np.uint8))
            g.compute(hip, g.set_rows(a, g.tensor(gl.F32, width, n, n2, n3, data=x), g.tensor(gl.I32, n, 2, 3, data=idx)))
            got = raw(g, a).reshape(n3, n2, rows, bytes_)
        for i3 in range(n3):
            for i2 in range(n2):
                want = expected(np.zeros((rows, bytes_), np.uint8), x[i3, i2], idx[i3 % 3, i2 % 2], type)
                assert np.array_equal(got[i3, i2], want), (type, i3, i2)


@pytest.mark.parametrize("type", [gl.F16, gl.Q4_0])
def test_set_rows_into_a_view(hip, type):
    """A cache inside a larger one, its rows apart; what lies between keeps its values."""
    rng = np.random.default_rng(7)
    x, idx = rng.standard_normal((3, 64)).astype(np.float32), np.array([4, 0, 2], np.int32)
    rb = row_bytes(type, 32)
    fill = stored(rng.standard_normal((40, 32)).astype(np.float32), type)
    with Graph(mem=1 << 20) as g:
        base = g.tensor(type, 32, 40, data=fill)
        a = g.view_2d(base, 64, 5, 7 * rb, 3 * rb)
        g.compute(hip, g.set_rows(a, g.tensor(gl.F32, 64, 3, data=x), g.tensor(gl.I32, 3, data=idx)))
        got = raw(g, base).reshape(40, rb)
    want = np.ascontiguousarray(fill).view(np.uint8).reshape(40, rb).copy()
    for r, at in enumerate(idx):
        want[3 + 7 * at:5 + 7 * at] = stored(x[r:r + 1], type).reshape(-1).view(np.uint8).reshape(2, rb)
    assert np.array_equal(got, want)


def test_set_rows_refuses_shared_memory(hip):
    with Graph(mem=1 << 20) as g:
        a = g.tensor(gl.F32, 64, 10, data=np.zeros((10, 64), np.float32))
        n = g.set_rows(g.view_2d(a, 64, 6, 256, 0), g.view_2d(a, 64, 3, 256, 5 * 256), g.tensor(gl.I32, 3, data=np.arange(3, dtype=np.int32)))
        with pytest.raises(AssertionError):
            g.compute(hip, n)


# ---- appends: keys rotated on the way ----
def append_graph(g, d, type, rotate, outputs):
    T, KV, D, W = d["T"], d["KV"], d["D"], d["W"]
    rows = g.tensor(gl.F32, W, T, data=d["x"])
    pos = g.tensor(gl.I32, d["pos"].size, data=d["pos"])
    idx = g.tensor(gl.I32, T, data=d["idx"])
    kc, vc = (g.tensor(type, KV * D, d["rows"], data=d["fill"]) for _ in "kv")
    view = lambda n, at: g.view_3d(rows, D, n, T, D * 4, W * 4, at * 4)  # noqa: E731
    q = rotate(g, view(2 * KV, 0), pos)
    k = rotate(g, view(KV, 2 * KV * D), pos)
    ks = g.set_rows(kc, g.reshape_2d(k, KV * D, T), idx)
    vs = g.set_rows(vc, g.view_2d(rows, KV * D, T, W * 4, 3 * KV * D * 4), idx)
    outs = [q, ks, vs] + ([k] if outputs else [])
    return outs, kc, vc


@pytest.mark.parametrize("type", [gl.F32, gl.F16, gl.Q8_0, gl.Q4_0])
@pytest.mark.parametrize("how", ["several", "neox", "normal", "partly"])
@pytest.mark.parametrize("T, KV, D", [(1, 8, 128), (5, 2, 64), (40, 3, 96)])
def test_append_as_the_operators_one_by_one(hip, type, how, T, KV, D):
    """Fused, the keys go into the cache unwritten elsewhere; the bits are those of a rotation and a set_rows."""
    rng = np.random.default_rng(T + KV)
    W, rows = 4 * KV * D + 8, 3 * T + 4
    d = dict(T=T, KV=KV, D=D, W=W, rows=rows, x=rng.standard_normal((T, W)).astype(np.float32),
             pos=positions(rng, T) if how == "several" else rng.integers(0, 5000, T).astype(np.int32),
             idx=rng.permutation(rows)[:T].astype(np.int32),
             fill=stored(rng.standard_normal((rows, KV * D)).astype(np.float32), type))
    if T > 4:
        d["idx"][2] = -1

    def rotate(g, x, pos):
        if how == "several":
            h = D // 2
            return multi(g, x, pos, D, (h // 4, h // 2, h - h // 4 - h // 2, 0), ref.MROPE)
        mode = gl.ROPE_NORMAL if how == "normal" else gl.ROPE_NEOX
        return g.rope_ext(x, pos, None, D // 2 if how == "partly" else D, mode, 0, 1e4, 1.0, 0.0, 1.0, 32.0, 1.0)

    got = []
    for fused in (True, False):
        gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, fused)
        with Graph(mem=1 << 20) as g:
            outs, kc, vc = append_graph(g, d, type, rotate, not fused)
            res = g.compute(hip, outs)
            got.append((res[0], raw(g, kc), raw(g, vc), None if fused else res[3]))
    gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, True)
    for a, b in zip(got[0][:3], got[1][:3]):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    cache = np.ascontiguousarray(d["fill"]).view(np.uint8).reshape(rows, -1)
    assert np.array_equal(got[0][1], expected(cache.copy(), got[1][3].reshape(T, KV * D), d["idx"], type).ravel())
    assert np.array_equal(got[0][2], expected(cache.copy(), np.ascontiguousarray(d["x"][:, 3 * KV * D:4 * KV * D]), d["idx"], type).ravel())


def test_append_in_order_with_what_reads_the_cache(hip):
    """A reader of the cache between the rotation and its set_rows sees the cache as it was; one behind it, as it is;
    two appends to one cache keep their order."""
    rng = np.random.default_rng(8)
    x, fill = rng.standard_normal((4, 2, 64)).astype(np.float32), rng.standard_normal((6, 128)).astype(np.float32)
    pos, idx = positions(rng, 4), np.array([3, 1, 0, 5], np.int32)
    with Graph(mem=1 << 20) as g:
        a, p, c = g.tensor(gl.F32, 64, 2, 4, data=x), g.tensor(gl.I32, 16, data=pos), g.tensor(gl.I32, 4, data=idx)
        cache = g.tensor(gl.F32, 128, 6, data=fill)
        k = multi(g, a, p, 64, (8, 12, 12, 0), ref.MROPE)
        g.core.ggml_set_output(k)
        before = g.scale(cache, 1.0)
        s1 = g.set_rows(cache, g.reshape_2d(k, 128, 4), c)
        s2 = g.set_rows(s1, g.reshape_2d(a, 128, 4), g.tensor(gl.I32, 4, data=np.array([0, 2, 3, 4], np.int32)))
        after = g.scale(s2, 1.0)
        got = g.compute(hip, [k, before, s1, s2, after])
    want = fill.copy()
    want[idx] = got[0].reshape(4, 128)
    want[[0, 2, 3, 4]] = x.reshape(4, 128)
    assert np.array_equal(got[1], fill.ravel())
    assert np.array_equal(got[4], want.ravel())


@pytest.mark.parametrize("how", ["several", "neox", "normal"])
@pytest.mark.parametrize("T, KV, D, moved", [(60, 2, 64, True), (300, 8, 128, True), (5, 30, 96, False), (40, 17, 96, False), (3, 24, 80, True)])
def test_rows_of_the_cache_itself(hip, how, T, KV, D, moved):
    """A cache's rows turned further and stored in it again, moved or where they were (heads across the border of what a
    workgroup reads): bits as without fusion, and all rows read before one is stored."""
    rng = np.random.default_rng(T + KV)
    rows, W = T + 7, KV * D
    fill, pos = rng.standard_normal((rows, W)).astype(np.float32), positions(rng, T, 5000)
    idx = (rng.permutation(rows)[:T] if moved else np.arange(3, T + 3)).astype(np.int64)
    got = []
    for fused in (True, False):
        gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, fused)
        with Graph(mem=1 << 20) as g:
            cache = g.tensor(gl.F32, W, rows, data=fill)
            x = g.view_3d(cache, D, KV, T, D * 4, W * 4, 3 * W * 4)
            if how == "several":
                k = multi(g, x, g.tensor(gl.I32, 4 * T, data=pos), D, (D // 8, D // 8, D // 4, 0), ref.MROPE)
            else:
                k = g.rope_ext(x, g.tensor(gl.I32, T, data=pos[0]), None, D, gl.ROPE_NORMAL if how == "normal" else gl.ROPE_NEOX,
                               0, 1e4, 1.0, 0.0, 1.0, 32.0, 1.0)
            out = g.set_rows(cache, g.reshape_2d(k, W, T), g.tensor(gl.I64, T, data=idx))
            res = g.compute(hip, out if fused else [out, k])
            got.append((g.read(cache).reshape(rows, W), None if fused else res[1].reshape(T, W)))
    gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, True)
    turned = got[1][1]
    if how == "several":
        near(turned, *ref.rope(fill[3:T + 3].reshape(T, KV, D), pos, D, (D // 8, D // 8, D // 4, 0), ref.MROPE, 1e6))
    want = fill.copy()
    want[idx] = turned
    assert np.array_equal(got[0][0], want) and np.array_equal(got[1][0], want)


@pytest.mark.parametrize("how", ["several", "neox"])
@pytest.mark.parametrize("T", [1, 3, 40])
def test_append_of_normed_keys(hip, how, T):
    """Queries and keys normed by head before they turn, values added to a bias: bits as without fusion."""
    rng = np.random.default_rng(T)
    x, w, bias = (rng.standard_normal(s).astype(np.float32) for s in ((T, 8, 64), 64, (T, 128)))
    idx = rng.permutation(T + 3)[:T].astype(np.int64)
    pos = positions(rng, T, 5000)
    got = []
    for fused in (True, False):
        gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, fused)
        with Graph(mem=1 << 20) as g:
            rows, tw = g.tensor(gl.F32, 64, 8, T, data=x), g.tensor(gl.F32, 64, data=w)
            p = g.tensor(gl.I32, 4 * T, data=pos) if how == "several" else g.tensor(gl.I32, T, data=pos[0])
            to = g.tensor(gl.I64, T, data=idx)
            kc, vc = (g.tensor(gl.Q4_0, 128, T + 3, data=quantize(np.zeros((T + 3, 128), np.float32), gl.Q4_0)) for _ in "kv")

            def normed(n, at):
                a = g.mul(g.rms_norm(g.cont_3d(g.view_3d(rows, 64, n, T, 256, 2048, 256 * at), 64, n, T), 1e-6), tw)
                return multi(g, a, p, 64, (8, 12, 12, 0), ref.MROPE) if how == "several" else \
                    g.rope_ext(a, p, None, 64, gl.ROPE_NEOX, 0, 1e4, 1.0, 0.0, 1.0, 32.0, 1.0)
            q, k = normed(4, 0), normed(2, 4)
            v = g.add(g.cont_2d(g.view_3d(rows, 64, 2, T, 256, 2048, 256 * 6), 128, T), g.tensor(gl.F32, 128, T, data=bias))
            res = g.compute(hip, [q, g.set_rows(kc, g.reshape_2d(k, 128, T), to), g.set_rows(vc, v, to)])
            got.append((res[0], raw(g, kc), raw(g, vc)))
    gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, True)
    for a, b in zip(*got):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    cache = quantize(np.zeros((T + 3, 128), np.float32), gl.Q4_0).view(np.uint8).reshape(T + 3, -1).copy()
    values = x[:, 6:].reshape(T, 128) + bias
    assert np.array_equal(got[0][2], expected(cache, values, idx, gl.Q4_0).ravel())


@pytest.mark.parametrize("D, n_dims", [(1024, 1024), (1028, 1026), (1100, 1030), (2048, 2048), (4096, 3000)])
@pytest.mark.parametrize("T", [2, 40])
def test_append_of_wide_heads(hip, D, n_dims, T):
    """Rotations of up to and past the pairs that a workgroup holds, beside rows stored by index: bits as without fusion."""
    rng = np.random.default_rng(D + T)
    x, pos = rng.standard_normal((T, 2, D)).astype(np.float32), rng.integers(0, 5000, T).astype(np.int32)
    idx = rng.permutation(T + 3)[:T].astype(np.int32)
    got = []
    for fused in (True, False):
        gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, fused)
        with Graph(mem=1 << 20) as g:
            a, p, c = g.tensor(gl.F32, D, 2, T, data=x), g.tensor(gl.I32, T, data=pos), g.tensor(gl.I32, T, data=idx)
            kc, vc = (g.tensor(gl.F16, 2 * D, T + 3, data=np.zeros((T + 3, 2 * D), np.float16)) for _ in "kv")
            q, k = (g.rope_ext(a, p, None, n_dims, mode, 0, 1e4, 1.0, 0.0, 1.0, 32.0, 1.0) for mode in (gl.ROPE_NORMAL, gl.ROPE_NEOX))
            res = g.compute(hip, [q, g.set_rows(kc, g.reshape_2d(k, 2 * D, T), c), g.set_rows(vc, g.reshape_2d(a, 2 * D, T), c)])
            got.append((res[0], raw(g, kc), raw(g, vc)))
    gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, True)
    for a, b in zip(*got):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    want = np.zeros((T + 3, 2 * D), np.float16)
    want[idx] = x.reshape(T, -1)
    assert np.array_equal(got[0][2], want.view(np.uint8).ravel())


@pytest.mark.parametrize("T, H, D", [(7, 5, 96), (3, 40, 64), (2, 9, 128)])
def test_rope_multi_in_place(hip, T, H, D):
    """Over its own rows, where a workgroup has whole heads: bits as into other memory."""
    rng = np.random.default_rng(T)
    x, pos = rng.standard_normal((T, H, D)).astype(np.float32), positions(rng, T)
    core = gl.libs()["core"]
    with Graph(mem=1 << 20) as g:
        a = g.tensor(gl.F32, D, H, T, data=x)
        n = multi(g, a, g.tensor(gl.I32, 4 * T, data=pos), D, (D // 8, D // 8, D // 4, 0), ref.MROPE)
        want = g.compute(hip, n)
        n.contents.data = a.contents.data
        gf = core.ggml_new_graph(g.ctx)
        core.ggml_build_forward_expand(gf, n)
        assert core.ggml_backend_graph_compute(hip, gf) == 0
        assert np.array_equal(want.view(np.uint32), g.read(a).view(np.uint32))


def test_rope_multi_in_place_is_written(hip):
    """Over its own rows, stored by index and read by another node through the rows' own tensor: bits as without fusion."""
    rng = np.random.default_rng(1)
    x, pos, core = rng.standard_normal((5, 3, 64)).astype(np.float32), positions(rng, 5), gl.libs()["core"]
    got = []
    for fused in (True, False):
        gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, fused)
        with Graph(mem=1 << 20) as g:
            a, c = g.tensor(gl.F32, 64, 3, 5, data=x), g.tensor(gl.I32, 5, data=np.array([4, 2, 0, 1, 3], np.int32))
            cache = g.tensor(gl.F32, 192, 5, data=np.zeros((5, 192), np.float32))
            k = multi(g, a, g.tensor(gl.I32, 20, data=pos), 64, (8, 8, 16, 0), ref.MROPE)
            s, y = g.set_rows(cache, g.reshape_2d(k, 192, 5), c), g.scale(a, 1.0)
            g.compute(hip, [])
            gf = core.ggml_new_graph(g.ctx)
            for n in (s, y):
                core.ggml_set_output(n)
                core.ggml_build_forward_expand(gf, n)
            k.contents.data = a.contents.data
            s.contents.src[0].contents.data = a.contents.data
            assert core.ggml_backend_graph_compute(hip, gf) == 0
            got.append((g.read(y).reshape(5, 192), g.read(cache).reshape(5, 192)))
    gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, True)
    assert all(np.array_equal(*pair) for pair in zip(*got))
    near(got[0][0], *(v.reshape(5, 192) for v in ref.rope(x, pos, 64, (8, 8, 16, 0), ref.MROPE, 1e6)))
    assert np.array_equal(got[0][1][[4, 2, 0, 1, 3]], got[0][0])


def test_rope_multi_refuses_shared_memory(hip):
    """Over parts of its rows, its positions or its factors, or its rows where a head goes over two workgroups."""
    core = gl.libs()["core"]
    with Graph(mem=1 << 20) as g:
        a, f = g.tensor(gl.F32, 96, 40, 6, data=np.ones((6, 40, 96), np.float32)), g.tensor(gl.F32, 48, data=np.ones(48, np.float32))
        p = g.tensor(gl.I32, 24, data=np.arange(24, dtype=np.int32))
        n = multi(g, g.view_3d(a, 96, 40, 5, 384, 384 * 40, 0), g.view_1d(p, 20, 0), 96, (16, 16, 16, 0), ref.MROPE, ff=f)
        g.compute(hip, n)
        gf = core.ggml_new_graph(g.ctx)
        core.ggml_build_forward_expand(gf, n)
        own = n.contents.data
        for at in (a.contents.data, a.contents.data + 96 * 40 * 4, p.contents.data, f.contents.data):
            n.contents.data = at
            assert core.ggml_backend_graph_compute(hip, gf) != 0
        n.contents.data = own
        assert core.ggml_backend_graph_compute(hip, gf) == 0


@pytest.mark.parametrize("D, H", [(96, 40), (64, 3)])
def test_rope_in_place_beside_rows(hip, D, H):
    """A rope_ext over its own rows, before rows stored by index: bits as without fusion."""
    rng = np.random.default_rng(D)
    T, core = 30, gl.libs()["core"]
    x, v = (rng.standard_normal((T, H, D)).astype(np.float32) for _ in "kv")
    pos, idx = rng.integers(0, 5000, T).astype(np.int32), rng.permutation(T + 2)[:T].astype(np.int32)
    got = []
    for fused in (True, False):
        gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, fused)
        with Graph(mem=1 << 20) as g:
            a, b, p, c = g.tensor(gl.F32, D, H, T, data=x), g.tensor(gl.F32, D * H, T, data=v), g.tensor(gl.I32, T, data=pos), g.tensor(gl.I32, T, data=idx)
            cache = g.tensor(gl.F32, D * H, T + 2, data=np.zeros((T + 2, D * H), np.float32))
            k = g.rope_ext(a, p, None, D, gl.ROPE_NEOX, 0, 1e4, 1.0, 0.0, 1.0, 32.0, 1.0)
            s = g.set_rows(cache, b, c)
            g.compute(hip, [])
            gf = core.ggml_new_graph(g.ctx)
            for n in (k, s):
                core.ggml_set_output(n)
                core.ggml_build_forward_expand(gf, n)
            k.contents.data = a.contents.data
            assert core.ggml_backend_graph_compute(hip, gf) == 0
            got.append((g.read(a), g.read(cache)))
    gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, True)
    assert all(np.array_equal(*pair) for pair in zip(*got))
    want = np.zeros((T + 2, D * H), np.float32)
    want[idx] = v.reshape(T, -1)
    assert np.array_equal(got[0][1].reshape(want.shape), want)


def test_rows_of_nothing(hip):
    """No heads, no tokens, no rows, no values."""
    with Graph(mem=1 << 20) as g:
        some = g.tensor(gl.F32, 64, 2, 3, data=np.ones((3, 2, 64), np.float32))
        pos = g.tensor(gl.I32, 12, data=np.zeros(12, np.int32))
        a = multi(g, g.tensor(gl.F32, 64, 0, 3), pos, 64, (8, 12, 12, 0), ref.MROPE)
        b = multi(g, g.tensor(gl.F32, 64, 2, 0), g.tensor(gl.I32, 0), 64, (8, 12, 12, 0), ref.MROPE)
        c = multi(g, some, pos, 64, (8, 12, 12, 0), ref.MROPE)
        cache = g.tensor(gl.F16, 64, 5, data=np.ones((5, 64), np.float16))
        d = g.set_rows(cache, g.tensor(gl.F32, 64, 0), g.tensor(gl.I64, 0))
        e = g.set_rows(g.tensor(gl.F32, 0, 5), g.tensor(gl.F32, 0, 3), g.tensor(gl.I64, 3, data=np.arange(3)))
        f = g.set_rows(g.tensor(gl.F32, 64, 5, 0), g.tensor(gl.F32, 64, 3, 0), g.tensor(gl.I64, 3, data=np.arange(3)))
        core, gf = g.core, g.core.ggml_new_graph(g.ctx)
        for t in (a, b, c, d, e, f):
            core.ggml_set_output(t)
            core.ggml_build_forward_expand(gf, t)
        g.buf = core.ggml_backend_alloc_ctx_tensors(g.ctx, hip)
        for t, x in g.inputs:
            core.ggml_backend_tensor_set(t, x.ctypes.data, 0, x.nbytes)
        assert core.ggml_backend_graph_compute(hip, gf) == 0
        assert (g.read(c) == 1).all() and (g.read(cache, np.float16) == 1).all()
