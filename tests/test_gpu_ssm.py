"""The state space mixers' operators on the HIP backend against float64 (ssm_ref, which carries the
bound that each value is held to)."""
import numpy as np
import pytest

import ssm_ref
from gl import Graph, cpu_backend, gl, ptr

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    b = gl.hip_backend(0)
    yield b
    gl.libs()["core"].ggml_backend_free(b)


def near(got, want, bound, what=""):
    """Each value within its bound; where the definition is not finite, the same kind of value."""
    got, want, bound = got.reshape(want.shape).astype(np.float64), want, np.broadcast_to(bound, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(got)), what
    off = np.abs(got - want)[fine] - (bound[fine] + 1e-37)
    assert off.size == 0 or off.max() <= 0, (what, off.max(), (np.abs(got - want)[fine] / (bound[fine] + 1e-37)).max())


def draw(rng, S, T, H, P, N, G, pool, a0, big_dt=False):
    d = dict(
        state=rng.standard_normal((pool, H, P, N)).astype(np.float32),
        x=rng.standard_normal((S, T, H, P)).astype(np.float32),
        dt=(rng.standard_normal((S, T, H)) * (8 if big_dt else 1) - (0 if big_dt else 3)).astype(np.float32),
        A=-(0.5 + 8 * rng.random((H, a0))).astype(np.float32),
        B=rng.standard_normal((S, T, G, N)).astype(np.float32),
        C=rng.standard_normal((S, T, G, N)).astype(np.float32),
        ids=rng.permutation(pool)[:S].astype(np.int32))
    return d


def scan_node(g, d):
    S, T, H, P = d["x"].shape
    pool, _, _, N = d["state"].shape
    G = d["B"].shape[2]
    t = lambda a, *ne: g.tensor(gl.F32, *ne, data=a)  # noqa: E731
    return g.ssm_scan(t(d["state"], N, P, H, pool), t(d["x"], P, H, T, S), t(d["dt"], H, T, S), t(d["A"], d["A"].shape[1], H),
                      t(d["B"], N, G, T, S), t(d["C"], N, G, T, S), g.tensor(gl.I32, S, data=d["ids"]), 1)


def check_scan(hip, d, what="", clamp=False):
    S, T, H, P = d["x"].shape
    N = d["B"].shape[3]
    with Graph(mem=1 << 20) as g:
        out = g.compute(hip, scan_node(g, d))
    ids = np.clip(d["ids"], 0, len(d["state"]) - 1) if clamp else d["ids"]
    y, h, ye, he = ssm_ref.scan(d["state"][ids], d["x"], d["dt"], d["A"], d["B"], d["C"])
    n = S * T * H * P
    near(out[:n], y, ye, ("y", what))
    near(out[n:], h, he, ("state", what))
    return out


# S, T, H, P, N, G, pool, A's extent
SCANS = [
    (1, 1, 1, 1, 1, 1, 1, 1), (1, 1, 5, 3, 7, 1, 1, 1), (3, 1, 6, 64, 128, 2, 5, 1), (2, 2, 4, 64, 128, 1, 2, 1),
    (1, 17, 3, 5, 13, 3, 2, 1), (2, 63, 2, 64, 128, 1, 2, 1), (1, 64, 4, 64, 128, 2, 1, 1), (1, 65, 2, 64, 128, 2, 1, 1),
    (2, 130, 2, 32, 16, 1, 3, 1), (1, 200, 3, 80, 96, 1, 1, 1), (1, 129, 2, 128, 256, 2, 1, 1), (1, 333, 2, 64, 64, 1, 1, 1),
    (4, 13000, 1, 16, 128, 1, 4, 1), (1, 64, 3, 130, 128, 1, 1, 1), (1, 300, 16, 64, 128, 8, 1, 1), (2, 150, 9, 16, 32, 3, 2, 1),
    (1, 200, 40, 32, 64, 8, 1, 1), (1, 2000, 3, 48, 128, 1, 1, 1), (1, 90, 1, 33, 100, 1, 1, 1), (1, 70, 2, 48, 200, 1, 1, 1), (5, 7, 3, 64, 128, 3, 9, 1), (1, 1100, 2, 64, 128, 1, 1, 1),
    # a decay per state: a head per channel, and heads of several channels
    (1, 1, 300, 1, 16, 1, 1, 16), (2, 50, 130, 1, 16, 1, 3, 16), (1, 257, 67, 1, 8, 1, 1, 8), (3, 3, 65, 1, 32, 1, 3, 32),
    (2, 100, 128, 1, 16, 2, 2, 16), (1, 40, 70, 1, 16, 1, 1, 1), (1, 17, 64, 1, 32, 1, 1, 32), (1, 9, 12, 1, 8, 3, 1, 8),
    (2, 16, 5, 4, 4, 1, 2, 1), (3, 2, 8, 8, 256, 2, 3, 256), (1, 5, 4, 2, 64, 2, 1, 1), (1, 40, 6, 1, 5, 2, 1, 5), (1, 33, 3, 4, 16, 1, 2, 16), (1, 25, 2, 2, 129, 2, 1, 129), (1, 1030, 64, 1, 16, 1, 1, 16),
]


@pytest.mark.parametrize("S, T, H, P, N, G, pool, a0", SCANS)
def test_scan(hip, S, T, H, P, N, G, pool, a0):
    rng = np.random.default_rng(S * 1000 + T * 7 + H + P + N)
    check_scan(hip, draw(rng, S, T, H, P, N, G, pool, a0))


@pytest.mark.parametrize("P, N, a0", [(64, 128, 1), (1, 16, 16), (5, 7, 1)])
def test_scan_extreme_steps(hip, P, N, a0):
    """Time steps from none (dt far below zero) to decays that forget everything."""
    d = draw(np.random.default_rng(9), 2, 150, 3, P, N, 1, 2, a0, big_dt=True)
    d["dt"][0, 5:9] = -200
    d["dt"][0, 80:84] = 60
    d["dt"][1, 0] = 1e4
    check_scan(hip, d)


@pytest.mark.parametrize("P, N, a0", [(64, 128, 1), (1, 16, 16), (5, 7, 1)])
@pytest.mark.parametrize("big", [1e12, 2e38])
def test_scan_steps_that_forget_everything(hip, P, N, a0, big):
    """A time step of any size that leaves nothing of the state is as good as a step of 60 (e^-240) with the
    same d x: neither its own token nor the later ones lose bits to its exponent, or become NaN where that
    leaves the range. (60 x / d rounds once: u of d x B, within the 4 u that the bound has for it.)"""
    d = draw(np.random.default_rng(8), 2, 150, 3, P, N, 1, 2, a0)
    d["A"] = (d["A"] / 2 - 4).astype(np.float32)
    same = {k: v.copy() for k, v in d.items()}
    for at in (3, 4, 70, 71, 72, 149):
        d["dt"][:, at] = np.float32(big)
        same["dt"][:, at] = 60
        d["x"][:, at] = (d["x"][:, at].astype(np.float64) * (60 / float(np.float32(big)))).astype(np.float32)
    with Graph(mem=1 << 20) as g:
        out = g.compute(hip, scan_node(g, d))
    y, h, ye, he = ssm_ref.scan(same["state"][same["ids"]], same["x"], same["dt"], same["A"], same["B"], same["C"])
    near(out[:y.size], y, ye, "y")
    near(out[y.size:], h, he, "state")


@pytest.mark.parametrize("T", [0, 1, 100])
@pytest.mark.parametrize("P, N, a0", [(64, 128, 1), (1, 16, 16), (5, 7, 7)])
def test_scan_of_no_sequences(hip, T, P, N, a0):
    """A graph whose batch is empty runs, beside one that is not."""
    d = draw(np.random.default_rng(15), 1, T, 3, P, N, 1, 1, a0)
    none = dict(d, **{k: d[k][:0] for k in ("x", "dt", "B", "C", "ids")})
    with Graph(mem=1 << 20) as g:
        empty, one = scan_node(g, none), scan_node(g, d)
        assert empty.contents.ne[0] == 0
        got = g.compute(hip, [empty, one])
        assert got[0].size == 0
    y, h, ye, he = ssm_ref.scan(d["state"][d["ids"]], d["x"], d["dt"], d["A"], d["B"], d["C"])
    near(got[1][:y.size], y, ye)
    near(got[1][y.size:], h, he)


@pytest.mark.parametrize("T", [0, 1, 100])
def test_scan_decay_of_one_and_growth(hip, T):
    d = draw(np.random.default_rng(10), 1, T, 3, 64, 128, 1, 1, 1)
    d["A"][0], d["A"][1] = 0, 0.05                    # a state that keeps everything, one that grows
    out = check_scan(hip, d)
    if T == 0:
        assert np.array_equal(out, d["state"].ravel())   # no token: the states as they are


@pytest.mark.parametrize("T", [1, 70])
def test_scan_ids(hip, T):
    """Two sequences of one row, and ids outside the pool (clamped, never followed)."""
    d = draw(np.random.default_rng(11), 4, T, 2, 64, 128, 1, 3, 1)
    d["ids"] = np.array([2, 2, -1, 7], np.int32)
    check_scan(hip, d, clamp=True)


@pytest.mark.parametrize("T, at", [(1, 0), (100, 0), (100, 37), (100, 70), (200, 199)])
@pytest.mark.parametrize("P, N, a0", [(64, 128, 1), (1, 16, 16)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_scan_keeps_what_came_before_a_bad_value(hip, T, at, P, N, a0, bad):
    """A value that is not finite reaches its own head's outputs from its token on, and nothing else:
    earlier tokens, other heads and other sequences keep theirs."""
    d = draw(np.random.default_rng(12), 2, T, 3, P, N, 1, 2, a0)
    clean = check_scan(hip, d)
    d["x"][1, at, 2, 0] = bad
    with Graph(mem=1 << 20) as g:
        out = g.compute(hip, scan_node(g, d))
    n = d["x"].size
    y, was = out[:n].reshape(d["x"].shape), clean[:n].reshape(d["x"].shape)
    fine = np.ones(y.shape, bool)
    fine[1, at:, 2, 0] = False
    assert not np.isfinite(y[~fine]).any()
    h, h0 = out[n:].reshape(2, 3, P, N), clean[n:].reshape(2, 3, P, N)
    hf = np.ones(h.shape, bool)
    hf[1, 2, 0] = False
    assert not np.isfinite(h[~hf]).any()
    y64, h64, ye, he = ssm_ref.scan(d["state"][d["ids"]], np.where(np.isfinite(d["x"]), d["x"], 0), d["dt"], d["A"], d["B"], d["C"])
    near(y[fine], y64[fine], ye[fine])
    near(h[hf], h64[hf], he[hf])


def with_outliers(d, kind, size):
    """Operands of unequal size: values of one token, of one state, or of an input and a token."""
    H, P, N, G = d["x"].shape[2], d["x"].shape[3], d["B"].shape[3], d["B"].shape[2]
    h, p, n, g = H // 2, P // 3, N // 3, G - 1
    if kind in ("late x", "early x"):
        d["x"][0, 50 if kind == "late x" else 3, h, p] *= size
    if kind == "x of all channels":
        d["x"][0, 50] *= size
    if kind in ("B", "C"):
        d[kind][0, 50, g, n] *= size
    if kind in ("row of B", "row of C"):
        d[kind[-1]][0, 50] *= size
    if kind in ("state of B", "state of C"):
        d["B"][..., n] *= size if kind[-1] == "B" else 1 / size
        d["C"][..., n] *= size if kind[-1] == "C" else 1 / size
    if kind == "first state":
        d["state"][:, h, p, n] *= size
    if kind == "small inputs first":
        d["state"][:] = 0
        d["x"][:, :40] /= size
    if kind == "x and B":
        d["x"][0, 20, h, p] *= size
        d["B"][0, 45, g, n] *= size
    if kind == "every eighth x":
        d["state"][:] = 0
        d["x"][:, 7::8] *= size
    return d


@pytest.mark.parametrize("size", [1e5, 1e6, 1e8, 1e11, 1e18])
@pytest.mark.parametrize("kind", ["late x", "early x", "x of all channels", "B", "C", "row of B", "row of C", "state of B", "state of C",
                                  "first state", "small inputs first", "x and B", "every eighth x"])
@pytest.mark.parametrize("S, T, H, P, N, G, a0", [(2, 150, 2, 64, 128, 1, 1), (1, 400, 2, 20, 30, 2, 1), (1, 70, 3, 5, 256, 1, 1), (1, 150, 66, 1, 16, 1, 16)])
def test_scan_of_operands_of_unequal_size(hip, S, T, H, P, N, G, a0, kind, size):
    """A value far larger than the others, finite, takes bits from no other token, channel or state: each
    output is held to the bound of its own terms."""
    rng = np.random.default_rng(T + P + N)
    d = draw(rng, S, T, H, P, N, G, S, a0)
    check_scan(hip, with_outliers(d, kind, np.float32(size)))


@pytest.mark.parametrize("T, a", [(150, 2.0), (70, 15.0), (200, 0.3), (64, 20.0)])
def test_scan_that_grows(hip, T, a):
    """Decays above 1: a chunk's last tokens are far larger than its first, which keep their bits."""
    d = draw(np.random.default_rng(14), 1, T, 3, 64, 128, 1, 1, 1)
    d["A"][:] = np.float32(a) * np.array([[1.0], [0.5], [-1.0]], np.float32)
    d["dt"][:] = np.minimum(d["dt"], -2.5)
    check_scan(hip, d)


@pytest.mark.parametrize("N", [8, 16])
@pytest.mark.parametrize("inputs", [False, True])
def test_scan_of_long_segments(hip, N, inputs):
    """Many channels of one each take few segments of some 200 tokens, whose decays are one sum of time steps: what
    that rounds may not grow with the tokens, also where they are all alike (the same dt for every token, by a stride
    of none, so that every rounding may go the same way). A sample of the channels against the recurrence."""
    rng = np.random.default_rng(N)
    H, T = 40960, 1400
    dt = (rng.standard_normal((1, 1, H)) * 0.5 - 2).astype(np.float32)
    A = -(0.5 + 1.5 * rng.random((H, N))).astype(np.float32)
    state = rng.standard_normal((1, H, 1, N)).astype(np.float32)
    x = (rng.standard_normal((1, T, 1, 1)) * inputs).astype(np.float32)
    B, Cm = (rng.standard_normal((1, T, 1, N)).astype(np.float32) for _ in range(2))
    with Graph(mem=1 << 20) as g:
        xt = g.view_4d(g.tensor(gl.F32, T, data=x), 1, 1, T, 1, 4, 4, 4 * T, 0)
        dtt = g.view_3d(g.tensor(gl.F32, H, data=dt), H, 1, 1, 4 * H, 4 * H, 0)
        for t, many in ((xt, H), (dtt, T)):
            t.contents.ne[1], t.contents.nb[1] = many, 0
        out = g.compute(hip, g.ssm_scan(g.tensor(gl.F32, N, 1, H, 1, data=state), xt, dtt, g.tensor(gl.F32, N, H, data=A),
                                        g.tensor(gl.F32, N, 1, T, 1, data=B), g.tensor(gl.F32, N, 1, T, 1, data=Cm),
                                        g.tensor(gl.I32, 1, data=np.zeros(1, np.int32)), 1))
    some = np.sort(rng.permutation(H)[:256])
    y, h, ye, he = ssm_ref.scan(state[:, some], np.broadcast_to(x, (1, T, 256, 1)), np.broadcast_to(dt[:, :, some], (1, T, 256)),
                                A[some], B, Cm)
    near(out[:T * H].reshape(1, T, H, 1)[:, :, some], y, ye, "y")
    near(out[T * H:].reshape(1, H, 1, N)[:, some], h, he, "state")


# few tokens, channels and states at the edges of what a lane, a wave or a group of rows takes
FEW = [
    (3, 1, 67, 1, 16, 1, 3, 16), (2, 1, 64, 1, 8, 1, 2, 8), (3, 2, 130, 1, 32, 1, 3, 32), (2, 5, 129, 1, 16, 1, 2, 16), (1, 8, 1, 1, 16, 1, 1, 1),
    (2, 4, 192, 1, 8, 3, 2, 8), (1, 3, 96, 1, 16, 3, 1, 16), (2, 39, 65, 1, 16, 1, 2, 16), (2, 48, 65, 1, 16, 1, 2, 16), (3, 41, 200, 1, 32, 1, 3, 32),
    (5, 3, 7, 3, 20, 1, 5, 1), (3, 1, 5, 1, 64, 1, 3, 64), (4, 2, 3, 3, 12, 1, 4, 12), (3, 4, 3, 6, 128, 1, 3, 1), (2, 24, 3, 64, 128, 1, 2, 1),
    (2, 25, 3, 64, 128, 1, 2, 1), (1, 48, 2, 4, 256, 1, 1, 1), (1, 49, 2, 4, 256, 1, 1, 1), (33, 17, 32, 64, 20, 1, 33, 1), (2, 7, 6, 2, 36, 3, 2, 1),
]


@pytest.mark.parametrize("S, T, H, P, N, G, pool, a0", FEW)
@pytest.mark.parametrize("odd", [False, True])
def test_scan_of_few_tokens(hip, S, T, H, P, N, G, pool, a0, odd):
    """Whole tensors, and slices of rows whose addresses and strides are no multiple of 16 bytes."""
    d = draw(np.random.default_rng(S + T * 3 + H + P * N), S, T, H, P, N, G, pool, a0)
    if not odd:
        check_scan(hip, d)
        return
    rows = lambda a, n: a.reshape(-1, n)  # noqa: E731
    wide = np.concatenate([np.zeros((S * T, 1), np.float32), rows(d["x"], H * P), rows(d["B"], G * N), rows(d["C"], G * N)], 1)
    w = wide.shape[1] + 1 if wide.shape[1] % 2 == 0 else wide.shape[1]
    wide = np.pad(wide, ((0, 0), (0, w - wide.shape[1])))
    per = H * P * N + 1
    states = np.pad(rows(d["state"], H * P * N), ((0, 0), (0, 1)))
    with Graph(mem=1 << 20) as g:
        r = g.tensor(gl.F32, w, T, S, data=wide)
        x = g.view_4d(r, P, H, T, S, P * 4, w * 4, T * w * 4, 4)
        B, Cm = (g.view_4d(r, N, G, T, S, N * 4, w * 4, T * w * 4, 4 * a) for a in (1 + H * P, 1 + H * P + G * N))
        s = g.view_4d(g.tensor(gl.F32, per, pool, data=states), N, P, H, pool, N * 4, N * P * 4, per * 4, 0)
        dt, A = g.tensor(gl.F32, H, T, S, data=d["dt"]), g.tensor(gl.F32, a0, H, data=d["A"])
        out = g.compute(hip, g.ssm_scan(s, x, dt, A, B, Cm, g.tensor(gl.I32, S, data=d["ids"]), 1))
    y, h, ye, he = ssm_ref.scan(d["state"][d["ids"]], d["x"], d["dt"], d["A"], d["B"], d["C"])
    near(out[:y.size], y, ye)
    near(out[y.size:], h, he)


def test_scan_of_strided_operands(hip):
    """x, B and C as slices of one projection, dt of another, A of a table, a pool of wider rows."""
    rng = np.random.default_rng(13)
    S, T, H, P, N, G = 2, 75, 4, 64, 128, 2
    d = draw(rng, S, T, H, P, N, G, 3, 1)
    w = H * P + 2 * G * N + 3
    rows = rng.standard_normal((S, T, w)).astype(np.float32)
    steps = np.concatenate([rng.standard_normal((S, T, 5)).astype(np.float32), d["dt"]], 2)
    d["x"] = rows[:, :, :H * P].reshape(S, T, H, P)
    d["B"] = rows[:, :, H * P:H * P + G * N].reshape(S, T, G, N)
    d["C"] = rows[:, :, H * P + G * N:w - 3].reshape(S, T, G, N)
    with Graph(mem=1 << 20) as g:
        r = g.tensor(gl.F32, w, T, S, data=rows)
        x = g.view_4d(r, P, H, T, S, P * 4, w * 4, T * w * 4, 0)
        B, Cm = (g.view_4d(r, N, G, T, S, N * 4, w * 4, T * w * 4, a * 4) for a in (H * P, H * P + G * N))
        dt = g.view_3d(g.tensor(gl.F32, H + 5, T, S, data=steps), H, T, S, (H + 5) * 4, T * (H + 5) * 4, 20)
        table = np.concatenate([d["A"], np.ones((H, 2), np.float32)], 1)
        A = g.view_2d(g.tensor(gl.F32, 3, H, data=table), 1, H, 12, 0)
        pool = np.concatenate([d["state"].reshape(3, -1), np.ones((3, 4), np.float32)], 1)
        s = g.view_4d(g.tensor(gl.F32, pool.shape[1], 3, data=pool), N, P, H, 3, N * 4, N * P * 4, pool.shape[1] * 4, 0)
        out = g.compute(hip, g.ssm_scan(s, x, dt, A, B, Cm, g.tensor(gl.I32, S, data=d["ids"]), 1))
    y, h, ye, he = ssm_ref.scan(d["state"][d["ids"]], d["x"], d["dt"], d["A"], d["B"], d["C"])
    near(out[:y.size], y, ye)
    near(out[y.size:], h, he)


@pytest.mark.parametrize("K, T, D, S", [(4, 1, 1, 1), (4, 1, 300, 5), (1, 9, 5, 1), (2, 5, 64, 1), (4, 2, 33, 2), (4, 100, 129, 1),
                                       (3, 65, 64, 3), (7, 70, 40, 1), (4, 300, 1024, 1), (4, 0, 8, 1), (1, 70, 9, 2), (32, 130, 70, 1),
                                       (32, 1, 3, 2)])
def test_conv(hip, K, T, D, S):
    rng = np.random.default_rng(K + T + D)
    sx = rng.standard_normal((S, D, K - 1 + T)).astype(np.float32)
    w = rng.standard_normal((D, K)).astype(np.float32)
    with Graph(mem=1 << 20) as g:
        out = g.compute(hip, g.ssm_conv(g.tensor(gl.F32, K - 1 + T, D, S, data=sx), g.tensor(gl.F32, K, D, data=w)))
    near(out, *ssm_ref.conv(sx, w))


def test_conv_of_strided_operands(hip):
    """The rows channel by channel in memory (a transposed view), the filters with a gap between them."""
    rng = np.random.default_rng(21)
    K, T, D = 4, 37, 50
    rows = rng.standard_normal((K - 1 + T, D + 6)).astype(np.float32)
    w = rng.standard_normal((D, K + 1)).astype(np.float32)
    with Graph(mem=1 << 20) as g:
        sx = g.transpose(g.view_2d(g.tensor(gl.F32, D + 6, K - 1 + T, data=rows), D, K - 1 + T, (D + 6) * 4, 8))
        c = g.view_2d(g.tensor(gl.F32, K + 1, D, data=w), K, D, (K + 1) * 4, 0)
        out = g.compute(hip, g.ssm_conv(sx, c))
    near(out, *ssm_ref.conv(rows[:, 2:2 + D].T[None], w[:, :K]))


def test_conv_of_most_channels(hip):
    """2^30 + 5 channels of one token are more tiles than one dimension of a launch has; every channel reads the same
    rows and the same filter, by strides of none. The ends and a sample are read back."""
    K, T, D = 5, 1, (1 << 30) + 5
    rng = np.random.default_rng(22)
    sx, w = rng.standard_normal((1, 1, K - 1 + T)).astype(np.float32), rng.standard_normal((1, K)).astype(np.float32)
    with Graph(mem=1 << 20) as g:
        sxt = g.view_3d(g.tensor(gl.F32, K - 1 + T, data=sx), K - 1 + T, 1, 1, 4 * (K - 1 + T), 4 * (K - 1 + T), 0)
        wt = g.view_2d(g.tensor(gl.F32, K, data=w), K, 1, 4 * K, 0)
        for t in (sxt, wt):
            t.contents.ne[1], t.contents.nb[1] = D, 0
        n = g.ssm_conv(sxt, wt)
        gf = g.core.ggml_new_graph(g.ctx)
        g.core.ggml_build_forward_expand(gf, n)
        g.buf = g.core.ggml_backend_alloc_ctx_tensors(g.ctx, hip)
        assert g.buf
        for t, v in g.inputs:
            g.core.ggml_backend_tensor_set(t, ptr(v), 0, v.nbytes)
        assert g.core.ggml_backend_graph_compute(hip, gf) == 0
        y, bound = ssm_ref.conv(sx, w)
        for at in (0, (1 << 28) - 500, (1 << 28) + 64, 3 << 28, D - 1000):
            got = np.zeros(1000, np.float32)
            g.core.ggml_backend_tensor_get(n, ptr(got), 4 * at, got.nbytes)
            near(got, np.full(1000, y[0, 0, 0]), bound[0, 0, 0], at)


class Mixer:
    """The convolution with its state, bias and SiLU as a mixer's graph has it. In place: the new rows
    go back into the state they came from."""

    def __init__(self, g, state, rows, w, bias, in_place, act=True, D=None):
        S, T, W = rows.shape
        D, K = w.shape
        self.st = g.tensor(gl.F32, K - 1, D, S, data=state) if K > 1 else None
        x = g.view_3d(g.tensor(gl.F32, W, T, S, data=rows), D, T, S, W * 4, T * W * 4, 0)
        sx = g.concat(self.st, g.transpose(x), 0)
        nb = sx.contents.nb
        dest = self.st if in_place else g.tensor(gl.F32, K - 1, D, S, data=np.zeros_like(state))
        self.new = g.cpy(g.view_3d(sx, K - 1, D, S, nb[1], nb[2], T * 4), dest)
        y = g.ssm_conv(sx, g.tensor(gl.F32, K, D, data=w))
        if bias is not None:
            y = g.add(y, g.tensor(gl.F32, D, data=bias))
        self.y = g.silu(y) if act else y


@pytest.mark.parametrize("fusion", [True, False])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("K, T, D, S, W, bias, act", [
    (4, 1, 21, 3, 25, True, True), (3, 40, 259, 2, 261, True, True), (4, 9, 2, 1, 7, True, False), (2, 3, 1027, 2, 1027, False, True),
    (4, 1, 8, 1, 8, True, True), (4, 1, 260, 7, 300, True, True), (4, 2, 65, 2, 65, True, True), (4, 3, 64, 3, 70, False, True),
    (4, 64, 64, 1, 128, True, True), (4, 67, 130, 2, 131, True, True), (2, 5, 33, 1, 40, True, True), (3, 200, 512, 1, 1100, False, True),
    (4, 300, 1000, 1, 1000, True, False), (6, 4, 20, 2, 20, True, True), (9, 70, 70, 2, 71, True, True),
    (4, 21, 44, 1, 44, False, False)])
def test_conv_with_its_state(hip, fusion, in_place, K, T, D, S, W, bias, act):
    rng = np.random.default_rng(K * T + D)
    state = rng.standard_normal((S, D, K - 1)).astype(np.float32)
    rows = rng.standard_normal((S, T, W)).astype(np.float32)
    w = rng.standard_normal((D, K)).astype(np.float32)
    b = rng.standard_normal(D).astype(np.float32) if bias else None
    sx = np.concatenate([state, rows[:, :, :D].transpose(0, 2, 1)], 2)
    gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, fusion)
    try:
        with Graph(mem=1 << 20) as g:
            m = Mixer(g, state, rows, w, b, in_place, act)
            new, y = g.compute(hip, [m.new, m.y])
    finally:
        gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, True)
    assert np.array_equal(new.reshape(S, D, K - 1), sx[:, :, T:])
    near(y, *ssm_ref.conv(sx, w, b, act))


def test_conv_that_others_read(hip):
    """Graphs that the fused launch must leave alone: the joined rows are an output, the old state is
    read after the convolution and before the copy over it, the new state goes to another sequence's
    row of the same memory."""
    rng = np.random.default_rng(41)
    K, T, D, S = 4, 2, 24, 1
    state = rng.standard_normal((2, D, K - 1)).astype(np.float32)
    rows = rng.standard_normal((S, T, D)).astype(np.float32)
    w, b = rng.standard_normal((D, K)).astype(np.float32), rng.standard_normal(D).astype(np.float32)
    sx = np.concatenate([state[:1], rows.transpose(0, 2, 1)], 2)
    want, bound = ssm_ref.conv(sx, w, b, True)
    nb1, nb2 = (K - 1) * 4, (K - 1) * D * 4
    for kind in ("joined", "old", "shift"):
        with Graph(mem=1 << 20) as g:
            pool = g.tensor(gl.F32, K - 1, D, 2, data=state)
            st = g.view_3d(pool, K - 1, D, 1, nb1, nb2, 0)
            joined = g.concat(st, g.transpose(g.tensor(gl.F32, D, T, S, data=rows)), 0)
            y = g.silu(g.add(g.ssm_conv(joined, g.tensor(gl.F32, K, D, data=w)), g.tensor(gl.F32, D, data=b)))
            old = g.scale(g.reshape_2d(st, K - 1, D), 2.0) if kind == "old" else None
            nb = joined.contents.nb
            # one step into the pool: the new state lies over the end of the old one and the next row
            to = g.view_3d(pool, K - 1, D, 1, nb1, nb2, nb1 if kind == "shift" else 0)
            new = g.cpy(g.view_3d(joined, K - 1, D, S, nb[1], nb[2], T * 4), to)
            outs = [y] + ([joined] if kind == "joined" else [old] if kind == "old" else []) + [new]
            got = g.compute(hip, outs)
            near(got[0], want, bound, kind)
            assert np.array_equal(got[-1].reshape(D, K - 1), sx[0, :, T:]), kind
            if kind == "joined":
                assert np.array_equal(got[1].reshape(sx.shape), sx)
            if kind == "old":
                assert np.array_equal(got[1].reshape(D, K - 1), 2 * state[0])


@pytest.mark.parametrize("what", ["rows", "joined", "between"])
def test_conv_whose_result_takes_used_memory(hip, what):
    """A result that lies in memory which is free by its place in the graph, and not before: the new
    rows', the joined rows', that of another node's value."""
    rng = np.random.default_rng(43)
    K, T, D = 4, 300, 96
    state = rng.standard_normal((1, D, K - 1)).astype(np.float32)
    rows = rng.standard_normal((1, T, D)).astype(np.float32)
    w, b = rng.standard_normal((D, K)).astype(np.float32), rng.standard_normal(D).astype(np.float32)
    want, bound = ssm_ref.conv(np.concatenate([state, 2 * rows.transpose(0, 2, 1)], 2), w, b, True)
    with Graph(mem=1 << 20) as g:
        r = g.tensor(gl.F32, D, T, data=rows)
        x = g.scale(r, 2.0)
        joined = g.concat(g.tensor(gl.F32, K - 1, D, 1, data=state), g.transpose(x), 0)
        conv = g.ssm_conv(joined, g.tensor(gl.F32, K, D, data=w))
        between = g.scale(r, 3.0)
        used = g.scale(between, 0.5)
        y = g.silu(g.add(conv, g.tensor(gl.F32, D, data=b)))
        gf = g.core.ggml_new_graph(g.ctx)
        for t in (conv, used, y):
            g.core.ggml_build_forward_expand(gf, t)
        for t in (used, y):
            g.core.ggml_set_output(t)
        g.buf = g.core.ggml_backend_alloc_ctx_tensors(g.ctx, hip)
        for t, v in g.inputs:
            g.core.ggml_backend_tensor_set(t, ptr(v), 0, v.nbytes)
        y.contents.data = {"rows": x, "joined": joined, "between": between}[what].contents.data
        assert g.core.ggml_backend_graph_compute(hip, gf) == 0
        near(g.read(y), want, bound, what)
        assert np.array_equal(g.read(used), (rows * np.float32(3) * np.float32(0.5)).ravel())


def test_static_compute(hip):
    d = draw(np.random.default_rng(31), 1, 150, 2, 64, 128, 1, 1, 1)
    with Graph(mem=1 << 20) as g:
        n = scan_node(g, d)
        want = g.compute(hip, n)
        core = g.core
        gf = core.ggml_new_graph(g.ctx)
        core.ggml_build_forward_expand(gf, n)
        assert gl.libs()["hip"].ggml_backend_hip_graph_compute_static(hip, gf) == 0
        assert np.array_equal(g.read(n), want)


@pytest.mark.parametrize("fusion", [True, False])
@pytest.mark.parametrize("what", ["bias", "bias of the plain node", "filters"])
def test_conv_whose_operands_are_written_before_their_use(hip, what, fusion):
    """A copy into the bias between the convolution and its sum, or into the filters between the joined rows and
    the convolution, is seen."""
    rng = np.random.default_rng(44)
    K, T, D = 4, 30, 96
    state = rng.standard_normal((1, D, K - 1)).astype(np.float32)
    rows = rng.standard_normal((1, T, D)).astype(np.float32)
    w, b, w2, b2 = (rng.standard_normal(s).astype(np.float32) for s in ((D, K), D, (D, K), D))
    sx = np.concatenate([state, rows.transpose(0, 2, 1)], 2)
    gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, fusion)
    try:
        with Graph(mem=1 << 20) as g:
            if what == "bias of the plain node":
                joined = g.tensor(gl.F32, K - 1 + T, D, 1, data=sx)
            else:
                joined = g.concat(g.tensor(gl.F32, K - 1, D, 1, data=state), g.transpose(g.tensor(gl.F32, D, T, data=rows)), 0)
            wt, bt = g.tensor(gl.F32, K, D, data=w), g.tensor(gl.F32, D, data=b)
            conv = g.ssm_conv(joined, wt)
            copy = g.cpy(g.tensor(gl.F32, K, D, data=w2), wt) if what == "filters" else g.cpy(g.tensor(gl.F32, D, data=b2), bt)
            y = g.silu(g.add(conv, bt))
            gf = g.core.ggml_new_graph(g.ctx)
            for t in (joined, copy, conv, y) if what == "filters" else (conv, copy, y):
                g.core.ggml_build_forward_expand(gf, t)
            g.core.ggml_set_output(y)
            g.buf = g.core.ggml_backend_alloc_ctx_tensors(g.ctx, hip)
            for t, v in g.inputs:
                g.core.ggml_backend_tensor_set(t, ptr(v), 0, v.nbytes)
            assert g.core.ggml_backend_graph_compute(hip, gf) == 0
            y = g.read(y)
    finally:
        gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, True)
    near(y, *ssm_ref.conv(sx, w2 if what == "filters" else w, b if what == "filters" else b2, True))


def static(g, hip, *nodes):
    gf = g.core.ggml_new_graph(g.ctx)
    for n in nodes:
        g.core.ggml_build_forward_expand(gf, n)
    return gl.libs()["hip"].ggml_backend_hip_graph_compute_static(hip, gf)


@pytest.mark.parametrize("S, T, H, P, N, G, pool, a0", [(150, 50, 8, 4, 256, 8, 150, 1), (150, 130, 8, 4, 200, 8, 150, 1), (61, 70, 16, 5, 100, 16, 64, 1)])
def test_static_compute_of_many_sequences(hip, S, T, H, P, N, G, pool, a0):
    """One chunk of all sequences is more than the prepared operands' 64 MiB: they go through in passes, in the
    caller's scratch too, and each has its own operands, states and results."""
    d = draw(np.random.default_rng(33), S, T, H, P, N, G, pool, a0)
    want = check_scan(hip, d)
    with Graph(mem=1 << 20) as g:
        n = scan_node(g, d)
        g.buf = g.core.ggml_backend_alloc_ctx_tensors(g.ctx, hip)
        for t, v in g.inputs:
            g.core.ggml_backend_tensor_set(t, ptr(v), 0, v.nbytes)
        assert static(g, hip, n) == 0
        assert np.array_equal(g.read(n), want)


def test_scans_of_a_graph_share_their_scratch(hip):
    """Scans whose scratch would not fit the static area together, the larger ones later."""
    ds = [draw(np.random.default_rng(34 + S), S, 50, 8, 4, 256, 8, S, 1) for S in (20, 40, 50, 56)]
    with Graph(mem=1 << 20) as g:
        nodes = [scan_node(g, d) for d in ds]
        sizes = [gl.libs()["hip"].ggml_backend_hip_scan_scratch(n) for n in nodes]
        assert sum(sizes) > 136 << 20 and max(sizes) <= 96 << 20
        g.buf = g.core.ggml_backend_alloc_ctx_tensors(g.ctx, hip)
        for t, v in g.inputs:
            g.core.ggml_backend_tensor_set(t, ptr(v), 0, v.nbytes)
        assert static(g, hip, *nodes) == 0
        for n, d in zip(nodes, ds):
            y, h, ye, he = ssm_ref.scan(d["state"][d["ids"]], d["x"], d["dt"], d["A"], d["B"], d["C"])
            out = g.read(n)
            near(out[:y.size], y, ye)
            near(out[y.size:], h, he)


def test_refused_graphs_run_nothing(hip, capfd):
    """A refused node fails the whole graph before its first kernel: the copy beside it is not made."""
    with Graph(mem=1 << 20) as g:
        a = g.tensor(gl.F32, 16, data=np.ones(16, np.float32))
        b = g.tensor(gl.F32, 16, data=np.zeros(16, np.float32))
        d = draw(np.random.default_rng(5), 1, 2, 2, 4, 8, 1, 1, 1)
        s = g.tensor(gl.F32, 8, 4, 2, 1, data=d["state"])
        x = g.tensor(gl.F32, 4, 2, 2, 1, data=d["x"])
        dt = g.tensor(gl.F32, 2, 2, 1, data=d["dt"])
        bc = g.tensor(gl.F32, 8, 1, 2, 1, data=d["B"])
        n = g.ssm_scan(s, x, dt, g.tensor(gl.F32, 1, 2, data=d["A"]), bc, bc, g.tensor(gl.I32, 1, data=d["ids"]), 3)
        gf = g.core.ggml_new_graph(g.ctx)
        for t in (g.cpy(a, b), n):
            g.core.ggml_build_forward_expand(gf, t)
        g.buf = g.core.ggml_backend_alloc_ctx_tensors(g.ctx, hip)
        for t, v in g.inputs:
            g.core.ggml_backend_tensor_set(t, ptr(v), 0, v.nbytes)
        assert g.core.ggml_backend_graph_compute(hip, gf) == -1
        assert gl.libs()["hip"].ggml_backend_hip_graph_compute_static(hip, gf) == -1
        assert not g.read(b).any()
    assert "version 1 only" in capfd.readouterr().err


def run_with_state_copy(hip, d, kind, fusion):
    """y and the memory the final states are copied to; `kind`: what else the graph does with either."""
    S, T, H, P = d["x"].shape
    pool, _, _, N = d["state"].shape
    one = H * P * N
    gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, fusion)
    try:
        with Graph(mem=1 << 20) as g:
            n = scan_node(g, d)
            s = n.contents.src[0]
            y = g.view_1d(n, S * T * H * P, 0)
            states = g.view_1d(n, S * one, S * T * H * P * 4)
            other = g.tensor(gl.F32, S * one, data=np.zeros(S * one, np.float32))
            to = {"apart": other, "read_between": other}.get(kind)
            if to is None:
                to = g.view_1d(s, S * one, 0)
            outs = [g.scale(y, 1.0)]
            if kind == "old":
                outs.append(g.scale(g.reshape_2d(s, N * P, H * pool), 2.0))       # the pool's old rows, read after the scan
            if kind == "read_between":
                outs.append(g.scale(other, 2.0))
            if kind == "states":
                outs.append(g.scale(states, 3.0))
            if kind == "across":
                outs.append(g.scale(g.view_1d(n, 2 * H * P, max(S * T * H * P - H * P, 0) * 4), 2.0))
            copy = g.cpy(states, to)
            got = g.compute(hip, outs + [copy])
            return got, g.read(s)
    finally:
        gl.libs()["hip"].ggml_backend_hip_set_fusion(hip, True)


@pytest.mark.parametrize("kind", ["pool", "apart", "old", "read_between", "states", "across"])
@pytest.mark.parametrize("S, T, H, P, N, G, pool, a0", [
    (1, 1, 4, 64, 128, 2, 1, 1), (1, 5, 3, 3, 20, 1, 1, 20), (1, 100, 4, 64, 128, 1, 1, 1), (1, 1000, 4, 64, 128, 1, 1, 1),
    (1, 1, 130, 1, 16, 1, 1, 16), (1, 300, 130, 1, 16, 1, 1, 16), (1, 3, 5, 2, 7, 1, 1, 1), (3, 1, 4, 64, 128, 2, 3, 1),
    (3, 2, 65, 1, 16, 1, 4, 16), (2, 200, 4, 32, 64, 1, 2, 1)])
def test_scan_with_its_state_copied(hip, S, T, H, P, N, G, pool, a0, kind):
    """The copy of the final states into the pool or elsewhere, with and without fusion: the same values,
    whatever else reads the states, the old ones, or the memory that they go to."""
    d = draw(np.random.default_rng(S + T + H + N), S, T, H, P, N, G, pool, a0)
    want, pool_want = run_with_state_copy(hip, d, kind, False)
    got, pool_got = run_with_state_copy(hip, d, kind, True)
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
    assert np.array_equal(pool_got, pool_want)
    y, h, ye, he = ssm_ref.scan(d["state"][d["ids"]], d["x"], d["dt"], d["A"], d["B"], d["C"])
    near(got[0], y, ye)
    near(got[-1], h, he)


def test_refuses_memory_of_another_backend(hip, capfd):
    """Operands in host memory are named, not read."""
    cpu = cpu_backend(1)
    d = draw(np.random.default_rng(6), 1, 2, 2, 4, 8, 1, 1, 1)
    with Graph(mem=1 << 20) as g:
        n = scan_node(g, d)
        gf = g.core.ggml_new_graph(g.ctx)
        g.core.ggml_build_forward_expand(gf, n)
        g.buf = g.core.ggml_backend_alloc_ctx_tensors(g.ctx, cpu)
        assert g.core.ggml_backend_graph_compute(hip, gf) == -1
        assert gl.libs()["hip"].ggml_backend_hip_graph_compute_static(hip, gf) == -1
    gl.libs()["core"].ggml_backend_free(cpu)
    assert "not in this device's memory" in capfd.readouterr().err


@pytest.mark.parametrize("which", ["x", "result"])
def test_refuses_host_memory_without_a_buffer(hip, which, capfd):
    """A tensor that the caller placed itself has no buffer to tell its memory by: a context's own memory is
    named, not read or written; device memory runs."""
    d = draw(np.random.default_rng(7), 1, 2, 2, 4, 8, 1, 1, 1)
    host = np.zeros(4096, np.float32)
    with Graph(mem=1 << 20) as g:
        n = scan_node(g, d)
        want = g.compute(hip, n)
        gf = g.core.ggml_new_graph(g.ctx)
        g.core.ggml_build_forward_expand(gf, n)
        t = n if which == "result" else n.contents.src[1]
        held, at = t.contents.buffer, t.contents.data
        t.contents.buffer = None
        assert g.core.ggml_backend_graph_compute(hip, gf) == 0
        t.contents.data = host.ctypes.data
        assert g.core.ggml_backend_graph_compute(hip, gf) == -1
        assert gl.libs()["hip"].ggml_backend_hip_graph_compute_static(hip, gf) == -1
        t.contents.buffer, t.contents.data = held, at
        assert np.array_equal(g.read(n), want) and not host.any()
    assert capfd.readouterr().err.count("not in this device's memory") == 2
