"""ggml_backend_hip_logprobs against float64.

The bound (u = 2^-24): z = l - max rounds once (u |z|), e^z is off by 2 u (1 + |z|) of itself, and a
32-bit sum of n of them in at least 256 partial sums by (n / 256 + 10) u. So log S is off by
(n / 256 + 12 + 2 max|z| w) u plus its own rounding, with w |z| <= 1 for e^z's weight; a log
probability adds z's rounding and two of its own, the entropy (a weighted mean of z <= log n) the
same again, times log n.
"""
import numpy as np
import pytest

from gl import Graph, gl, ptr

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def hip():
    b = gl.hip_backend(0)
    yield b
    gl.libs()["core"].ggml_backend_free(b)


class Rows:
    def __init__(self, backend, rows, ne=None):
        rows = np.ascontiguousarray(rows, np.float32)
        self.g = Graph(mem=1 << 20)
        self.t = self.g.tensor(gl.F32, *(ne or rows.shape[::-1]))
        self.g.buf = self.g.core.ggml_backend_alloc_ctx_tensors(self.g.ctx, backend)
        self.g.core.ggml_backend_tensor_set(self.t, ptr(rows), 0, rows.nbytes)

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.g.close()


def reference(x):
    """log p, entropy and order of each row in float64; NaN where a row has no distribution."""
    x = np.asarray(x, np.float64)
    ok = ~np.isnan(x).any(1) & np.isfinite(x.max(1, initial=-np.inf, where=~np.isnan(x)))
    with np.errstate(all="ignore"):
        z = x - x.max(1, keepdims=True)
        p = np.exp(z)
        s = p.sum(1, keepdims=True)
        lp = z - np.log(s)
        ent = -(np.where(p > 0, p * lp, 0) / s).sum(1)
    lp[~ok], ent[~ok] = np.nan, np.nan
    order = np.argsort(-np.where(np.isnan(x), -np.inf, x), axis=1, kind="stable")
    return lp, ent, order


def check(hip, x, tokens, n_top, row=0, t=None):
    n = x.shape[1]
    if t is None:
        with Rows(hip, x) as r:
            got = gl.hip_logprobs(hip, r.t, tokens, row=row, n_top=n_top)
    else:
        got = gl.hip_logprobs(hip, t, tokens, row=row, n_top=n_top)
    lp, ent, order = reference(x[row:row + len(tokens)])
    at = np.arange(len(tokens))
    base = (n / 256 + 24 + 4 * np.log(n)) * U

    def close(got, want, bound):
        bad = ~np.isfinite(want)
        assert np.array_equal(got[bad], want[bad].astype(np.float32), equal_nan=True)
        assert (np.abs(got[~bad] - want[~bad]) <= np.broadcast_to(bound, want.shape)[~bad]).all()

    want = lp[at, tokens]
    close(got[0], want, base + 4 * U * np.abs(want))
    close(got[1], ent, base * (2 + np.log(n)))
    assert np.array_equal(got[2], order[:, :n_top])
    want = np.take_along_axis(lp, order[:, :n_top], 1)
    close(got[3], want, base + 4 * U * np.abs(want))
    return got


@pytest.mark.parametrize("n, rows, n_top", [(1, 1, 1), (2, 3, 2), (7, 4, 7), (64, 2, 0), (255, 5, 128), (257, 3, 20), (1000, 33, 5), (57345, 2, 20), (57345, 1, 128),
                                            (4099, 9, 128), (32064, 37, 20), (151936, 1, 20), (151936, 2, 128), (128256, 300, 1),
                                            (151936, 1, 0), (50257, 2, 64), (8192, 3, 100), (8193, 3, 100), (600001, 1, 128)])
def test_scores(hip, n, rows, n_top):
    rng = np.random.default_rng(n + rows)
    x = (rng.standard_normal((rows, n)) * 3).astype(np.float32)
    x[:, rng.integers(0, n)] += 9
    check(hip, x, rng.integers(0, n, rows), n_top)


@pytest.mark.parametrize("n", [5, 300, 5000, 40000])
@pytest.mark.parametrize("n_top", [0, 5])
def test_rows_of_every_kind(hip, n, n_top):
    """Equal logits, ascending and descending rows, banned tokens, one token left, large values, and
    rows without a distribution (nothing left, a NaN, an infinity)."""
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((12, n)) * 2).astype(np.float32)
    x[0] = 0.5
    x[1] = np.round(x[1] * 2) / 2
    x[2], x[3] = np.sort(x[2]), -np.sort(-x[3])
    x[4, rng.random(n) < 0.9] = -np.inf
    x[4, 1] = 0
    x[5] = -np.inf
    x[5, n // 2] = 3
    x[6] *= 1e30
    x[7] = -np.inf
    x[8, n // 3] = np.nan
    x[9, n - 1] = np.inf
    x[10] = np.finfo(np.float32).min
    x[11, :] = np.where(rng.random(n) < 0.5, -0.0, 0.0)
    check(hip, x, rng.integers(0, n, 12), n_top)


@pytest.mark.parametrize("n", [4500, 8192, 30000])
@pytest.mark.parametrize("n_top", [1, 3, 6, 12, 20, 40, 100])
def test_a_regular_pattern_of_banned_tokens(hip, n, n_top):
    """Every 1024 ids begin with 256 banned ones, or with 256 of one low value; the rest with and
    without equal values."""
    rng = np.random.default_rng(n + n_top)
    x = rng.standard_normal((6, n)).astype(np.float32)
    low = np.arange(n) % 1024 < 256
    x[0, low] = -np.inf
    x[1, low] = -5
    x[2] = np.round(x[2])
    x[2, low] = -np.inf
    x[3] = np.where(low, -np.inf, 1.0)
    x[4] = np.where(low, -4.0, np.where(np.arange(n) % 3 == 0, 1.0, 0.5))
    x[5, ~low] = -np.inf
    check(hip, x, rng.integers(0, n, 6), n_top)


@pytest.mark.parametrize("n", [700, 5000, 30000])
@pytest.mark.parametrize("n_top", [2, 7, 20, 33, 128])
def test_the_last_of_the_likeliest_among_equals(hip, n, n_top):
    """The n_top-th entry is one of many equal ones, of a sign that 0 has two of, next to the smallest
    floats or at the range's end; equal ones go by their ids."""
    rng = np.random.default_rng(n + n_top)
    x = -1 - rng.random((6, n), dtype=np.float32)
    some = [rng.permutation(n) for _ in range(6)]
    x[0, some[0][:200]] = np.where(rng.random(200) < 0.5, 0.0, -0.0)
    x[1, some[1][:200]] = np.where(rng.random(200) < 0.5, 1e-45, -1e-45)
    x[2] = -np.inf
    x[2, some[2][:300]] = -np.finfo(np.float32).max
    x[3] = rng.integers(0, 4, n)
    x[4] = 0
    x[5, some[5][:100]] = 1e-45
    x[5, some[5][100:200]] = 0.0
    for r in range(6):
        if r != 4:
            x[r, some[r][300:300 + n_top // 2]] = 3.0        # some above them
    check(hip, x, rng.integers(0, n, 6), n_top)


@pytest.mark.parametrize("n_top", [1, 20, 128])
def test_very_long_rows(hip, n_top):
    """Rows of so many segments that their lists are too long to compare each entry with all: an ordinary row, one
    with segments that hold nothing, one with few values that are all equal, and equal values throughout."""
    n = 4_200_001
    rng = np.random.default_rng(n_top)
    x = (rng.standard_normal((4, n), dtype=np.float32) * 3)
    x[1, 100_000:150_000] = -np.inf
    x[2] = -np.inf
    x[2, rng.permutation(n)[:n_top // 2 + 1]] = 1.0
    x[3] = np.round(x[3])
    check(hip, x, rng.integers(0, n, 4), n_top)


def test_a_banned_token(hip):
    x = np.array([[0, -np.inf, 1]], np.float32)
    got = check(hip, x, np.array([1]), 3)
    assert got[0][0] == -np.inf and list(got[2][0]) == [2, 0, 1] and got[3][0, 2] == -np.inf


def test_some_rows_and_some_outputs(hip):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((24, 700)).astype(np.float32)
    with Rows(hip, x, (700, 4, 3, 2)) as r:
        check(hip, x, rng.integers(0, 700, 5), 3, row=17, t=r.t)
        check(hip, x, rng.integers(0, 700, 24), 3, t=r.t)
        lib = gl.libs()["hip"]
        ent = np.zeros(2, np.float32)
        assert lib.ggml_backend_hip_logprobs(hip, r.t, 22, 2, None, 0, None, ptr(ent), None, None) == 0
        assert np.allclose(ent, reference(x[22:])[1], rtol=1e-4)
        ids = np.zeros((2, 4), np.int32)
        assert lib.ggml_backend_hip_logprobs(hip, r.t, 0, 2, None, 4, None, None, ptr(ids), None) == 0
        assert np.array_equal(ids, reference(x[:2])[2][:, :4])
        assert lib.ggml_backend_hip_logprobs(hip, r.t, 24, 0, None, 4, None, None, None, None) == 0
        out = gl.hip_logprobs(hip, r.t, None, row=3, n_rows=2, n_top=1)
        assert out[0] is None and np.array_equal(out[2], reference(x[3:5])[2][:, :1])


def test_strided_rows(hip):
    """Rows of a wider tensor that begin at any float, and a permuted order of them."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 1003)).astype(np.float32)
    with Graph(mem=1 << 20) as g:
        t = g.tensor(gl.F32, 1003, 6)
        v = g.view_2d(t, 997, 6, 1003 * 4, 5 * 4)
        p = g.permute(g.view_3d(t, 997, 3, 2, 1003 * 4, 3 * 1003 * 4, 0), 0, 2, 1, 3)
        g.buf = g.core.ggml_backend_alloc_ctx_tensors(g.ctx, hip)
        g.core.ggml_backend_tensor_set(t, ptr(x), 0, x.nbytes)
        check(hip, x[:, 5:5 + 997], rng.integers(0, 997, 6), 9, t=v)
        check(hip, x[[0, 3, 1, 4, 2, 5], :997], rng.integers(0, 997, 6), 9, t=p)


def test_more_rows_than_a_launch_takes(hip):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((16384 + 70, 12)).astype(np.float32)
    check(hip, x, rng.integers(0, 12, len(x)), 2)


def test_more_alternatives_than_the_download_area_holds(hip):
    """128 alternatives of each of 16384 + 70 rows are more than the pinned area's 16 MiB."""
    rng = np.random.default_rng(7)
    x = rng.standard_normal((16384 + 70, 130)).astype(np.float32)
    check(hip, x, rng.integers(0, 130, len(x)), 128)


def test_refuses_another_buffer(hip, capfd):
    with Graph(mem=1 << 20) as g:
        with pytest.raises(RuntimeError):
            gl.hip_logprobs(hip, g.tensor(gl.F32, 8, 2), [0, 1])
    assert "device buffer" in capfd.readouterr().err
