"""The state space mixers' operators without a device: the shapes their constructors give and what
the HIP backend refuses (ggml_backend_hip_refusal, the check graph_compute makes before it queues
anything)."""
import numpy as np
import pytest

import ssm_ref
from gl import Graph, gl


def refusal(node):
    why = gl.libs()["hip"].ggml_backend_hip_refusal(node)
    return why.decode() if why else None


def scan_operands(g, N=16, P=4, H=6, T=5, S=2, G=2, pool=3, a0=1, t=gl.F32):
    return dict(s=g.tensor(t, N, P, H, pool), x=g.tensor(t, P, H, T, S), dt=g.tensor(t, H, T, S), A=g.tensor(t, a0, H),
                B=g.tensor(t, N, G, T, S), C=g.tensor(t, N, G, T, S), ids=g.tensor(gl.I32, S))


def scan(g, version=1, **o):
    return g.ssm_scan(o["s"], o["x"], o["dt"], o["A"], o["B"], o["C"], o["ids"], version)


def test_scan_takes_states_from_a_pool():
    with Graph(mem=1 << 20) as g:
        n = scan(g, **scan_operands(g))
        assert n.contents.ne[0] == 4 * 6 * 5 * 2 + 16 * 4 * 6 * 2   # the two sequences' states, not the pool's three
        assert refusal(n) is None


@pytest.mark.parametrize("o", [dict(a0=16), dict(N=256), dict(P=1, a0=16, G=1), dict(T=0), dict(T=1, S=1, pool=1), dict(G=6)])
def test_scan_accepts(o):
    with Graph(mem=1 << 20) as g:
        assert refusal(scan(g, **scan_operands(g, **o))) is None


@pytest.mark.parametrize("change, says", [
    (dict(version=2), "version"),
    (dict(version=0), "version"),
    (dict(N=257), "states per channel"),
    (dict(a0=2), "extents"),
    (dict(G=4), "groups"),
])
def test_scan_refuses(change, says):
    with Graph(mem=1 << 20) as g:
        version = change.pop("version", 1)
        assert says in refusal(scan(g, version=version, **scan_operands(g, **change)))


@pytest.mark.parametrize("name, ne, t", [
    ("x", (4, 6, 5, 1), gl.F32), ("dt", (6, 4, 2), gl.F32), ("dt", (6, 5, 2), gl.F16), ("A", (1, 5), gl.F32),
    ("B", (16, 2, 5, 1), gl.F32), ("B", (8, 2, 5, 2), gl.F32), ("C", (16, 1, 5, 2), gl.F32), ("C", (16, 2, 6, 2), gl.F32),
    ("ids", (3,), gl.I32), ("ids", (2,), gl.F32), ("s", (16, 4, 5, 3), gl.F32), ("s", (16, 4, 6, 3), gl.F16),
])
def test_scan_refuses_an_operand(name, ne, t):
    with Graph(mem=1 << 20) as g:
        o = scan_operands(g)
        o[name] = g.tensor(t, *ne)
        assert refusal(scan(g, **o))


def test_scan_without_ids_is_built_and_refused():
    with Graph(mem=1 << 20) as g:
        o = dict(scan_operands(g), ids=None)
        n = scan(g, **o)
        assert n.contents.ne[0] == 4 * 6 * 5 * 2 + 16 * 4 * 6 * 3
        assert "missing" in refusal(n)


def test_scan_refuses_strides_it_cannot_read():
    with Graph(mem=1 << 20) as g:
        o = scan_operands(g)
        wide = g.tensor(gl.F32, 64 * 5 * 2)
        o["B"] = g.view_4d(wide, 16, 2, 5, 2, 64, 128, 640, 0)
        assert refusal(scan(g, **o)) is None
        for nb in ((66, 128, 640), (64, 128, 2000)):          # not whole floats; past the tensor's end
            o["B"] = g.view_4d(wide, 16, 2, 5, 2, *nb, 0)
            assert refusal(scan(g, **o))
        o["B"] = g.permute(g.tensor(gl.F32, 2, 16, 5, 2), 1, 0, 2, 3)   # states not contiguous
        assert refusal(scan(g, **o))


def test_conv_refuses():
    with Graph(mem=1 << 20) as g:
        w = g.tensor(gl.F32, 4, 16)
        assert refusal(g.ssm_conv(g.tensor(gl.F32, 7, 16, 2), w)) is None
        assert refusal(g.ssm_conv(g.tensor(gl.F32, 3, 16, 2), w)) is None            # no new tokens
        assert refusal(g.ssm_conv(g.transpose(g.tensor(gl.F32, 16, 7)), w)) is None  # any strides
        assert "F32" in refusal(g.ssm_conv(g.tensor(gl.F16, 7, 16, 2), w))
        assert "F32" in refusal(g.ssm_conv(g.tensor(gl.F32, 7, 16, 2), g.tensor(gl.F16, 4, 16)))
        assert "extents" in refusal(g.ssm_conv(g.tensor(gl.F32, 7, 16, 2), g.tensor(gl.F32, 4, 16, 2)))
        assert "extents" in refusal(g.ssm_conv(g.tensor(gl.F32, 7, 16, 2, 2), w))
        wide = g.tensor(gl.F32, 7 * 16)
        assert refusal(g.ssm_conv(g.tensor(gl.F32, 32, 16), g.tensor(gl.F32, 32, 16))) is None
        assert "taps" in refusal(g.ssm_conv(g.tensor(gl.F32, 33, 16), g.tensor(gl.F32, 33, 16)))
        assert "past" in refusal(g.ssm_conv(g.view_3d(wide, 7, 16, 1, 32, 448, 0), w))
        assert "whole elements" in refusal(g.ssm_conv(g.view_3d(wide, 5, 16, 1, 22, 352, 0), w))


def test_refuses_what_no_launch_takes():
    with Graph(mem=1 << 20) as g:
        conv = lambda D, T: refusal(g.ssm_conv(g.tensor(gl.F32, 3 + T, D), g.tensor(gl.F32, 4, D)))  # noqa: E731
        assert conv(10240, 1 << 20) is None and conv(1, 1 << 26) is None and conv(1 << 30, 1) is None
        assert "too many" in conv(10240, 1 << 21) and "too many" in conv(1, (1 << 26) + 1) and "too many" in conv(1 << 31, 0)
        many = lambda S, H, P: refusal(scan(g, **scan_operands(g, S=S, H=H, P=P, T=1, G=1, pool=1)))  # noqa: E731
        assert many(4096, 128, 64) is None and many(1, 1 << 25, 1) is None
        assert "channels" in many(4097, 128, 64) and "channels" in many(1, (1 << 25) + 1, 1) and "channels" in many(1, 1 << 20, 1 << 12)


@pytest.mark.parametrize("T", [1, 17, 64, 65, 4096, 1 << 17])
@pytest.mark.parametrize("S", [1, 2, 33, 96, 512, 4095, 70000])
@pytest.mark.parametrize("N, P, H, G, a0", [(128, 64, 128, 8, 1), (256, 64, 16, 16, 1), (256, 1, 600, 600, 1), (16, 1, 512, 1, 16), (32, 1, 64, 1, 32),
                                            (64, 1000, 8, 2, 1), (1, 1, 1, 1, 1)])
def test_scan_scratch_is_bounded(S, T, N, P, H, G, a0):
    """96 MiB, and for more than a block of tokens two copies of the states, whatever the number of sequences."""
    with Graph(mem=1 << 20) as g:
        n = scan(g, **scan_operands(g, N=N, P=P, H=H, T=T, S=S, G=G, pool=1, a0=a0))
        got = gl.libs()["hip"].ggml_backend_hip_scan_scratch(n)
        if refusal(n):
            assert got == 0
        elif T <= 64:
            assert got <= 96 << 20
        else:
            assert got <= (96 << 20) + 2 * S * N * P * H * 4


@pytest.mark.parametrize("P, a0", [(4, 1), (1, 16)])
def test_scan_of_no_sequences_takes_no_scratch(P, a0):
    with Graph(mem=1 << 20) as g:
        n = scan(g, **scan_operands(g, S=0, T=100, P=P, H=64, G=1, a0=a0))
        assert refusal(n) is None and gl.libs()["hip"].ggml_backend_hip_scan_scratch(n) == 0


def test_scan_scratch_of_other_nodes():
    with Graph(mem=1 << 20) as g:
        lib = gl.libs()["hip"]
        assert lib.ggml_backend_hip_scan_scratch(None) == 0
        assert lib.ggml_backend_hip_scan_scratch(g.silu(g.tensor(gl.F32, 8))) == 0
        assert lib.ggml_backend_hip_scan_scratch(scan(g, version=2, **scan_operands(g, T=100))) == 0
        assert lib.ggml_backend_hip_scan_scratch(scan(g, **scan_operands(g, T=1))) == 0
        assert lib.ggml_backend_hip_scan_scratch(scan(g, **scan_operands(g, T=100))) > 0


def test_other_nodes_are_not_refused():
    with Graph(mem=1 << 20) as g:
        a = g.tensor(gl.F32, 8, 3)
        assert refusal(g.silu(a)) is None
        assert refusal(None)


def test_reference_scan_is_the_closed_form():
    """One channel, constant inputs: h_t = b (1 - a^t) / (1 - a) + a^t h_0."""
    T, d, A, B, x, h0 = 9, 0.3, -0.7, 1.5, 2.0, 0.25
    dt = np.log(np.expm1(d))
    one = np.ones((1, T, 1, 1))
    y, h, ye, he = ssm_ref.scan(np.full((1, 1, 1, 1), h0), x * one, np.full((1, T, 1), dt), np.full((1, 1), A), B * one, one)
    a, b = np.exp(d * A), d * x * B
    want = b * (1 - a ** np.arange(1, T + 1)) / (1 - a) + a ** np.arange(1, T + 1) * h0
    assert np.allclose(y.ravel(), want, rtol=1e-13) and np.allclose(h.ravel(), want[-1:], rtol=1e-13)
    assert (ye > 0).all() and ye.max() < 1e-3
