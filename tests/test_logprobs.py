"""What ggml_backend_hip_logprobs refuses, without a device: every check of the arguments comes
before the backend is looked at."""
import ctypes as C

import numpy as np
import pytest

from gl import Graph, gl, ptr

F = np.float32


def call(t, row=0, n_rows=1, tokens=(0,), n_top=0, logprob=True):
    toks = None if tokens is None else np.asarray(tokens, np.int32)
    out = np.full(max(len(toks) if toks is not None else 1, 1), 7, F)
    st = gl.libs()["hip"].ggml_backend_hip_logprobs(None, t, row, n_rows, None if toks is None else ptr(toks), n_top,
                                                    ptr(out) if logprob else None, None, None, None)
    assert st == -1 and (out == 7).all()


@pytest.mark.parametrize("args, says", [
    (dict(row=-1), "rows out of range"), (dict(row=3), "rows out of range"), (dict(n_rows=4), "rows out of range"),
    (dict(row=2, n_rows=2, tokens=(0, 0)), "rows out of range"), (dict(n_rows=-1), "rows out of range"),
    (dict(row=2 ** 62, n_rows=2 ** 62), "rows out of range"),
    (dict(n_top=-1), "n_top"), (dict(n_top=9), "n_top"), (dict(tokens=(8,)), "token out of range"),
    (dict(tokens=(-1,)), "token out of range"), (dict(n_rows=2, tokens=(0, 99)), "token out of range"),
    (dict(tokens=None), "no tokens"), (dict(), "not a HIP backend"), (dict(tokens=None, logprob=False), "not a HIP backend"),
    (dict(row=2, n_rows=1, n_top=8), "not a HIP backend"), (dict(row=3, n_rows=0, tokens=()), "not a HIP backend"),
])
def test_refusals(args, says, capfd):
    with Graph(mem=1 << 20) as g:
        call(g.tensor(gl.F32, 8, 3), **args)
    assert says in capfd.readouterr().err


def test_refuses_other_tensors(capfd):
    with Graph(mem=1 << 20) as g:
        call(None)
        assert "null" in capfd.readouterr().err
        a = g.tensor(gl.F32, 300, 3)
        for t in (g.tensor(gl.F16, 8, 3), g.transpose(a), g.view_2d(a, 8, 3, 34, 0), g.view_2d(a, 8, 3, 2000, 0)):
            call(t)
            assert "contiguous rows" in capfd.readouterr().err
        call(g.tensor(gl.F32, 8, 3), n_top=9)
        call(a, n_top=129)
        assert capfd.readouterr().err.count("n_top") == 2


def test_python_wrapper_checks():
    with Graph(mem=1 << 20) as g:
        t = g.tensor(gl.F32, 8, 3)
        with pytest.raises(ValueError):
            gl.hip_logprobs(None, t, None)
        with pytest.raises(ValueError):
            gl.hip_logprobs(None, t, [1, 2], n_rows=3)
        with pytest.raises(RuntimeError):
            gl.hip_logprobs(None, t, [1, 2])


@pytest.mark.parametrize("tokens", [[2 ** 32 + 1], np.array([2 ** 32 + 1]), np.array([-2 ** 32], np.int64), np.array([2 ** 32 - 1], np.uint32),
                                    [1.5], np.array([1.0], F), [True], ["1"], [[1]], np.array([2 ** 64 - 1], np.uint64)])
def test_python_wrapper_takes_no_token_for_another(tokens):
    """A token that is no 32-bit integer is refused, not cut to one that is in range."""
    with Graph(mem=1 << 20) as g:
        with pytest.raises(ValueError):
            gl.hip_logprobs(None, g.tensor(gl.F32, 8, 3), tokens)


@pytest.mark.parametrize("tokens", [[1], (1,), np.array([1], np.int64), np.array([1], np.uint8), []])
def test_python_wrapper_takes_integers_of_any_kind(tokens, capfd):
    with Graph(mem=1 << 20) as g:
        with pytest.raises(RuntimeError):
            gl.hip_logprobs(None, g.tensor(gl.F32, 8, 3), tokens)
    assert "not a HIP backend" in capfd.readouterr().err
