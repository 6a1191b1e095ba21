"""The state space mixers' operators in float64, each with a bound on the error of a float32
evaluation that is carried through the same recurrence (u = 2^-24, half a step of float32).

scan: a step forms exp(d A) from a softplus (a series and a 2^x instruction: 4 u of it, 4 u with the
product by A and by log2 e, so 8 u |d A| with both) and another 2^x (2 u), multiplies and adds (2 u),
and adds d x B (4 u). Decays over up to 128 tokens may be formed from one running sum of their
exponents, whose rounding (8 u of the sum of |d A| over them) every such decay inherits. The output
adds N products: at most (2 + 8 + N / 8) u of their absolute sum, for lanes that hold up to N / 8 of
them, or 32 u where one lane holds up to 32; a state that matrix products form adds up to 64 products
per pass, 64 u of the absolute state, which covers that too.
"""
import numpy as np

U = 2.0 ** -24


def softplus(x):
    x = np.asarray(x, np.float64)
    return np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x)))


def silu(x):
    return x / (1 + np.exp(-x))


def conv(sx, w, bias=None, act=False):
    """sx [S, D, K - 1 + T], w [D, K] -> y [S, T, D] and its bound."""
    sx, w = np.asarray(sx, np.float64), np.asarray(w, np.float64)
    K = w.shape[1]
    T = sx.shape[2] - K + 1
    y, mag = np.zeros((sx.shape[0], T, sx.shape[1])), np.zeros((sx.shape[0], T, sx.shape[1]))
    for k in range(K):
        part = (sx[:, :, k:k + T] * w[:, k][None, :, None]).transpose(0, 2, 1)
        y += part
        mag += np.abs(part)
    if bias is not None:
        y, mag = y + bias, mag + np.abs(bias)
    err = (K + 2) * U * mag
    if act:
        out = silu(y)
        # |silu'| <= 1.1; e^-y is off by up to 2 u (1 + |y|) of itself, the sum and quotient by 3 u
        return out, 1.1 * err + (6 + 2 * np.abs(y)) * U * np.abs(out)
    return y, err


def scan(h0, x, dt, A, B, C):
    """h0 [S, H, P, N], x [S, T, H, P], dt [S, T, H], A [H, N or 1], B, C [S, T, G, N] ->
    y [S, T, H, P], h [S, H, P, N] and the two bounds."""
    x, A, B, C = (np.asarray(a, np.float64) for a in (x, A, B, C))
    S, T, H, P = x.shape
    N, per = B.shape[3], H // B.shape[2]
    d = softplus(dt)
    h = np.asarray(h0, np.float64).copy()
    mag, err = np.abs(h), np.zeros_like(h)
    y, ye = np.zeros(x.shape), np.zeros(x.shape)
    expo = d[..., None] * np.abs(A)                                    # [S, T, H, 1 or N]
    run = np.concatenate([np.zeros((S, 1) + expo.shape[2:]), np.cumsum(expo, 1)], 1)
    for t in range(T):
        b, c = (np.repeat(m[:, t], per, 1)[:, :, None] for m in (B, C))
        a = np.exp(d[:, t, :, None] * A)[:, :, None]
        new = (d[:, t, :, None] * x[:, t])[..., None] * b
        step = (8 * expo[:, t][:, :, None] + 4) * U
        err = a * (err + mag * step) + 4 * U * np.abs(new)
        h = a * h + new
        mag = a * mag + np.abs(new)
        window = run[:, t + 1] - run[:, max(0, t + 1 - 128)]
        here = err + mag * U * (8 * window[:, :, None] + 64)
        y[:, t] = (h * c).sum(3)
        ye[:, t] = (np.abs(c) * (here + mag * U * (10 + N / 8))).sum(3)
    window = run[:, T] - run[:, max(0, T - 128)]
    return y, h, ye, err + mag * U * (8 * window[:, :, None] + 64)
