"""What the operators of the paged cache compute, in float64 numpy, each with a bound on how far 32-bit
results may be off (derived beside it)."""
import numpy as np

MROPE, VISION, IMROPE = 8, 24, 40
U32, U64 = 2.0 ** -24, 2.0 ** -53


# ---- rotations of several axes ----
def corr_dims(n_dims, n_ctx_orig, base, beta_fast, beta_slow):
    at = lambda rot: n_dims * np.log(n_ctx_orig / (rot * 2 * np.pi)) / (2 * np.log(base))  # noqa: E731
    return max(np.floor(at(beta_fast)), 0), min(np.ceil(at(beta_slow)), n_dims - 1)


def rope_angles(pos, n_dims, sections, mode, base, freq_scale=1.0, ext=0.0, attn=1.0, beta_fast=32.0, beta_slow=1.0,
                n_ctx_orig=0, ff=None):
    """(angles [T, pairs], the factor of cosines and sines) for positions [4, T]."""
    base, freq_scale, ext, attn = (float(np.float32(v)) for v in (base, freq_scale, ext, attn))
    pairs = n_dims if mode == VISION else n_dims // 2
    theta = np.zeros((pos.shape[1], pairs))
    mscale = attn * (1 + 0.1 * np.log(1 / freq_scale)) if ext else attn
    for i in range(pairs):
        sector, axis, e = i % sum(sections), 0, i
        if mode == IMROPE:
            axis = sector % 3 if sector < 3 * sections[sector % 3] else 3
        else:
            ends = np.cumsum(sections)
            axis = int(np.searchsorted(ends, sector, side="right"))
            if mode == VISION:
                e = sector - (ends[axis] - sections[axis])
        t = pos[axis].astype(np.float64) * base ** (-2.0 * e / n_dims)
        if ff is not None:
            t = t / float(ff[i])
        m = freq_scale
        if ext:
            lo, hi = corr_dims(n_dims, n_ctx_orig, base, beta_fast, beta_slow)
            mix = (1 - min(1, max(0, (i - lo) / max(0.001, hi - lo)))) * ext
            m = freq_scale * (1 - mix) + mix
        theta[:, i] = t * m
    return theta, mscale


def rope(x, pos, n_dims, sections, mode, base, **kw):
    """x [T, H, D] -> (y, bound). Turns are a product of three rounded factors (and a quotient): 4 units of 64 bits of
    the angle here and as much there; the rotation is rounded to 32 bits once."""
    theta, mscale = rope_angles(pos, n_dims, sections, mode, base, **kw)
    pairs = theta.shape[1]
    y, x = x.astype(np.float64).copy(), x.astype(np.float64)
    c, s = np.cos(theta)[:, None] * mscale, np.sin(theta)[:, None] * mscale
    a, b = x[:, :, :pairs], x[:, :, pairs:2 * pairs]
    y[:, :, :pairs], y[:, :, pairs:2 * pairs] = a * c - b * s, a * s + b * c
    bound = U32 * np.abs(y)
    off = (8 * np.abs(theta)[:, None] + 16) * U64 * np.hypot(a, b) * abs(mscale)
    bound[:, :, :pairs] += off
    bound[:, :, pairs:2 * pairs] += off
    bound[:, :, 2 * pairs:] = 0
    return y, bound


# ---- attention over pages ----
def attention(q, k, v, pages, q_start, kv_len, scale):
    """q [T, H, D]; k, v [n_pages, page, KV, D] (the values held); pages [S, max]. -> (o [T, H, D], bound, listed [T])

    The bound: scores are sums of D products of 24-bit values whose parts (a query in two halves of 11 bits, a sum a
    block, its scale) are off by less than 8 units of 32 bits of sum |q k|, and so is log2(e) times them; p = e^(s - m)
    is off by that and by 2 units more; a term p v by 4 (p d in two halves of 11 bits); sums in parts of at most 64 terms,
    then joined, by 64 + 40. Numerator and denominator both: 2 max_j(8 scale sum |q k| + 2) + 2 (4 + 104) units of
    sum p |v| / sum p. What is absolute: p below 2^-126 ends the range of 32-bit floats, and operands of the
    products in two halves of 11 bits end at 2^-25, half the smallest F16. They are scaled so that the largest p (it may
    be 2^4 times the one that is divided by) and the largest scale d make at most 2^15: where d's largest is at 2^9 or
    more, a term p d c, |c| <= 8, may lose 2^-34 max |v|, max |v| = 8 max d, and a scale far below the largest of its kind
    as much again: 2^-33 max |v| for each of the n terms, and sum p >= 1 divides it."""
    T, H, D = q.shape
    page, KV = k.shape[1:3]
    o, bound, listed = np.zeros(q.shape), np.zeros(q.shape), np.zeros(T, bool)
    scale = float(np.float32(scale))
    for s in range(len(kv_len)):
        a = min(max(int(q_start[s]), 0), T)
        b = min(max(int(q_start[s + 1]), a), T)
        n = min(max(int(kv_len[s]), 0), pages.shape[1] * page)
        at = np.arange(n)
        pg = pages[s][at // page]
        there = (pg >= 0) & (pg < len(k))
        kk, vv = (x[np.where(there, pg, 0), at % page].astype(np.float64) for x in (k, v))
        for t in range(a, b):
            listed[t] = True
            see = there & (at <= int(kv_len[s]) - (b - a) + (t - a))
            if not see.any():
                continue
            for h in range(H):
                kh, vh, qh = kk[see, h // (H // KV)], vv[see, h // (H // KV)], q[t, h].astype(np.float64)
                z = scale * (kh @ qh)
                p = np.exp(z - z.max())
                w = p / p.sum()
                o[t, h] = w @ vh
                most = (abs(scale) * (np.abs(kh) @ np.abs(qh))).max()
                lost = see.sum() * 2.0 ** -33 * np.abs(vv[see]).max()
                bound[t, h] = U32 * (16 * most + 4 + 216) * (w @ np.abs(vh)) + lost
    return o, bound, listed


# ---- drafted tokens ----
def verify(p, q, drafted, tokens, u):
    """p [sum(n + 1), V], q [sum(n), V] or None -> (accepted, token) of each sequence."""
    accepted, picked, r, d = [], [], 0, 0
    for n in drafted:
        n, k = int(n), 0
        while k < n:
            tok = int(tokens[d + k])
            qd = 1.0 if q is None else float(q[d + k, tok])
            if not float(u[r + k]) * qd < float(p[r + k, tok]):
                break
            k += 1
        w = np.maximum(p[r + k].astype(np.float64), 0)
        if k < n:
            less = w.copy()
            if q is None:
                less[int(tokens[d + k])] = 0
            else:
                less = np.maximum(p[r + k].astype(np.float64) - q[d + k].astype(np.float64), 0)
            if less.sum() != 0:
                w = less
        total = w.sum()
        if not (np.isfinite(total) and total > 0):
            picked.append(-1)
        else:
            c = np.cumsum(w)
            picked.append(min(int((c <= float(u[r + n]) * c[-1]).sum()), int(np.nonzero(w > 0)[0][-1])))
        accepted.append(k)
        r += n + 1
        d += n
    return np.array(accepted, np.int32), np.array(picked, np.int32)
