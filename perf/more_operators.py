"""Performance cases of serving several sequences from a paged cache.

Four kinds of work:

* ``rope``    rotation of query and key rows by positions of several axes (time, height, width)
* ``append``  keys and values of new tokens stored into the rows of a cache that the caller names
              (a page's row for each token), the keys rotated on the way; the cache in 4 bits or F16
* ``attn``    attention of the new tokens of several sequences over a cache held in 4 bits, each
              sequence's positions on pages of its own in any order
* ``verify``  drafted tokens accepted or replaced by the target's probabilities, from given random
              numbers

A token per sequence is a decoding step, a few are drafted tokens to be verified, hundreds a part of
a prompt. Rows come as a model has them: slices of one wide projection of queries, keys and values.

``run`` computes each in plain torch operations, or, where ``own`` is set, through the package's
graph operators and entry points.
"""
from __future__ import annotations

import ctypes as C
import importlib.util
import math
import os
import random
import sys
import zlib

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
F16, F32, F64, I32, U8 = torch.float16, torch.float32, torch.float64, torch.int32, torch.uint8
MROPE, VISION, IMROPE = 8, 24, 40
TYPE_F16, TYPE_Q4_0 = 1, 2
BASE = 1e6


# ---------------------------------------------------------------------------------------------
# the cases
#
# rope: T tokens of H heads of D values, in projections of H + 2 * KV heads; mode and sections
# append: T tokens of KV heads of D values, S sequences' pages of P rows in a cache of `pool` pages
# attn: S sequences of up to L positions (`even`: all of them near L), N new tokens each (`ragged`:
#       up to N), H query heads over KV heads of D values, pages of P rows
# verify: S sequences of up to N drafted tokens, V tokens to choose from; `q`: whether the drafts
#         come with their probabilities

def listed():
    return [
        # one decoding step of 16 sequences; a prompt of text and images
        dict(name="rope_step_16", kind="rope", T=16, H=32, KV=8, D=128, mode=IMROPE, sections="24,20,20,0"),
        dict(name="rope_prompt_2100", kind="rope", T=2100, H=32, KV=8, D=128, mode=MROPE, sections="16,24,24,0"),
        # decoding one sequence; a batch of decoding sequences with idle places, into an F16 cache; a prompt
        dict(name="append_step_1", kind="append", T=1, KV=8, D=128, P=16, pool=512, type=TYPE_Q4_0, idle=0),
        dict(name="append_step_96", kind="append", T=96, KV=8, D=128, P=64, pool=300, type=TYPE_F16, idle=5),
        dict(name="append_prompt_4096", kind="append", T=4096, KV=8, D=128, P=64, pool=256, type=TYPE_Q4_0, idle=0),
        # decoding one sequence, and a batch of sequences of very different lengths
        dict(name="attn_step_1", kind="attn", S=1, L=4113, N=1, H=32, KV=8, D=128, P=16, even=True, ragged=False),
        dict(name="attn_step_32", kind="attn", S=32, L=16384, N=1, H=24, KV=8, D=128, P=64, even=False, ragged=False),
        # every query head with a KV head of its own
        dict(name="attn_step_8_mha", kind="attn", S=8, L=2000, N=1, H=32, KV=32, D=96, P=32, even=False, ragged=False),
        # drafted tokens of 16 sequences, eight query heads over a KV head; a part of two prompts
        dict(name="attn_draft_16", kind="attn", S=16, L=8192, N=5, H=32, KV=4, D=128, P=16, even=False, ragged=True),
        dict(name="attn_prompt_2", kind="attn", S=2, L=8192, N=700, H=32, KV=8, D=128, P=64, even=True, ragged=True),
        # one sequence's drafts, and those of a batch
        dict(name="verify_1", kind="verify", S=1, N=4, V=151936, q=True),
        dict(name="verify_64", kind="verify", S=64, N=6, V=128256, q=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    kind = rng.choice(("rope", "append", "append", "attn", "attn", "attn", "verify"))
    if kind == "verify":
        return dict(kind=kind, S=_log(rng, 1, 64), N=rng.randint(1, 8), V=_log(rng, 500, 152000), q=rng.random() < 0.7)
    D, KV = rng.choice((64, 96, 128, 128)), rng.choice((1, 2, 4, 8, 8, 12))
    if kind == "rope":
        mode = rng.choice((MROPE, VISION, IMROPE))
        h = D // 2
        if mode == VISION:
            s = (h // 2, h - h // 2, 0, 0)
        elif mode == MROPE:
            t = rng.randint(1, h - 2)
            a = rng.randint(1, h - t - 1)
            s = (t, a, h - t - a, 0)
        else:
            a = rng.randint(1, h // 3)
            s = (h - 2 * a, a, a, 0)
        return dict(kind=kind, T=_log(rng, 1, 2100), H=KV * rng.choice((1, 2, 4)), KV=KV, D=D, mode=mode,
                    sections=",".join(map(str, s)))
    if kind == "append":
        T, P = _log(rng, 1, 4096), rng.choice((1, 16, 16, 24, 64, 128))
        return dict(kind=kind, T=T, KV=KV, D=D, P=P, pool=-(-T // P) + _log(rng, 2, 200),
                    type=rng.choice((TYPE_F16, TYPE_Q4_0)), idle=rng.choice((0, 0, rng.randint(0, T // 4))))
    S, N = rng.choice(((1, 1), (_log(rng, 2, 32), 1), (_log(rng, 1, 16), rng.randint(2, 8)), (rng.randint(1, 3), _log(rng, 20, 700))))
    return dict(kind=kind, S=S, L=max(_log(rng, 20, 16384), N), N=N, H=KV * rng.choice((1, 2, 3, 4, 8)), KV=KV, D=D,
                P=rng.choice((8, 16, 16, 48, 64, 100)), even=rng.random() < 0.5, ragged=N > 1 and rng.random() < 0.5)


def draw(rng: random.Random):
    most = {}
    for c in listed():
        for key, v in work(c).items():
            most[c["kind"], key] = max(v, most.get((c["kind"], key), 0))
    while True:
        case = _drawn(rng)
        if all(v <= most[case["kind"], key] for key, v in work(case).items()):
            return case


def _lengths(c):
    """New tokens and positions (the new ones among them) of each sequence, of the case alone."""
    r = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    S, L, N = c["S"], c["L"], c["N"]
    new = [max(1, N - r.randint(0, N // 2)) if c["ragged"] and i else N for i in range(S)]
    low = 0.9 * L if c["even"] else L / 60
    seen = [L] + [int(round(math.exp(r.uniform(math.log(max(1, low)), math.log(L))))) for _ in range(S - 1)]
    return new, [max(n, s) for n, s in zip(new, seen)]


def _drafted(c):
    r = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    return [c["N"]] + [r.randint(0, c["N"]) for _ in range(c["S"] - 1)]


# ---------------------------------------------------------------------------------------------
# seeded inputs

def _gen(seed, name):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) << 32) + zlib.crc32(name.encode()))
    return g


def _randn(seed, name, *shape):
    return torch.randn(*shape, generator=_gen(seed, name), device=DEV)


def _rand(seed, name, *shape):
    return torch.rand(*shape, generator=_gen(seed, name), device=DEV)


def _sections(c):
    return tuple(int(v) for v in c["sections"].split(","))


def _positions(c, seed):
    """[4, T]: text with images in between, whose tokens share a time and walk over a grid."""
    r, T = random.Random(seed), c["T"]
    pos, at = [], r.randint(0, 60000)
    while len(pos) < T:
        if r.random() < 0.5:
            n = r.randint(1, 300)
            pos += [(at + i,) * 3 for i in range(n)]
            at += n
        else:
            h, w = r.randint(4, 40), r.randint(4, 40)
            pos += [(at, at + y, at + x) for y in range(h) for x in range(w)]
            at += max(h, w)
    p = torch.tensor(pos[:T], dtype=I32).T
    return torch.cat([p, torch.zeros(1, T, dtype=I32)]).contiguous().to(DEV)


def _rope_inputs(c, seed):
    W = (c["H"] + 2 * c["KV"]) * c["D"]
    return dict(rows=_randn(seed, "rows", c["T"], W), pos=_positions(c, seed))


def _append_inputs(c, seed):
    T, KV, D, P = c["T"], c["KV"], c["D"], c["P"]
    G = 4
    d = dict(rows=_randn(seed, "rows", T, (G + 2) * KV * D), pos=_positions(c, seed))
    # a few channels of the keys stand out
    d["rows"][:, G * KV * D:(G + 1) * KV * D] *= torch.exp(0.5 * _randn(seed, "channels", KV * D))
    pages = _rand(seed, "pages", c["pool"]).argsort()[:-(-T // P)]
    rows = (pages[:, None] * P + torch.arange(P, device=DEV)).flatten()[:T]
    if T <= 256:
        # one token for each of T sequences: any rows of the pool
        rows = _rand(seed, "slots", c["pool"] * P).argsort()[:T]
    rows = rows.to(I32)
    if c["idle"]:
        rows[_rand(seed, "idle", T).argsort()[:c["idle"]]] = -1
    d["slots"] = rows
    return d


def _attn_inputs(c, seed):
    S, H, KV, D, P = (c[k] for k in ("S", "H", "KV", "D", "P"))
    new, seen = _lengths(c)
    used = [-(-s // P) for s in seen]
    pool = sum(used) + 3
    order = _rand(seed, "pages", pool).argsort().to(I32)
    table = torch.zeros(S, max(used), dtype=I32, device=DEV)
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    d = dict(q=1.7 * _randn(seed, "q", sum(new), H, D), table=table, start=torch.from_numpy(start).to(DEV),
             seen=torch.tensor(seen, dtype=I32, device=DEV))
    for name in ("k", "v"):
        x = _randn(seed, name, pool * P, KV, D)
        x *= torch.exp(0.4 * _randn(seed, name + "_channels", KV, D))
        d[name + "_d"], d[name + "_q"] = _quantized(x.view(pool * P, KV * D // 32, 32))
    # where each sequence's new tokens stand among all of them (the places past its last: its first)
    i = np.arange(max(new))
    d["place"] = torch.from_numpy(start[:-1, None] + np.where(i < np.array(new)[:, None], i, 0)).to(DEV)
    d["real"] = torch.from_numpy(np.flatnonzero((i < np.array(new)[:, None]).ravel())).to(DEV)
    return d


def _verify_inputs(c, seed):
    S, V = c["S"], c["V"]
    k = _drafted(c)
    rows, drafts = sum(k) + S, sum(k)
    logits = 2.5 * _randn(seed, "logits", rows, V)
    logits.scatter_add_(1, (_rand(seed, "peaks", rows, 8) * V).long(), 5 + 3 * _randn(seed, "heights", rows, 8))
    first = np.cumsum([0] + [n + 1 for n in k])
    of_draft = torch.from_numpy(np.concatenate([first[s] + np.arange(n) for s, n in enumerate(k)]).astype(np.int64)).to(DEV)
    d = dict(p=torch.softmax(logits, 1), drafted=torch.tensor(k, dtype=I32, device=DEV))
    guess = torch.softmax(logits[of_draft] + 0.7 * _randn(seed, "guess", drafts, V), 1)
    # the draft model's own choice
    d["tokens"] = (torch.log(guess) - torch.log(-torch.log(_rand(seed, "choice", drafts, V).clamp(1e-9, 1 - 1e-6)))).argmax(1).to(I32)
    if c["q"]:
        d["q"] = guess
    u = torch.rand(rows, generator=_gen(seed, "u"), device=DEV, dtype=F64)
    d["u"] = u
    n = np.array(k)
    i = np.arange(c["N"])
    has = i < n[:, None]
    d["has"] = torch.from_numpy(has).to(DEV)
    d["row"] = torch.from_numpy(first[:-1, None] + np.arange(c["N"] + 1).clip(max=n[:, None])).to(DEV)
    d["draft"] = torch.from_numpy(np.concatenate([[0], np.cumsum(n)])[:-1, None] + np.where(has, i, 0)).clamp(max=max(drafts - 1, 0)).to(DEV)
    return d


INPUTS = {"rope": _rope_inputs, "append": _append_inputs, "attn": _attn_inputs, "verify": _verify_inputs}


# ---------------------------------------------------------------------------------------------
# the plain forms

def _quantized(x):
    """4-bit blocks of 32 along the last extent: scales F16 [...], values 0 to 15 as U8 [..., 32]."""
    at = x.abs().argmax(-1, keepdim=True)
    d = x.gather(-1, at) / -8.0
    inv = torch.where(d != 0, 1.0 / d, 0.0)
    q = (x * inv + 8.5).to(torch.int8).clamp(max=15)
    return d[..., 0].to(F16), q.to(U8)


def _values(d, q):
    return d.to(F32)[..., None] * (q.to(F32) - 8.0)


def _angles(c, pos):
    """[T, D / 2] in 64 bits: each pair's position on its axis times its frequency."""
    D, mode = c["D"], c.get("mode", MROPE)
    s = _sections(c) if "sections" in c else (D // 8, D // 4 - D // 16, D // 2 - D // 8 - (D // 4 - D // 16), 0)
    pair = torch.arange(D // 2, device=DEV)
    if mode == VISION:
        axis = (pair >= s[0]).long()
        freq = torch.exp(-2 * math.log(BASE) / (D // 2) * torch.where(axis == 0, pair, pair - s[0]).to(F64))
    else:
        freq = torch.exp(-2 * math.log(BASE) / D * pair.to(F64))
        if mode == MROPE:
            axis = (pair >= s[0]).long() + (pair >= s[0] + s[1]) + (pair >= s[0] + s[1] + s[2])
        else:
            axis = torch.full_like(pair, 3)
            for a in (0, 1, 2):
                axis = torch.where((pair % 3 == a) & (pair < 3 * s[a]), a, axis)
    return pos[axis].T.to(F64) * freq


def _rotated(x, angle):
    """x [T, heads, D], pairs (i, i + D / 2)."""
    x = x.to(F64)
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x.chunk(2, 2)
    return torch.cat([a * c - b * s, a * s + b * c], 2).to(F32)


def _rope_plain(c, d):
    H, KV, D = c["H"], c["KV"], c["D"]
    q, k, _ = d["rows"].split((H * D, KV * D, KV * D), 1)
    angle = _angles(c, d["pos"])
    return [_rotated(q.unflatten(1, (H, D)), angle), _rotated(k.unflatten(1, (KV, D)), angle)]


def _append_plain(c, d):
    T, KV, D = c["T"], c["KV"], c["D"]
    _, k, v = d["rows"].split((4 * KV * D, KV * D, KV * D), 1)
    k = _rotated(k.unflatten(1, (KV, D)), _angles(c, d["pos"])).flatten(1)
    slots = d["slots"].long()
    out = []
    for cache, x in ((d["kc"], k), (d["vc"], v)):
        # a row of -1 is the one behind the cache
        if c["type"] == TYPE_F16:
            cache[slots] = x.to(F16)
            out.append(cache[:-1])
        else:
            cache[0][slots], cache[1][slots] = _quantized(x.unflatten(1, (KV * D // 32, 32)))
            at = slots.clamp(min=0)
            out.append(_values(cache[0][at], cache[1][at]).flatten(1))
    return out


def _attn_plain(c, d):
    S, H, KV, D, P = (c[k] for k in ("S", "H", "KV", "D", "P"))
    G = H // KV
    L, N = d["table"].shape[1] * P, d["place"].shape[1]
    rows = (d["table"][:, :, None] * P + torch.arange(P, device=DEV)).reshape(S, L)
    k, v = (_values(d[n + "_d"][rows], d[n + "_q"][rows]).view(S, L, KV, D).transpose(1, 2).contiguous() for n in "kv")
    q = d["q"][d["place"]].view(S, N, KV, G, D).permute(0, 2, 1, 3, 4).reshape(S, KV, N * G, D)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(D)).view(S, KV, N, G, L)
    new = d["start"][1:] - d["start"][:-1]
    last = (d["seen"] - new)[:, None] + torch.arange(N, device=DEV)
    hidden = torch.arange(L, device=DEV) > last[:, :, None]                       # [S, N, L]
    s.masked_fill_(hidden[:, None, :, None], -math.inf)
    e = torch.exp(s - s.amax(4, keepdim=True))
    total = e.sum(4, keepdim=True).view(S, KV, N * G, 1)
    o = torch.matmul(e.view(S, KV, N * G, L), v) / total
    o = o.view(S, KV, N, G, D).permute(0, 2, 1, 3, 4).reshape(S * N, H, D)
    return o[d["real"]]


def _verify_plain(c, d):
    S, N, V = c["S"], c["N"], c["V"]
    if d["tokens"].numel():
        tok = d["tokens"].long()[d["draft"]]                                      # [S, N]
        p = d["p"][d["row"][:, :N], tok].to(F64)
        q = d["q"][d["draft"], tok].to(F64) if c["q"] else 1.0
        u = d["u"][d["row"][:, :N]]
        ok = d["has"] & (u * q < p)
        accepted = ok.long().cumprod(1).sum(1)
    else:
        accepted = torch.zeros(S, dtype=torch.int64, device=DEV)
    drafted = d["drafted"].long()
    one = torch.arange(S, device=DEV)
    w = d["p"][d["row"][one, accepted]].to(F64)                                   # [S, V]
    if d["tokens"].numel():
        refused = (accepted < drafted)[:, None]
        at = accepted.clamp(max=N - 1)
        if c["q"]:
            less = (w - d["q"][d["draft"][one, at]].to(F64)).clamp(min=0)
        else:
            less = w.scatter(1, tok[one, at][:, None], 0.0)
        w = torch.where(refused & (less.sum(1, keepdim=True) > 0), less, w)
    cum = w.cumsum(1)
    u = d["u"][d["row"][one, drafted]]
    pick = (cum <= (u * cum[:, -1])[:, None]).sum(1)
    last = V - 1 - (w.flip(1) > 0).long().argmax(1)
    return [accepted.to(I32), torch.minimum(pick, last).to(I32)]


PLAIN = {"rope": _rope_plain, "append": _append_plain, "attn": _attn_plain, "verify": _verify_plain}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits

def _rope_exact_rows(c, x, pos):
    """x [T, heads, D] rotated pair by pair."""
    D, mode = c["D"], c.get("mode", MROPE)
    s = _sections(c) if "sections" in c else (D // 8, D // 4 - D // 16, D // 2 - D // 8 - (D // 4 - D // 16), 0)
    y = x.to(F64).clone()
    for j in range(D // 2):
        n, power = D, j
        if mode == VISION:
            n, axis = D // 2, 0 if j < s[0] else 1
            power = j if j < s[0] else j - s[0]
        elif mode == MROPE:
            axis = 0 if j < s[0] else 1 if j < s[0] + s[1] else 2 if j < s[0] + s[1] + s[2] else 3
        else:
            axis = j % 3 if j < 3 * s[j % 3] else 3
        theta = pos[axis].to(F64) * BASE ** (-2.0 * power / n)
        co, si = torch.cos(theta)[:, None], torch.sin(theta)[:, None]
        a, b = x[:, :, j].to(F64), x[:, :, j + D // 2].to(F64)
        y[:, :, j], y[:, :, j + D // 2] = a * co - b * si, b * co + a * si
    return y


def _rope_exact(c, seed):
    d = _rope_inputs(c, seed)
    H, KV, D = c["H"], c["KV"], c["D"]
    x = d["rows"][:, :(H + KV) * D].view(c["T"], H + KV, D)
    y = _rope_exact_rows(c, x, d["pos"])
    return [y[:, :H], y[:, H:]]


def _append_exact(c, seed):
    d = _append_inputs(c, seed)
    T, KV, D = c["T"], c["KV"], c["D"]
    x = d["rows"].view(T, 6, KV, D)
    rows = [_rope_exact_rows(c, x[:, 4], d["pos"]).reshape(T, KV * D), x[:, 5].reshape(T, KV * D).to(F64)]
    out = []
    for r in rows:
        if c["type"] == TYPE_F16:
            cache = torch.zeros(c["pool"] * c["P"], KV * D, dtype=F64, device=DEV)
            keep = d["slots"] >= 0
            cache[d["slots"][keep].long()] = r[keep]
            out.append(cache)
            continue
        # blocks are formed of 32-bit values by 32-bit steps
        b = r.to(F32).cpu().numpy().reshape(T, -1, 32)
        big = np.take_along_axis(b, np.abs(b).argmax(2)[:, :, None], 2)
        scale = big / np.float32(-8)
        with np.errstate(divide="ignore"):
            inverse = np.where(scale != 0, np.float32(1) / scale, np.float32(0))
        n = np.minimum(np.trunc(b * inverse + np.float32(8.5)), 15).astype(np.float64)
        values = torch.from_numpy(((n - 8) * scale.astype(np.float16).astype(np.float64)).reshape(T, KV * D)).to(DEV)
        # an idle token reads the cache's first row
        at = d["slots"].long()
        first = (at == 0).nonzero()[:, 0]
        values[at < 0] = values[first[0]] if len(first) else 0.0
        out.append(values)
    return out


def _attn_exact(c, seed):
    d = _attn_inputs(c, seed)
    S, H, KV, D, P = (c[k] for k in ("S", "H", "KV", "D", "P"))
    new, seen = _lengths(c)
    G, out, at = H // KV, [], 0
    for s in range(S):
        pages = d["table"][s, :-(-seen[s] // P)].long()
        rows = (pages[:, None] * P + torch.arange(P, device=DEV)).flatten()[:seen[s]]
        k, v = (((d[n + "_q"][rows].to(F64) - 8) * d[n + "_d"][rows].to(F64)[..., None]).reshape(seen[s], KV, D) for n in "kv")
        past = seen[s] - new[s]
        o = torch.empty(new[s], H, D, dtype=F64, device=DEV)
        visible = torch.arange(seen[s], device=DEV) <= past + torch.arange(new[s], device=DEV)[:, None]
        for h in range(H):
            logits = d["q"][at:at + new[s], h].to(F64) @ k[:, h // G].T.contiguous() / D ** 0.5
            p = torch.softmax(torch.where(visible, logits, -math.inf), 1)
            o[:, h] = p @ v[:, h // G].contiguous()
        out.append(o)
        at += new[s]
    return torch.cat(out)


EXACT = {"rope": _rope_exact, "append": _append_exact, "attn": _attn_exact}


# ---------------------------------------------------------------------------------------------
# the package's operators

def _package():
    if "ggml_loader_amd" not in sys.modules:
        spec = importlib.util.spec_from_file_location(
            "ggml_loader_amd", os.path.join(ROOT, "ggml-loader_amd", "__init__.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules["ggml_loader_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["ggml_loader_amd"]


_held = {}


def _backend():
    """One backend for the process, as a program keeps it."""
    if "backend" not in _held:
        _held["backend"] = _package().hip_backend(0)
    return _held["backend"]


class _Memory:
    def __init__(self, owner, data, shape, kind):
        self.owner = owner
        self.__cuda_array_interface__ = dict(shape=tuple(shape), typestr=kind, data=(data, False), version=3)


class _Graph:
    """A graph as a program builds it once and computes it again, with its tensors on the device."""

    def __init__(self):
        self.gl = _package()
        self.core, self.ctx, self.buf = self.gl.libs()["core"], None, None
        self.ctx = self.core.ggml_init(self.gl.ggml_init_params(1 << 20, None, True))
        self.gf = self.core.ggml_new_graph(self.ctx)
        self.data = []

    def __getattr__(self, name):
        fn = getattr(self.core, "ggml_" + name)
        return lambda *args: fn(self.ctx, *args)

    def new(self, type, *ne):
        return getattr(self.core, f"ggml_new_tensor_{len(ne)}d")(self.ctx, type, *ne)

    def tensor(self, x):
        """A tensor with x's shape and values, for x [..., ne1, ne0]."""
        t = self.new(self.gl.I32 if x.dtype == I32 else self.gl.F32, *x.shape[::-1])
        self.data.append((t, x))
        return t

    def blocks(self, d, q, *ne):
        """A 4-bit tensor of scales d and values q [blocks, 32]."""
        t = self.new(self.gl.Q4_0, *ne)
        nibbles = q[:, :16] | (q[:, 16:] << 4)
        self.data.append((t, torch.cat([d[:, None].view(U8), nibbles], 1)))
        return t

    def output(self, t):
        self.core.ggml_set_output(t)
        self.core.ggml_build_forward_expand(self.gf, t)

    def finish(self):
        self.buf = self.core.ggml_backend_alloc_ctx_tensors(self.ctx, _backend())
        if not self.buf:
            raise MemoryError("out of memory for a graph")
        self.core.ggml_backend_buffer_clear(self.buf, 0)
        for t, x in self.data:
            if x.dtype == F32:
                self.view(t, x.shape).copy_(x)
            else:
                a = np.ascontiguousarray(x.cpu().numpy())
                self.core.ggml_backend_tensor_set(t, a.ctypes.data_as(C.c_void_p), 0, a.nbytes)
        self.data = []

    def view(self, t, shape, kind="<f4"):
        """The tensor's device memory as a torch tensor."""
        return torch.as_tensor(_Memory(self, t.contents.data, shape, kind), device=DEV)

    def rope(self, x, pos, c):
        s = _sections(c) if "sections" in c else None
        D = c["D"]
        if s is None:
            s = (D // 8, D // 4 - D // 16, D // 2 - D // 8 - (D // 4 - D // 16), 0)
        mode = c.get("mode", MROPE)
        return self.rope_multi(x, pos, None, D // 2 if mode == VISION else D, (C.c_int * 4)(*s), mode, 0,
                               BASE, 1.0, 0.0, 1.0, 32.0, 1.0)

    def __del__(self):
        if self.buf:
            self.core.ggml_backend_buffer_free(self.buf)
        if self.ctx:
            self.core.ggml_free(self.ctx)


def _rope_graph(c, d):
    T, H, KV, D = (c[k] for k in ("T", "H", "KV", "D"))
    W = (H + 2 * KV) * D
    g = _Graph()
    rows, pos = g.tensor(d["rows"]), g.tensor(d["pos"].flatten())
    q = g.rope(g.view_3d(rows, D, H, T, D * 4, W * 4, 0), pos, c)
    k = g.rope(g.view_3d(rows, D, KV, T, D * 4, W * 4, H * D * 4), pos, c)
    g.output(q)
    g.output(k)
    g.finish()
    return g, [g.view(q, (T, H, D)), g.view(k, (T, KV, D))]


def _append_graph(c, d):
    T, KV, D, n = c["T"], c["KV"], c["D"], c["pool"] * c["P"]
    W = 6 * KV * D
    g = _Graph()
    rows, pos, slots = g.tensor(d["rows"]), g.tensor(d["pos"].flatten()), g.tensor(d["slots"])
    kc, vc = g.new(c["type"], KV * D, n), g.new(c["type"], KV * D, n)
    k = g.rope(g.view_3d(rows, D, KV, T, D * 4, W * 4, 4 * KV * D * 4), pos, c)
    v = g.view_2d(rows, KV * D, T, W * 4, 5 * KV * D * 4)
    k, v = g.set_rows(kc, g.reshape_2d(k, KV * D, T), slots), g.set_rows(vc, v, slots)
    if c["type"] != TYPE_F16:
        at = g.tensor(d["slots"].clamp(min=0))
    for x in (k, v):
        g.output(x)
    if c["type"] == TYPE_F16:
        g.finish()
        return g, [g.view(x, (n, KV * D), "<f2") for x in (kc, vc)]
    out = [g.get_rows(x, at) for x in (k, v)]
    for x in out:
        g.output(x)
    g.finish()
    return g, [g.view(x, (T, KV * D)) for x in out]


def _attn_graph(c, d):
    S, H, KV, D, P = (c[k] for k in ("S", "H", "KV", "D", "P"))
    T, n = d["q"].shape[0], d["k_d"].shape[0] // P
    g = _Graph()
    k, v = (g.blocks(d[x + "_d"].flatten(), d[x + "_q"].view(-1, 32), D, KV, P, n) for x in "kv")
    o = g.flash_attn_paged(g.tensor(d["q"]), k, v, g.tensor(d["table"]), g.tensor(d["start"]), g.tensor(d["seen"]), 1 / math.sqrt(D))
    g.output(o)
    g.finish()
    return g, g.view(o, (T, H, D))


def _verify_tensors(c, d):
    g = _Graph()
    p, q = g.tensor(d["p"]), g.tensor(d["q"]) if c["q"] and d["q"].numel() else None
    g.finish()
    return g, (p, q, d["drafted"].cpu().numpy(), d["tokens"].cpu().numpy(), d["u"].cpu().numpy())


OWN = {"rope": _rope_graph, "append": _append_graph, "attn": _attn_graph, "verify": _verify_tensors}


# ---------------------------------------------------------------------------------------------
# what the measurement calls

def prepare(case, seed):
    d = INPUTS[case["kind"]](case, seed)
    if own:
        # the same values in the backend's buffer, and the graph over them
        g, rest = OWN[case["kind"]](case, d)
        return case, g, _backend(), rest
    if case["kind"] == "append":
        n, w = case["pool"] * case["P"] + 1, case["KV"] * case["D"]
        if case["type"] == TYPE_F16:
            d["kc"], d["vc"] = (torch.zeros(n, w, dtype=F16, device=DEV) for _ in "kv")
        else:
            d["kc"], d["vc"] = ((torch.zeros(n, w // 32, dtype=F16, device=DEV),
                                 torch.full((n, w // 32, 32), 8, dtype=U8, device=DEV)) for _ in "kv")
    return case, d


def run(state):
    if not own:
        case, d = state
        return PLAIN[case["kind"]](case, d)
    case, g, backend, rest = state
    if case["kind"] == "verify":
        p, q, drafted, tokens, u = rest
        return list(g.gl.hip_verify(backend, p, drafted, tokens, u, draft_probs=q))
    if g.core.ggml_backend_graph_compute_async(backend, g.gf) != 0:
        raise RuntimeError("graph compute failed")
    return rest


def exact(case, seed):
    # the verified tokens are whole numbers
    return EXACT[case["kind"]](case, seed) if case["kind"] in EXACT else None


def work(case):
    """Inputs and outputs once each, of a cache the positions that are seen; the definition's operations. Of
    the probabilities a sequence needs the rows, of the target and of the draft, that its last token is drawn from."""
    c = case
    if c["kind"] == "verify":
        return {"bytes": c["S"] * c["V"] * (8 if c["q"] else 4), "flops": 3 * c["S"] * c["V"]}
    if c["kind"] == "rope":
        n = c["T"] * (c["H"] + c["KV"]) * c["D"]
        return {"bytes": 8 * n + 16 * c["T"], "flops": 3 * n}
    if c["kind"] == "append":
        n = 2 * c["T"] * c["KV"] * c["D"]
        held = 2 if c["type"] == TYPE_F16 else 18 / 32
        return {"bytes": int(n * (4 + held)) + 20 * c["T"], "flops": n * 3}
    new, seen = _lengths(c)
    H, KV, D = c["H"], c["KV"], c["D"]
    pairs = sum(n * s - n * (n - 1) // 2 for n, s in zip(new, seen))
    return {"bytes": int(sum(seen) * KV * D * 36 / 32) + 8 * sum(new) * H * D, "flops": 4 * pairs * H * D}
