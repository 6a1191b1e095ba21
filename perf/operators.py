"""Performance cases of the recurrent mixer's operators and of the token scores.

Four kinds of work:

* ``conv``   the short causal convolution of a state space mixer: the last d_conv - 1 rows of a
             sequence joined before its new rows, one filter of d_conv taps per channel, the bias,
             SiLU, and the rows that the next step starts from
* ``scan1``  the selective scan with a decay per channel and state (each channel a head of its own)
* ``scan2``  the selective scan with one decay per head of several channels
* ``score``  log probabilities of given tokens under rows of logits, with each row's entropy and its
             likeliest tokens

One new row per sequence is a decoding step, hundreds to thousands a prompt. Rows come as a mixer
has them: slices of wider projections (the convolution's input beside the gate and the time steps,
B and C beside the scan's input), states as rows of a pool in which each sequence names its own.

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
F32, F64 = torch.float32, torch.float64


# ---------------------------------------------------------------------------------------------
# the cases
#
# conv: S sequences of T new rows of D channels in projections of W values a row, K taps
# scan: S sequences of T new rows, H heads of P channels, N states a channel, G groups of B and C
# score: R rows of V logits, the k likeliest tokens of each; the last `pad` ids can't be drawn

def listed():
    return [
        # decoding one sequence: the smallest calls, all latency
        dict(name="conv_step_1", kind="conv", S=1, T=1, D=2560, W=5120, K=4),
        # a batch of 64 decoding sequences
        dict(name="conv_step_64", kind="conv", S=64, T=1, D=5120, W=10304, K=4),
        # a ragged prompt, and a long one through a wide mixer
        dict(name="conv_prompt_777", kind="conv", S=1, T=777, D=2560, W=5120, K=4),
        dict(name="conv_prompt_4096", kind="conv", S=1, T=4096, D=10240, W=18560, K=4),
        # decoding with a decay per channel and state; a prompt of that kind
        dict(name="scan1_step_1", kind="scan1", S=1, T=1, H=5120, P=1, N=16, G=1),
        dict(name="scan1_prompt_1500", kind="scan1", S=1, T=1500, H=5120, P=1, N=16, G=1),
        # decoding with a decay per head: 32 sequences, whose states are most of what is read
        dict(name="scan2_step_32", kind="scan2", S=32, T=1, H=80, P=64, N=128, G=1),
        # a ragged prompt through few heads, and a long one through many
        dict(name="scan2_prompt_333", kind="scan2", S=1, T=333, H=24, P=64, N=128, G=1),
        dict(name="scan2_prompt_4096", kind="scan2", S=1, T=4096, H=128, P=64, N=128, G=8),
        # one step's scores, those of a short text and of a prompt
        dict(name="score_1", kind="score", R=1, V=151936, k=20, pad=267),
        dict(name="score_37", kind="score", R=37, V=32064, k=5, pad=0),
        dict(name="score_512", kind="score", R=512, V=128256, k=20, pad=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    kind = rng.choice(("conv", "scan1", "scan2", "scan2", "score"))
    if kind == "score":
        V = _log(rng, 1000, 152000)
        return dict(kind=kind, R=_log(rng, 1, 512), V=V, k=rng.choice((0, 1, 5, 20, rng.randint(2, 64))),
                    pad=rng.choice((0, rng.randint(1, 500))))
    if rng.random() < 0.35:
        S, T = _log(rng, 1, 96), rng.choice((1, 1, 2, 4, 7))
    else:
        S, T = rng.choice((1, 1, 1, 2, 3, 5)), _log(rng, 8, 4096)
    if kind == "conv":
        D = _log(rng, 200, 10240)
        return dict(kind=kind, S=S, T=T, D=D, W=D + rng.choice((0, _log(rng, 16, 8320))), K=rng.choice((2, 3, 4, 4, 4)))
    if kind == "scan1":
        return dict(kind=kind, S=S, T=T, H=_log(rng, 200, 8192), P=1, N=rng.choice((8, 16, 16, 32)), G=1)
    G = rng.choice((1, 1, 2, 4, 8))
    return dict(kind=kind, S=S, T=T, H=G * _log(rng, 2, 128 // G), P=rng.choice((32, 48, 64, 64, 80, 128)),
                N=rng.choice((16, 64, 96, 128, 128, 256)), G=G)


def draw(rng: random.Random):
    most = {}
    for c in listed():
        for key, v in work(c).items():
            most[c["kind"], key] = max(v, most.get((c["kind"], key), 0))
    while True:
        case = _drawn(rng)
        if all(v <= most[case["kind"], key] for key, v in work(case).items()):
            return case


# ---------------------------------------------------------------------------------------------
# seeded inputs

def _randn(seed, name, *shape):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) << 32) + zlib.crc32(name.encode()))
    return torch.randn(*shape, generator=g, device=DEV)


def _rand(seed, name, *shape):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) << 32) + zlib.crc32(name.encode()))
    return torch.rand(*shape, generator=g, device=DEV)


def _conv_inputs(c, seed):
    S, T, D, W, K = (c[k] for k in "STDWK")
    return dict(rows=_randn(seed, "rows", S, T, W), state=_randn(seed, "state", S, D, K - 1),
                w=_randn(seed, "w", D, K) / math.sqrt(K), bias=0.1 * _randn(seed, "bias", D))


def _scan_inputs(c, seed):
    S, T, H, P, N, G = (c[k] for k in "STHPNG")
    # time steps whose softplus is 0.001 to 0.1 with each row's own part on top
    dt = torch.exp(_rand(seed, "dt", H) * math.log(100) + math.log(1e-3))
    dt = dt + torch.log(-torch.expm1(-dt)) + 0.5 * _randn(seed, "dt_rows", S, T, H)
    pool = S + 2
    ids = _rand(seed, "ids", pool).argsort()[:S].to(torch.int32)
    d = dict(state=0.3 * _randn(seed, "state", pool, H, P, N), ids=ids)
    if c["kind"] == "scan1":
        # the scan's input is the convolution's whole output; B and C are slices of a small projection
        rank = -(-H // 32)
        d["x"] = torch.nn.functional.silu(_randn(seed, "x", S, T, H))
        d["bc"] = _randn(seed, "bc", S, T, rank + 2 * N)
        d["dt"] = dt
        d["A"] = -torch.arange(1, N + 1, device=DEV, dtype=F32).repeat(H, 1) * torch.exp(0.1 * _randn(seed, "A", H, N))
    else:
        # the scan's input, B and C are slices of the convolution's output, the time steps of the projection
        d["xbc"] = torch.nn.functional.silu(_randn(seed, "x", S, T, H * P + 2 * G * N))
        d["dt"] = torch.cat([_randn(seed, "gate", S, T, 16), dt], 2)
        d["A"] = -(1 + 15 * _rand(seed, "A", H, 1))
    return d


def _scan_views(c, d):
    """x [S, T, H, P], dt [S, T, H], B and C [S, T, G, N] as slices of what they come in."""
    S, T, H, P, N, G = (c[k] for k in "STHPNG")
    if c["kind"] == "scan1":
        r = d["bc"].shape[2] - 2 * N
        return (d["x"].unsqueeze(3), d["dt"], d["bc"][:, :, r:r + N].unsqueeze(2), d["bc"][:, :, r + N:].unsqueeze(2))
    x, B, Cm = d["xbc"].split((H * P, G * N, G * N), 2)
    return x.unflatten(2, (H, P)), d["dt"][:, :, 16:], B.unflatten(2, (G, N)), Cm.unflatten(2, (G, N))


def _score_inputs(c, seed):
    R, V, pad = c["R"], c["V"], c["pad"]
    # logits of a language model: a normal bulk and a few likely tokens per row
    x = 2.5 * _randn(seed, "logits", R, V)
    peak = (_rand(seed, "peaks", R, 8) * (V - pad)).long()
    x.scatter_add_(1, peak, 4 + 3 * _randn(seed, "heights", R, 8))
    if pad:
        x[:, V - pad:] = -math.inf
    pick = torch.where(_rand(seed, "pick", R) < 0.7, peak[:, 0], (_rand(seed, "other", R) * (V - pad)).long())
    return dict(logits=x, tokens=pick.to(torch.int32))


INPUTS = {"conv": _conv_inputs, "scan1": _scan_inputs, "scan2": _scan_inputs, "score": _score_inputs}


# ---------------------------------------------------------------------------------------------
# the plain forms

def _conv_plain(c, d):
    D, T, K = c["D"], c["T"], c["K"]
    sx = torch.cat([d["state"], d["rows"][:, :, :D].transpose(1, 2)], 2)          # [S, D, K - 1 + T]
    y = (sx.unfold(2, K, 1) * d["w"][:, None]).sum(3) + d["bias"][:, None]
    y = y / (1 + torch.exp(-y))
    return [y.transpose(1, 2).contiguous(), sx[:, :, T:].contiguous()]


def _softplus(x):
    return x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))


def _scan_step_plain(h0, x, dt, A, B, Cm):
    """One new row."""
    h = h0 * torch.exp(dt[:, 0, :, None] * A)[:, :, None] + (dt[:, 0, :, None] * x[:, 0])[..., None] * B[:, 0, :, None]
    return (h * Cm[:, 0, :, None]).sum(3)[:, None], h


def _scan1_plain(h0, x, dt, A, B, Cm):
    """All rows at once: pairs (decay, input) joined over 1, 2, 4, ... rows."""
    T = x.shape[1]
    a = torch.exp(dt[..., None] * A)                                              # [S, T, H, N]
    b = (dt * x[..., 0])[..., None] * B
    b[:, 0] += a[:, 0] * h0[:, :, 0]
    shift = 1
    while shift < T:
        b = torch.cat([b[:, :shift], b[:, shift:] + a[:, shift:] * b[:, :-shift]], 1)
        a = torch.cat([a[:, :shift], a[:, shift:] * a[:, :-shift]], 1)
        shift *= 2
    return (b * Cm).sum(3)[..., None], b[:, -1].unsqueeze(2)


def _scan2_plain(h0, x, dt, A, B, Cm):
    """Products of 64 rows at a time, joined by the decays between the chunks."""
    (S, T, H, P), (G, N) = x.shape, B.shape[2:]
    Q, nc = 64, -(-T // 64)
    pad = nc * Q - T

    def chunks(t):                                                                # [S, nc, heads, Q, ...]
        t = torch.cat([t, t.new_zeros(S, pad, *t.shape[2:])], 1) if pad else t
        return t.unflatten(1, (nc, Q)).transpose(2, 3)

    cum = chunks((dt.to(F64) * A[:, 0]).contiguous()).cumsum(3)                    # [S, nc, H, Q]
    lower = torch.ones(Q, Q, device=DEV, dtype=torch.bool).tril()
    decay = torch.exp((cum[..., :, None] - cum[..., None, :]).masked_fill(~lower, -math.inf).to(F32))
    xs = chunks(dt[..., None] * x)                                                # [S, nc, H, Q, P]
    Bc, Cc = chunks(B), chunks(Cm)                                                # [S, nc, G, Q, N]
    per = H // G
    g = torch.matmul(Cc, Bc.transpose(3, 4).contiguous()).repeat_interleave(per, 2)
    y = torch.matmul(g * decay, xs)
    left = torch.exp((cum[..., -1:] - cum).to(F32))
    part = torch.matmul((xs * left[..., None]).transpose(3, 4).contiguous(), Bc.repeat_interleave(per, 2))
    total = torch.cat([cum.new_zeros(S, 1, H), cum[..., -1].cumsum(1)], 1).transpose(1, 2)   # [S, H, nc + 1]
    later = torch.ones(nc + 1, nc + 1, device=DEV, dtype=torch.bool).tril()
    across = torch.exp((total[..., :, None] - total[..., None, :]).masked_fill(~later, -math.inf).to(F32))
    held = torch.cat([h0[:, None], part], 1).transpose(1, 2).flatten(3)           # [S, H, nc + 1, P * N]
    held = torch.matmul(across, held).unflatten(3, (P, N)).transpose(1, 2)
    y = y + torch.matmul(Cc.repeat_interleave(per, 2), held[:, :-1].transpose(3, 4).contiguous()) * torch.exp(cum.to(F32))[..., None]
    return y.transpose(2, 3).flatten(1, 2)[:, :T], held[:, -1]


def _scan_plain(c, d):
    x, dt, B, Cm = _scan_views(c, d)
    h0 = d["state"][d["ids"].long()]
    dt = _softplus(dt)
    if c["T"] == 1:
        per = c["H"] // c["G"]
        y, h = _scan_step_plain(h0, x, dt, d["A"], B.repeat_interleave(per, 2), Cm.repeat_interleave(per, 2))
    else:
        y, h = (_scan1_plain if c["kind"] == "scan1" else _scan2_plain)(h0, x, dt, d["A"], B, Cm)
    return [y.contiguous(), h.contiguous()]


def _score_plain(c, d):
    x, k = d["logits"], c["k"]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, dtype=F64)
    lse = top[:, 0].to(F64) + torch.log(total)
    logprob = x.gather(1, d["tokens"].long()[:, None])[:, 0] - lse
    mean = torch.where(e > 0, e * (x - top), 0).sum(1, dtype=F64) / total
    out = [logprob.to(F32), (torch.log(total) - mean).to(F32)]
    if k:
        # the order of the values, and of the ids where values are equal
        bits = x.view(torch.int32).to(torch.int64)
        order = torch.where(bits < 0, -2147483648 - bits - 1, bits)
        key = (order << 32) + (c["V"] - 1 - torch.arange(c["V"], device=DEV))
        ids = c["V"] - 1 - (key.topk(k, 1)[0] & 0xFFFFFFFF)
        out += [ids.to(torch.int32), (x.gather(1, ids) - lse[:, None]).to(F32)]
    return out


PLAIN = {"conv": _conv_plain, "scan1": _scan_plain, "scan2": _scan_plain, "score": _score_plain}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits

def _conv_exact(c, seed):
    d = _conv_inputs(c, seed)
    D, T, K = c["D"], c["T"], c["K"]
    seen = torch.cat([d["state"].to(F64).transpose(1, 2), d["rows"][:, :, :D].to(F64)], 1)   # [S, K - 1 + T, D]
    y = d["bias"].to(F64).expand(c["S"], T, D).clone()
    for k in range(K):
        y += seen[:, k:k + T] * d["w"][:, k].to(F64)
    return [y * torch.sigmoid(y), seen[:, T:].transpose(1, 2).contiguous()]


def _scan_exact(c, seed):
    d = _scan_inputs(c, seed)
    x, dt, B, Cm = (t.to(F64) for t in _scan_views(c, d))
    dt = torch.nn.functional.softplus(dt, threshold=200)
    A, per = d["A"].to(F64), c["H"] // c["G"]
    h = d["state"][d["ids"].long()].to(F64)                                       # [S, H, P, N]
    y = torch.empty_like(x)
    for t in range(c["T"]):
        b, cm = (m[:, t].repeat_interleave(per, 1)[:, :, None] for m in (B, Cm))  # [S, H, 1, N]
        h = h * torch.exp(dt[:, t, :, None] * A)[:, :, None] + (dt[:, t, :, None] * x[:, t])[..., None] * b
        y[:, t] = (h * cm).sum(3)
    return [y, h]


def _score_exact(c, seed):
    d = _score_inputs(c, seed)
    p = torch.log_softmax(d["logits"].to(F64), 1)
    out = [p.gather(1, d["tokens"].long()[:, None])[:, 0], -torch.special.xlogy(p.exp(), p.exp()).sum(1)]
    if c["k"]:
        ids = torch.cat([r.sort(descending=True, stable=True)[1][None, :c["k"]] for r in d["logits"]])
        out += [ids.to(torch.int32), p.gather(1, ids)]
    return out


EXACT = {"conv": _conv_exact, "scan1": _scan_exact, "scan2": _scan_exact, "score": _score_exact}


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
    def __init__(self, owner, data, shape):
        self.owner = owner
        self.__cuda_array_interface__ = dict(shape=tuple(shape), typestr="<f4", data=(data, False), version=3)


class _Graph:
    """A graph as a program builds it once and computes it again, with its tensors on the device."""

    def __init__(self):
        self.gl = _package()
        self.core, self.ctx, self.buf = self.gl.libs()["core"], None, None
        self.core.ggml_backend_graph_compute_async.restype = C.c_int
        self.core.ggml_backend_graph_compute_async.argtypes = [C.c_void_p, C.c_void_p]
        self.ctx = self.core.ggml_init(self.gl.ggml_init_params(1 << 20, None, True))
        self.gf = self.core.ggml_new_graph(self.ctx)
        self.data, self.outputs = [], []

    def __getattr__(self, name):
        fn = getattr(self.core, "ggml_" + name)
        return lambda *args: fn(self.ctx, *args)

    def tensor(self, x):
        """A tensor with x's shape and values, for x [..., ne1, ne0]."""
        ne = x.shape[::-1]
        t = getattr(self.core, f"ggml_new_tensor_{len(ne)}d")(
            self.ctx, self.gl.I32 if x.dtype == torch.int32 else self.gl.F32, *ne)
        self.data.append((t, x))
        return t

    def output(self, t):
        self.core.ggml_set_output(t)
        self.core.ggml_build_forward_expand(self.gf, t)

    def finish(self):
        self.buf = self.core.ggml_backend_alloc_ctx_tensors(self.ctx, _backend())
        if not self.buf:
            raise MemoryError("out of memory for a graph")
        for t, x in self.data:
            if x.dtype == torch.int32:
                a = np.ascontiguousarray(x.cpu().numpy())
                self.core.ggml_backend_tensor_set(t, a.ctypes.data_as(C.c_void_p), 0, a.nbytes)
            else:
                self.view(t, x.shape).copy_(x)
        self.data = []

    def view(self, t, shape, offset=0):
        """The tensor's device memory as a torch tensor."""
        return torch.as_tensor(_Memory(self, t.contents.data + offset, shape), device=DEV)

    def __del__(self):
        if self.buf:
            self.core.ggml_backend_buffer_free(self.buf)
        if self.ctx:
            self.core.ggml_free(self.ctx)


def _conv_graph(c, d):
    S, T, D, W, K = (c[k] for k in "STDWK")
    g = _Graph()
    rows = g.view_3d(g.tensor(d["rows"]), D, T, S, W * 4, T * W * 4, 0)
    sx = g.concat(g.tensor(d["state"]), g.transpose(rows), 0)
    nb = sx.contents.nb
    new = g.cpy(g.view_3d(sx, K - 1, D, S, nb[1], nb[2], T * 4), g.tensor(torch.zeros_like(d["state"])))
    y = g.silu(g.add(g.ssm_conv(sx, g.tensor(d["w"])), g.tensor(d["bias"])))
    for t in (y, new):
        g.output(t)
    g.finish()
    return g, [g.view(y, (S, T, D)), g.view(new, (S, D, K - 1))]


def _scan_graph(c, d):
    S, T, H, P, N, G = (c[k] for k in "STHPNG")
    g = _Graph()
    dt = g.tensor(d["dt"])
    w = d["dt"].shape[2]
    dt = g.view_3d(dt, H, T, S, w * 4, T * w * 4, (w - H) * 4)
    if c["kind"] == "scan1":
        x, r, bc = g.reshape_4d(g.tensor(d["x"]), 1, H, T, S), d["bc"].shape[2], g.tensor(d["bc"])
        at = (r - 2 * N, r - N)
    else:
        r, bc = d["xbc"].shape[2], g.tensor(d["xbc"])
        x = g.view_4d(bc, P, H, T, S, P * 4, r * 4, T * r * 4, 0)
        at = (H * P, H * P + G * N)
    B, Cm = (g.view_4d(bc, N, G, T, S, N * 4, r * 4, T * r * 4, a * 4) for a in at)
    y = g.ssm_scan(g.tensor(d["state"]), x, dt, g.tensor(d["A"]), B, Cm, g.tensor(d["ids"]), 1)
    g.output(y)
    g.finish()
    return g, [g.view(y, (S, T, H, P)), g.view(y, (S, H, P, N), S * T * H * P * 4)]


def _score_tensor(c, d):
    g = _Graph()
    logits = g.tensor(d["logits"])
    g.finish()
    return g, (logits, d["tokens"].cpu().numpy())


OWN = {"conv": _conv_graph, "scan1": _scan_graph, "scan2": _scan_graph, "score": _score_tensor}


# ---------------------------------------------------------------------------------------------
# what the measurement calls

def prepare(case, seed):
    d = INPUTS[case["kind"]](case, seed)
    if own:
        # the same values in the backend's buffer, and the graph over them
        g, rest = OWN[case["kind"]](case, d)
        return case, g, _backend(), rest
    return case, d


def run(state):
    if not own:
        case, d = state
        return PLAIN[case["kind"]](case, d)
    case, g, backend, rest = state
    if case["kind"] == "score":
        logits, tokens = rest
        out = g.gl.hip_logprobs(backend, logits, tokens, n_top=case["k"])
        return list(out if case["k"] else out[:2])
    if g.core.ggml_backend_graph_compute_async(backend, g.gf) != 0:
        raise RuntimeError("graph compute failed")
    return rest


def exact(case, seed):
    return EXACT[case["kind"]](case, seed)


def work(case):
    """Inputs and outputs once each; the definition's operations (two per state for the update and two
    for the output of a scan's row)."""
    c = case
    if c["kind"] == "score":
        return {"bytes": 4 * c["R"] * (c["V"] + 3 + 2 * c["k"]), "flops": 4 * c["R"] * c["V"]}
    S, T = c["S"], c["T"]
    if c["kind"] == "conv":
        D, K = c["D"], c["K"]
        return {"bytes": 4 * (2 * S * T * D + 2 * S * D * (K - 1) + D * (K + 1)), "flops": S * T * D * (2 * K + 5)}
    H, P, N, G = (c[k] for k in "HPNG")
    return {"bytes": 4 * (2 * S * T * H * P + S * T * H + 2 * S * T * G * N + 2 * S * H * P * N + c["H"] * (N if P == 1 else 1)),
            "flops": S * T * H * P * N * (6 if P == 1 else 4)}
