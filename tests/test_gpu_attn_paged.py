"""Attention over a 4-bit cache on pages, on the HIP backend, against float64 (serving_ref.attention, which carries
the bound that each value is held to)."""
import numpy as np
import pytest

import serving_ref as ref
from gl import Graph, dequantize, gl, quantize

pytestmark = pytest.mark.gpu
MARK = np.float32(-12345.5)


@pytest.fixture(scope="module")
def hip():
    b = gl.hip_backend(0)
    yield b
    gl.libs()["core"].ggml_backend_free(b)


def draw(rng, new, seen, H, KV, D, P, spare=3, pad=0, sharp=1.5, pool=None):
    """Sequences with `new` tokens, the last of `seen` positions, on shuffled pages; `pad` tokens behind the last."""
    used = [-(-s // P) for s in seen]
    n_pages = sum(used) + spare
    order = rng.permutation(n_pages)
    pages = np.full((len(seen), max(used + [1]) + 1), 10 ** 6, np.int32)       # unused entries point nowhere
    at = 0
    for s, n in enumerate(used):
        pages[s, :n] = order[at:at + n]
        at += n
    blocks = {}
    for name in "kv":
        x = (rng.standard_normal((n_pages, P, KV, D)) * np.exp(0.5 * rng.standard_normal((KV, D)))).astype(np.float32)
        raw = quantize(x, gl.Q4_0)
        blocks[name] = raw
        blocks[name + "_values"] = dequantize(raw, gl.Q4_0, x.size).reshape(x.shape)
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = (sharp * rng.standard_normal((int(start[-1]) + pad, H, D))).astype(np.float32)
    return dict(q=q, pages=pages, start=start, seen=np.array(seen, np.int32), scale=D ** -0.5, P=P, **blocks)


def cache(g, d, name, order):
    n, P, KV, D = d[name + "_values"].shape
    if order == "heads":       # a page's heads one after another
        raw = np.ascontiguousarray(d[name].reshape(n, P, KV, -1).transpose(0, 2, 1, 3))
        return g.permute(g.tensor(gl.Q4_0, D, P, KV, n, data=raw), 0, 2, 1, 3)
    if order == "odd":         # behind other blocks, the pages and positions apart
        bs, nb = 18, D // 32
        wide = np.zeros((n, P + 1, KV * nb + 1, bs), np.uint8)
        wide[:, :P, 1:] = d[name].reshape(n, P, KV * nb, bs)
        t = g.tensor(gl.Q4_0, 32 * wide.size // bs, data=wide)
        return g.view_4d(t, D, KV, P, n, nb * bs, (KV * nb + 1) * bs, (P + 1) * (KV * nb + 1) * bs, bs)
    return g.tensor(gl.Q4_0, D, KV, P, n, data=d[name])


def node(g, d, order="", q=None):
    T, H, D = d["q"].shape
    S, most = d["pages"].shape
    q = g.tensor(gl.F32, D, H, T, data=d["q"]) if q is None else q
    return g.flash_attn_paged(q, cache(g, d, "k", order), cache(g, d, "v", order), g.tensor(gl.I32, most, S, data=d["pages"]),
                              g.tensor(gl.I32, S + 1, data=d["start"]), g.tensor(gl.I32, S, data=d["seen"]), d["scale"])


def computed(hip, d, order=""):
    """The node's result, its memory filled with a mark before."""
    core = gl.libs()["core"]
    with Graph(mem=1 << 20) as g:
        n = node(g, d, order)
        gf = core.ggml_new_graph(g.ctx)
        core.ggml_set_output(n)
        core.ggml_build_forward_expand(gf, n)
        g.buf = core.ggml_backend_alloc_ctx_tensors(g.ctx, hip)
        for t, a in g.inputs:
            core.ggml_backend_tensor_set(t, a.ctypes.data, 0, a.nbytes)
        fill = np.full(d["q"].shape, MARK)
        if fill.size:
            core.ggml_backend_tensor_set(n, fill.ctypes.data, 0, fill.nbytes)
        assert core.ggml_backend_graph_compute(hip, gf) == 0
        first = g.read(n)
        assert core.ggml_backend_graph_compute(hip, gf) == 0
        assert np.array_equal(first.view(np.uint32), g.read(n).view(np.uint32))       # the same bits again
        return first.reshape(d["q"].shape)


def check(hip, d, order=""):
    got = computed(hip, d, order)
    want, bound, listed = ref.attention(d["q"], d["k_values"], d["v_values"], d["pages"], d["start"], d["seen"], d["scale"])
    assert (got[~listed] == MARK).all()
    off = np.abs(got - want)[listed]
    assert (off <= bound[listed]).all(), (off - bound[listed]).max()
    return got


@pytest.mark.parametrize("new, seen, H, KV, D, P", [
    ([1], [1], 1, 1, 64, 16), ([1], [2], 4, 1, 128, 1), ([1], [63], 8, 8, 64, 16), ([1], [64], 8, 2, 96, 16), ([1], [65], 8, 2, 128, 16),
    ([1], [129], 32, 8, 128, 100), ([1], [1000], 24, 8, 128, 64), ([1], [4113], 32, 8, 128, 16), ([1], [5000], 5, 5, 96, 48),
    ([1, 1, 1], [5, 700, 64], 32, 4, 128, 16), ([1] * 9, [1, 3, 17, 64, 65, 128, 500, 1023, 2048], 6, 2, 64, 24),
    ([2], [2], 4, 4, 64, 16), ([5], [300], 32, 4, 128, 16), ([4, 1, 3], [4, 90, 1025], 12, 3, 96, 7), ([3, 2], [64, 65], 17, 1, 128, 8),
    ([16], [16], 8, 2, 64, 16), ([70], [70], 8, 2, 128, 16), ([64, 3], [64, 500], 4, 1, 64, 100), ([100], [1500], 8, 8, 96, 64),
    ([33, 200, 1], [33, 260, 900], 16, 4, 128, 16), ([129], [257], 3, 1, 64, 1),
])
def test_attention(hip, new, seen, H, KV, D, P):
    check(hip, draw(np.random.default_rng(sum(seen) + H + D), new, seen, H, KV, D, P))


@pytest.mark.parametrize("new, seen, H, KV, D, P", [
    ([300, 1, 40], [500, 300, 40], 32, 8, 64, 16), ([150, 2, 1, 1], [1100, 64, 700, 1], 32, 2, 128, 16), ([200], [200], 48, 16, 96, 10),
    ([60, 50, 70], [64, 300, 70], 40, 40, 64, 64),
])
def test_attention_of_many_tokens(hip, new, seen, H, KV, D, P):
    """Prompts' parts beside single tokens, joined by team."""
    assert sum(new) * H > 4096
    check(hip, draw(np.random.default_rng(sum(seen) + H + D), new, seen, H, KV, D, P))


@pytest.mark.parametrize("D", [64, 96])
def test_attention_of_many_tokens_of_many_sequences(hip, D):
    """More sequences than lanes, one of them longer than the others together."""
    rng = np.random.default_rng(70 + D)
    new = rng.integers(0, 50, 70)
    new[66] = 900
    seen = new + rng.integers(0, 60, 70)
    check(hip, draw(rng, [int(n) for n in new], [int(n) for n in seen], 4, 1, D, 16))


@pytest.mark.parametrize("new, seen, H, KV, D, P", [
    ([25], [180], 1000, 1, 64, 16), ([26], [26], 1024, 8, 96, 10), ([200], [270], 128, 16, 128, 16), ([26], [90], 1000, 4, 128, 7),
    ([500, 1, 310, 3, 0], [560, 300, 310, 70, 9], 32, 8, 64, 64), ([20, 1, 9], [150, 40, 33], 840, 20, 96, 16),
    ([410, 2, 1, 400, 1], [500, 400, 1, 400, 129], 32, 4, 128, 24),
])
def test_attention_of_prompts(hip, new, seen, H, KV, D, P):
    """Tiles of 128 rows, beside sequences of few rows and without: last tiles in part, a missing page, scales of V that
    are no numbers at positions that no token sees, and at the last that one does."""
    assert sum(new) * H > 24576 and sum(new) * (H // KV) > 64 * len(new)
    d = draw(np.random.default_rng(sum(seen) + D), new, seen, H, KV, D, P)
    if seen[0] > new[0] + 2 * P:
        d["pages"][0, 1] = -1
    want, bound, _ = ref.attention(d["q"], d["k_values"], d["v_values"], d["pages"], d["start"], d["seen"], d["scale"])
    last, row = d["pages"][0, (seen[0] - 1) // P], (seen[0] - 1) % P
    raw = d["v"].reshape(*d["v_values"].shape[:3], -1, 18)
    raw[last, row + 1:, :, :, :2] = np.array([np.nan], np.float16).view(np.uint8)
    off = np.abs(computed(hip, d) - want)
    assert (off <= bound).all(), (off - bound).max()
    raw[last, row, :, :, :2] = np.array([np.inf], np.float16).view(np.uint8)
    got = computed(hip, d)
    others = np.arange(len(got)) != new[0] - 1
    assert not np.isfinite(got[new[0] - 1]).any()
    assert (np.abs(got - want)[others] <= bound[others]).all()


@pytest.mark.parametrize("order", ["heads", "odd"])
@pytest.mark.parametrize("new, seen, D", [([1, 1], [90, 200], 128), ([6, 2], [70, 2], 96), ([80], [200], 64)])
def test_attention_of_other_cache_layouts(hip, order, new, seen, D):
    check(hip, draw(np.random.default_rng(D), new, seen, 8, 2, D, 16), order)


def test_attention_of_wider_rows_of_queries(hip):
    rng = np.random.default_rng(2)
    d = draw(rng, [1, 3], [50, 129], 8, 2, 64, 16)
    T, H, D = d["q"].shape
    wide = rng.standard_normal((T, H + 3, D + 1)).astype(np.float32)
    d["q"] = np.ascontiguousarray(wide[:, 2:2 + H, 1:])
    with Graph(mem=1 << 20) as g:
        t = g.tensor(gl.F32, D + 1, H + 3, T, data=wide)
        q = g.view_3d(t, D, H, T, (D + 1) * 4, (D + 1) * (H + 3) * 4, (2 * (D + 1) + 1) * 4)
        got = g.compute(hip, node(g, d, q=q)).reshape(T, H, D)
    want, bound, _ = ref.attention(d["q"], d["k_values"], d["v_values"], d["pages"], d["start"], d["seen"], d["scale"])
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("D", [64, 96, 128])
def test_attention_of_empty_and_unlisted_rows(hip, D):
    """Sequences of no tokens or no positions, tokens before the first position, tokens behind the last sequence."""
    d = draw(np.random.default_rng(D), [1, 0, 3, 2, 0, 70], [5, 40, 1, 0, 0, 50], 4, 2, D, 8, pad=9)
    got = check(hip, d)
    assert (got[1:3] == 0).all() and (got[4:6] == 0).all() and (got[6:26] == 0).all() and (got[26] != 0).any()


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 4, 1], [90, 2, 70]])
def test_attention_of_bad_pages_and_bounds(hip, new):
    """Positions on pages that are not there do not exist; lengths past the table and starts past the tokens are cut."""
    d = draw(np.random.default_rng(5), new, [300, 130, 77], 8, 2, 64, 16)
    d["pages"][0, [0, 5, 18]] = -1, 2 ** 31 - 1, len(d["k_values"])
    d["pages"][1, :9] = -7
    check(hip, d)
    d["seen"][:] = 2 ** 31 - 1, -3, 10 ** 6
    d["start"] = np.array([-5, 1, 10 ** 6, 2 ** 31 - 1], np.int32)
    check(hip, d)


@pytest.mark.parametrize("new, H, KV, D, P, n", [
    ([1], 8, 1, 64, 8, 5), ([1, 1], 4, 4, 96, 7, 3), ([1], 8, 2, 128, 16, 3), ([1], 8, 2, 128, 1, 33),          # few rows, narrow
    ([1], 16, 1, 64, 16, 5), ([2, 1], 24, 3, 96, 16, 1), ([1], 32, 4, 128, 48, 1),                              # wide, on pages of sixteens
    ([2, 3], 8, 2, 128, 7, 6), ([1], 9, 1, 64, 100, 1),                                                         # wide, on others
    ([1, 100], 8, 2, 64, 8, 5), ([1, 2, 150], 8, 2, 128, 16, 3), ([40], 8, 2, 96, 16, 5),                       # beside tiles, in tiles
])
def test_attention_of_lengths_past_the_table(hip, new, H, KV, D, P, n):
    """Lengths are cut to a table that is full of pages, also where it ends inside a step of positions."""
    d = draw(np.random.default_rng(n * P + H), new, [n * P] * len(new), H, KV, D, P)
    d["pages"] = np.ascontiguousarray(d["pages"][:, :n])
    check(hip, d)
    for seen in (n * P + 1, n * P + 40, 1000, 2 ** 31 - 1, -2 ** 31):
        d["seen"][:] = seen
        check(hip, d)


def test_attention_of_values_at_the_edges(hip):
    """Scores that leave all weight on one position, equal scores, queries and scales of any size; infinities and NaN in
    places that are masked, or on pages of others."""
    rng = np.random.default_rng(6)
    for big in (1e-30, 1e-6, 1.0, 300.0, 1e6):
        d = draw(rng, [1, 2, 66], [200, 65, 90], 8, 2, 64, 16, sharp=big)
        check(hip, d)
    d = draw(rng, [1, 2, 66], [200, 65, 90], 8, 2, 64, 16)
    d["q"][1] = 0
    for name in "kv":
        raw = d[name].reshape(-1, 18)
        f = raw[:, :2].view(np.float16)
        f *= np.exp2(rng.integers(-10, 6, f.shape)).astype(np.float16)          # blocks of very different scales
        raw[::7, :2].view(np.float16)[:] = 0
        d[name + "_values"] = dequantize(d[name], gl.Q4_0, d[name + "_values"].size).reshape(d[name + "_values"].shape)
    good = check(hip, d)
    # the rows past each sequence's last position, and the spare pages
    n, P = d["k_values"].shape[:2]
    hidden = np.ones((n, P), bool)
    for s, seen in enumerate(d["seen"]):
        for j in range(seen):
            hidden[d["pages"][s, j // P], j % P] = False
    for name in "kv":
        raw = d[name].reshape(n, P, -1, 18)
        raw[hidden, :, :2] = np.array([np.nan if name == "k" else np.inf], np.float16).view(np.uint8)
        raw[hidden, ::2, :2] = np.array([np.inf if name == "k" else np.nan], np.float16).view(np.uint8)
    again = computed(hip, d)
    assert np.array_equal(good.view(np.uint32), again.view(np.uint32))


def test_attention_keeps_later_positions_out(hip):
    """A NaN in the last position's keys and values reaches the token that sees it and no other."""
    for new, seen in (([5], [69]), ([80], [100]), ([1, 5], [30, 64])):
        d = draw(np.random.default_rng(7), new, seen, 4, 1, 128, 16)
        want, bound, _ = ref.attention(d["q"], d["k_values"], d["v_values"], d["pages"], d["start"], d["seen"], d["scale"])
        last = seen[-1] - 1
        for name in "kv":
            raw = d[name].reshape(*d[name + "_values"].shape[:3], -1, 18)
            raw[d["pages"][-1, last // 16], last % 16, :, :, :2] = np.array([np.nan], np.float16).view(np.uint8)
        got = computed(hip, d)
        assert np.isnan(got[-1]).all()
        assert (np.abs(got[:-1] - want[:-1]) <= bound[:-1]).all()


@pytest.mark.parametrize("new, H, D", [([2], 4, 64), ([2], 2, 128), ([3], 1, 96), ([5], 4, 128), ([4], 3, 64), ([80], 4, 128)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_attention_of_scales_that_are_not_finite_later(hip, new, H, D, bad):
    """A scale of V that is no number reaches the token that sees it, and costs the others, of small values, no bits."""
    d = draw(np.random.default_rng(D + H), new, [100], H, 1, D, 16)
    raw = d["v"].reshape(*d["v_values"].shape[:3], -1, 18)
    raw[..., :2].view(np.float16)[:] *= np.float16(2.0 ** -9)
    d["v_values"] = dequantize(d["v"], gl.Q4_0, d["v_values"].size).reshape(d["v_values"].shape)
    want, bound, _ = ref.attention(d["q"], d["k_values"], d["v_values"], d["pages"], d["start"], d["seen"], d["scale"])
    raw[d["pages"][0, 99 // 16], 99 % 16, :, :, :2] = np.array([bad], np.float16).view(np.uint8)
    got = computed(hip, d)
    assert not np.isfinite(got[-1]).any()
    assert (np.abs(got[:-1] - want[:-1]) <= bound[:-1]).all()


def test_attention_of_a_long_cache(hip):
    """Blocks past 2^31 bytes and rows past 2^32 values of the cache: pages at its far end."""
    D, KV, P = 128, 8, 64
    n_pages = 70000                                        # 4.6e9 values, 2.6 GB each for K and V
    rng = np.random.default_rng(8)
    far = np.array([0, n_pages - 1, n_pages // 2, n_pages - 7], np.int32)
    d = draw(rng, [1, 3], [120, 100], 16, KV, D, P, spare=0)
    small = len(d["k_values"])
    core = gl.libs()["core"]
    with Graph(mem=1 << 20) as g:
        k, v = (g.tensor(gl.Q4_0, D, KV, P, n_pages) for _ in "kv")
        pages = far[d["pages"].clip(0, small - 1)]
        n = g.flash_attn_paged(g.tensor(gl.F32, D, 16, 4, data=d["q"]), k, v, g.tensor(gl.I32, pages.shape[1], 2, data=pages),
                               g.tensor(gl.I32, 3, data=d["start"]), g.tensor(gl.I32, 2, data=d["seen"]), d["scale"])
        gf = core.ggml_new_graph(g.ctx)
        core.ggml_set_output(n)
        core.ggml_build_forward_expand(gf, n)
        g.buf = core.ggml_backend_alloc_ctx_tensors(g.ctx, hip)
        for t, a in g.inputs:
            core.ggml_backend_tensor_set(t, a.ctypes.data, 0, a.nbytes)
        size = P * KV * D // 32 * 18
        for t, name in ((k, "k"), (v, "v")):
            raw = np.ascontiguousarray(d[name]).reshape(small, size)
            for i in range(small):
                core.ggml_backend_tensor_set(t, raw[i].ctypes.data, int(far[i]) * size, size)
        assert core.ggml_backend_graph_compute(hip, gf) == 0
        got = g.read(n).reshape(d["q"].shape)
    want, bound, _ = ref.attention(d["q"], d["k_values"], d["v_values"], d["pages"], d["start"], d["seen"], d["scale"])
    assert (np.abs(got - want) <= bound).all()


def test_attention_in_the_static_scratch(hip):
    """graph_compute_static gives the same bits."""
    core, h = gl.libs()["core"], gl.libs()["hip"]
    for new, seen in (([1] * 4, [3000, 10, 700, 64]), ([90, 3], [500, 400])):
        d = draw(np.random.default_rng(9), new, seen, 8, 2, 128, 16)
        with Graph(mem=1 << 20) as g:
            n = node(g, d)
            want = g.compute(hip, n)
            gf = core.ggml_new_graph(g.ctx)
            core.ggml_build_forward_expand(gf, n)
            assert h.ggml_backend_hip_graph_compute_static(hip, gf) == 0
            assert np.array_equal(want.view(np.uint32), g.read(n).view(np.uint32))


def test_attention_refuses_shared_memory(hip):
    """A result over its queries, its cache or its lengths is refused before anything runs."""
    d = draw(np.random.default_rng(10), [1, 6], [30, 50], 8, 2, 64, 16)
    core = gl.libs()["core"]
    with Graph(mem=1 << 20) as g:
        n = node(g, d)
        want = g.compute(hip, n)
        gf = core.ggml_new_graph(g.ctx)
        core.ggml_build_forward_expand(gf, n)
        own = n.contents.data
        for k in range(6):
            n.contents.data = n.contents.src[k].contents.data
            assert core.ggml_backend_graph_compute(hip, gf) != 0
        n.contents.data = n.contents.src[0].contents.data + d["q"].nbytes - 4          # its last value alone
        assert core.ggml_backend_graph_compute(hip, gf) != 0
        n.contents.data = own
        assert core.ggml_backend_graph_compute(hip, gf) == 0
        assert np.array_equal(want.view(np.uint32), g.read(n).view(np.uint32))
