"""Rotary positions in a trained block, and causal attention token by token over a paged
cache, as a user builds them from pico's ops; against float64 (tests/_paged.py)."""
import ctypes

import numpy as np
import pytest
import torch

import _paged as O
from pico_amd.pico import Pico, PicoError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def P():
    return Pico()


# ------------------------------------------------------------- positions, trained
B, T, H, HD, ROT = 2, 24, 3, 32, 24
D = H * HD
SHAPES = {"x": (B * T, D), "wqkv": (D, 3 * D), "wo": (D, D)}
POS = np.tile(np.arange(T), B) * 5


def _values(seed):
    g = torch.Generator().manual_seed(seed)
    return {k: torch.randn(*s, generator=g) * (s[0] ** -0.5 if k[0] == "w" else 1.0) for k, s in SHAPES.items()}


def _block(P, p, rope, pos=POS):
    """an attention layer with positions; its gradient reaches x by two ways"""
    q, k, v = P.split_cols(P.matmul(p["x"], p["wqkv"]), 3)
    a = P.attention_causal(P.rope(q, rope, pos, H), P.rope(k, rope, pos, H), P.rope(v, rope, pos, H), B, H)
    return P.matmul_add(a, p["wo"], p["x"])


def _exact(v, inter, m):
    v = {k: t.double().requires_grad_() for k, t in v.items()}
    f = torch.tensor(O.freqs(ROT))
    a = torch.tensor(POS).double()[:, None] * f
    c, s = m * torch.cos(a)[:, None], m * torch.sin(a)[:, None]
    i1 = torch.arange(ROT // 2) * (2 if inter else 1)
    i2 = i1 + (1 if inter else ROT // 2)

    def turn(t):
        t = t.reshape(B * T, H, HD)
        y = t.clone()
        y[..., i1] = t[..., i1] * c - t[..., i2] * s
        y[..., i2] = t[..., i2] * c + t[..., i1] * s
        return y.view(B, T, H, HD).transpose(1, 2)

    q, k, u = (turn(t) for t in (v["x"] @ v["wqkv"]).split(D, 1))
    z = q @ k.transpose(2, 3) / HD ** 0.5
    z = z.masked_fill(torch.ones(T, T, dtype=torch.bool).triu(1), -np.inf)
    o = (torch.softmax(z, 3) @ u).transpose(1, 2).reshape(B * T, D)
    return v, v["x"] + o @ v["wo"]


@pytest.mark.parametrize("inter", [False, True])
def test_gradients(P, inter):
    vals = _values(1)
    v, y = _exact(vals, inter, 1.25)
    y.sum().backward()
    p = {k: P.param(list(t.shape), t.numpy()) for k, t in vals.items()}
    rope = P.rope_init(ROT, interleaved=inter, magnitude=1.25)
    with P.arena():
        out = _block(P, p, rope)
        P.backward(out)
        # four products, a softmax and three turns of fewer than 300 terms on the way: 1e-4
        # is over 100 times 8 * 300 u / sqrt(300)
        for got, want in [(P.value(out), y)] + [(P.grad_value(p[k]), v[k].grad) for k in SHAPES]:
            want = want.detach()
            assert float((torch.from_numpy(got).double() - want).norm() / want.norm()) <= 1e-4
        P.sync()
    P.lib.pico_rope_free(rope)
    for t in p.values():
        P.free(t)


def test_gradient_of_a_tensor_turned_twice(P):
    """y = turn(x, a) + turn(x, b): both contributions reach x, bit for bit the sum of the two
    turned back"""
    x = np.random.default_rng(2).standard_normal((40, 64)).astype(np.float32)
    a, b = np.arange(40), np.arange(40) * 7 + 3
    rope = P.rope_init(32)
    t = P.param([40, 64], x)
    grads = []
    for pair in ((a,), (b,), (a, b)):
        P.set_grad(t, np.zeros((40, 64)))
        with P.arena():
            y = P.rope(t, rope, pair[0], 2)
            if len(pair) == 2:
                y = P.add(y, P.rope(t, rope, pair[1], 2))
            P.backward(y)
            grads.append(P.grad(t))
    np.testing.assert_allclose(grads[2], grads[0] + grads[1], rtol=0, atol=2.0 ** -22)
    P.lib.pico_rope_free(rope)
    P.free(t)


def test_capture_beside_a_live_eager_graph(P):
    """a training step captured while an eager graph of the same leaves, its backward done,
    is kept; that graph's second backward between the replays"""
    vals = _values(3)
    p = {k: P.param(list(t.shape), t.numpy()) for k, t in vals.items()}
    opt = P.lib.pico_optim_sgd_init(0.0)
    for t in p.values():
        P.lib.pico_optim_sgd_add(opt, t)
    rope = P.rope_init(ROT)
    grads = lambda: {k: P.grad_value(t) for k, t in p.items()}  # noqa: E731
    with P.arena() as keep:
        pos32 = POS.astype(np.int32)
        dev = P.lib.pico_ids_to_device(pos32.ctypes.data_as(ctypes.c_void_p), len(POS))
        with P.arena() as a:
            eager = _block(P, p, rope, dev)
            P.lib.pico_optim_sgd_zero_grad(opt)
            P.lib.pico_backward(a, eager)
            want = grads()
            with P.arena() as b:
                out = _block(P, p, rope, dev)
                P.lib.pico_backward(b, out)
                P.reset(b)
                assert P.lib.pico_graph_begin() == 0
                out = _block(P, p, rope, dev)
                P.lib.pico_optim_sgd_zero_grad(opt)
                P.lib.pico_backward(b, out)
                graph = P.lib.pico_graph_end()
                assert graph, P.lib.pico_gpu_last_error()
                for _ in range(3):
                    assert P.lib.pico_graph_launch(graph) == 0
                    got = grads()
                    for k in SHAPES:
                        assert np.array_equal(got[k], want[k]), k
                    P.lib.pico_optim_sgd_zero_grad(opt)
                    P.lib.pico_backward(a, eager)
                    assert np.isfinite(P.grad_value(p["wo"])).all()
                P.lib.pico_graph_free(graph)
    assert not P.lib.pico_gpu_last_error()
    P.lib.pico_rope_free(rope)
    P.lib.pico_optim_sgd_free(opt)
    for t in p.values():
        P.free(t)


# ------------------------------------------------------------- token by token
class Model:
    """the oracle of a cache of several layers, page numbers of its own"""

    def __init__(self, layers, kvh, hd, page, seqs, length):
        width = -(-length // page)
        table = np.arange(seqs * width).reshape(seqs, width)
        self.layers = [O.Cache(seqs * width, kvh, page, hd, table) for _ in range(layers)]
        self.lens = np.zeros(seqs, int)
        self.kvh, self.hd = kvh, hd

    def step(self, new, inputs, heads, turn):
        """[(o, tol)] of every layer, for its (q, k, v) [N, heads, hd]; turn(x, pos): as
        pico_rope does it, so that the keys' 8 bits are the same"""
        offsets = np.concatenate([[0], np.cumsum(new)])
        pos = np.concatenate([np.arange(a, a + n) for a, n in zip(self.lens, new)]).astype(np.int32)
        out = []
        for c, (q, k, v) in zip(self.layers, inputs):
            c.append(turn(k, pos), v, self.lens, offsets)
            out.append(c.attend(turn(q, pos).astype(np.float64), self.lens, offsets, heads))
        self.lens = self.lens + new
        return out


def _step(P, kv, rope, new, inputs, heads):
    N = P.kv_begin(kv, new)
    assert N == sum(new)
    got = []
    for layer, qkv in enumerate(inputs):
        q, k, v = (P.tensor([N, x.shape[1] * x.shape[2]], x) for x in qkv)
        got.append(P.value(P.attention_cached(kv, layer, q, k, v, heads, rope)))
    return got


def _inputs(rng, layers, N, heads, kvh, hd):
    return [tuple(rng.standard_normal((N, n, hd)).astype(np.float32) for n in (heads, kvh, kvh))
            for _ in range(layers)]


@pytest.mark.parametrize("kvh,heads,hd,page,turn", [(2, 4, 64, 16, True), (1, 3, 40, 32, False), (3, 3, 128, 64, False)])
def test_steps_of_a_model(P, kvh, heads, hd, page, turn):
    """prompts, single tokens, a sequence that waits, one that is dropped and begins anew"""
    rng = np.random.default_rng(hd)
    layers, seqs, length = 2, 3, 200
    kv = P.kv_init(layers, kvh, hd, page, 3 * -(-length // page), seqs, length)
    rope = P.rope_init(2 * (hd // 4)) if turn else None

    def turned(x, pos):
        if not turn:
            return x
        with P.arena():
            t = P.rope(P.tensor([len(x), x.shape[1] * hd], x), rope, pos, x.shape[1])
            return P.value(t).reshape(x.shape)

    model = Model(layers, kvh, hd, page, seqs, length)
    for new in ([70, 0, 5], [1, 1, 1], [0, 33, 1], None, [1, 4, 1], [100, 1, 0]):
        if new is None:
            assert P.lib.pico_kv_drop(kv, 0) == 0
            assert P.lib.pico_kv_length(kv, 0) == 0
            model.lens[0] = 0
            continue
        inputs = _inputs(rng, layers, sum(new), heads, kvh, hd)
        with P.arena():
            got = _step(P, kv, rope, new, inputs, heads)
        assert [P.lib.pico_kv_length(kv, b) for b in range(seqs)] == list(model.lens + new)
        for x, (want, tol) in zip(got, model.step(np.array(new), inputs, heads, turned)):
            assert (np.abs(x.reshape(want.shape) - want) <= tol).all()
    if rope:
        P.lib.pico_rope_free(rope)
    P.lib.pico_kv_free(kv)


def test_views_of_one_projection(P):
    """q, k and v as column views of one product give what contiguous ones give"""
    rng = np.random.default_rng(4)
    H, hd = 3, 64
    x = rng.standard_normal((6, 3 * H * hd)).astype(np.float32)
    rope = P.rope_init(hd, interleaved=True)
    out = []
    for views in (True, False):
        kv = P.kv_init(1, H, hd, 16, 8, 2, 64)
        with P.arena():
            assert P.kv_begin(kv, [2, 4]) == 6
            if views:
                q, k, v = P.split_cols(P.tensor(list(x.shape), x), 3)
            else:
                q, k, v = (P.tensor([6, H * hd], np.ascontiguousarray(t)) for t in np.split(x, 3, axis=1))
            out.append(P.value(P.attention_cached(kv, 0, q, k, v, H, rope)))
        P.lib.pico_kv_free(kv)
    assert np.array_equal(out[0], out[1])
    P.lib.pico_rope_free(rope)


def test_pages_run_out_and_come_back(P):
    kv = P.kv_init(1, 1, 32, 16, 4, 2, 64)
    one = np.zeros((1, 32), np.float32)
    with P.arena():
        assert P.kv_begin(kv, [40, 16]) == 56  # 3 and 1 pages: all
        for bad in ([0, 1], [9, 0], [-1, 0], [0, 100]):
            with pytest.raises(PicoError):
                P.kv_begin(kv, bad)
            assert [P.lib.pico_kv_length(kv, b) for b in (0, 1)] == [40, 16]
        assert P.kv_begin(kv, [8, 0]) == 8  # room on a page that it has
        assert P.lib.pico_kv_drop(kv, 0) == 0
        t = P.tensor([1, 32], one)
        with pytest.raises(PicoError):  # no step since
            P.attention_cached(kv, 0, t, t, t, 1, None)
        assert P.kv_begin(kv, [1, 30]) == 31
        assert P.kv_begin(kv, [0, 0]) == 0
        e = P.tensor([0, 32], np.zeros((0, 32)))
        assert P.value(P.attention_cached(kv, 0, e, e, e, 1, None)).size == 0
        with pytest.raises(PicoError):
            P.kv_begin(kv, [0, 64])  # past max_length
    assert P.lib.pico_kv_length(kv, 2) == -1
    assert P.lib.pico_kv_drop(kv, 2) != 0
    P.lib.pico_kv_free(kv)


def test_refusals(P):
    kv = P.kv_init(2, 2, 32, 16, 4, 1, 64)
    rope, wide = P.rope_init(32), P.rope_init(64)
    with P.arena():
        q, k = P.tensor([3, 128], np.zeros((3, 128))), P.tensor([3, 64], np.zeros((3, 64)))
        with pytest.raises(PicoError):  # no step begun
            P.attention_cached(kv, 0, q, k, k, 4, rope)
        P.kv_begin(kv, [3])
        for args in ((2, q, k, k, 4, rope), (-1, q, k, k, 4, rope), (0, q, k, k, 3, rope), (0, q, k, k, 0, rope),
                     (0, k, k, k, 4, rope), (0, q, q, k, 4, rope), (0, q, k, q, 4, rope), (0, q, k, k, 4, wide),
                     (0, P.tensor([2, 128], np.zeros((2, 128))), k, k, 4, rope)):
            with pytest.raises(PicoError):
                P.attention_cached(kv, *args)
        assert P.shape(P.attention_cached(kv, 0, q, k, k, 4, rope)) == (3, 128)
        with pytest.raises(PicoError):
            P.rope(k, wide, [0, 1, 2], 2)  # heads of 32
        with pytest.raises(PicoError):
            P.rope(k, rope, [0, 1, 2], 3)
        with pytest.raises(PicoError):
            P._check(P.lib.pico_rope(k, None, P.ids([0, 1, 2]), 2), "pico_rope")
        with pytest.raises(PicoError):
            P._check(P.lib.pico_rope(k, rope, None, 2), "pico_rope")
        assert P.lib.pico_graph_begin() == 0
        with pytest.raises(PicoError):
            P.kv_begin(kv, [1])
        assert not P.lib.pico_graph_end()
        assert P.lib.pico_kv_length(kv, 0) == 3
    P.lib.pico_gpu_clear_error()
    for r in (rope, wide):
        P.lib.pico_rope_free(r)
    P.lib.pico_kv_free(kv)


def test_captured_step(P):
    """a step of two layers captured once and replayed after each pico_kv_begin, a sequence
    growing into new pages, against eager steps of a cache of its own"""
    rng = np.random.default_rng(5)
    kvh, heads, hd, seqs = 2, 4, 64, 2
    rope = P.rope_init(hd)
    kvs = [P.kv_init(2, kvh, hd, 16, 40, seqs, 300) for _ in range(2)]
    leaves = {n: P.param([seqs, w * hd]) for n, w in (("q", heads), ("k", kvh), ("v", kvh))}

    def layer(kv):
        x = P.attention_cached(kv, 0, leaves["q"], leaves["k"], leaves["v"], heads, rope)
        return P.attention_cached(kv, 1, x, leaves["k"], leaves["v"], heads, rope)

    prompt = [rng.standard_normal((35, w * hd)).astype(np.float32) for w in (heads, kvh, kvh)]
    for kv in kvs:
        with P.arena():
            P.kv_begin(kv, [30, 5])
            q, k, v = (P.tensor(list(x.shape), x) for x in prompt)
            for i in range(2):
                P.attention_cached(kv, i, q, k, v, heads, rope)
            P.sync()
    with P.arena() as a:
        P.kv_begin(kvs[0], [1, 1])
        P.kv_begin(kvs[1], [1, 1])
        layer(kvs[0])
        with P.arena():
            layer(kvs[1])
            P.sync()
        P.reset(a)
        assert P.lib.pico_graph_begin() == 0
        out = layer(kvs[0])
        graph = P.lib.pico_graph_end()
        assert graph, P.lib.pico_gpu_last_error()
        for i in range(20):
            for t, w in (("q", heads), ("k", kvh), ("v", kvh)):
                P.set(leaves[t], rng.standard_normal((seqs, w * hd)))
            for kv in kvs:
                P.kv_begin(kv, [1, 1])
            assert P.lib.pico_graph_launch(graph) == 0
            got = P.value(out)
            with P.arena():
                want = P.value(layer(kvs[1]))
            assert np.array_equal(got, want), i
        P.lib.pico_graph_free(graph)
    assert not P.lib.pico_gpu_last_error()
    P.lib.pico_rope_free(rope)
    for kv in kvs:
        P.lib.pico_kv_free(kv)
    for t in leaves.values():
        P.free(t)


def test_max_length_within_a_page(P):
    """max_length holds, though the last page has room for more"""
    kv = P.kv_init(1, 1, 32, 16, 8, 2, 20)
    assert P.kv_begin(kv, [19, 0]) == 19
    for bad in ([2, 0], [0, 21], [13, 1]):
        with pytest.raises(PicoError):
            P.kv_begin(kv, bad)
        assert [P.lib.pico_kv_length(kv, b) for b in (0, 1)] == [19, 0]
    assert P.kv_begin(kv, [1, 20]) == 21
    with pytest.raises(PicoError):
        P.kv_begin(kv, [1, 0])
    assert P.kv_begin(kv, [0, 0]) == 0
    assert P.lib.pico_kv_drop(kv, 0) == 0
    assert P.kv_begin(kv, [20, 0]) == 20
    P.lib.pico_kv_free(kv)


def test_arrays_of_another_length(P):
    """fewer positions than rows, or counts than sequences, are not read past their end"""
    kv, rope = P.kv_init(1, 1, 32, 16, 8, 2, 64), P.rope_init(32)
    with P.arena():
        x = P.tensor([3, 32], np.zeros((3, 32)))
        for pos in ([0, 1], [], [0, 1, 2, 3], np.zeros((2, 3))):
            with pytest.raises(ValueError):
                P.rope(x, rope, pos, 1)
        assert P.shape(P.rope(x, rope, [[0], [1], [2]], 1)) == (3, 32)
    for new in ([1], [], [1, 1, 1]):
        with pytest.raises(ValueError):
            P.kv_begin(kv, new)
        assert [P.lib.pico_kv_length(kv, b) for b in (0, 1)] == [0, 0]
    assert P.kv_begin(kv, np.array([2, 1], np.int64)) == 3
    P.lib.pico_rope_free(rope)
    P.lib.pico_kv_free(kv)
