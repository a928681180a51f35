"""A recurrent mixture-of-experts block as a user builds it from pico's ops: layer norm,
gated recurrence over a projection's column views, layer norm, router and experts.
Trained eagerly and as a captured step, whose replays must equal the eager steps bit
for bit; gradients against float64 autograd."""
import numpy as np
import pytest
import torch

from pico_amd.pico import Pico

pytestmark = pytest.mark.gpu

B, T, D, F, E, TOPK, EPS = 3, 21, 32, 40, 5, 2, 1e-5
N = B * T
SHAPES = {"x": (N, D), "g1": (D,), "b1": (D,), "wfx": (D, 2 * D), "wo": (D, D), "h0": (B, D), "g2": (D,),
          "b2": (D,), "wr": (D, E), "w13": (E, D, 2 * F), "w2": (E, F, D)}


@pytest.fixture(scope="module")
def P():
    return Pico()


def _values(seed):
    g = torch.Generator().manual_seed(seed)
    v = {k: torch.randn(*s, generator=g) * (s[-2] ** -0.5 if k.startswith("w") else 1.0)
         for k, s in SHAPES.items()}
    for k in ("g1", "g2"):
        v[k] = 1 + 0.1 * v[k]
    return v


def _block(P, p):
    h = P.layernorm(p["x"], p["g1"], p["b1"], EPS)
    f, u = P.split_cols(P.matmul(h, p["wfx"]), 2)
    x = P.matmul_add(P.gated_scan(f, u, p["h0"], B), p["wo"], p["x"])
    h = P.layernorm(x, p["g2"], p["b2"], EPS)
    gates, route = P.route_topk(P.matmul(h, p["wr"]), TOPK)
    gu = P.expert_matmul(P.expert_gather(h, route), p["w13"], route)
    ys = P.expert_matmul(P.swiglu(*P.split_cols(gu, 2)), p["w2"], route)
    return P.expert_combine(ys, gates, route, x), route


def _exact(v):
    v = {k: t.double().requires_grad_() for k, t in v.items()}

    def norm(x, g, b):
        m = x.mean(1, keepdim=True)
        return (x - m) / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + EPS) * g + b

    f, u = (norm(v["x"], v["g1"], v["b1"]) @ v["wfx"]).view(B, T, 2 * D).split(D, 2)
    s, state, hs = torch.sigmoid(f), v["h0"], []
    for t in range(T):
        state = s[:, t] * state + (1 - s[:, t]) * u[:, t]
        hs.append(state)
    x = v["x"] + torch.stack(hs, 1).reshape(N, D) @ v["wo"]
    h = norm(x, v["g2"], v["b2"])
    z = h @ v["wr"]
    top = torch.sort(z, dim=1, descending=True, stable=True)
    gates, experts = torch.softmax(top.values[:, :TOPK], 1), top.indices[:, :TOPK]
    y = x
    for e in range(E):
        t, j = torch.nonzero(experts == e, as_tuple=True)
        gate, up = (h[t] @ v["w13"][e]).split(F, 1)
        y = y.index_add(0, t, ((torch.nn.functional.silu(gate) * up) @ v["w2"][e]) * gates[t, j][:, None])
    gap = (top.values[:, TOPK - 1] - top.values[:, TOPK]).min()
    return v, y, float(gap.detach())


def test_gradients(P):
    vals = _values(1)
    v, y, gap = _exact(vals)
    assert gap > 1e-4  # no choice hangs on a rounding
    y.sum().backward()
    p = {k: P.param(list(t.shape), t.numpy()) for k, t in vals.items()}
    with P.arena():
        out, _ = _block(P, p)
        P.backward(out)
        # eleven products, norms and sums of fewer than 200 terms on the way: 1e-4 is
        # over 100 times 11 * 200 u / sqrt(200)
        for got, want in [(P.value(out), y)] + [(P.grad_value(p[k]), v[k].grad) for k in SHAPES]:
            want = want.detach()
            err = (torch.from_numpy(got).double() - want).norm() / want.norm()
            assert float(err) <= 1e-4
    for t in p.values():
        P.free(t)


def test_training_steps_captured_and_replayed(P):
    """five SGD steps, four of them from a graph, and five eager ones: the same parameters bit for
    bit; eager work between the replays, and a second graph of the same leaves"""
    vals = _values(2)

    def make():
        p = {k: P.param(list(t.shape), t.numpy()) for k, t in vals.items()}
        opt = P.lib.pico_optim_sgd_init(1e-6)
        for t in p.values():
            P.lib.pico_optim_sgd_add(opt, t)
        return p, opt

    def step(arena, p, opt):
        out, route = _block(P, p)
        P.lib.pico_optim_sgd_zero_grad(opt)
        P.lib.pico_backward(arena, out)
        P.lib.pico_optim_sgd_step(opt)
        return out, route

    p, opt = make()
    with P.arena() as a:
        eager = []
        for _ in range(5):
            out, _ = step(a, p, opt)
            eager.append(P.data(out))
            P.reset(a)
        want = {k: P.data(t) for k, t in p.items()}
    assert not P.lib.pico_gpu_last_error()
    q, opt2 = make()
    with P.arena() as a:
        out, _ = step(a, q, opt2)
        got = [P.data(out)]
        P.reset(a)
        assert P.lib.pico_graph_begin() == 0
        out, route = step(a, q, opt2)
        graph = P.lib.pico_graph_end()
        assert graph, P.lib.pico_gpu_last_error()
        with P.arena() as b:  # another graph, of a forward pass over the same leaves
            warm, _ = _block(P, q)
            P.reset(b)
            assert P.lib.pico_graph_begin() == 0
            other, _ = _block(P, q)
            second = P.lib.pico_graph_end()
            assert second, P.lib.pico_gpu_last_error()
            for i in range(4):
                assert P.lib.pico_graph_launch(graph) == 0
                got.append(P.data(out))
                assert P.lib.pico_graph_launch(second) == 0
                after = P.data(other)
                with P.arena():
                    assert np.array_equal(P.data(_block(P, q)[0]), after)
                experts, offsets = P.route_to_host(route, N, TOPK, E)
                assert offsets[E] == N * TOPK and (experts >= 0).all()
            P.lib.pico_graph_free(second)
        for x, y in zip(got, eager):
            assert np.array_equal(x, y)
        for k, t in q.items():
            assert np.array_equal(P.data(t), want[k]), k
        P.lib.pico_graph_free(graph)
    for o, d in ((opt, p), (opt2, q)):
        P.lib.pico_optim_sgd_free(o)
        for t in d.values():
            P.free(t)


def test_capture_beside_a_live_eager_graph(P):
    """a step captured while an eager graph of the same leaves, its backward done, is kept;
    that graph's second backward between the replays"""
    vals = _values(3)
    p = {k: P.param(list(t.shape), t.numpy()) for k, t in vals.items()}
    grads = lambda: {k: P.grad_value(t) for k, t in p.items()}
    opt = P.lib.pico_optim_sgd_init(0.0)
    for t in p.values():
        P.lib.pico_optim_sgd_add(opt, t)
    with P.arena() as a:
        eager, _ = _block(P, p)
        P.lib.pico_optim_sgd_zero_grad(opt)
        P.lib.pico_backward(a, eager)
        want = grads()
        with P.arena() as b:
            out, _ = _block(P, p)  # the arena's blocks
            P.lib.pico_optim_sgd_zero_grad(opt)
            P.lib.pico_backward(b, out)
            P.reset(b)
            assert P.lib.pico_graph_begin() == 0
            out, _ = _block(P, p)
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
                assert np.isfinite(P.grad_value(p["w13"])).all()
            P.lib.pico_graph_free(graph)
    assert not P.lib.pico_gpu_last_error()
    P.lib.pico_optim_sgd_free(opt)
    for t in p.values():
        P.free(t)


def test_no_tokens(P):
    """an empty batch: empty results, and gradients of zero"""
    d, e, k = 8, 4, 2
    w = P.param([e, d, d], np.ones((e, d, d), np.float32))
    g, b = P.param([d], np.ones(d, np.float32)), P.param([d], np.ones(d, np.float32))
    with P.arena():
        x = P.layernorm(P.tensor([0, d], np.zeros((0, d))), g, b, EPS)
        x = P.gated_scan(x, P.tensor([0, d], np.zeros((0, d))), None, 3)
        gates, route = P.route_topk(P.tensor([0, e], np.zeros((0, e))), k)
        y = P.expert_combine(P.expert_matmul(P.expert_gather(x, route), w, route), gates, route, x)
        assert P.data(y).size == 0
        experts, offsets = P.route_to_host(route, 0, k, e)
        assert experts.size == 0 and not offsets.any()
        P.backward(y)
        for t in (w, g, b):
            assert not P.grad_value(t).any()
    for t in (w, g, b):
        P.free(t)
