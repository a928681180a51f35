"""The recurrence, the last token, the router and the experts over column views, weights that
are no parameters, and a stream of the caller's; against float64 autograd.

Bounds: every result passes at most four products, norms or sums of fewer than 200 terms;
1e-4 of its 2-norm is over 100 times 4 * 200 u / sqrt(200), u = 2^-24."""
import numpy as np
import pytest
import torch

from pico_amd.pico import Pico

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def P():
    return Pico()


def _near(got, want, what):
    want = want.detach()
    err = (torch.as_tensor(got).double() - want).norm() / want.norm()
    assert float(err) <= 1e-4, (what, float(err))


def _values(seed, **shapes):
    g = torch.Generator().manual_seed(seed)
    return {k: torch.randn(*s, generator=g) for k, s in shapes.items()}


def test_last_token_of_a_column_view(P):
    """the last token of one half of a projection, beside the other half used whole"""
    B, T, C = 3, 5, 8
    v = _values(1, x=(B * T, C), w=(C, 2 * C), d=(B, C), e=(B * T, C))
    leaves = {k: v[k].double().requires_grad_() for k in ("x", "w")}
    y = leaves["x"] @ leaves["w"]
    last = y[:, C:].reshape(B, T, C)[:, -1]
    ((last * v["d"].double()).sum() + (torch.nn.functional.silu(y[:, :C]) * y[:, C:] * v["e"].double()).sum()).backward()
    x, w = P.param([B * T, C], v["x"].numpy()), P.param([C, 2 * C], v["w"].numpy())
    with P.arena():
        a, b = P.split_cols(P.matmul(x, w), 2)
        got = P.last_token(b, B)
        _near(P.value(got), last, "last")
        one = P.mul(got, P.tensor([B, C], v["d"].numpy()))
        two = P.mul(P.swiglu(a, b), P.tensor([B * T, C], v["e"].numpy()))
        total = P.add(P.matmul(P.matmul(P.tensor([1, B], np.ones(B)), one), P.tensor([C, 1], np.ones(C))),
                      P.matmul(P.matmul(P.tensor([1, B * T], np.ones(B * T)), two), P.tensor([C, 1], np.ones(C))))
        P.backward(total)
        for t, k in ((x, "x"), (w, "w")):
            _near(P.grad_value(t), leaves[k].grad, k)
    for t in (x, w):
        P.free(t)


def _experts(v, tokens, k, d, E):
    """[x | logits | rest] = a w, routed by the logits: the layer, in float64"""
    y = v["a"] @ v["w"]
    x, z = y[:, :d], y[:, d:d + E]
    top = torch.sort(z, dim=1, descending=True, stable=True)
    gates, experts = torch.softmax(top.values[:, :k], 1), top.indices[:, :k]
    out = 0
    for e in range(E):
        t, j = torch.nonzero(experts == e, as_tuple=True)
        out = out + torch.zeros(tokens, d, dtype=torch.float64).index_add(0, t, (x[t] @ v["we"][e]) *
                                                                          gates[t, j][:, None])
    gap = (top.values[:, k - 1] - top.values[:, k]).min()
    return out, float(gap.detach())


@pytest.mark.parametrize("own_stream", [False, True])
@pytest.mark.parametrize("weights", ["parameters", "tensors", "a product"])
def test_views_and_weights_that_are_no_parameters(P, weights, own_stream):
    """tokens and logits as column views of one projection; the experts' weights as
    parameters, or as tensors of the arena; on the library's stream and on a caller's"""
    tokens, k, d, E = 45, 2, 12, 12
    vals = _values(8, a=(tokens, 20), w=(20, 2 * d), we=(E, d, d), dy=(tokens, d))
    v = {n: t.double().requires_grad_() for n, t in vals.items() if n != "dy"}
    want, gap = _experts(v, tokens, k, d, E)
    assert gap > 1e-4  # no choice hangs on a rounding
    (want * vals["dy"].double()).sum().backward()
    stream = torch.cuda.Stream()
    if own_stream:
        torch.cuda.synchronize()
        P.lib.pico_gpu_set_stream(stream.cuda_stream)
    try:
        made = {n: P.param(list(t.shape), t.numpy()) for n, t in vals.items() if n != "dy"}
        with P.arena():
            p = dict(made)
            if weights == "tensors":
                p = {n: P.tensor(list(vals[n].shape), vals[n].numpy()) for n in made}
            elif weights == "a product":
                p["we"] = P.mul(made["we"], P.tensor([E, d, d], np.ones((E, d, d))))
            x, z = P.split_cols(P.matmul(p["a"], p["w"]), 2)
            gates, route = P.route_topk(z, k)
            ys = P.expert_matmul(P.expert_gather(x, route), p["we"], route)
            out = P.expert_combine(ys, gates, route, None)
            P.backward(P.mul(out, P.tensor([tokens, d], vals["dy"].numpy())))
            _near(P.value(out), want, "y")
            for n in v:
                _near(P.grad_value(p[n]), v[n].grad, n)
                if weights == "a product":
                    _near(P.grad_value(made[n]), v[n].grad, n)
        for t in made.values():
            P.free(t)
    finally:
        P.sync()
        if own_stream:
            P.lib.pico_gpu_set_stream(None)
    assert not P.lib.pico_gpu_last_error()
