"""The mixture of experts (pk_route_topk_*, pk_expert_*, pk_gemm_experts_*, and pico's
ops on them) against float64.

Bounds, u = 2^-24.  Products: an fp32 product of K terms is within (K + 8) 2 u of the
sum of |a||b| (24-bit products, fp32 sums that may drop a last bit); bf16 products
are exact for the rounded operands, so the same with operands rounded; of three bf16
products the operands' halves leave 2^-17 each and lo.lo 2^-16.  A softmax over k logits:
(|z - top| + k + 8) u.  Weighted sums of k rows and dot products of d values: one u for
every addition on the way, at most d/64 + 8 of a dot product.
"""
import numpy as np
import pytest
import torch

from pico_amd import _lib
from pico_amd import kernels as K
from pico_amd.pico import Pico, PicoError

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = float("inf")


@pytest.fixture(scope="module")
def P():
    return Pico()


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _empty(*shape, dtype=torch.float32):
    return torch.full(shape, 7, device="cuda:0", dtype=dtype)


def _close(got, want, tol, what):
    ratio = (got.double().cpu() - want).abs() / (tol + 1e-37)
    assert bool((ratio <= 1).all()), (what, float(ratio.max()))


# -------------------------------------------------------------------- router
def _choose(z, k):
    """by hand: experts (int32) and gates (float64) of every token"""
    R, E = z.shape
    experts, gates = np.full((R, k), -1, np.int32), np.zeros((R, k))
    for t in range(R):
        row = z[t].tolist()
        key = [(0 if v != v else 1, 0.0 if v != v else -v, e) for e, v in enumerate(row)
               if v != -INF]
        top = [e for _, _, e in sorted(key)[:k]]
        experts[t, :len(top)] = top
        if top:
            v = np.array([row[e] for e in top])
            with np.errstate(all="ignore"):
                w = np.exp(v - v[0])
                gates[t, :len(top)] = w / w.sum()
    return experts, gates


ROUTES = [(1, 1, 1), (1, 2, 1), (5, 2, 2), (64, 8, 2), (33, 8, 8), (7, 9, 3), (100, 16, 4), (31, 17, 17),
          (50, 32, 6), (65, 33, 2), (257, 64, 8), (40, 64, 64), (20, 65, 2), (30, 128, 8), (9, 129, 5),
          (17, 256, 8), (8, 512, 10), (6, 777, 64), (5, 1024, 3)]


@pytest.mark.parametrize("R,E,k", ROUTES)
def test_router(dev, R, E, k):
    z = torch.randn(R, E, generator=_gen(R + E)) * 2
    z = (z * 4).round() / 4  # with ties
    z[R // 2, : E // 2] = -INF
    if R > 2:
        z[R - 1] = -INF  # nothing to choose
        z[R - 2] = torch.finfo(torch.float32).min  # all equal, and choosable
        z[0, E // 3] = torch.finfo(torch.float32).min
    want_e, want_g = _choose(z, k)
    zd = torch.full((R, E + 3), 9.0)
    zd[:, :E] = z
    zd = zd.cuda()
    experts, gates = _empty(R + 1, k, dtype=torch.int32), _empty(R + 1, k)
    K.route_topk(zd[:, :E], experts[:R], gates[:R])
    assert np.array_equal(experts[:R].cpu().numpy(), want_e)
    drop = np.where(want_e < 0, 0, np.take_along_axis(z.numpy().astype(np.float64),
                                                      np.maximum(want_e, 0), 1))
    spread = np.where(want_e < 0, 0, drop[:, :1] - drop)
    tol = want_g * (spread + k + 8) * U
    _close(gates[:R], torch.from_numpy(want_g), torch.from_numpy(tol), "gates")
    assert bool((gates[R] == 7).all()) and bool((experts[R] == 7).all())
    # the gradient, written and added
    dg = torch.randn(R, k, generator=_gen(3)).cuda()
    g64, d64 = torch.from_numpy(want_g), dg.double().cpu()
    mixed = (g64 * d64).sum(1, keepdim=True)
    want = torch.zeros(R, E + 1, dtype=torch.float64)
    bound = torch.zeros(R, E + 1, dtype=torch.float64)
    at = torch.from_numpy(np.where(want_e < 0, E, want_e)).long()
    want.scatter_add_(1, at, g64 * (d64 - mixed))
    rel = torch.from_numpy(spread) + 3 * k + 20
    bound.scatter_add_(1, at, g64 * U * (rel * (d64.abs() + mixed.abs()) +
                                         (rel.amax(1, keepdim=True) * (g64 * d64).abs().sum(1, keepdim=True))))
    dz = _empty(R, E + 3)
    K.route_topk_bwd(experts[:R], gates[:R], dg, dz[:, :E])
    _close(dz[:, :E], want[:, :E], bound[:, :E], "dlogits")
    assert bool((dz[:, E:] == 7).all())
    base = torch.randn(R, E, generator=_gen(4)).cuda()
    acc = base.clone()
    K.route_topk_bwd(experts[:R], gates[:R], dg, acc, accum=True)
    assert torch.equal(acc, base + dz[:, :E])


def test_router_bad_values(dev):
    """NaN is above all and leaves its token's gates NaN, +inf as a softmax has it"""
    z = torch.tensor([[1.0, float("nan"), 3.0, 2.0], [0.0, INF, 1.0, 2.0], [1.0, 1.0, 1.0, 1.0],
                      [-0.0, 0.0, -1.0, 0.0]]).cuda()
    experts, gates = _empty(4, 2, dtype=torch.int32), _empty(4, 2)
    K.route_topk(z, experts, gates)
    assert experts.tolist() == [[1, 2], [1, 3], [0, 1], [0, 1]]
    assert bool(torch.isnan(gates[0]).all()) and bool(torch.isnan(gates[1, 0]))
    assert gates[2:].tolist() == [[0.5, 0.5], [0.5, 0.5]]


def test_router_gradient_against_differences(dev):
    R, E, k = 6, 10, 3
    z = torch.randn(R, E, generator=_gen(1))
    dg = torch.randn(R, k, generator=_gen(2))
    experts, gates, dz = _empty(R, k, dtype=torch.int32), _empty(R, k), _empty(R, E)
    K.route_topk(z.cuda(), experts, gates)
    K.route_topk_bwd(experts, gates, dg.cuda(), dz)
    for i in range(0, R * E, 3):
        step = []
        for d in (1e-5, -1e-5):
            moved = z.double()
            moved.view(-1)[i] += d
            step.append((torch.from_numpy(_choose(moved, k)[1]) * dg.double()).sum())
        diff = float((step[0] - step[1]) / 2e-5)
        assert abs(float(dz.view(-1)[i]) - diff) <= 2e-5


# ---------------------------------------------------------------------- plan
def _plan(experts, E):
    flat = experts.reshape(-1).tolist()
    lists = [[i for i, e in enumerate(flat) if e == x] for x in range(E)] if E * len(flat) < 1e6 else None
    if lists is None:
        lists = [[] for _ in range(E)]
        for i, e in enumerate(flat):
            if 0 <= e < E:
                lists[e].append(i)
    order = [i for group in lists for i in group]
    offsets = np.cumsum([0] + [len(group) for group in lists])
    place = np.full(len(flat), -1)
    place[order] = np.arange(len(order))
    order += [i for i, e in enumerate(flat) if not 0 <= e < E]
    return offsets, np.array(order, int), place


@pytest.mark.parametrize("n,E", [(1, 1), (2, 3), (63, 2), (64, 64), (65, 7), (1000, 8), (1024, 16),
                                 (1025, 63), (2047, 64), (5000, 65), (8192, 256), (8193, 3), (10241, 129),
                                 (40000, 1000), (300, 1023), (9001, 1024), (70001, 8)])
def test_plan(dev, n, E):
    g = _gen(n + E)
    share = torch.rand(E, generator=g) ** 3 + 1e-6
    if E > 2:
        share[E // 2] = 0
    experts = torch.multinomial(share, n, replacement=True, generator=g).to(torch.int32)
    drop = torch.rand(n, generator=g)
    experts[drop < 0.05] = -1
    experts[(drop > 0.05) & (drop < 0.07)] = E
    experts[(drop > 0.07) & (drop < 0.08)] = 2 ** 31 - 1
    offsets, order, place = (_empty(m + 1, dtype=torch.int32) for m in (E + 1, n, n))
    K.expert_plan(experts.cuda(), offsets[:-1], order[:-1], place[:-1])
    for got, want in zip((offsets, order, place), _plan(experts, E)):
        assert np.array_equal(got[:-1].cpu().numpy(), want)
        assert int(got[-1]) == 7


def test_plan_of_one_expert_and_of_none(dev):
    for fill in (2, -1):
        experts = torch.full((3000,), fill, dtype=torch.int32).cuda()
        offsets, order, place = (_empty(m, dtype=torch.int32) for m in (6, 3000, 3000))
        K.expert_plan(experts, offsets, order, place)
        for got, want in zip((offsets, order, place), _plan(experts.cpu(), 5)):
            assert np.array_equal(got.cpu().numpy(), want)
    none = torch.empty(0, dtype=torch.int32, device="cuda:0")
    offsets = _empty(6, dtype=torch.int32)
    K.expert_plan(none, offsets, none, none)
    assert not offsets.any()


# ---------------------------------------------------------------------- rows
def _routing(R, k, E, seed, dropped=0.1):
    g = _gen(seed)
    experts = torch.randint(0, E, (R, k), generator=g).to(torch.int32)
    experts[torch.rand(R, k, generator=g) < dropped] = -1
    if R > 1:
        experts[R // 2] = -1  # a token without any
    n = R * k
    offsets, order, place = (_empty(m, dtype=torch.int32) for m in (E + 1, n, n))
    K.expert_plan(experts.cuda(), offsets, order, place)
    return experts, offsets, order, place


@pytest.mark.parametrize("R,k,E,d", [(1, 1, 1, 1), (3, 2, 4, 5), (64, 2, 8, 64), (50, 3, 5, 63), (33, 1, 7, 260),
                                     (100, 8, 16, 96), (17, 2, 3, 1030), (1000, 2, 64, 36)])
@pytest.mark.parametrize("pad", [0, 1, 4])
def test_gather_and_combine(dev, R, k, E, d, pad):
    experts, offsets, order, place = _routing(R, k, E, R + d)
    g = _gen(d)
    n, kept = R * k, int(offsets[E])

    def rows(m):
        full = torch.randn(m, d + pad, generator=g).cuda()
        return full[:, :d], full

    x, _ = rows(R)
    out, guard = rows(n)
    guard.fill_(7)
    K.expert_gather(x, k, offsets, order, out)
    src = (order.long() // k)[:kept]
    assert torch.equal(out[:kept], x[src]) and not out[kept:].any()
    assert bool((guard[:, d:] == 7).all())
    # combine, with and without the residual and the gates
    ys, _ = rows(n)
    ys[kept:] = float("nan")  # never read
    c, _ = rows(R)
    gates = torch.rand(R, k, generator=g).cuda()
    p = place.long().view(R, k).cpu()
    picked = torch.where((p < 0)[:, :, None], 0.0, ys.double().cpu()[p])
    for residual in (None, c):
        for weights in (gates, None):
            w = torch.ones(R, k, dtype=torch.float64) if weights is None else weights.double().cpu()
            terms = picked * w[:, :, None]
            want = terms.sum(1) + (0 if residual is None else residual.double().cpu())
            bound = (k + 2) * U * (terms.abs().sum(1) + (0 if residual is None else residual.double().cpu().abs()))
            got, guard = rows(R)
            guard.fill_(7)
            K.expert_combine(place, weights, ys, got, c=residual)
            _close(got, want, bound, "combine")
            assert bool((guard[:, d:] == 7).all())
    inplace = c.clone()
    K.expert_combine(place, gates, ys, inplace, c=inplace)
    again, _ = rows(R)
    K.expert_combine(place, gates, ys, again, c=c.clone())
    assert torch.equal(inplace, again)
    # gradients
    dout, _ = rows(R)
    dys, dguard = rows(n)
    dguard.fill_(7)
    dgates = _empty(R, k)
    K.expert_combine_bwd(offsets, order, gates, ys, dout, dys, dgates)
    flat = gates.view(-1)[order.long()][:kept]
    assert torch.equal(dys[:kept], flat[:, None] * dout[src]) and not dys[kept:].any()
    prods = picked * dout.double().cpu()[:, None]
    _close(dgates, prods.sum(2), (d / 64 + 9) * U * prods.abs().sum(2), "dgates")
    assert bool((dguard[:, d:] == 7).all())
    b1, b2 = torch.randn(n, d, generator=g).cuda(), torch.randn(R, k, generator=g).cuda()
    a1, a2 = b1.clone(), b2.clone()
    K.expert_combine_bwd(offsets, order, gates, ys, dout, a1, None, accum_dys=True)
    K.expert_combine_bwd(offsets, order, gates, ys, dout, None, a2, accum_dgates=True)
    assert bool(((a1 - (b1 + dys)).abs() <= 2 * U * (b1.abs() + dys.abs())).all())
    # (unaligned rows add the dot product in another order)
    assert bool(((a2 - (b2 + dgates)).abs().double().cpu() <=
                 2 * (d / 64 + 10) * U * prods.abs().sum(2) + 2 * U * b2.abs().double().cpu()).all())


# ------------------------------------------------------------------ products
def _offsets(sizes, extra=0):
    o = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    return torch.from_numpy(o).cuda(), int(o[-1]) + extra


def _rounded(t, precision):
    return t.bfloat16().double() if precision == "bf16" else t.double()


def _factor(k, precision):
    return (k + 8) * 2 * U + (2.0 ** -15 + 4 * k * U if precision == "bf16x3" else 0)


SIZES = [([1], 8, 8), ([3, 0, 2], 5, 7), ([64], 64, 64), ([0, 0, 1], 33, 65), ([17, 40, 0, 130], 96, 100),
         ([300, 1, 2, 0, 0, 77], 130, 257), ([256, 512, 0, 256], 256, 256), ([1, 1, 1, 1, 1, 1, 1, 1], 768, 128),
         ([700, 90, 13], 1000, 33), ([5] * 70, 40, 36), ([2000, 3, 500], 64, 520), ([129] * 3, 1, 1),
         ([40, 2], 2, 300), ([60, 0, 61], 3, 1),
         # many rows: whole tiles of 256 apart from the rest, with and without bounds
         ([1500, 700, 0, 900], 64, 256), ([1025, 511], 40, 300), ([2048], 32, 512), ([512, 1024], 96, 256),
         # a few rows, streamed weights: sizes around the vectors' and steps'
         ([4, 4], 128, 64), ([5, 3, 9], 131, 68), ([1], 4, 4), ([2, 7], 130, 66), ([30, 2], 515, 6),
         ([4] * 5, 512, 260), ([3] * 9, 1030, 36), ([9, 2, 4], 769, 33), ([6] * 40, 256, 300), ([2] * 20, 385, 700),
         ([128] * 3, 96, 85), ([36], 419, 85), ([64, 65, 0, 90], 100, 100), ([120], 515, 130),
         # more experts than a wave's lanes, tiles of several rows each
         ([45] * 70, 96, 130), ([0] * 40 + [200] * 30, 32, 40)]


@pytest.mark.parametrize("sizes,kk,nn", SIZES)
@pytest.mark.parametrize("precision", ["fp32", "bf16", "bf16x3"])
@pytest.mark.parametrize("pad", [0, 3])
def test_products(dev, sizes, kk, nn, precision, pad):
    """Y, its input gradient and the weights' gradients; rows behind the last expert's,
    and strided operands"""
    E = len(sizes)
    offsets, n = _offsets(sizes, extra=5)
    kept = n - 5
    g = _gen(n + kk)

    def strided(*shape):
        full = torch.randn(*shape[:-1], shape[-1] + pad, generator=g).cuda()
        return full[..., :shape[-1]]

    x, w, dy = strided(n, kk), strided(E, kk, nn), strided(n, nn)
    y, dx, dw = (strided(*s) for s in ((n, nn), (n, kk), (E, kk, nn)))
    guards = []
    for t in (y, dx, dw):
        t.fill_(7)
        if pad:
            guards.append(torch.as_strided(t, t.shape[:-1] + (pad,), t.stride(), t.storage_offset() + t.shape[-1]))
            guards[-1].fill_(7)
    K.gemm_experts("N", x, w, offsets, y, precision=precision)
    K.gemm_experts("T", dy, w, offsets, dx, precision=precision)
    K.gemm_experts_dw(x, dy, offsets, dw, precision=precision)
    for t in guards:
        assert bool((t == 7).all())
    xr, wr, dr = (_rounded(t.cpu(), precision) for t in (x, w, dy))
    at = offsets.tolist()
    for e in range(E):
        r = slice(at[e], at[e + 1])
        for got, a, b in ((y[r], xr[r], wr[e]), (dx[r], dr[r], wr[e].t()), (dw[e], xr[r].t(), dr[r])):
            _close(got, a @ b, _factor(a.shape[1], precision) * (a.abs() @ b.abs()), e)
    assert not y[kept:].any() and not dx[kept:].any()
    base = [torch.randn(t.shape, generator=g).cuda() for t in (y, dx, dw)]
    acc = [t.clone() for t in base]
    K.gemm_experts("N", x, w, offsets, acc[0], precision=precision, accum=True)
    K.gemm_experts("T", dy, w, offsets, acc[1], precision=precision, accum=True)
    K.gemm_experts_dw(x, dy, offsets, acc[2], precision=precision, accum=True)
    for a, b, t in zip(acc, base, (y, dx, dw)):
        assert bool(((a - (b + t)).abs() <= 2 * U * (b.abs() + t.abs())).all())
    assert torch.equal(acc[0][kept:], base[0][kept:]) and torch.equal(acc[1][kept:], base[1][kept:])


def test_products_of_many_experts(dev):
    """more experts than a wave has lanes, most of them without rows"""
    g = _gen(5)
    for E in (64, 65, 200, 1024):
        sizes = (torch.rand(E, generator=g) < 0.2) * torch.randint(0, 90, (E,), generator=g)
        offsets, n = _offsets(sizes.numpy())
        x, w = torch.randn(n, 24, generator=g).cuda(), torch.randn(E, 24, 40, generator=g).cuda()
        y, dw = _empty(n, 40), _empty(E, 24, 40)
        K.gemm_experts("N", x, w, offsets, y)
        K.gemm_experts_dw(x, y, offsets, dw)
        e = torch.repeat_interleave(torch.arange(E), sizes.long())
        xd, wd = x.double().cpu(), w.double().cpu()
        want = (xd[:, :, None] * wd[e]).sum(1)
        _close(y, want, _factor(24, "fp32") * (xd[:, :, None] * wd[e]).abs().sum(1), E)
        yd = y.double().cpu()
        outer = xd[:, :, None] * yd[:, None]
        wantw = torch.zeros(E, 24, 40, dtype=torch.float64).index_add_(0, e, outer)
        boundw = torch.zeros(E, 24, 40, dtype=torch.float64).index_add_(0, e, outer.abs())
        _close(dw, wantw, _factor(90, "fp32") * boundw, E)


def test_products_keep_bad_values_to_their_rows(dev):
    """NaN and infinities of one row, or of one expert's weights, reach no other row
    and no other expert; the other rows of a block that holds one are computed again
    on the fp32 cores, so they keep their bound, not their bits"""
    offsets, n = _offsets([30, 34, 0, 70], extra=3)
    g = _gen(8)
    x, w, dy = (torch.randn(*s, generator=g).cuda() for s in ((n, 48), (4, 48, 80), (n, 80)))
    clean = [_empty(n, 80), _empty(n, 48), _empty(4, 48, 80)]

    def run(out):
        K.gemm_experts("N", x, w, offsets, out[0])
        K.gemm_experts("T", dy, w, offsets, out[1])
        K.gemm_experts_dw(x, dy, offsets, out[2])

    run(clean)
    x[10, 5], x[29, 47], dy[63, 0], w[2] = float("nan"), INF, float("nan"), INF
    x[n - 1] = float("nan")  # behind the last expert
    got = [_empty(n, 80), _empty(n, 48), _empty(4, 48, 80)]
    run(got)
    rows = torch.ones(n, dtype=torch.bool, device="cuda:0")
    rows[[10, 29]] = False
    near = 2 * _factor(80, "fp32") * 80 * 30  # (values below 6 in sums of at most 80)
    assert float((got[0][rows] - clean[0][rows]).abs().max()) <= near
    assert torch.equal(got[0][64:], clean[0][64:])
    assert bool(torch.isnan(got[0][10]).all()) and not bool(torch.isfinite(got[0][29]).any())
    rows = torch.ones(n, dtype=torch.bool, device="cuda:0")
    rows[63] = False
    assert float((got[1][rows] - clean[1][rows]).abs().max()) <= near
    assert torch.equal(got[1][64:], clean[1][64:]) and bool(torch.isnan(got[1][63]).all())
    assert torch.equal(got[2][2:], clean[2][2:])
    assert not got[0][-3:].any() and not got[1][-3:].any() and not got[2][2].any()


def test_shared_weights_and_no_rows(dev):
    g = _gen(9)
    offsets, n = _offsets([4, 9])
    x, w = torch.randn(n, 8, generator=g).cuda(), torch.randn(1, 8, 12, generator=g).cuda()
    y, plain = _empty(n, 12), _empty(n, 12)
    K.gemm_experts("N", x, w.expand(2, 8, 12), offsets, y)
    K.gemm_experts("N", x, w.repeat(2, 1, 1), offsets, plain)
    assert torch.equal(y, plain)
    none, zero = torch.empty(0, 8, device="cuda:0"), torch.zeros(3, dtype=torch.int32, device="cuda:0")
    dw = _empty(2, 8, 12)
    K.gemm_experts("N", none, w.repeat(2, 1, 1), zero, torch.empty(0, 12, device="cuda:0"))
    K.gemm_experts_dw(none, torch.empty(0, 12, device="cuda:0"), zero, dw)
    assert not dw.any()


def test_layer_captured_and_replayed_with_other_routings(dev):
    """router, plan, products and their gradients in one graph: group sizes are read
    on the device, so each replay takes that routing's"""
    R, E, k, d, f = 90, 6, 2, 32, 48
    g = _gen(2)
    n = R * k
    z, x = torch.randn(R, E, generator=g).cuda(), torch.randn(R, d, generator=g).cuda()
    w1, w2 = torch.randn(E, d, f, generator=g).cuda(), torch.randn(E, f, d, generator=g).cuda()
    experts, gates = _empty(R, k, dtype=torch.int32), _empty(R, k)
    offsets, order, place = (_empty(m, dtype=torch.int32) for m in (E + 1, n, n))
    xs, h, ys, out = _empty(n, d), _empty(n, f), _empty(n, d), _empty(R, d)
    dys, dgates, dh, dw2, dz = _empty(n, d), _empty(R, k), _empty(n, f), _empty(E, f, d), _empty(R, E)
    outs = [gates, xs, h, ys, out, dys, dgates, dh, dw2, dz]
    ws = torch.empty(max(1, K.expert_plan_workspace(n, E), K.gemm_experts_dw_workspace(n, f, d, E)),
                     dtype=torch.uint8, device="cuda:0")

    def step():
        K.route_topk(z, experts, gates)
        K.expert_plan(experts, offsets, order, place, ws=ws)
        K.expert_gather(x, k, offsets, order, xs)
        K.gemm_experts("N", xs, w1, offsets, h)
        K.gemm_experts("N", h, w2, offsets, ys)
        K.expert_combine(place, gates, ys, out, c=x)
        K.expert_combine_bwd(offsets, order, gates, ys, x, dys, dgates)
        K.gemm_experts("T", dys, w2, offsets, dh)
        K.gemm_experts_dw(h, dys, offsets, dw2, ws=ws)
        K.route_topk_bwd(experts, gates, dgates, dz)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    seen = set()
    for i in range(4):
        z.copy_(torch.randn(R, E, generator=g) + 3 * torch.randn(E, generator=g))
        if i == 2:
            z[:50] = -INF
        graph.replay()
        torch.cuda.synchronize()
        seen.add(tuple(offsets.tolist()))
        got = [t.clone() for t in outs]
        for t in outs:
            t.fill_(7)
        step()
        assert all(torch.equal(a, b) for a, b in zip(got, outs))
    assert len(seen) == 4


@pytest.mark.parametrize("bad", [[-7, 3, 2, 400], [0, 1 << 30, 1 << 30, 1 << 30], [90, 60, 30, 0],
                                 [-(1 << 31)] * 4])
@pytest.mark.parametrize("kk,nn", [(64, 256), (40, 20)])
def test_offsets_out_of_range_stay_in_bounds(dev, bad, kk, nn):
    """offsets are held to the rows there are and to increase: nothing outside the
    outputs is written, and rows that one expert has alone are right"""
    n, E = 100, 3
    g = _gen(3)
    offsets = torch.tensor(bad, dtype=torch.int32).cuda()
    x, w = torch.randn(n, kk, generator=g).cuda(), torch.randn(E, kk, nn, generator=g).cuda()
    y, dw = _empty(n + 2, nn), _empty(E + 2, kk, nn)
    K.gemm_experts("N", x, w, offsets, y[1:n + 1])
    dy = torch.randn(n, nn, generator=g).cuda()
    K.gemm_experts_dw(x, dy, offsets, dw[1:E + 1])
    assert bool((y[[0, n + 1]] == 7).all()) and bool((dw[[0, E + 1]] == 7).all())
    lo = [min(max(b, 0), n) for b in bad]
    hi = [max(lo[e + 1], lo[e]) for e in range(E)]
    own = torch.zeros(n, dtype=torch.int32)
    for e in range(E):
        own[lo[e]:hi[e]] += 1
        a, b = x[lo[e]:hi[e]].double().cpu(), dy[lo[e]:hi[e]].double().cpu()
        _close(dw[e + 1], a.t() @ b, _factor(len(a), "fp32") * (a.t().abs() @ b.abs()), e)
    for e in range(E):
        r = [i for i in range(lo[e], hi[e]) if own[i] == 1 and i < lo[E]]
        a, b = x[r].double().cpu(), w[e].double().cpu()
        _close(y[1:n + 1][r], a @ b, _factor(kk, "fp32") * (a.abs() @ b.abs()), e)


def test_dw_workspace_is_optional(dev):
    """few tiles and many rows: split with a workspace, unsplit without; both right"""
    offsets, n = _offsets([3000, 0, 5000])
    g = _gen(4)
    x, dy = torch.randn(n, 64, generator=g).cuda(), torch.randn(n, 48, generator=g).cuda()
    need = K.gemm_experts_dw_workspace(n, 64, 48, 3)
    assert need > 0
    out = []
    for size in (need, need - 1, 1):
        dw = _empty(3, 64, 48)
        K.gemm_experts_dw(x, dy, offsets, dw, ws=torch.empty(size, dtype=torch.uint8, device="cuda:0"))
        out.append(dw)
        for e, r in ((0, slice(0, 3000)), (1, slice(0, 0)), (2, slice(3000, 8000))):
            a, b = x[r].double().cpu(), dy[r].double().cpu()
            _close(dw[e], a.t() @ b, _factor(len(a), "fp32") * (a.t().abs() @ b.abs()), (size, e))
    assert torch.equal(out[1], out[2])


def test_rows_past_32_bit_offsets(dev):
    """1100 rows 2^21 values apart: element offsets beyond 2^31, byte offsets beyond 2^33"""
    n, E, ld, kk, nn = 1100, 3, 1 << 21, 36, 40
    g = _gen(8)
    far = torch.empty(n, ld, device="cuda:0")
    x, y, dys = far[:, :kk], far[:, 64:64 + nn], far[:, 128:128 + kk]
    x.copy_(torch.randn(n, kk, generator=g).cuda())
    experts = torch.randint(0, E, (n, 1), generator=g, dtype=torch.int32).cuda()
    offsets, order, place = (_empty(m, dtype=torch.int32) for m in (E + 1, n, n))
    K.expert_plan(experts, offsets, order, place)
    w = torch.randn(E, kk, nn, generator=g).cuda()
    gates, dout = torch.rand(n, 1, generator=g).cuda(), torch.randn(n, kk, generator=g).cuda()
    near = x.contiguous()
    for a, b in ((lambda t, o: K.expert_gather(t, 1, offsets, order, o), kk),
                 (lambda t, o: K.gemm_experts("N", t, w, offsets, o), nn),
                 (lambda t, o: K.expert_combine(place, gates, t, o), kk)):
        out = far[:, 192:192 + b]
        want = _empty(n, b)
        a(near, want)
        a(x, out)
        assert torch.equal(out, want)
    dw, want, dgates, dwant = _empty(E, kk, kk), _empty(E, kk, kk), _empty(n, 1), _empty(n, 1)
    K.expert_combine_bwd(offsets, order, gates, x, dout, dys, dgates)
    ndys = _empty(n, kk)
    K.expert_combine_bwd(offsets, order, gates, near, dout, ndys, dwant)
    assert torch.equal(dys, ndys) and torch.equal(dgates, dwant)
    K.gemm_experts_dw(x, dys, offsets, dw)
    K.gemm_experts_dw(near, ndys, offsets, want)
    assert torch.equal(dw, want)
    logits, dlogits = far[:, 256:256 + E], far[:, 320:320 + E]
    logits.copy_(torch.randn(n, E, generator=g).cuda())
    out = [(_empty(n, 2, dtype=torch.int32), _empty(n, 2)) for _ in range(2)]
    K.route_topk(logits, *out[0])
    K.route_topk(logits.contiguous(), *out[1])
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    dg, dz = torch.randn(n, 2, generator=g).cuda(), _empty(n, E)
    K.route_topk_bwd(*out[0], dg, dlogits)
    K.route_topk_bwd(*out[0], dg, dz)
    assert torch.equal(dlogits, dz)


def test_two_streams(dev):
    """the same layer on two streams at once, each with other tokens, as on one"""
    E, k, d, f = 6, 2, 96, 160
    g = _gen(9)
    w, w2 = torch.randn(E, d, f, generator=g).cuda(), torch.randn(E, f, d, generator=g).cuda()
    inputs = [(torch.randn(R, d, generator=g).cuda(), torch.randn(R, E, generator=g).cuda()) for R in (700, 3000)]

    def layer(x, z):
        R = len(x)
        experts, gates = _empty(R, k, dtype=torch.int32), _empty(R, k)
        offsets, order, place = (_empty(m, dtype=torch.int32) for m in (E + 1, R * k, R * k))
        K.route_topk(z, experts, gates)
        K.expert_plan(experts, offsets, order, place)
        xs, h, ys, y = _empty(R * k, d), _empty(R * k, f), _empty(R * k, d), _empty(R, d)
        K.expert_gather(x, k, offsets, order, xs)
        K.gemm_experts("N", xs, w, offsets, h)
        K.gemm_experts("N", h, w2, offsets, ys)
        K.expert_combine(place, gates, ys, y, c=x)
        dw = _empty(E, d, f)
        K.gemm_experts_dw(xs, h, offsets, dw)
        return y, dw

    want = [layer(*i) for i in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for st, i in zip(streams, inputs):
            with torch.cuda.stream(st):
                got.append(layer(*i))
    torch.cuda.synchronize()
    for i, pair in enumerate(got):
        for a, b in zip(pair, want[i % 2]):
            assert torch.equal(a, b)


def test_transpose_flag(dev):
    offsets, n = _offsets([4, 9])
    for tb in ("n", "t", "C", ""):
        with pytest.raises(ValueError):
            K.gemm_experts(tb, _empty(n, 8), _empty(2, 8, 8), offsets, _empty(n, 8))


def test_refusals(dev):
    offsets, n = _offsets([4, 9])
    x, w, y = _empty(n, 8), _empty(2, 8, 12), _empty(n, 12)
    for bad in (lambda: K.gemm_experts("N", x[:, :7], w, offsets, y),
                lambda: K.gemm_experts("N", x, w, offsets[:2], y),
                lambda: K.gemm_experts("N", x, w, offsets, y[:-1]),
                lambda: K.gemm_experts("N", x, w.transpose(1, 2), offsets, y),
                lambda: K.gemm_experts("T", x, w, offsets, y),
                lambda: K.gemm_experts_dw(x, y[:-1], offsets, w),
                lambda: K.expert_gather(x, 2, offsets, _empty(n, dtype=torch.int32), y),
                lambda: K.route_topk(x, _empty(n, 2, dtype=torch.int32), _empty(n, 3))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: K.gemm_experts("N", x, w, offsets.long(), y),
                lambda: K.gemm_experts("N", x.half(), w, offsets, y)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(_lib.PkError):  # gradients that would overlap
        K.gemm_experts_dw(x, y, offsets, w[:1].expand(2, 8, 12))
    with pytest.raises(_lib.PkError):
        K.route_topk(x, _empty(n, 9, dtype=torch.int32), _empty(n, 9))


# ------------------------------------------------------------------- pico's API
def _layer(x, z, w13, w2, k, f):
    """the layer in float64 with autograd: out"""
    experts, _ = _choose(z.detach(), k)
    experts = torch.from_numpy(experts).long()
    picked = torch.gather(z, 1, experts.clamp(min=0))
    gone = experts < 0
    gates = torch.where(gone, 0.0, torch.softmax(torch.where(gone, -1e300, picked), 1))
    y = x
    for e in range(w13.shape[0]):
        t, j = torch.nonzero(experts == e, as_tuple=True)
        gate, up = (x[t] @ w13[e]).split(f, 1)
        y = y.index_add(0, t, ((torch.nn.functional.silu(gate) * up) @ w2[e]) * gates[t, j][:, None])
    return y


@pytest.mark.parametrize("R,E,k,d,f", [(40, 4, 2, 32, 48), (65, 8, 1, 36, 20), (30, 3, 3, 64, 64)])
def test_pico_layer(P, R, E, k, d, f):
    """a whole feed-forward of experts and its gradients, one expert without tokens,
    a padding token; then a second backward and a second layer on the same tokens"""
    g = _gen(R)
    x, z = torch.randn(R, d, generator=g), torch.randn(R, E, generator=g)
    w13, w2 = torch.randn(E, d, 2 * f, generator=g) * d ** -0.5, torch.randn(E, f, d, generator=g) * f ** -0.5
    if E > k:
        z[:, 1] = -INF
    z[3] = -INF
    dy = torch.randn(R, d, generator=g)
    leaves = [t.double().requires_grad_() for t in (x, z, w13, w2)]
    y = _layer(*leaves, k, f)
    (y * dy.double()).sum().backward()
    ps = [P.param(list(t.shape), t.numpy()) for t in (x, z, w13, w2)]
    xp, zp, ap, bp = ps
    with P.arena():
        gates, route = P.route_topk(zp, k)
        experts, offsets = P.route_to_host(route, R, k, E)
        assert np.array_equal(experts, _choose(z, k)[0])
        assert offsets[E] == (experts >= 0).sum()
        gu = P.expert_matmul(P.expert_gather(xp, route), ap, route)
        ys = P.expert_matmul(P.swiglu(*P.split_cols(gu, 2)), bp, route)
        out = P.expert_combine(ys, gates, route, xp)
        P.backward(P.mul(out, P.tensor([R, d], dy.numpy())))
        # every value passes at most five products and sums of at most d + 2f + R terms
        # whose absolute values are within 40 times the largest result's
        bound = 40 * (d + 2 * f + R + 50) * 2 * U
        _close(torch.from_numpy(P.value(out)), y.detach(), bound * y.detach().abs().max(), "y")
        for t, leaf, name in zip(ps, leaves, ("dx", "dlogits", "dw13", "dw2")):
            want = torch.nan_to_num(leaf.grad)
            _close(torch.from_numpy(P.grad_value(t)), want, bound * want.abs().max(), name)
        for bad in ((xp, None), (P.tensor([R + 1, d], np.zeros((R + 1, d))), route), (None, route)):
            with pytest.raises(PicoError):
                P.expert_gather(*bad)
        for bad in ((xp, ap, route) if k > 1 else (ys, xp, route), (ys, bp, route) if f != d else (ys, xp, route),
                    (ys, None, route)):
            with pytest.raises(PicoError):
                P.expert_matmul(*bad)
        for bad in ((ys, xp, route, None), (xp, gates, route, None) if k > 1 else (gates, gates, route, None),
                    (ys, gates, route, ys) if k > 1 else (ys, gates, None, None)):
            with pytest.raises(PicoError):
                P.expert_combine(*bad)
        for bad in (0, E + 1):
            with pytest.raises(PicoError):
                P.route_topk(zp, bad)
    for t in ps:
        P.free(t)


@pytest.mark.parametrize("precision", [0, 1, 2, 3])
def test_pico_product_precisions(P, precision):
    """the product and its gradients in the precision set when it ran (fp8: bf16)"""
    R, E, kk, nn = 50, 3, 40, 72
    g = _gen(6)
    z, x = torch.randn(R, E, generator=g), torch.randn(R, kk, generator=g)
    w, dy = torch.randn(E, kk, nn, generator=g), torch.randn(R, nn, generator=g)
    name = {0: "fp32", 1: "bf16", 2: "bf16x3", 3: "bf16"}[precision]
    zp, xp, wp = (P.param(list(t.shape), t.numpy()) for t in (z, x, w))
    with P.arena():
        _, route = P.route_topk(zp, 1)
        experts, offsets = P.route_to_host(route, R, 1, E)
        P.lib.pico_set_matmul_precision(precision)
        y = P.expert_matmul(xp, wp, route)
        P.lib.pico_set_matmul_precision(0)
        P.backward(P.mul(y, P.tensor([R, nn], dy.numpy())))
        xr, wr, dr = (_rounded(t, name) for t in (x, w, dy))
        gy, gx, gw = (torch.from_numpy(a) for a in (P.value(y), P.grad_value(xp), P.grad_value(wp)))
        for e in range(E):
            r = slice(offsets[e], offsets[e + 1])
            for got, a, b in ((gy[r], xr[r], wr[e]), (gx[r], dr[r], wr[e].t()), (gw[e], xr[r].t(), dr[r])):
                _close(got, a @ b, _factor(a.shape[1], name) * (a.abs() @ b.abs()), e)
    for t in (zp, xp, wp):
        P.free(t)


def test_pico_shared_weights_padding_and_two_backwards(P):
    """two layers over one route with the same weights and gates, a padded batch, and the
    gradients of two backward passes added up"""
    R, E, k, d = 37, 4, 2, 48
    g = _gen(12)
    x, z = torch.randn(R, d, generator=g), torch.randn(R, E, generator=g)
    w = torch.randn(E, d, d, generator=g) * d ** -0.5
    z[30:] = -INF
    dy = torch.randn(R, d, generator=g)
    vx, vz, vw = leaves = [t.double().requires_grad_() for t in (x, z, w)]
    experts = torch.from_numpy(_choose(z, k)[0]).long()
    gone = experts < 0
    picked = torch.gather(torch.where(vz == -INF, 0.0, vz), 1, experts.clamp(min=0))
    gates = torch.where(gone, 0.0, torch.softmax(picked, 1))

    def layer(h):
        y = h
        for e in range(E):
            t, j = torch.nonzero(experts == e, as_tuple=True)
            y = y.index_add(0, t, (h[t] @ vw[e]) * gates[t, j][:, None])
        return y

    y = layer(layer(vx))
    (2 * y * dy.double()).sum().backward()
    xp, zp, wp = ps = [P.param(list(t.shape), t.numpy()) for t in (x, z, w)]
    for _ in range(2):
        with P.arena():
            gp, route = P.route_topk(zp, k)
            h = xp
            for _ in range(2):
                h = P.expert_combine(P.expert_matmul(P.expert_gather(h, route), wp, route), gp, route, h)
            P.backward(P.mul(h, P.tensor([R, d], dy.numpy())))
            got = P.value(h)
    assert np.array_equal(got[30:], x[30:].numpy())  # no expert: the residual alone
    # every value passes at most four products, of at most d + R terms, whose absolute
    # values are within 40 times the largest result's
    bound = 40 * (2 * d + 2 * R + 50) * 2 * U
    _close(torch.from_numpy(got), y.detach(), bound * y.detach().abs().max(), "y")
    for t, leaf, name in zip(ps, leaves, ("dx", "dlogits", "dw")):
        _close(torch.from_numpy(P.grad_value(t)), leaf.grad, bound * leaf.grad.abs().max(), name)
    assert not P.grad_value(zp)[30:].any()
    for t in ps:
        P.free(t)


def test_pico_weight_gradient_workspace(P):
    """the workspace of split weight gradients is taken by the backward, not by the forward;
    where it cannot be had, or under capture, the rows are not split and nothing fails"""
    R, E, kk, nn = 4096, 4, 96, 128
    g = _gen(13)
    z, x = torch.randn(R, E, generator=g), torch.randn(R, kk, generator=g)
    w = torch.randn(E, kk, nn, generator=g)
    need = K.gemm_experts_dw_workspace(R, kk, nn, E)
    assert need > 2 << 20
    zp, xp, wp = (P.param(list(t.shape), t.numpy()) for t in (z, x, w))
    xr = x.double()

    def check():
        got = torch.from_numpy(P.grad_value(wp))
        for e in range(E):
            a = xr[offsets[e]:offsets[e + 1]]
            want, mag = a.sum(0)[:, None].expand(kk, nn), a.abs().sum(0)[:, None].expand(kk, nn)
            _close(got[e], want, _factor(len(a), "fp32") * mag, e)

    opt = P.lib.pico_optim_sgd_init(0.0)
    P.lib.pico_optim_sgd_add(opt, wp)
    with P.arena(1 << 20) as arena:
        _, route = P.route_topk(zp, 1)
        _, offsets = P.route_to_host(route, R, 1, E)
        before = P.memory()[0]
        y = P.expert_matmul(xp, wp, route)
        # its values and gradients, each in a block of its own
        assert P.memory()[0] - before <= 2 * 4 * R * nn + 4096
        before = P.memory()[0]
        P.lib.pico_gpu_fail_next_workspaces(1)
        P.backward(y)
        P.lib.pico_gpu_fail_next_workspaces(0)
        assert P.memory()[0] == before and not P.lib.pico_gpu_last_error()
        check()
        P.lib.pico_optim_sgd_zero_grad(opt)
        y = P.expert_matmul(xp, wp, route)
        before = P.memory()[0]
        P.backward(y)
        assert P.memory()[0] - before >= need
        check()
        # captured with no room for it: the forward's blocks are there, the workspace is not
        with P.arena(1 << 20) as other:
            P.expert_matmul(xp, wp, route)
            P.reset(other)
            P.lib.pico_optim_sgd_zero_grad(opt)
            P.sync()
            before = P.memory()[0]
            assert P.lib.pico_graph_begin() == 0
            P.lib.pico_optim_sgd_zero_grad(opt)
            y = P.expert_matmul(xp, wp, route)
            P.lib.pico_backward(other, y)
            graph = P.lib.pico_graph_end()
            assert graph, P.lib.pico_gpu_last_error()
            assert P.memory()[0] == before
            for _ in range(3):
                assert P.lib.pico_graph_launch(graph) == 0
                check()
            P.lib.pico_graph_free(graph)
    P.lib.pico_optim_sgd_free(opt)
    for t in (zp, xp, wp):
        P.free(t)


@pytest.mark.parametrize("sizes,nn", [([4] * 8, 768), ([0, 1, 2, 3, 4, 6, 7, 9], 768), ([8] * 3, 1280), ([5] * 8, 704),
                                      ([1] * 13, 768), ([6] * 8, 770)])
@pytest.mark.parametrize("precision", ["fp32", "bf16"])
def test_few_rows_of_long_sums(dev, sizes, nn, precision):
    """a few rows an expert, on both sides of where the columns of a workgroup change"""
    kk = 2048
    offsets, n = _offsets(sizes, extra=2)
    g = _gen(nn + len(sizes))
    x, w = torch.randn(n, kk, generator=g).cuda(), torch.randn(len(sizes), kk, nn, generator=g).cuda()
    y = _empty(n, nn)
    K.gemm_experts("N", x, w, offsets, y, precision=precision)
    at = offsets.tolist()
    xr, wr = _rounded(x.cpu(), precision), _rounded(w.cpu(), precision)
    for e in range(len(sizes)):
        r = slice(at[e], at[e + 1])
        _close(y[r], xr[r] @ wr[e], _factor(kk, precision) * (xr[r].abs() @ wr[e].abs()), e)
    assert not y[at[-1]:].any()
