"""Layer norm (pk_layernorm_*, pico_layernorm) against float64.

Bounds, with u = 2^-24 and D = C/64 + 8 (no sum over a row adds more terms than
that one after another): the mean is off by D u max|x|, so x - mean by
e = (D + 2) u max|x|; rstd by the relative e rstd + (D + 7)/2 u; xh = (x - mean) rstd by
Ex = e rstd (1 + |xh|) + |xh| (D + 10) u.  From these follow the bounds of y, dx and
the column sums (R terms each); a factor of 2 covers their products.
"""
import numpy as np
import pytest
import torch

from pico_amd import _lib
from pico_amd import kernels as K
from pico_amd.pico import Pico, PicoError

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5


@pytest.fixture(scope="module")
def P():
    return Pico()


def _data(R, C, seed, shift=0.5, dev="cuda:0"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, C, generator=g) * 2 + shift * torch.randn(R, 1, generator=g)
    t = [x, 1 + 0.1 * torch.randn(C, generator=g), torch.randn(C, generator=g),
         torch.randn(R, C, generator=g)]
    return [a.to(dev) for a in t]


def _reference(x, g, b, dy, eps=EPS):
    x, g, dy = x.double(), g.double(), dy.double()
    R, C = x.shape
    m = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - m) * r
    y = xh * g + (0 if b is None else b.double())
    gd = g * dy
    s1, s2 = gd.mean(1, keepdim=True), (gd * xh).mean(1, keepdim=True)
    dx = r * (gd - s1 - xh * s2)
    dg, db = (dy * xh).sum(0), dy.sum(0)
    D = C / 64 + 8
    e = (D + 2) * U * x.abs().amax(1, keepdim=True)
    ex = e * r * (1 + xh.abs()) + xh.abs() * (D + 10) * U
    tol = {
        "y": 2 * g.abs() * ex + 3 * U * (y.abs() + (0 if b is None else b.double().abs())),
        "dx": 2 * (r * ((D + 2) * U * gd.abs().mean(1, keepdim=True) +
                        xh.abs() * ((D + 4) * U * (gd * xh).abs().mean(1, keepdim=True) +
                                    (gd.abs() * ex).mean(1, keepdim=True)) +
                        ex * s2.abs() + 5 * U * (gd.abs() + s1.abs() + (xh * s2).abs())) +
                   (e * r + (D + 7) * U) * dx.abs()),
        "dg": 2 * (R * U * (dy * xh).abs().sum(0) + (dy.abs() * ex).sum(0)) + 4 * U * dg.abs(),
        "db": 2 * R * U * dy.abs().sum(0),
    }
    return {"y": y, "dx": dx, "dg": dg, "db": db}, tol


def _close(got, want, tol, what):
    bad = (got.double() - want).abs() > tol + 1e-37
    assert not bad.any(), (what, int(bad.sum()),
                           float(((got.double() - want).abs() / (tol + 1e-37)).max()))


def _empty(*shape):
    return torch.full(shape, 7.0, device="cuda:0")


SHAPES = [(1, 1), (3, 1), (1, 2), (5, 3), (64, 63), (7, 64), (64, 128), (2, 255), (33, 256),
          (513, 257), (300, 768), (1030, 1000), (65, 1024), (129, 1503), (40, 2048), (31, 2052),
          (77, 4096), (19, 4097), (9, 8192), (5, 8200), (6, 16384), (3, 20001), (2, 65540)]


@pytest.mark.parametrize("R,C", SHAPES)
@pytest.mark.parametrize("bias", [True, False])
def test_forward_and_gradients(dev, R, C, bias):
    x, g, b, dy = _data(R, C, R * 7 + C)
    b = b if bias else None
    want, tol = _reference(x, g, b, dy)
    y, dx = _empty(R + 1, C), _empty(R + 1, C)
    mean, rstd, dg, db = _empty(R + 1), _empty(R + 1), _empty(C + 1), _empty(C + 1)
    K.layernorm_fwd(x, g, b, y[:R], mean[:R], rstd[:R], EPS)
    K.layernorm_bwd(x, g, mean[:R], rstd[:R], dy, dx[:R], dg[:C], db[:C])
    _close(y[:R], want["y"], tol["y"], "y")
    _close(dx[:R], want["dx"], tol["dx"], "dx")
    _close(dg[:C], want["dg"], tol["dg"], "dg")
    _close(db[:C], want["db"], tol["db"], "db")
    for t in (y[R], dx[R], mean[R], rstd[R], dg[C], db[C]):
        assert bool((t == 7.0).all())  # nothing behind the outputs is written



# one launch for all the gradients up to 16384 values, and just past that
FEW = [(1, 4), (1, 16384), (4096, 4), (4097, 4), (3276, 5), (2000, 5), (1024, 16), (256, 64), (257, 64), (31, 512),
       (31, 528), (33, 496), (15, 1024), (17, 1024), (2, 8192), (3, 5003), (29, 131)]


@pytest.mark.parametrize("R,C", FEW)
def test_gradients_of_few_values(dev, R, C):
    """all three at once, each by itself, and added to what is there: the same bits"""
    x, g, b, dy = _data(R, C, R * 3 + C)
    want, tol = _reference(x, g, b, dy)
    y, mean, rstd = _empty(R, C), _empty(R), _empty(R)
    K.layernorm_fwd(x, g, b, y, mean, rstd, EPS)
    dx, dg, db = _empty(R + 1, C), _empty(C + 1), _empty(C + 1)
    K.layernorm_bwd(x, g, mean, rstd, dy, dx[:R], dg[:C], db[:C])
    for t, k in ((dx[:R], "dx"), (dg[:C], "dg"), (db[:C], "db")):
        _close(t, want[k], tol[k], k)
    for t in (dx[R], dg[C], db[C]):
        assert bool((t == 7.0).all())
    for n in range(3):
        one = [torch.full_like(t, 5.0) if i == n else None for i, t in enumerate((dx[:R], dg[:C], db[:C]))]
        K.layernorm_bwd(x, g, mean, rstd, dy, *one)
        assert torch.equal(one[n], (dx[:R], dg[:C], db[:C])[n])
    base = [torch.randn_like(t) for t in (dg[:C], db[:C])]
    acc, inplace = [t.clone() for t in base], torch.randn_like(dx[:R])
    given = inplace.clone()
    K.layernorm_bwd(x, g, mean, rstd, dy, inplace, *acc, dx_in=inplace, accum_dg=True, accum_db=True)
    assert torch.equal(acc[0], base[0] + dg[:C]) and torch.equal(acc[1], base[1] + db[:C])
    # one more rounding, of the sum
    assert bool(((inplace - (given + dx[:R])).abs() <= 3 * U * (given.abs() + dx[:R].abs())).all())


def test_many_short_rows_take_no_longer_than_a_square(dev):
    """16384 values as 4096 rows of 4 and as 64 of 256, the backward in a graph: by rows one
    after another the first would take 40 times the second"""
    times = []
    for R, C in ((4096, 4), (64, 256)):
        x, g, b, dy = _data(R, C, 1)
        y, mean, rstd, dx, dg, db = _empty(R, C), _empty(R), _empty(R), _empty(R, C), _empty(C), _empty(C)
        ws = torch.empty(K.layernorm_bwd_workspace(R, C), dtype=torch.uint8, device="cuda:0")
        K.layernorm_fwd(x, g, b, y, mean, rstd, EPS)
        K.layernorm_bwd(x, g, mean, rstd, dy, dx, dg, db, ws=ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(20):
                K.layernorm_bwd(x, g, mean, rstd, dy, dx, dg, db, ws=ws)
        best = 1e9
        for _ in range(5):
            a, z = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            graph.replay()
            z.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(z))
        times.append(best)
    assert times[0] < 8 * times[1], times


@pytest.mark.parametrize("R,C", [(64, 128), (50, 1503), (300, 768), (9, 4096), (3, 20001)])
def test_accumulation_and_single_gradients(dev, R, C):
    x, g, b, dy = _data(R, C, 5)
    mean, rstd, y = _empty(R), _empty(R), _empty(R, C)
    K.layernorm_fwd(x, g, b, y, mean, rstd, EPS)
    dx, dg, db = _empty(R, C), _empty(C), _empty(C)
    K.layernorm_bwd(x, g, mean, rstd, dy, dx, dg, db)
    base = torch.randn(R, C, device="cuda:0")
    other = _empty(R, C)
    K.layernorm_bwd(x, g, mean, rstd, dy, other, None, None, dx_in=base)
    # one more rounding, of the sum
    assert bool(((other - (base + dx)).abs() <= 3 * U * (base.abs() + dx.abs())).all())
    inplace = base.clone()
    K.layernorm_bwd(x, g, mean, rstd, dy, inplace, None, None, dx_in=inplace)
    assert torch.equal(inplace, other)
    g2, b2 = torch.randn(C, device="cuda:0"), torch.randn(C, device="cuda:0")
    ag, ab = g2.clone(), b2.clone()
    K.layernorm_bwd(x, g, mean, rstd, dy, None, ag, ab, accum_dg=True, accum_db=True)
    assert torch.equal(ag, g2 + dg) and torch.equal(ab, b2 + db)
    only = _empty(C)
    K.layernorm_bwd(x, g, mean, rstd, dy, None, None, only)
    assert torch.equal(only, db)
    K.layernorm_bwd(x, g, mean, rstd, dy, None, only, None)
    assert torch.equal(only, dg)
    # deterministic, on another stream too
    again = [_empty(R, C), _empty(C), _empty(C)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        K.layernorm_bwd(x, g, mean, rstd, dy, *again)
    s.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(again, (dx, dg, db)))


def test_no_rows(dev):
    x = torch.empty(0, 40, device="cuda:0")
    g = torch.ones(40, device="cuda:0")
    none = torch.empty(0, device="cuda:0")
    dg, db = _empty(40), _empty(40)
    K.layernorm_fwd(x, g, g, x, none, none, EPS)
    K.layernorm_bwd(x, g, none, none, x, x, dg, db)
    assert not dg.any() and not db.any()
    dg, db = _empty(40), _empty(40)
    K.layernorm_bwd(x, g, none, none, x, x, dg, db, accum_dg=True, accum_db=True)
    assert bool((dg == 7).all()) and bool((db == 7).all())


@pytest.mark.parametrize("C", [64, 333, 1024, 4096])
def test_far_mean_constant_rows_and_bad_values(dev, C):
    """a mean far from zero keeps the difference (the variance is not taken from
    squares); a constant row gives the bias; a NaN or infinite row stays alone"""
    x, g, b, dy = _data(6, C, 9)
    x[0] += 1e4
    x[1] = 3.25
    want, tol = _reference(x, g, b, dy)
    x[3, C // 2] = float("nan")
    x[4, 0] = float("inf")
    y, mean, rstd, dx = _empty(6, C), _empty(6), _empty(6), _empty(6, C)
    K.layernorm_fwd(x, g, b, y, mean, rstd, EPS)
    K.layernorm_bwd(x, g, mean, rstd, dy, dx, None, None)
    for r in (0, 1, 2, 5):
        _close(y[r], want["y"][r], tol["y"][r], f"y {r}")
        _close(dx[r], want["dx"][r], tol["dx"][r], f"dx {r}")
    assert torch.equal(y[1], b)
    for r in (3, 4):
        assert bool(torch.isnan(y[r]).all()) and bool(torch.isnan(dx[r]).all())


def test_gradients_against_differences(dev):
    R, C = 4, 37
    x, g, b, dy = _data(R, C, 3)

    def loss(x, g, b):
        m = x.mean(1, keepdim=True)
        r = 1 / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + EPS)
        return (((x - m) * r * g + b) * dy.double()).sum()

    y, mean, rstd, dx, dg, db = (_empty(R, C), _empty(R), _empty(R), _empty(R, C), _empty(C),
                                 _empty(C))
    K.layernorm_fwd(x, g, b, y, mean, rstd, EPS)
    K.layernorm_bwd(x, g, mean, rstd, dy, dx, dg, db)
    args = [t.double() for t in (x, g, b)]
    for k, got in enumerate((dx, dg, db)):
        for i in range(0, args[k].numel(), 7):
            step = []
            for h in (1e-5, -1e-5):
                moved = [t.clone() for t in args]
                moved[k].view(-1)[i] += h
                step.append(loss(*moved))
            diff = float((step[0] - step[1]) / 2e-5)
            # differences: h^2 times the third derivative, below 1e-7 here
            assert abs(float(got.view(-1)[i]) - diff) <= 2e-5 * (1 + abs(diff))


def test_captured_and_replayed(dev):
    R, C = 70, 900
    x, g, b, dy = _data(R, C, 1)
    out = [_empty(R, C), _empty(R), _empty(R), _empty(R, C), _empty(C), _empty(C)]
    ws = torch.empty(K.layernorm_bwd_workspace(R, C), dtype=torch.uint8, device="cuda:0")

    def step():
        K.layernorm_fwd(x, g, b, out[0], out[1], out[2], EPS)
        K.layernorm_bwd(x, g, out[1], out[2], dy, out[3], out[4], out[5], ws=ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        x.copy_(_data(R, C, 20 + i)[0])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for t in out:
            t.fill_(7.0)
        step()
        assert all(torch.equal(a, c) for a, c in zip(got, out))


def test_values_past_32_bit_offsets(dev):
    """more than 2^31 values: the last rows as by themselves"""
    R, C = 1100000, 2048
    x = torch.empty(R, C, device="cuda:0")
    last = torch.randn(64, C, generator=torch.Generator().manual_seed(1)).cuda()
    x.fill_(1)
    x[-64:] = last
    g, b = torch.randn(C, device="cuda:0"), torch.randn(C, device="cuda:0")
    y, mean, rstd = torch.empty_like(x), torch.empty(R, device="cuda:0"), torch.empty(R, device="cuda:0")
    K.layernorm_fwd(x, g, b, y, mean, rstd, 1e-5)
    want, m, r = torch.empty_like(last), torch.empty(64, device="cuda:0"), torch.empty(64, device="cuda:0")
    K.layernorm_fwd(last, g, b, want, m, r, 1e-5)
    assert torch.equal(y[-64:], want) and torch.equal(mean[-64:], m) and torch.equal(rstd[-64:], r)
    assert torch.equal(y[:-64].amax(0), b) and torch.equal(y[:-64].amin(0), b)
    # the same rows' gradients; those of the others are zero
    dy = y.zero_()
    dy[-64:] = want
    dg, db, dg1, db1 = (torch.empty(C, device="cuda:0") for _ in range(4))
    dx, dx1 = torch.full_like(x, 7), torch.empty_like(last)
    K.layernorm_bwd(x, g, mean, rstd, dy, dx, dg, db)
    K.layernorm_bwd(last, g, m, r, want, dx1, dg1, db1)
    assert torch.equal(dx[-64:], dx1) and not dx[:-64].any()
    # (64 values a column, added in two orders)
    for a, c, each in ((dg, dg1, want * (last - m[:, None]) * r[:, None]), (db, db1, want)):
        assert bool(((a - c).abs() <= 2 * 66 * 2.0 ** -24 * each.abs().sum(0)).all())


def test_refusals(dev):
    x, g, b, dy = _data(4, 8, 2)
    m = _empty(4)
    with pytest.raises(ValueError):
        K.layernorm_fwd(x, g[:7], b, x, m, m, EPS)
    with pytest.raises(ValueError):
        K.layernorm_fwd(x.t(), g, b, x, m, m, EPS)
    with pytest.raises(TypeError):
        K.layernorm_fwd(x.half(), g, b, x, m, m, EPS)
    with pytest.raises(_lib.PkError):
        K.layernorm_bwd(x, g, m, m, dy, _empty(4, 8), _empty(8), None,
                        ws=torch.empty(4, device="cuda:0"))


# ------------------------------------------------------------------- pico's API
@pytest.mark.parametrize("bias", [True, False])
def test_pico_op(P, bias):
    R, C = 50, 96
    x, g, b, dy = (t.cpu().numpy() for t in _data(R, C, 4))
    want, tol = _reference(*(torch.from_numpy(a) for a in (x, g)),
                           torch.from_numpy(b) if bias else None, torch.from_numpy(dy))
    xp, gp, bp = P.param([R, C], x), P.param([C], g), P.param([C], b)
    with P.arena() as a:
        y = P.layernorm(xp, gp, bp if bias else None, EPS)
        z = P.mul(y, P.tensor([R, C], dy))
        P.backward(z)
        _close(torch.from_numpy(P.value(y)), want["y"], tol["y"], "y")
        for t, k in ((xp, "dx"), (gp, "dg"), (bp, "db")):
            if t is bp and not bias:
                assert not P.grad(t).any()
                continue
            _close(torch.from_numpy(P.grad_value(t)), want[k], tol[k], k)
        # a second backward adds the same again
        one = [P.grad(t) for t in (xp, gp)]
        P.backward(z)
        # (z's and y's own gradients doubled meanwhile: pico accumulates there too)
        assert np.abs(P.grad(gp)).sum() > np.abs(one[1]).sum()
        for bad in ((xp, xp, None), (xp, gp, gp), (xp, xp, bp), (None, gp, bp)):
            with pytest.raises(PicoError):
                P.layernorm(*bad, EPS)
        view = P.split_cols(P.matmul(P.tensor([4, 3], np.ones((4, 3))), P.tensor([3, 2 * C])), 2)[0]
        with pytest.raises(PicoError):
            P.layernorm(view, gp, None, EPS)
    for t in (xp, gp, bp):
        P.free(t)
