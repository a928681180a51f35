"""The gated linear recurrence (pk_gated_scan_*, pico_gated_scan) against float64.

Bounds, with u = 2^-24: s and 1 - s are off by 10 u of themselves, so a step of the
recurrence, in whatever order its products are taken, by 20 u of the absolute values
that go in.  With H_t = s H_{t-1} + q |x_t| and the same of the gradients, the errors
follow E_t = s E_{t-1} + 20 u (H_t + s H_{t-1}).
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


def _data(B, T, C, seed, keep=2.0, dev="cuda:0"):
    g = torch.Generator().manual_seed(seed)
    f = torch.randn(B * T, C, generator=g) + keep
    t = [f, torch.randn(B * T, C, generator=g), torch.randn(B, C, generator=g),
         torch.randn(B * T, C, generator=g)]
    return [a.to(dev) for a in t]


def _reference(B, f, x, h0, dh):
    N, C = x.shape
    T = N // B
    f, x, dh = (t.double().reshape(B, T, C) for t in (f, x, dh))
    s, q = torch.sigmoid(f), torch.sigmoid(-f)
    start = torch.zeros(B, C, dtype=torch.float64, device=x.device) if h0 is None else h0.double()
    h, eh = torch.empty_like(x), torch.empty_like(x)
    p, ab, e = start, start.abs(), torch.zeros_like(start)
    for t in range(T):
        e = s[:, t] * e + 20 * U * s[:, t] * ab
        ab = s[:, t] * ab + q[:, t] * x[:, t].abs()
        e = e + 20 * U * ab
        p = s[:, t] * p + q[:, t] * x[:, t]
        h[:, t], eh[:, t] = p, e
    G, eG, aG = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    u, eu, au = (torch.zeros_like(start) for _ in range(3))
    for t in range(T - 1, -1, -1):
        G[:, t], aG[:, t] = dh[:, t] + u, dh[:, t].abs() + au
        eG[:, t] = eu + 20 * U * aG[:, t]
        u, au, eu = s[:, t] * G[:, t], s[:, t] * aG[:, t], s[:, t] * (eG[:, t] + 20 * U * aG[:, t])
    hp = torch.cat([start[:, None], h[:, :-1]], 1)
    ehp = torch.cat([torch.zeros_like(start)[:, None], eh[:, :-1]], 1)
    want = {"h": h, "dx": q * G, "df": G * (hp - x) * s * q, "dh0": u}
    tol = {"h": eh, "dx": q * (eG + 12 * U * aG),
           "df": s * q * (eG * (hp - x).abs() + aG * ehp + 30 * U * aG * (hp.abs() + x.abs())),
           "dh0": eu}
    rows = {k: (v if k == "dh0" else v.reshape(N, C)) for k, v in want.items()}
    return rows, {k: (v if k == "dh0" else v.reshape(N, C)) for k, v in tol.items()}


def _close(got, want, tol, what):
    ratio = (got.double() - want).abs() / (tol + 1e-37)
    assert bool((ratio <= 1).all()), (what, float(ratio.max()))


def _empty(*shape):
    return torch.full(shape, 7.0, device="cuda:0")


SHAPES = [(1, 1, 1), (2, 1, 3), (64, 1, 768), (3, 2, 5), (1, 3, 64), (2, 7, 63), (5, 8, 100),
          (2, 9, 65), (1, 33, 257), (3, 64, 128), (2, 65, 16), (1, 127, 4), (4, 128, 12), (2, 200, 333),
          (8, 256, 96), (1, 257, 1), (2, 300, 130), (1, 1000, 48), (3, 1001, 33), (1, 2049, 64),
          (1, 5000, 7), (1, 9000, 20), (70, 130, 20), (1, 16385, 4), (2, 4096, 36), (513, 20, 8),
          # many short sequences: token after token
          (1030, 16, 36), (1030, 17, 12), (4100, 40, 8), (4100, 41, 5)]


@pytest.mark.parametrize("B,T,C", SHAPES)
@pytest.mark.parametrize("state", [True, False])
def test_forward_and_gradients(dev, B, T, C, state):
    f, x, h0, dh = _data(B, T, C, B + T + C)
    h0 = h0 if state else None
    want, tol = _reference(B, f, x, h0, dh)
    N = B * T
    h, df, dx, dh0 = _empty(N + 1, C), _empty(N + 1, C), _empty(N + 1, C), _empty(B + 1, C)
    K.gated_scan_fwd(B, f, x, h[:N], h0=h0)
    _close(h[:N], want["h"], tol["h"], "h")
    K.gated_scan_bwd(B, f, x, h[:N], dh, df[:N], dx[:N], h0=h0, dh0=dh0[:B] if state else None)
    _close(df[:N], want["df"], tol["df"], "df")
    _close(dx[:N], want["dx"], tol["dx"], "dx")
    if state:
        _close(dh0[:B], want["dh0"], tol["dh0"], "dh0")
    for t in (h[N], df[N], dx[N], dh0[B]):
        assert bool((t == 7.0).all())  # nothing behind the outputs is written



@pytest.mark.parametrize("lo,hi", [(0.0, 1.0), (1.0, 20.0), (20.0, 87.3), (87.3, 110.0)])
def test_the_gates_themselves(dev, lo, hi):
    """s and 1 - s over the range of f, read off single tokens: a state of 1 with x = 0 and
    an empty one with x = 1.  The larger is within 3.5 u of itself (two roundings and half
    of the exponential's 3 u, which are an ulp of the hardware's and a rounding), the
    smaller within 6 u (those 3 u, which 1 + t takes part of back, and three roundings), or
    0 below 2^-126"""
    C = 1 << 20
    g = torch.Generator(device="cuda:0").manual_seed(5)
    f = torch.rand(1, C, device="cuda:0", generator=g) * (hi - lo) + lo
    f[:, ::2] *= -1
    one, zero, s, q = (torch.full((1, C), v, device="cuda:0") for v in (1.0, 0.0, 7.0, 7.0))
    K.gated_scan_fwd(1, f, zero, s, h0=one)
    K.gated_scan_fwd(1, f, one, q)
    for got, want, large in ((s, torch.sigmoid(f.double()), f >= 0), (q, torch.sigmoid(-f.double()), f < 0)):
        off = (got.double() - want).abs()
        assert bool((off[large] <= 3.5 * U * want[large]).all())
        assert bool((off[~large] <= 6 * U * want[~large] + 2.0 ** -126).all())
        assert bool((got[~large & (f.abs() >= 87.34)] == 0).all())


def _chain(a, b):
    """y_t = a_t y_{t-1} + b_t along dim 0 from zero, in log2(T) passes"""
    step = 1
    a, b = a.clone(), b.clone()
    while step < a.shape[0]:
        b[step:] = b[step:] + a[step:] * b[:-step]
        a[step:] = a[step:] * a[:-step]
        step *= 2
    return b


def test_larger_than_the_caches(dev):
    """one sequence of 25 million values a tensor, which takes the backward's own kernel"""
    T, C = 50000, 512
    g = torch.Generator(device="cuda:0").manual_seed(1)
    f = torch.randn(T, C, device="cuda:0", generator=g) + 2
    x, dh = (torch.randn(T, C, device="cuda:0", generator=g) for _ in range(2))
    h, df, dx = _empty(T, C), _empty(T, C), _empty(T, C)
    K.gated_scan_fwd(1, f, x, h)
    K.gated_scan_bwd(1, f, x, h, dh, df, dx)
    for c in range(0, C, 64):
        cut = slice(c, c + 64)
        fd, xd, gd = (t[:, cut].double() for t in (f, x, dh))
        s, q = torch.sigmoid(fd), torch.sigmoid(-fd)
        zero = torch.zeros_like(s[:1])
        want, ab = _chain(s, q * xd), _chain(s, q * xd.abs())
        eh = _chain(s, 20 * U * (ab + s * torch.cat([zero, ab[:-1]])))
        _close(h[:, cut], want, eh, "h")
        after = torch.cat([s[1:], zero]).flip(0)
        G, aG = _chain(after, gd.flip(0)).flip(0), _chain(after, gd.abs().flip(0)).flip(0)
        eG = _chain(after, 40 * U * aG.flip(0)).flip(0)
        _close(dx[:, cut], q * G, q * (eG + 12 * U * aG), "dx")
        hp, ehp = torch.cat([zero, want[:-1]]), torch.cat([zero, eh[:-1]])
        _close(df[:, cut], G * (hp - xd) * s * q,
               s * q * (eG * (hp - xd).abs() + aG * ehp + 30 * U * aG * (hp.abs() + xd.abs())), "df")


@pytest.mark.parametrize("B,T", [(1, 1100), (275, 4)])
def test_rows_past_32_bit_offsets(dev, B, T):
    """rows 2^21 values apart: element offsets beyond 2^31"""
    C = 20
    far = torch.empty(B * T, 1 << 21, device="cuda:0")
    f, x, h0, dh = _data(B, T, C, 3)
    ff, fx, fdf, fdx = (far[:, i:i + C] for i in (0, 64, 128, 192))
    ff.copy_(f)
    fx.copy_(x)
    h, want = _empty(B * T, C), _empty(B * T, C)
    K.gated_scan_fwd(B, ff, fx, h, h0=h0)
    K.gated_scan_fwd(B, f, x, want, h0=h0)
    assert torch.equal(h, want)
    df, dx, d0, d1 = _empty(B * T, C), _empty(B * T, C), _empty(B, C), _empty(B, C)
    K.gated_scan_bwd(B, ff, fx, h, dh, fdf, fdx, h0=h0, dh0=d0)
    K.gated_scan_bwd(B, f, x, h, dh, df, dx, h0=h0, dh0=d1)
    assert torch.equal(fdf, df) and torch.equal(fdx, dx) and torch.equal(d0, d1)


@pytest.mark.parametrize("B,T,C", [(2, 70, 24), (1, 3000, 17), (3, 1, 64), (4, 600, 64)])
def test_views_accumulation_and_single_gradients(dev, B, T, C):
    """f and x as column blocks of one projection, the gradients as columns of its
    gradient; each gradient alone and added to what is there; another stream"""
    N = B * T
    f, x, h0, dh = _data(B, T, C, 11)
    fx = torch.cat([f, x, dh], 1)
    h, df, dx, dh0 = _empty(N, C), _empty(N, C), _empty(N, C), _empty(B, C)
    K.gated_scan_fwd(B, f, x, h, h0=h0)
    K.gated_scan_bwd(B, f, x, h, dh, df, dx, h0=h0, dh0=dh0)
    h2, grad = _empty(N, C), _empty(N, 3 * C)
    K.gated_scan_fwd(B, fx[:, :C], fx[:, C:2 * C], h2, h0=h0)
    K.gated_scan_bwd(B, fx[:, :C], fx[:, C:2 * C], h2, dh, grad[:, :C], grad[:, C:2 * C], h0=h0)
    # (the order of the sums may differ with the alignment)
    want, tol = _reference(B, f, x, h0, dh)
    _close(h2, want["h"], tol["h"], "h")
    _close(grad[:, :C], want["df"], tol["df"], "df")
    _close(grad[:, C:2 * C], want["dx"], tol["dx"], "dx")
    assert bool((grad[:, 2 * C:] == 7).all())
    base = [torch.randn_like(t) for t in (df, dx, dh0)]
    acc = [t.clone() for t in base]
    K.gated_scan_bwd(B, f, x, h, dh, acc[0], None, h0=h0, accum_df=True)
    K.gated_scan_bwd(B, f, x, h, dh, None, acc[1], h0=h0, accum_dx=True)
    K.gated_scan_bwd(B, f, x, h, dh, None, None, h0=h0, dh0=acc[2], accum_dh0=True)
    for a, b, g in zip(acc, base, (df, dx, dh0)):
        assert bool(((a - (b + g)).abs() <= 3 * U * (b.abs() + g.abs())).all())
    again = [_empty(N, C), _empty(N, C), _empty(B, C)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        K.gated_scan_bwd(B, f, x, h, dh, again[0], again[1], h0=h0, dh0=again[2])
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, (df, dx, dh0)))


@pytest.mark.parametrize("B,T,C", [(3, 50, 40), (2, 777, 20)])
def test_token_by_token_is_the_whole_sequence(dev, B, T, C):
    f, x, h0, dh = _data(B, T, C, 2)
    want, tol = _reference(B, f, x, h0, dh)
    f3, x3 = f.view(B, T, C), x.view(B, T, C)
    state = h0.clone()
    for t in range(T):
        K.gated_scan_fwd(B, f3[:, t].contiguous(), x3[:, t].contiguous(), state, h0=state)
        _close(state, want["h"].view(B, T, C)[:, t], tol["h"].view(B, T, C)[:, t], t)
    # in two parts, the second from the first one's last token
    cut = T // 3
    a, b = _empty(B * cut, C), _empty(B * (T - cut), C)
    K.gated_scan_fwd(B, f3[:, :cut].reshape(-1, C), x3[:, :cut].reshape(-1, C), a, h0=h0)
    last = a.view(B, cut, C)[:, -1].contiguous()
    K.gated_scan_fwd(B, f3[:, cut:].reshape(-1, C), x3[:, cut:].reshape(-1, C), b, h0=last)
    got = torch.cat([a.view(B, cut, C), b.view(B, T - cut, C)], 1).view(-1, C)
    _close(got, want["h"], tol["h"], "parts")


@pytest.mark.parametrize("B,C", [(1, 1), (64, 768), (3, 41)])
def test_state_in_place(dev, B, C):
    """one token at a time, the new state over the old one"""
    f, x, state, _ = _data(B, 1, C, 4)
    want = _empty(B, C)
    K.gated_scan_fwd(B, f, x, want, h0=state)
    K.gated_scan_fwd(B, f, x, state, h0=state)
    assert torch.equal(state, want)


@pytest.mark.parametrize("T", [9, 500, 3000])
def test_closed_and_open_gates(dev, T):
    """f = -inf starts anew at a token, f = +inf and large f hold the state, the type's
    lowest value is a closed gate; what is bad in one channel or sequence stays there"""
    B, C = 2, 36
    f, x, h0, dh = _data(B, T, C, 6)
    f3 = f.view(B, T, C)
    f3[:, T // 2, :8] = -float("inf")
    f3[:, T // 2, 8:12] = torch.finfo(torch.float32).min
    f3[0, :, 12:16] = float("inf")
    f3[1, T // 3:, 12:16] = 40.0
    want, tol = _reference(B, f, x, h0, dh)
    x.view(B, T, C)[0, 1, 20] = float("nan")
    h, df, dx, dh0 = _empty(B * T, C), _empty(B * T, C), _empty(B * T, C), _empty(B, C)
    K.gated_scan_fwd(B, f, x, h, h0=h0)
    K.gated_scan_bwd(B, f, x, h, dh, df, dx, h0=h0, dh0=dh0)
    ok = torch.ones(B, T, C, dtype=torch.bool, device="cuda:0")
    ok[0, :, 20] = False
    ok = ok.view(-1, C)
    for got, k in ((h, "h"), (df, "df"), (dx, "dx")):
        ratio = (got.double() - want[k]).abs() / (tol[k] + 1e-37)
        assert bool((ratio[ok] <= 1).all()), k
    assert torch.equal(h.view(B, T, C)[:, T // 2, :8], x.view(B, T, C)[:, T // 2, :8])
    assert torch.equal(h.view(B, T, C)[0, -1, 12:16], h0[0, 12:16])
    assert bool(torch.isnan(h.view(B, T, C)[0, 1:, 20]).all())
    assert not bool(torch.isnan(h.view(B, T, C)[0, :1, 20]).any())



# serial, one tile, tiles, chunks of one tile and of several; V of 1 and of 4 channels
@pytest.mark.parametrize("B,T,C", [(3, 7, 20), (2, 100, 37), (2, 777, 20), (1, 1001, 33), (1, 9000, 20), (2, 3000, 3),
                                   (8, 600, 200), (1, 40000, 64)])
@pytest.mark.parametrize("closed", [-INF, -100.0])
def test_a_closed_gate_keeps_bad_values_out(dev, B, T, C, closed):
    """documents packed into one sequence, each starting with a closed gate: infinities and NaN
    of one's tokens, gates or gradients stay in it, forward, backward and added to what is
    there"""
    g = torch.Generator().manual_seed(T + C)
    f, x, h0, dh = (t.cpu() for t in _data(B, T, C, 21))
    cuts = sorted({0, T} | set(torch.randint(1, T, (min(9, T // 2),), generator=g).tolist()))
    f3, x3, dh3 = f.view(B, T, C), x.view(B, T, C), dh.view(B, T, C)
    f3[:, cuts[1:-1]] = closed
    docs = list(zip(cuts, cuts[1:]))
    want, tol = ({k: torch.zeros(B, T, C, dtype=torch.float64) for k in ("h", "df", "dx")} for _ in range(2))
    for n, (lo, hi) in enumerate(docs):
        rows, bound = _reference(B, f3[:, lo:hi].reshape(-1, C), x3[:, lo:hi].reshape(-1, C), h0 if n == 0 else None,
                                 dh3[:, lo:hi].reshape(-1, C))
        for k in want:
            want[k][:, lo:hi], tol[k][:, lo:hi] = (t[k].view(B, hi - lo, C) for t in (rows, bound))
    # every other document is spoilt in every third channel
    bad_h, bad_g = (torch.zeros(B, T, C, dtype=torch.bool) for _ in range(2))
    for n, (lo, hi) in enumerate(docs):
        if n % 2:
            continue
        at = int(torch.randint(lo, hi, (1,), generator=g))
        cols = torch.arange(n % 3, C, 3)
        kind = (n // 2) % 4
        if kind == 0:
            x3[:, at, cols] = float("nan")
        elif kind == 1:
            x3[:, at, cols] = INF if at % 2 else -INF
        if kind < 2:
            bad_h[:, at:hi, cols] = True
        elif kind == 2:
            dh3[:, at, cols] = float("nan")
            bad_g[:, lo:at + 1, cols] = True
        else:
            dh3[:, at, cols] = -INF
            bad_g[:, lo:at + 1, cols] = True
    fd, xd, hd, dhd = (t.to(dev) for t in (f, x, h0, dh))
    h, df, dx, dh0 = _empty(B * T, C), _empty(B * T, C), _empty(B * T, C), _empty(B, C)
    K.gated_scan_fwd(B, fd, xd, h, h0=hd)
    K.gated_scan_bwd(B, fd, xd, h, dhd, df, dx, h0=hd, dh0=dh0)
    base = [torch.randn(B * T, C, generator=g).to(dev) for _ in range(2)]
    acc = [t.clone() for t in base]
    K.gated_scan_bwd(B, fd, xd, h, dhd, acc[0], acc[1], h0=hd, accum_df=True, accum_dx=True)
    got = {"h": h, "df": df, "dx": dx}
    # df of a document takes its h; a token's dx and df with a closed gate are dh and 0
    spoilt = {"h": bad_h, "dx": bad_g, "df": bad_g | bad_h}
    for k, t in got.items():
        t = t.view(B, T, C).cpu()
        ok = ~spoilt[k]
        ratio = (t.double() - want[k]).abs() / (tol[k] + 1e-37)
        assert bool((ratio[ok] <= 1).all()), (k, float(ratio[ok].nan_to_num(INF).max()))
    assert not bool(torch.isfinite(h.view(B, T, C).cpu()[bad_h]).any())
    assert not bool(torch.isfinite(dx.view(B, T, C).cpu()[bad_g]).any())
    assert bool(torch.isfinite(dh0.cpu()[:, ~bad_g[0, 0]]).all())
    # (a tile done again may round a token's gradient otherwise than in the call above: the
    # bound is the gradient's own and u of the sum, which is at most |b| + |want| + tol)
    for a, b, k in zip(acc, base, ("df", "dx")):
        ok = ~spoilt[k].view(-1, C)
        a, b, w, e = a.double().cpu()[ok], b.double().cpu()[ok], want[k].view(-1, C)[ok], tol[k].view(-1, C)[ok]
        assert bool(((a - (b + w)).abs() <= (1 + U) * e + U * (b.abs() + w.abs()) + 1e-37).all()), k


@pytest.mark.parametrize("B,T,C", [(3, 7, 20), (2, 777, 20), (1, 9000, 20), (2, 3000, 3)])
@pytest.mark.parametrize("opened", [INF, 100.0])
def test_an_open_gate_passes_bad_tokens_over(dev, B, T, C, opened):
    """a token with f = +inf leaves the state as it is, whatever x holds, and gets no gradient"""
    f, x, h0, dh = _data(B, T, C, 22)
    f3, x3 = f.view(B, T, C), x.view(B, T, C)
    at = list(range(1, T, 5)) + [T - 1]
    f3[:, at] = opened
    want, tol = _reference(B, f, x, h0, dh)
    x3[:, at[::2]], x3[:, at[1::2]] = float("nan"), -INF
    h, df, dx, dh0 = _empty(B * T, C), _empty(B * T, C), _empty(B * T, C), _empty(B, C)
    K.gated_scan_fwd(B, f, x, h, h0=h0)
    K.gated_scan_bwd(B, f, x, h, dh, df, dx, h0=h0, dh0=dh0)
    for t, k in ((h, "h"), (dx, "dx"), (dh0, "dh0")):
        _close(t, want[k], tol[k], k)
    skipped = torch.zeros(B, T, C, dtype=torch.bool, device="cuda:0")
    skipped[:, at] = True
    skipped = skipped.view(-1, C)
    assert not df[skipped].any() and not dx[skipped].any()
    ratio = (df.double() - want["df"]).abs() / (tol["df"] + 1e-37)
    assert bool((ratio[~skipped] <= 1).all())


def test_bad_values_go_on_to_the_end(dev):
    """without a closed gate an infinity or NaN reaches every token behind it, also where
    the product of the gates between has come to 0 in fp32, and NaN gates too"""
    T, C = 20000, 64
    f, x, h0, dh = _data(1, T, C, 23, keep=-1.0)
    x[5, ::2] = INF
    f[17, 1::2] = float("nan")
    dh[T - 9] = float("nan")
    h, df, dx, dh0 = _empty(T, C), _empty(T, C), _empty(T, C), _empty(1, C)
    K.gated_scan_fwd(1, f, x, h, h0=h0)
    K.gated_scan_bwd(1, f, x, h, dh, df, dx, h0=h0, dh0=dh0)
    assert bool(torch.isfinite(h[:5]).all()) and not bool(torch.isfinite(h[17:]).any())
    assert bool(torch.isfinite(dx[T - 8:]).all()) and not bool(torch.isfinite(dx[:T - 8]).any())
    assert not bool(torch.isfinite(dh0).any())


def test_nothing(dev):
    e = torch.empty(0, 8, device="cuda:0")
    dh0 = _empty(3, 8)
    h0 = torch.zeros(3, 8, device="cuda:0")
    K.gated_scan_fwd(3, e, e, e, h0=h0)
    K.gated_scan_bwd(3, e, e, e, e, e, e, h0=h0, dh0=dh0)
    assert not dh0.any()


def test_gradients_against_differences(dev):
    B, T, C = 2, 11, 5
    f, x, h0, dh = _data(B, T, C, 8, keep=0.5)

    def loss(f, x, h0):
        s = torch.sigmoid(f.view(B, T, C))
        p, total = h0, 0
        for t in range(T):
            p = s[:, t] * p + (1 - s[:, t]) * x.view(B, T, C)[:, t]
            total = total + (p * dh.double().view(B, T, C)[:, t]).sum()
        return total

    h, df, dx, dh0 = _empty(B * T, C), _empty(B * T, C), _empty(B * T, C), _empty(B, C)
    K.gated_scan_fwd(B, f, x, h, h0=h0)
    K.gated_scan_bwd(B, f, x, h, dh, df, dx, h0=h0, dh0=dh0)
    args = [t.double() for t in (f, x, h0)]
    for k, got in enumerate((df, dx, dh0)):
        for i in range(0, args[k].numel(), 3):
            step = []
            for d in (1e-5, -1e-5):
                moved = [t.clone() for t in args]
                moved[k].view(-1)[i] += d
                step.append(loss(*moved))
            diff = float((step[0] - step[1]) / 2e-5)
            assert abs(float(got.reshape(-1)[i]) - diff) <= 2e-5 * (1 + abs(diff))


@pytest.mark.parametrize("B,T,C", [(1, 3000, 32), (4, 40, 70)])
def test_captured_and_replayed(dev, B, T, C):
    f, x, h0, dh = _data(B, T, C, 1)
    out = [_empty(B * T, C) for _ in range(3)] + [_empty(B, C)]
    ws = torch.empty(max(1, K.gated_scan_workspace(B, T, C)), dtype=torch.uint8, device="cuda:0")

    def step():
        K.gated_scan_fwd(B, f, x, out[0], h0=h0, ws=ws)
        K.gated_scan_bwd(B, f, x, out[0], dh, out[1], out[2], h0=h0, dh0=out[3], ws=ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        for t, v in zip((f, x, h0, dh), _data(B, T, C, 30 + i)):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for t in out:
            t.fill_(7.0)
        step()
        assert all(torch.equal(a, b) for a, b in zip(got, out))


def test_refusals(dev):
    f, x, h0, dh = _data(2, 6, 8, 1)
    h = _empty(12, 8)
    for bad in (lambda: K.gated_scan_fwd(5, f, x, h), lambda: K.gated_scan_fwd(2, f[:6], x, h),
                lambda: K.gated_scan_fwd(2, f, x, h, h0=h0[:1]),
                lambda: K.gated_scan_fwd(2, f.t().contiguous().t(), x, h),
                lambda: K.gated_scan_fwd(2, f[:1].expand(12, 8), x, h)):
        with pytest.raises(ValueError):
            bad()
    need = K.gated_scan_workspace(1, 60000, 8)
    if need:
        f, x, _, _ = _data(1, 60000, 8, 1)
        with pytest.raises(_lib.PkError):
            K.gated_scan_fwd(1, f, x, _empty(60000, 8),
                             ws=torch.empty(need - 1, dtype=torch.uint8, device="cuda:0"))


# ------------------------------------------------------------------- pico's API
def test_pico_op(P):
    """over the two column halves of one projection, with a state, and going on from
    the last token; every gradient"""
    B, T, C = 3, 40, 24
    f, x, h0, dh = (t.cpu() for t in _data(B, T, C, 4))
    want, tol = _reference(B, f, x, h0, dh)
    eye = np.eye(2 * C, dtype=np.float32)  # an exact projection
    fx = P.param([B * T, 2 * C], torch.cat([f, x], 1).numpy())
    sp, w = P.param([B, C], h0.numpy()), P.param([2 * C, 2 * C], eye)
    with P.arena():
        fv, xv = P.split_cols(P.matmul(fx, w), 2)
        h = P.gated_scan(fv, xv, sp, B)
        P.backward(P.mul(h, P.tensor([B * T, C], dh.numpy())))
        _close(torch.from_numpy(P.value(h)), want["h"], tol["h"], "h")
        g = torch.from_numpy(P.grad_value(fx))
        # (through the identity product: one more rounding in 24 bits)
        _close(g[:, :C], want["df"], tol["df"] + 2.0 ** -22 * want["df"].abs(), "df")
        _close(g[:, C:], want["dx"], tol["dx"] + 2.0 ** -22 * want["dx"].abs(), "dx")
        _close(torch.from_numpy(P.grad_value(sp)), want["dh0"], tol["dh0"], "dh0")
        last = P.last_token(h, B)
        assert np.array_equal(P.value(last), P.value(h).reshape(B, T, C)[:, -1])
    P.free(fx), P.free(sp), P.free(w)


def test_pico_parts_equal_the_whole(P):
    """a sequence in two parts, the state handed over by pico_last_token, has the whole
    sequence's values and gradients; one token at a time too"""
    B, T, C, cut = 2, 30, 8, 12
    f, x, h0, dh = (t.cpu() for t in _data(B, T, C, 5))
    want, tol = _reference(B, f, x, h0, dh)

    def part(t, lo, hi):
        return P.param([B * (hi - lo), C], t.view(B, T, C)[:, lo:hi].reshape(-1, C).numpy())

    ps = [part(t, lo, hi) for lo, hi in ((0, cut), (cut, T)) for t in (f, x)]
    sp = P.param([B, C], h0.numpy())
    with P.arena():
        a = P.gated_scan(ps[0], ps[1], sp, B)
        b = P.gated_scan(ps[2], ps[3], P.last_token(a, B), B)
        wa = P.tensor([B * cut, C], dh.view(B, T, C)[:, :cut].reshape(-1, C).numpy())
        wb = P.tensor([B * (T - cut), C], dh.view(B, T, C)[:, cut:].reshape(-1, C).numpy())
        # both parts' weighted sums as one entry: ones . (a wa) . ones + the same of b
        la = P.matmul(P.matmul(P.tensor([1, B * cut], np.ones(B * cut)), P.mul(a, wa)),
                      P.tensor([C, 1], np.ones(C)))
        lb = P.matmul(P.matmul(P.tensor([1, B * (T - cut)], np.ones(B * (T - cut))), P.mul(b, wb)),
                      P.tensor([C, 1], np.ones(C)))
        P.backward(P.add(la, lb))
        for k, v in (("df", 0), ("dx", 1)):
            got = torch.cat([torch.from_numpy(P.grad_value(ps[i])).view(B, -1, C)
                             for i in (v, v + 2)], 1).reshape(-1, C)
            _close(got, want[k], tol[k], k)
        _close(torch.from_numpy(P.grad_value(sp)), want["dh0"], tol["dh0"], "dh0")
    for t in ps + [sp]:
        P.free(t)


def test_pico_shared_operands_and_refusals(P):
    """one tensor as f and x, and as the state: the gradients add up"""
    B, C = 4, 6
    f, x, h0, dh = (t.cpu() for t in _data(B, 1, C, 6))
    t = P.param([B, C], x.numpy())
    v = x.double().requires_grad_()
    s = torch.sigmoid(v)
    ((s * v + (1 - s) * v) * dh.double()).sum().backward()
    with P.arena():
        h = P.gated_scan(t, t, t, B)
        P.backward(P.mul(h, P.tensor([B, C], dh.numpy())))
        got = torch.from_numpy(P.grad_value(t))
        # three gradients of at most (1 + |x|) |dh| each
        assert bool(((got - v.grad).abs() <= 60 * U * (1 + x.abs()) * dh.abs()).all())
        other = P.tensor([B, C + 1], np.zeros((B, C + 1)))
        for bad in ((t, other, None, B), (t, t, other, B), (t, t, None, 3), (t, t, None, 0),
                    (None, t, None, B)):
            with pytest.raises(PicoError):
                P.gated_scan(*bad)
        for bad in ((t, 3), (t, 0), (t, 8), (None, 1)):
            with pytest.raises(PicoError):
                P.last_token(*bad)
    P.free(t)


def test_pico_a_tensor_and_its_only_view(P):
    """a projection and the one column view of it share a gradient, to which each adds"""
    B, C = 4, 6
    f, x, h0, dh = (t.cpu() for t in _data(B, 1, C, 7))
    v = x.double().requires_grad_()
    s = torch.sigmoid(v)
    ((s * h0.double() + (1 - s) * v) * dh.double()).sum().backward()
    ((lambda u: torch.sigmoid(u) * u + (1 - torch.sigmoid(u)) * x.double())(v) * dh.double()).sum().backward()
    leaf, sp = P.param([B, C], x.numpy()), P.param([B, C], h0.numpy())
    one = P.param([C], np.ones(C, np.float32))
    with P.arena():
        for operands in (lambda t, u: (t, u, sp), lambda t, u: (t, sp, u)):
            t = P.matmul(leaf, P.tensor([C, C], np.eye(C)))
            f_, x_, h_ = operands(t, P.split_cols(t, 1)[0])
            if x_ is sp:  # the token itself as the state, and another one's values
                x_ = P.tensor([B, C], x.numpy())
            P.backward(P.mul(P.gated_scan(f_, x_, h_, B), P.tensor([B, C], dh.numpy())))
        got = torch.from_numpy(P.grad_value(leaf))
        # four gradients of at most (1 + |x| + |h0|) |dh| each
        assert bool(((got - v.grad).abs() <= 100 * U * (1 + x.abs() + h0.abs()) * dh.abs()).all())
        row = P.matmul(P.tensor([1, C], np.ones((1, C))), P.tensor([C, C], np.eye(C)))
        view = P.split_cols(row, 1)[0]
        for bad in ((row, view, one), (view, row, None), (P.tensor([3, C]), row, view)):
            with pytest.raises(PicoError):
                P.layernorm(*bad, 1e-5)
        col = P.matmul(P.tensor([B, C], np.ones((B, C))), P.tensor([C, 1], np.ones((C, 1))))
        gates, route = P.route_topk(P.tensor([B, 2], np.zeros((B, 2))), 1)
        with pytest.raises(PicoError):
            P.expert_combine(col, P.split_cols(col, 1)[0], route, None)
        # two views of one tensor have columns of their own
        two = P.split_cols(P.matmul(P.tensor([B, C], np.ones((B, C))), P.tensor([C, 2 * C], np.ones((C, 2 * C)))), 2)
        P.gated_scan(two[0], two[1], None, B)
    for t in (leaf, sp, one):
        P.free(t)
