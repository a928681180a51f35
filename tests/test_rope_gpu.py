"""Rotary positions (pk_rope_f32) against float64.

Tolerance: sine and cosine are each rounded once (2^-24 relative), and so are the two
products and their sum: |y - exact| <= m (|x1| + |x2|) (1/2 + 1/2 + 1) 2^-23, and half of
2^-23 |y| for the sum, of which |y| <= m (|x1| + |x2|); the angle, in float64, is off by
|position| 2^-52 at most.
"""
import numpy as np
import pytest
import torch

import _paged as O
from pico_amd import kernels as K
from pico_amd._lib import PkError

pytestmark = pytest.mark.gpu


def _cuda(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def _bound(x, pos, f, interleaved, m):
    n = len(f)
    b = np.zeros(x.shape)
    i1 = np.arange(n) * 2 if interleaved else np.arange(n)
    i2 = i1 + 1 if interleaved else i1 + n
    s = abs(m) * (np.abs(x[..., i1]) + np.abs(x[..., i2])) * (
        1.5 * 2.0 ** -23 + np.abs(np.asarray(pos, np.float64))[:, None, None] * 2.0 ** -51)
    b[..., i1] = b[..., i2] = s
    return b


# tokens, heads, head, turned, interleaved, largest position, scaling
SHAPES = [(1, 1, 2, 2, False, 1, "none"), (1, 12, 64, 64, False, 9, "none"), (64, 12, 64, 64, False, 1024, "none"),
          (7, 3, 80, 80, True, 5000, "linear"), (130, 5, 96, 48, False, 1 << 20, "parts"),
          (33, 2, 128, 64, True, 1 << 20, "ntk"), (65, 3, 36, 12, True, 77, "none"), (65, 3, 36, 8, False, 77, "none"),
          (20, 3, 7, 4, False, 50, "none"), (20, 3, 7, 6, True, 50, "none"), (9, 2, 50, 50, False, 50, "none"),
          (5, 2, 256, 256, False, 4096, "none"), (3, 1, 1024, 1024, False, 999, "none"), (3, 2, 1000, 6, True, 9, "none"),
          (17, 2, 64, 0, False, 9, "none"), (5000, 4, 32, 32, True, 3000, "none"), (1030, 24, 64, 64, False, 1024, "none"),
          (2, 5000, 8, 8, False, 4, "none"), (40, 3, 50, 22, False, 900, "none"), (11, 5, 130, 6, True, 900, "none"),
          (9, 4, 19, 10, True, 40, "none"), (700, 6, 128, 6, False, 900, "none"), (2, 524287, 2, 2, False, 9, "none"),
          (3, 349525, 3, 2, True, 9, "none"),
          # rows of fewer than 4 values
          (70, 1, 3, 2, False, 900, "none"), (70, 1, 3, 2, True, 900, "none"), (5, 3, 1, 0, False, 9, "none"), (600, 1, 2, 2, True, 9, "none")]


@pytest.mark.parametrize("N,H,hd,rot,inter,far,scaling", SHAPES)
def test_against_float64(dev, N, H, hd, rot, inter, far, scaling):
    rng = np.random.default_rng(N * 31 + hd)
    x = rng.standard_normal((N, H, hd)).astype(np.float32)
    pos = rng.integers(0, far, N).astype(np.int32)
    m = 1.25 if scaling == "parts" else 1.0
    fr = K.rope_freqs(rot, 10000.0, scaling, factor=16.0, length=max(1, far) / 16.0, device=dev)
    r = K.Rope(fr, inter, m)
    f = fr.cpu().numpy()
    for back in (False, True):
        y = torch.full((N, H * hd), 7.0, device=dev)
        K.rope(r, H, _cuda(x.reshape(N, -1), dev), _cuda(pos, dev), y, backward=back)
        got = y.cpu().numpy().reshape(N, H, hd)
        want = O.turned(x, pos, f, inter, m, back)
        assert (np.abs(got - want) <= _bound(x, pos, f, inter, m)).all()
        np.testing.assert_array_equal(got[..., rot:], x[..., rot:])


def test_backward_is_the_transpose(dev):
    """<dy, y(x)> = <dx(dy), x>, and the difference quotient of a sum along a direction"""
    N, H, hd, rot = 40, 3, 64, 32
    g = torch.Generator(device=dev).manual_seed(3)
    x, dy, d = (torch.randn(N, H * hd, device=dev, generator=g) for _ in range(3))
    pos = torch.arange(N, device=dev, dtype=torch.int32) * 37
    r = K.Rope(K.rope_freqs(rot, device=dev), True, 1.5)
    y, dx, y2 = (torch.empty_like(x) for _ in range(3))
    K.rope(r, H, x, pos, y)
    K.rope(r, H, dy, pos, dx, backward=True)
    a, b = (dy.double() * y.double()).sum(), (dx.double() * x.double()).sum()
    # sums of 7680 products of values off by 3 2^-24 (|x1| + |x2|) at most, each about 1
    assert abs(a - b) <= 2.0 ** -20 * (dy.double().abs() * y.double().abs()).sum()
    h = 0.125
    K.rope(r, H, x + h * d, pos, y2)
    num = ((dy.double() * (y2.double() - y.double())).sum()) / h
    want = (dx.double() * d.double()).sum()
    assert abs(num - want) <= 2.0 ** -18 * (dy.double().abs() * y.double().abs()).sum() / h


@pytest.mark.parametrize("H,hd,rot", [(4, 64, 48), (4, 64, 6), (3, 45, 10)])
@pytest.mark.parametrize("inter", [False, True])
def test_layouts_accumulation_and_place(dev, inter, H, hd, rot):
    N = 37
    g = torch.Generator(device=dev).manual_seed(5)
    wide = torch.randn(N, 3 * H * hd + 2, device=dev, generator=g)
    pos = torch.randint(0, 9999, (N,), device=dev, dtype=torch.int32, generator=g)
    r = K.Rope(K.rope_freqs(rot, device=dev), inter)
    want = torch.empty(N, H * hd, device=dev)
    for off in (0, H * hd, H * hd + 1):  # (the last: not 16-byte aligned)
        x = wide[:, off:off + H * hd]
        K.rope(r, H, x.contiguous(), pos, want)
        out = torch.full_like(wide, 3.0)
        K.rope(r, H, x, pos, out[:, off:off + H * hd])
        assert torch.equal(out[:, off:off + H * hd], want)
        assert (out[:, :off] == 3.0).all() and (out[:, off + H * hd:] == 3.0).all()
        # onto what is there: one rounding of the sum
        acc = torch.randn(N, H * hd, device=dev, generator=g)
        both = acc.clone()
        K.rope(r, H, x, pos, both, accum=True)
        assert torch.equal(both, want + acc)
        mine = x.contiguous()
        K.rope(r, H, mine, pos, mine)
        assert torch.equal(mine, want)


def test_positions_of_any_sign_and_size(dev):
    """cos is even, sin odd; the largest int32 stay on the circle"""
    N, hd = 6, 8
    x = torch.randn(N, hd, device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    pos = torch.tensor([5, -5, 2 ** 31 - 1, -2 ** 31, 0, 123456789], device=dev, dtype=torch.int32)
    r = K.Rope(K.rope_freqs(hd, device=dev))
    y, z = torch.empty_like(x), torch.empty_like(x)
    K.rope(r, 1, x, pos, y)
    K.rope(r, 1, y, pos, z, backward=True)
    torch.testing.assert_close(z, x, rtol=0, atol=float(x.abs().max()) * 8 * 2.0 ** -23)
    assert torch.equal(y[4], x[4])
    k = torch.empty_like(x)
    K.rope(r, 1, x[:1].expand(2, hd).contiguous(), pos[:2].contiguous(), k[:2], backward=False)
    back = torch.empty_like(x)
    K.rope(r, 1, x[:1].contiguous(), pos[:1].contiguous(), back[:1], backward=True)
    assert torch.equal(back[0], k[1])


def test_infinities_stay_in_their_pair(dev):
    x = torch.ones(1, 12, device=dev)
    x[0, 1], x[0, 11] = float("inf"), float("nan")
    pos = torch.ones(1, device=dev, dtype=torch.int32)
    y = torch.empty_like(x)
    K.rope(K.Rope(K.rope_freqs(8, device=dev)), 1, x, pos, y)
    bad = ~torch.isfinite(y[0])
    assert bad.nonzero().view(-1).tolist() == [1, 5, 11]


def test_empty_and_refused(dev):
    r = K.Rope(K.rope_freqs(8, device=dev))
    none = torch.empty(0, 16, device=dev)
    i = torch.empty(0, device=dev, dtype=torch.int32)
    K.rope(r, 2, none, i, none)
    x = torch.zeros(4, 16, device=dev)
    pos = torch.zeros(4, device=dev, dtype=torch.int32)
    with pytest.raises(ValueError):
        K.rope(r, 3, x, pos, x)  # 16 is not 3 heads
    with pytest.raises(ValueError):
        K.rope(r, 2, x, pos[:3], x)
    with pytest.raises(ValueError):
        K.rope(r, 2, x, pos, x[:, :8])
    with pytest.raises(TypeError):
        K.rope(r, 2, x, pos.long(), x)
    with pytest.raises(TypeError):
        K.rope(r, 2, x.double(), pos, x)
    with pytest.raises(PkError):
        K.rope(r, 4, x, pos, x)  # heads of 4 values, 8 to turn
    with pytest.raises(TypeError):
        K.Rope(torch.zeros(4, dtype=torch.float64))


def test_other_stream_and_captured(dev):
    N, H, hd = 300, 6, 64
    g = torch.Generator(device=dev).manual_seed(8)
    x = torch.randn(N, H * hd, device=dev, generator=g)
    pos = torch.randint(0, 4096, (N,), device=dev, dtype=torch.int32, generator=g)
    r = K.Rope(K.rope_freqs(hd, device=dev))
    want, y = torch.empty_like(x), torch.empty_like(x)
    K.rope(r, H, x, pos, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.rope(r, H, x, pos, y)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.rope(r, H, x, pos, y)
    for shift in (0, 5, 9):
        pos.add_(shift)
        x.mul_(1.5)
        y.zero_()
        graph.replay()
        K.rope(r, H, x, pos, want)
        assert torch.equal(y, want)
