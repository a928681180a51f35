"""The paged e4m3 cache (pk_kv_append_f32) and the attention over it (pk_attn_paged_f32)
against float64, token by token (tests/_paged.py, which derives the tolerances)."""
import numpy as np
import pytest
import torch

import _paged as O
from pico_amd import kernels as K
from pico_amd._lib import PkError

pytestmark = pytest.mark.gpu
NAN = 0x7f


def _cuda(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def _i32(a, dev):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=dev)


class Pair:
    """a cache on the device and the oracle's, with the same contents"""

    def __init__(self, dev, rng, lens, new, page, kvh, hd, spare=3, fill=None, width=0):
        self.dev, self.kvh, self.hd, self.page = dev, kvh, hd, page
        need = sum(-(-(a + n) // page) for a, n in zip(lens, new))
        table, self.offsets = O.layout(lens, new, page, need + spare, rng)
        if table.shape[1] < width:
            table = np.pad(table, ((0, 0), (0, width - table.shape[1])), constant_values=-1)
        self.lens = np.asarray(lens)
        self.o = O.Cache(need + spare, kvh, page, hd, table)
        for pool, exps in ((self.o.k, self.o.k_exp), (self.o.v, self.o.v_exp)):
            pool[...] = rng.integers(0, 256, pool.shape) if fill is None else fill
            pool[(pool & 127) == 127] = 0x3c
            exps[...] = rng.integers(122, 130, exps.shape)
        self.o.k[..., hd:] = 0
        self.upload()

    def upload(self):
        o = self.o
        self.t = [_cuda(a, self.dev) for a in (o.k, o.v, o.k_exp, o.v_exp, o.table.astype(np.int32))]
        self.lens_t, self.offsets_t = _i32(self.lens, self.dev), _i32(self.offsets, self.dev)
        self.c = K.PagedKV(*self.t, self.lens_t, self.offsets_t, self.hd)

    def same(self):
        for name, got, want in zip(("k", "v", "k_exp", "v_exp"), self.t, (self.o.k, self.o.v, self.o.k_exp, self.o.v_exp)):
            np.testing.assert_array_equal(got.cpu().numpy(), want, err_msg=name)


def _rows(rng, N, heads, hd):
    return rng.standard_normal((N, heads, hd)).astype(np.float32)


# lens, new, page, kv heads, head
APPENDS = [([0], [1], 16, 1, 64), ([0, 5, 16], [1, 1, 1], 16, 2, 64), ([3, 0, 15, 31], [0, 40, 1, 17], 16, 3, 80),
           ([63, 64, 100], [1, 1, 200], 64, 2, 128), ([7, 127], [121, 2], 128, 2, 256), ([1], [300], 32, 1, 96),
           ([5] * 70, [i % 4 for i in range(70)], 16, 1, 32), ([9, 2], [3, 30], 32, 2, 7), ([0] * 3, [0, 0, 0], 16, 1, 32),
           ([12], [129], 128, 1, 33), ([2], [1], 128, 16, 64),
           # many tokens of one sequence among others that wait
           ([5] + [0] * 99, [70] + [0] * 99, 64, 2, 64), ([37] + [3] * 40, [60] + [0] * 39 + [1], 16, 1, 256),
           # more pages and heads than are written to at once
           ([0, 37], [500, 700], 16, 8, 96), ([50, 3], [600, 200], 128, 60, 250)]


@pytest.mark.parametrize("lens,new,page,kvh,hd", APPENDS)
def test_append(dev, lens, new, page, kvh, hd):
    """without positions every byte is determined: equal to the oracle's, and nothing else
    is touched"""
    rng = np.random.default_rng(len(lens) * 7 + hd)
    p = Pair(dev, rng, lens, new, page, kvh, hd)
    N = int(p.offsets[-1])
    k, v = _rows(rng, N, kvh, hd), _rows(rng, N, kvh, hd)
    k *= 2.0 ** rng.integers(-8, 8, (N, 1, 1)).astype(np.float32)  # pages' scales grow
    K.kv_append(p.c, _cuda(k.reshape(N, kvh * hd), dev), _cuda(v.reshape(N, kvh * hd), dev))
    p.o.append(k, v, lens, p.offsets)
    p.same()


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("hd,rot,H", [(64, 64, 4), (80, 40, 2), (128, 128, 6), (96, 6, 2), (33, 32, 2), (7, 6, 4)])
def test_append_turns_as_rope_does(dev, hd, rot, H, inter):
    rng = np.random.default_rng(hd + rot)
    lens, new, page, kvh = [100, 0, 37, 4000], [3, 20, 0, 1], 16, 2
    p = Pair(dev, rng, lens, new, page, kvh, hd)
    N = int(p.offsets[-1])
    k, v, q = (_cuda(_rows(rng, N, n, hd).reshape(N, -1), dev) for n in (kvh, kvh, H))
    pos = np.concatenate([np.arange(a, a + n) for a, n in zip(lens, new)]).astype(np.int32)
    r = K.Rope(K.rope_freqs(rot, device=dev), inter, 1.25)
    kt, qt, q_out = torch.empty_like(k), torch.empty_like(q), torch.full_like(q, 9.0)
    K.rope(r, kvh, k, _cuda(pos, dev), kt)
    K.rope(r, H, q, _cuda(pos, dev), qt)
    K.kv_append(p.c, k, v, r, H=H, q=q, q_out=q_out)
    assert torch.equal(q_out, qt)
    p.o.append(kt.cpu().numpy().reshape(N, kvh, hd), v.cpu().numpy().reshape(N, kvh, hd), lens, p.offsets)
    p.same()
    mine = q.clone()  # in place
    K.kv_append(p.c, k, v, r, H=H, q=mine, q_out=mine)
    assert torch.equal(mine, qt)
    p.same()  # (the same tokens again: the same bytes)


@pytest.mark.parametrize("lens,new,page,kvh,hd,rot", [([100, 7], [300, 1], 128, 2, 256, 256), ([50], [900], 128, 44, 250, 100),
                                                      ([5] + [0] * 99, [130] + [0] * 99, 64, 2, 96, 96), ([0, 37], [500, 700], 16, 8, 64, 64)])
def test_append_turns_pages_in_parts(dev, lens, new, page, kvh, hd, rot):
    """values that are read twice, and waves with a page each, turned as pk_rope_f32 does"""
    rng = np.random.default_rng(hd + kvh)
    p = Pair(dev, rng, lens, new, page, kvh, hd)
    N = int(p.offsets[-1])
    k, v = (_cuda(_rows(rng, N, kvh, hd).reshape(N, -1), dev) for _ in range(2))
    pos = np.concatenate([np.arange(a, a + n) for a, n in zip(lens, new)]).astype(np.int32)
    r = K.Rope(K.rope_freqs(rot, device=dev))
    kt = torch.empty_like(k)
    K.rope(r, kvh, k, _cuda(pos, dev), kt)
    K.kv_append(p.c, k, v, r)
    p.o.append(kt.cpu().numpy().reshape(N, kvh, hd), v.cpu().numpy().reshape(N, kvh, hd), lens, p.offsets)
    p.same()


def test_append_one_by_one_and_at_once(dev):
    """a page filled token by token holds what it holds filled at once where its scale does
    not grow, and values off by a step of the last rounding where it does"""
    rng = np.random.default_rng(1)
    hd, kvh, page, T = 64, 2, 32, 75
    once, steps = (Pair(dev, np.random.default_rng(2), [0], [T], page, kvh, hd, fill=0) for _ in range(2))
    k, v = (_cuda(_rows(rng, T, kvh, hd).reshape(T, -1), dev) for _ in range(2))
    K.kv_append(once.c, k, v)
    for t in range(T):
        steps.lens_t.fill_(t)
        steps.offsets_t.copy_(_i32([0, 1], dev))
        K.kv_append(steps.c, k[t:t + 1], v[t:t + 1])
    for i in range(2):
        assert torch.equal(once.t[2 + i], steps.t[2 + i])
        a, b = (O.CODES[c.t[i].cpu().numpy()] for c in (once, steps))
        # values above 2^-6 of the scale keep their codes; below, a second rounding
        assert (np.abs(a - b) <= 2.0 ** -9).all()
        assert (a == b)[np.abs(a) >= 2.0 ** -6].all()


def test_append_of_many_rows(dev):
    """a million rows, whose queries have more heads than a launch has workgroups"""
    N, H, page = 1 << 20, 32, 128
    pages = N // page
    pool = K.kv_pool(pages, 1, page, 1, dev)
    table = torch.arange(pages, device=dev, dtype=torch.int32).view(1, -1)
    c = K.PagedKV(*pool, table, _i32([0], dev), _i32([0, N], dev), 1)
    k = torch.ones(N, 1, device=dev)
    q = torch.arange(N * H, device=dev, dtype=torch.float32).view(N, H)
    out = torch.zeros_like(q)
    K.kv_append(c, k, 3 * k, None, H=H, q=q, q_out=out)
    assert torch.equal(out, q)
    one = torch.tensor(1.0).to(torch.float8_e4m3fn)
    for x, e, want in ((pool[0][:, 0, :, 0], pool[2], 1.0), (pool[1][:, 0, 0, :], pool[3], 3.0)):
        assert (x.view(one.dtype).float() * torch.exp2(e.float() - 127) == want).all()


def test_append_odd_values(dev):
    rng = np.random.default_rng(4)
    p = Pair(dev, rng, [5], [12], 16, 2, 64)
    k, v = _rows(rng, 12, 2, 64), _rows(rng, 12, 2, 64)
    k[0, 0, 3], k[1, 0, 4], k[2, 1, 5] = np.inf, -np.inf, np.nan
    v[:, 1] = 0.0
    v[3, 0, :] = np.nan
    v[11, 0, 7] = 1e30  # beyond 448 * 2^40
    k[11, 1] = 1e-30
    K.kv_append(p.c, _cuda(k.reshape(12, -1), dev), _cuda(v.reshape(12, -1), dev))
    p.o.append(k, v, [5], p.offsets)
    for got, want in ((p.t[0], p.o.k), (p.t[1], p.o.v)):
        np.testing.assert_array_equal(O.CODES[got.cpu().numpy()], O.CODES[want])
    for got, want in ((p.t[2], p.o.k_exp), (p.t[3], p.o.v_exp)):
        np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_append_out_of_range(dev):
    """pages that are none, positions behind the table, rows behind the inputs: nothing is
    written for them"""
    rng = np.random.default_rng(6)
    p = Pair(dev, rng, [0, 10, 40, 3], [20, 20, 20, 4], 16, 2, 64)
    p.o.table[0, 1], p.o.table[1, 0] = -7, 10 ** 6
    p.o.table = np.ascontiguousarray(p.o.table[:, :3])  # sequence 2 ends behind it
    p.upload()
    N = int(p.offsets[-1])
    k, v = _rows(rng, N, 2, 64), _rows(rng, N, 2, 64)
    kt, vt = _cuda(k.reshape(N, -1), dev), _cuda(v.reshape(N, -1), dev)
    K.kv_append(p.c, kt, vt)
    p.o.append(k, v, p.lens, p.offsets)
    p.same()
    for lens, offsets in (([-5, 10 ** 9, 0, 0], [0, 20, 40, 60, 64]), ([0, 0, 0, 0], [-9, -3, -3, -3, -1]),
                          ([0, 0, 0, 0], [64, 64, 70, 10 ** 9, 65]), ([2 ** 31 - 1, -2 ** 31, 0, 0], [5, 5, 5, 5, 5])):
        before = [t.clone() for t in p.t]
        p.lens_t.copy_(_i32(lens, dev))
        p.offsets_t.copy_(_i32(offsets, dev))
        q = torch.full((N, 128), 2.0, device=dev)
        K.kv_append(p.c, kt, vt, K.Rope(K.rope_freqs(64, device=dev)), H=2, q=q, q_out=q)
        torch.cuda.synchronize()
        if lens[0] != -5:
            assert all(torch.equal(a, b) for a, b in zip(before, p.t))
            assert (q == 2.0).all()


# lens, new, page, kv heads, query heads a kv head, head
ATTENDS = [([0], [1], 16, 1, 1, 64), ([1, 15, 16, 17], [1, 1, 1, 1], 16, 2, 1, 64),
           ([63, 64, 65, 1000], [1, 1, 1, 1], 64, 2, 4, 128), ([200, 3, 77], [3, 0, 2], 16, 2, 5, 96),
           ([300, 0], [1, 1], 32, 1, 8, 32), ([300, 130], [1, 1], 128, 2, 16, 64), ([90], [7], 16, 3, 3, 80),
           ([0, 50], [33, 20], 16, 2, 2, 64), ([5000], [1], 128, 1, 2, 256), ([700], [4], 32, 1, 24, 256),
           ([31] * 70, [i % 3 for i in range(70)], 32, 1, 2, 7), ([0], [200], 64, 2, 1, 128), ([513], [130], 16, 1, 3, 33),
           ([0, 0, 0], [1, 0, 5], 128, 2, 2, 64), ([100], [90], 32, 1, 2, 256),
           # caches beyond 2048 tokens: units shared out evenly, tiles in parts
           ([2300, 700, 64], [1, 1, 1], 64, 1, 3, 64), ([2100, 2500], [2, 1], 16, 1, 8, 96),
           ([2200, 1, 0, 900], [1, 1, 0, 2], 128, 1, 1, 32), ([3000], [1], 64, 1, 16, 128), ([1500], [5], 16, 1, 7, 256),
           ([20] * 66 + [2100], [1] * 67, 128, 1, 4, 128), ([3000], [40], 64, 1, 4, 64),
           # tiles of 128 rows
           ([0], [700], 64, 2, 18, 64), ([40, 0, 7], [333, 0, 400], 16, 1, 17, 128), ([5], [530], 32, 1, 48, 33),
           ([300], [1040], 128, 12, 1, 96), ([77, 3], [500, 20], 16, 2, 12, 80), ([0], [530], 64, 1, 16, 256),
           # and these with a tile's tokens split over workgroups
           ([2600], [260], 64, 1, 16, 64), ([1500, 0, 900], [200, 0, 150], 16, 1, 36, 96), ([1300], [140], 32, 1, 60, 256),
           ([2000], [129], 128, 1, 32, 32), ([1500, 1], [1, 400], 32, 1, 31, 128),
           ([9000], [65], 128, 1, 64, 32)]


@pytest.mark.parametrize("lens,new,page,kvh,group,hd", ATTENDS)
def test_attention(dev, lens, new, page, kvh, group, hd):
    rng = np.random.default_rng(hd + len(lens))
    p = Pair(dev, rng, lens, new, page, kvh, hd)
    # what lies behind every sequence's last token may be anything
    for b, (a, n) in enumerate(zip(lens, new)):
        end = a + n
        if end % page:
            pid = p.o.table[b, end // page]
            if pid >= 0:
                p.o.k[pid, :, end % page:] = NAN
                p.o.v[pid, :, :, end % page:] = NAN
    p.upload()
    N, H = int(p.offsets[-1]), kvh * group
    q = _rows(rng, N, H, hd) * 2.0 ** rng.integers(-3, 2, (N, H, 1)).astype(np.float32)
    o = torch.full((N + 3, H * hd), 5.0, device=dev)
    qt = torch.cat([_cuda(q.reshape(N, -1), dev), torch.full((3, H * hd), float("nan"), device=dev)])
    scale = hd ** -0.5 / 16  # (values of a page are up to 448 times its scale)
    K.attn_paged(p.c, H, qt, o, scale=scale)
    got = o.cpu().numpy()
    assert (got[N:] == 5.0).all()  # rows of no sequence
    want, tol = p.o.attend(q.astype(np.float64), lens, p.offsets, H, scale)
    err = np.abs(got[:N].reshape(N, H, hd) - want)
    assert (err <= tol + 1e-30).all(), float((err / (tol + 1e-30)).max())


def test_attention_layouts_and_default_scale(dev):
    rng = np.random.default_rng(9)
    lens, new, H, kvh, hd = [40, 9], [2, 1], 4, 2, 64
    p = Pair(dev, rng, lens, new, 16, kvh, hd)
    N = 3
    q = _rows(rng, N, H, hd) / 64
    want, tol = p.o.attend(q.astype(np.float64), lens, p.offsets, H)
    for off in (0, 4, 1):  # (1: not 16-byte aligned)
        wide = torch.zeros(N, H * hd + 8, device=dev)
        wide[:, off:off + H * hd] = _cuda(q.reshape(N, -1), dev)
        out = torch.full_like(wide, 3.0)
        K.attn_paged(p.c, H, wide[:, off:off + H * hd], out[:, off:off + H * hd])
        got = out[:, off:off + H * hd].cpu().numpy().reshape(N, H, hd)
        assert (np.abs(got - want) <= tol).all()
        assert (out[:, :off] == 3.0).all() and (out[:, off + H * hd:] == 3.0).all()


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [30, 40, 1, 25], [150, 140, 1, 130]])
def test_attention_over_absent_pages(dev, new, hd):
    """pages that are none count as absent: in the middle, at the end, and all of them (a row
    without a key gets zeros); NaN in the pages that are read in their place does not matter"""
    rng = np.random.default_rng(10)
    lens = [100, 70, 40, 5]
    # (tables for 4096 tokens: with many rows, tiles of 128 in parts)
    p = Pair(dev, rng, lens, new, 16, 2, hd, width=256)
    p.o.table[0, 2], p.o.table[1, (70 + new[1] - 1) // 16] = -1, 10 ** 7
    p.o.table[2, :] = -1
    p.o.table[3, 0] = 2 ** 31 - 1
    used = set(p.o.table[(p.o.table >= 0) & (p.o.table < p.o.k.shape[0])].tolist())
    if 0 not in used:
        p.o.k[0], p.o.v[0] = NAN, NAN
    p.upload()
    N = int(p.offsets[-1])
    H = 24 if N > 400 else 4  # (24: tiles of 128 rows)
    q = _rows(rng, N, H, hd) / 64
    o = torch.full((N, H * hd), 5.0, device=dev)
    K.attn_paged(p.c, H, _cuda(q.reshape(N, -1), dev), o)
    want, tol = p.o.attend(q.astype(np.float64), lens, p.offsets, H)
    assert (np.abs(o.cpu().numpy().reshape(N, H, hd) - want) <= tol).all()
    assert (o[p.offsets[2]:p.offsets[3]] == 0).all()


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("new", [4, 50, 150])
def test_attention_nan_reaches_the_rows_that_see_it(dev, new, hd):
    """NaN among a later token's keys or values does not reach the rows before it"""
    rng = np.random.default_rng(11)
    lens, kvh, page = [90], 1, 16
    H = 32 if new == 150 else 2  # (150: tiles of 128 rows)
    for what in ("k", "v"):
        p = Pair(dev, rng, lens, [new], page, kvh, hd, width=256)  # (as above)
        t = 90 + new // 2  # this token's
        pid = p.o.table[0, t // page]
        if what == "k":
            p.o.k[pid, 0, t % page, 5] = NAN
        else:
            p.o.v[pid, 0, 7, t % page] = NAN | 128
        p.upload()
        q = _rows(rng, new, H, hd) / 64
        o = torch.empty(new, H * hd, device=dev)
        K.attn_paged(p.c, H, _cuda(q.reshape(new, -1), dev), o)
        got = o.cpu().numpy().reshape(new, H, hd)
        first = new // 2
        clean, tol = p.o.attend(q[:first].astype(np.float64), lens, [0, first], H)
        assert (np.abs(got[:first] - clean) <= tol).all()
        if what == "k":
            assert np.isnan(got[first:]).all()
        else:
            assert np.isnan(got[first:, :, 7]).all()
            assert np.isfinite(np.delete(got[first:], 7, axis=2)).all()


def test_attention_extreme_scales(dev):
    """pages whose values differ by 2^60 in scale, pages of zeros, queries of any size: the
    weighted sum keeps its relative exactness where the largest weights have the smallest
    values"""
    rng = np.random.default_rng(12)
    lens, new, page, kvh, hd, H = [127, 60], [1, 1], 16, 1, 64, 2
    p = Pair(dev, rng, lens, new, page, kvh, hd)
    p.o.v_exp[:, 0] = rng.choice([87, 97, 127, 147], p.o.v_exp.shape[0])
    p.o.k_exp[:, 0] = 119
    zero = p.o.table[0, 3]
    p.o.v[zero], p.o.v_exp[zero] = 0, 87
    p.upload()
    for size in (0.0, 1e-38, 1.0, 30.0, 1e-42):
        q = _rows(rng, 2, H, hd) * np.float32(size)
        o = torch.empty(2, H * hd, device=dev)
        K.attn_paged(p.c, H, _cuda(q.reshape(2, -1), dev), o, scale=0.01)
        want, tol = p.o.attend(q.astype(np.float64), lens, p.offsets, H, 0.01)
        assert (np.abs(o.cpu().numpy().reshape(2, H, hd) - want) <= tol).all()


def test_attention_queries_that_are_not_finite(dev):
    rng = np.random.default_rng(13)
    p = Pair(dev, rng, [40, 40], [1, 1], 16, 1, 64)
    q = _rows(rng, 2, 2, 64) / 64
    q[0, 0, 3], q[1, 1, 9] = np.inf, np.nan
    o = torch.empty(2, 128, device=dev)
    K.attn_paged(p.c, 2, _cuda(q.reshape(2, -1), dev), o)
    got = o.cpu().numpy().reshape(2, 2, 64)
    assert np.isnan(got[0, 0]).all() and np.isnan(got[1, 1]).all()
    want, tol = p.o.attend(np.nan_to_num(q).astype(np.float64), [40, 40], p.offsets, 2)
    for b, h in ((0, 1), (1, 0)):
        assert (np.abs(got[b, h] - want[b, h]) <= tol[b, h]).all()


@pytest.mark.parametrize("new", [1, 6, 200])
def test_attention_is_repeatable(dev, new):
    rng = np.random.default_rng(14)
    p = Pair(dev, rng, [3000, 17, 900], [new, new, new], 64, 2, 64)
    N, H = 3 * new, 8
    q = _cuda(_rows(rng, N, H, 64).reshape(N, -1), dev)
    a, b = torch.empty_like(q), torch.empty_like(q)
    K.attn_paged(p.c, H, q, a)
    for _ in range(3):
        K.attn_paged(p.c, H, q, b)
        assert torch.equal(a, b)


@pytest.mark.parametrize("past", [10, 3000])
def test_attention_bad_arrays(dev, past):
    """lengths and offsets of any value reach nothing out of bounds"""
    rng = np.random.default_rng(15)
    p = Pair(dev, rng, [past, 10, 10], [4, 4, 4], 16, 2, 64)
    q = torch.randn(12, 128, device=dev)
    for lens, offsets in (([-5, 10 ** 9, 0], [0, 4, 8, 12]), ([0, 0, 0], [-9, -3, -3, -1]),
                          ([0, 0, 0], [12, 70, 10 ** 9, 5]), ([9, 9, 9], [0, 12, 0, 12]), ([2 ** 31 - 1, -2 ** 31, 7], [0, 12, 3, 40])):
        p.lens_t.copy_(_i32(lens, dev))
        p.offsets_t.copy_(_i32(offsets, dev))
        o = torch.empty_like(q)
        K.attn_paged(p.c, 2, q, o)
        torch.cuda.synchronize()


@pytest.mark.parametrize("inter", [False, True])
def test_a_sequence_token_by_token_and_as_a_prompt(dev, inter):
    """positions, cache and attention together, as a layer of a model uses them: a prompt,
    then tokens one by one, against the whole sequence in one call"""
    rng = np.random.default_rng(16)
    B, T, first, kvh, H, hd, page = 2, 150, 130, 2, 4, 64, 16
    r = K.Rope(K.rope_freqs(32, device=dev), inter)
    k, v, q = (_rows(rng, B * T, n, hd).reshape(B, T, -1) for n in (kvh, kvh, H))
    whole, steps = (Pair(dev, np.random.default_rng(17), [0] * B, [T] * B, page, kvh, hd, fill=0) for _ in range(2))

    def call(p, lens, a, b):
        n = b - a
        p.lens_t.fill_(lens)
        p.offsets_t.copy_(_i32([i * n for i in range(B + 1)], dev))
        x = [_cuda(t[:, a:b].reshape(B * n, -1), dev) for t in (k, v, q)]
        o = torch.empty_like(x[2])
        K.kv_append(p.c, x[0], x[1], r, H=H, q=x[2], q_out=x[2])
        K.attn_paged(p.c, H, x[2], o)
        return o.cpu().numpy().reshape(B, n, H, hd)

    call(steps, 0, 0, first)
    got = [call(steps, t, t, t + 1) for t in range(first, T)]
    pos = np.tile(np.arange(T), B)
    turn = lambda x, n: O.turned(x.reshape(B * T, n, hd), pos, O.freqs(32), inter)  # noqa: E731
    want = call(whole, 0, 0, T)
    for p in (whole, steps):
        for i, n in enumerate(("k", "v", "k_exp", "v_exp")):
            setattr(p.o, n, p.t[i].cpu().numpy())
    exact, tol = whole.o.attend(turn(q, H), [0] * B, [0, T, 2 * T], H)
    exact, tol = exact.reshape(B, T, H, hd), tol.reshape(B, T, H, hd)
    # (the turned query is off by 3 2^-24 of its pair besides: as much as 2^-22 of sum |q k|)
    assert (np.abs(want - exact) <= 2 * tol).all()
    exact, tol = steps.o.attend(turn(q, H), [0] * B, [0, T, 2 * T], H)
    exact, tol = exact.reshape(B, T, H, hd), tol.reshape(B, T, H, hd)
    # (the cache's page may have been rounded again since an earlier token read it: only the
    # last page's last token has read the cache as it is now)
    last = got[-1][:, 0]
    assert (np.abs(last - exact[:, -1]) <= 2 * tol[:, -1]).all()


def test_captured_step_replays_with_other_sequences(dev):
    rng = np.random.default_rng(18)
    lens, kvh, H, hd, page = [60, 3, 200], 2, 4, 64, 16
    p = Pair(dev, rng, lens, [10, 10, 10], page, kvh, hd)
    r = K.Rope(K.rope_freqs(hd, device=dev))
    p.offsets_t.copy_(_i32([0, 1, 2, 3], dev))
    k, v, q = (torch.randn(3, n * hd, device=dev) / 16 for n in (kvh, kvh, H))
    o, qr, o2 = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q)
    ws = torch.empty(K.attn_paged_workspace(p.c, 3, H), dtype=torch.uint8, device=dev)

    def step(out):
        K.kv_append(p.c, k, v, r, H=H, q=q, q_out=qr)
        K.attn_paged(p.c, H, qr, out, ws=ws)

    start = [t.clone() for t in p.t]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(o)
    for i in range(4):
        for t in (k, v, q):
            t.copy_(torch.randn_like(t) / 16)
        p.lens_t.copy_(_i32([60 + i, 3 + 2 * i, 200 - i], dev))
        if i == 2:
            p.offsets_t.copy_(_i32([0, 0, 2, 3], dev))
        for t, s in zip(p.t, start):
            t.copy_(s)
        o.zero_()
        graph.replay()
        pools = [t.clone() for t in p.t]
        for t, s in zip(p.t, start):
            t.copy_(s)
        o2.zero_()
        step(o2)
        assert torch.equal(o, o2)
        assert all(torch.equal(a, b) for a, b in zip(pools, p.t))


def test_two_streams_with_workspaces_of_their_own(dev):
    rng = np.random.default_rng(19)
    H = 8
    pairs = [Pair(dev, rng, [4000 + 9 * i, 100], [1, 1], 64, 2, 64) for i in range(2)]
    q = torch.randn(2, H * 64, device=dev) / 16
    want = []
    for p in pairs:
        o = torch.empty_like(q)
        K.attn_paged(p.c, H, q, o)
        want.append(o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in pairs]
    outs = [torch.empty_like(q) for _ in pairs]
    for _ in range(5):
        for s, p, o in zip(streams, pairs, outs):
            with torch.cuda.stream(s):
                K.attn_paged(p.c, H, q, o)
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("new,H", [(1, 8), (300, 16)])
def test_two_graphs_share_a_workspace(dev, new, H):
    """replayed in turn on a stream, each leaves the other nothing that it reads"""
    rng = np.random.default_rng(22)
    pairs = [Pair(dev, rng, [4000 + 900 * i, 130, 2500], [new, new, new], 64, 2, 64) for i in range(2)]
    q = torch.randn(3 * new, H * 64, device=dev) / 16
    size = [K.attn_paged_workspace(p.c, 3 * new, H) for p in pairs]
    assert min(size) > 0
    ws = torch.full((max(size),), 255, dtype=torch.uint8, device=dev)  # (NaN to begin with)
    outs, graphs = [torch.empty_like(q) for _ in pairs], []
    for p, o in zip(pairs, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            K.attn_paged(p.c, H, q, o, ws=ws)
    for i in range(3):
        q.copy_(torch.randn_like(q) / 16)
        for p in pairs:
            p.lens_t.copy_(_i32([3000 - 700 * i, 100 + i, 2500 - 64 * i], dev))
        for g in graphs:
            g.replay()
        for p, o in zip(pairs, outs):
            want = torch.empty_like(q)
            K.attn_paged(p.c, H, q, want)
            assert torch.equal(o, want)


def test_pages_shared_for_reading(dev):
    """sequences that begin alike read the same pages, and write to their own"""
    rng = np.random.default_rng(23)
    lens, new, kvh, H, hd, page = [64, 64, 64], [1, 20, 3], 2, 8, 64, 32
    p = Pair(dev, rng, lens, new, page, kvh, hd)
    p.o.table[1:, :2] = p.o.table[0, :2]
    p.upload()
    N = sum(new)
    k, v, q = (_rows(rng, N, n, hd) / 8 for n in (kvh, kvh, H))
    K.kv_append(p.c, _cuda(k.reshape(N, -1), dev), _cuda(v.reshape(N, -1), dev))
    p.o.append(k, v, lens, p.offsets)
    p.same()
    o = torch.empty(N, H * hd, device=dev)
    K.attn_paged(p.c, H, _cuda(q.reshape(N, -1), dev), o)
    want, tol = p.o.attend(q.astype(np.float64), lens, p.offsets, H)
    assert (np.abs(o.cpu().numpy().reshape(N, H, hd) - want) <= tol).all()


def test_offsets_past_32_bits(dev):
    """a cache of more than 2^32 bytes of keys, its last pages in use"""
    kvh, hd, page = 16, 256, 128
    pages = (1 << 32) // (kvh * hd * page) + 40
    k, v, ke, ve = K.kv_pool(pages, kvh, page, hd, dev)
    ke.fill_(127)
    ve.fill_(127)
    ids = [pages - 1, 3, pages - 2]
    for pool in (k, v):
        for i in ids:
            pool[i].fill_(0)
    table = _i32([ids], dev)
    c = K.PagedKV(k, v, ke, ve, table, _i32([0], dev), _i32([0, 300], dev), hd)
    g = torch.Generator(device=dev).manual_seed(20)
    kk, vv = (torch.randn(300, kvh * hd, device=dev, generator=g) for _ in range(2))
    K.kv_append(c, kk, vv)
    q = torch.randn(300, kvh * hd, device=dev, generator=g)
    o = torch.empty_like(q)
    K.attn_paged(c, kvh, q, o)

    def dense(pool, exps, turn):
        x = pool[ids].view(torch.float8_e4m3fn).double() * torch.exp2(exps[ids].double() - 127)[..., None, None]
        x = x.transpose(2, 3) if turn else x
        return x.transpose(0, 1).flatten(1, 2)[:, :300].contiguous()  # [heads, 300, hd]

    kd, vd = dense(k, ke, False), dense(v, ve, True)
    # every value within half a step of what was given: 2^-4 of it, or 2^-10 of the scale
    top = vv.view(300, kvh, hd).transpose(0, 1).double()
    assert ((vd - top).abs() <= top.abs() * 2.0 ** -4 + 2.0 ** -10 * 2.0 ** -6).all()
    qd = q.view(300, kvh, hd).transpose(0, 1).double()
    mask = torch.ones(300, 300, device=dev, dtype=torch.bool).triu(1)
    for h in (0, kvh - 1):
        s = (qd[h] @ kd[h].t().contiguous()) / 16
        want = torch.softmax(s.masked_fill(mask, -float("inf")), 1) @ vd[h]
        ds = (qd[h].abs() @ kd[h].abs().t().contiguous()).max() / 16 * (2.0 ** -22 + 260 * 2.0 ** -24)
        tol = (2 * ds + 2.0 ** -21 + 2 * 308 * 2.0 ** -24) * vd[h].abs().max()
        got = o.view(300, kvh, hd)[:, h].double()
        assert (got - want).abs().max() <= tol


def test_refused_by_the_bindings(dev):
    p = Pair(dev, np.random.default_rng(21), [4], [2], 16, 2, 64)
    k = torch.zeros(2, 128, device=dev)
    with pytest.raises(ValueError):
        K.kv_append(p.c, k[:, :64], k[:, :64])
    with pytest.raises(ValueError):
        K.kv_append(p.c, k, k[:1])
    with pytest.raises(ValueError):
        K.kv_append(p.c, k, k, H=2, q=k)
    with pytest.raises(ValueError):
        K.attn_paged(p.c, 3, k, k)
    with pytest.raises(PkError, match="heads"):
        K.attn_paged(p.c, 3, torch.zeros(2, 192, device=dev), torch.zeros(2, 192, device=dev))
    with pytest.raises(TypeError):
        K.attn_paged(p.c, 2, k.double(), k)
    far = K.PagedKV(*p.t[:4], torch.full((1, 4096), -1, device=dev, dtype=torch.int32), p.lens_t, p.offsets_t, 64)
    with pytest.raises(PkError, match="workspace"):
        K.attn_paged(far, 2, k, k.clone(), ws=torch.empty(16, dtype=torch.uint8, device=dev))
    t = p.t
    for bad in ([t[0][:, :1].contiguous()] + t[1:], [t[0], t[0]] + t[2:], t[:2] + [t[2][:1].contiguous()] + t[3:]):
        with pytest.raises(ValueError):
            K.PagedKV(*bad, p.lens_t, p.offsets_t, 64)
    with pytest.raises(ValueError):
        K.PagedKV(*t, p.lens_t, p.lens_t, 64)
    with pytest.raises(ValueError):
        K.PagedKV(*t, p.lens_t, p.offsets_t, 65)
    with pytest.raises(TypeError):
        K.PagedKV(*t, p.lens_t.long(), p.offsets_t, 64)


def _spare_page_0(p):
    """a Pair whose sequences do not use page 0, and pages behind every sequence's last that
    its table names already"""
    t, pages = p.o.table, p.o.k.shape[0]
    free = [i for i in range(pages) if i not in t]
    if 0 not in free:
        t[t == 0] = free[-1]
    free = [i for i in range(pages) if i not in t]
    for b in range(len(t)):
        behind = np.flatnonzero(t[b] < 0)
        t[b, behind[0]] = free[b % len(free)]
    return free


@pytest.mark.parametrize("byte", [255, 254, 0])
@pytest.mark.parametrize("lens,new,page,kvh,group,hd", [
    ([20, 3], [1, 1], 16, 2, 2, 64), ([40, 0, 17], [3, 0, 20], 32, 1, 4, 128), ([70], [5], 64, 1, 2, 256),
    # units shared out evenly
    ([2300, 700], [1, 1], 16, 1, 3, 96), ([2500], [2], 32, 2, 4, 32),
    # tiles of 128 rows, whole and in parts
    ([0], [650], 16, 2, 20, 64), ([2600], [260], 16, 1, 16, 64), ([1300], [140], 32, 1, 60, 256)])
def test_powers_of_pages_without_keys(dev, lens, new, page, kvh, group, hd, byte):
    """the exponents of pages that hold no key of a sequence may be anything: of the page that
    is read in an absent one's place, and of those named ahead"""
    rng = np.random.default_rng(24 + hd)
    p = Pair(dev, rng, lens, new, page, kvh, hd)
    for i in _spare_page_0(p):
        p.o.k_exp[i] = p.o.v_exp[i] = byte
    p.upload()
    N, H = int(p.offsets[-1]), kvh * group
    q = _rows(rng, N, H, hd)
    o = torch.full((N, H * hd), 5.0, device=dev)
    scale = hd ** -0.5 / 16
    K.attn_paged(p.c, H, _cuda(q.reshape(N, -1), dev), o, scale=scale)
    want, tol = p.o.attend(q.astype(np.float64), lens, p.offsets, H, scale)
    assert (np.abs(o.cpu().numpy().reshape(N, H, hd) - want) <= tol + 1e-30).all()


@pytest.mark.parametrize("new,H", [(1, 2), (150, 24)])
def test_powers_beyond_their_range(dev, new, H):
    """an exponent's byte beyond -40 and 40 counts as the nearest, for the attention and for
    tokens that join such a page"""
    rng = np.random.default_rng(25)
    lens, kvh, hd, page = [5, 300], 1, 64, 16
    p = Pair(dev, rng, lens, [new, new], page, kvh, hd, width=256)
    p.o.k_exp[p.o.table[0, 0]], p.o.v_exp[p.o.table[0, 0]] = 3, 255
    p.o.k_exp[p.o.table[1, 2]], p.o.v_exp[p.o.table[1, 2]] = 86, 168
    p.upload()
    for x in (p.o.k_exp, p.o.v_exp):
        x[...] = x.clip(87, 167)
    q = _rows(rng, 2 * new, H, hd) / 64
    o = torch.empty(2 * new, H * hd, device=dev)
    for _ in range(2):
        K.attn_paged(p.c, H, _cuda(q.reshape(2 * new, -1), dev), o)
        want, tol = p.o.attend(q.astype(np.float64), lens, p.offsets, H)
        assert (np.abs(o.cpu().numpy().reshape(want.shape) - want) <= tol + 1e-30).all()
        k, v = _rows(rng, 2 * new, kvh, hd), _rows(rng, 2 * new, kvh, hd)
        K.kv_append(p.c, _cuda(k.reshape(2 * new, -1), dev), _cuda(v.reshape(2 * new, -1), dev))
        p.o.append(k, v, lens, p.offsets)
    for i, x in ((0, p.o.k), (1, p.o.v)):
        np.testing.assert_array_equal(p.t[i].cpu().numpy(), x)


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("past,new,H", [(0, 1, 1), (40, 1, 3), (100, 20, 2), (3000, 1, 2), (0, 660, 40), (2600, 200, 32)])
def test_attention_of_scores_far_below_zero(dev, past, new, H, hd):
    """scores of -1e35 are scores: a single key's row is its value, and a row of equal keys,
    whose scores' last bits decide between them, lies between the values that it sees"""
    rng = np.random.default_rng(26)
    p = Pair(dev, rng, [past], [new], 16, 1, hd)
    p.o.k[..., :hd], p.o.k_exp[...], p.o.v_exp[...] = 0x38, 150, 120  # keys of 2^23
    p.upload()
    q = np.full((new, H, hd), -1e28, np.float32)
    o = torch.empty(new, H * hd, device=dev)
    K.attn_paged(p.c, H, _cuda(q.reshape(new, -1), dev), o, scale=1.0 / hd)
    v = p.o.dense(0, past + new, 0)[1]
    lo, hi = (f.accumulate(v)[past:, None] for f in (np.minimum, np.maximum))
    # numerator and denominator are sums of L terms of weights of 22 bits, and a division is
    # rounded
    tol = (2.0 ** -21 + 2 * (past + new + 8) * 2.0 ** -24) * np.maximum(np.abs(lo), np.abs(hi))
    got = o.cpu().numpy().reshape(new, H, hd)
    assert (got >= lo - tol).all() and (got <= hi + tol).all()


def test_a_cache_of_no_sequence(dev):
    """an empty batch: nothing is written, and rows of no sequence are left"""
    pool = K.kv_pool(2, 1, 16, 64, dev)
    for t in pool:
        t.fill_(7)
    c = K.PagedKV(*pool, torch.empty(0, 4, dtype=torch.int32, device=dev), _i32([], dev), _i32([0], dev), 64)
    x = torch.full((3, 64), 2.0, device=dev)
    K.kv_append(c, x, x)
    K.attn_paged(c, 1, torch.zeros_like(x), x)
    assert K.attn_paged_workspace(c, 3, 1) == 0
    assert (x == 2.0).all() and all((t == 7).all() for t in pool)


def _guarded(t, byte=0xa5, rows=64):
    """(t's copy in the middle of a larger tensor, that tensor)"""
    big = torch.full((t.shape[0] + 2 * rows, *t.shape[1:]), byte, dtype=t.dtype, device=t.device)
    big[rows:-rows] = t
    return big[rows:-rows], big


@pytest.mark.parametrize("new,width", [(4, 0), (4, 256), (50, 256)])  # tiles of 16 rows, shared ones, of 128
@pytest.mark.parametrize("lens,offsets", [((-5, 10 ** 9, 7), (0, 1, 2, 3)), ((0, 0, 0), (-9, -3, 2 / 3, 10 ** 9)),
                                          ((2, 30, 0), (1, 2, 2, 5 / 2)), ((0, 30, 0), (3, 70, 10 ** 9, 5)), ((9, 9, 9), (0, 3, 0, 3)),
                                          ((2 ** 31 - 1, -2 ** 31, 7), (0, 3, 1, 40))])
def test_bad_arrays_reach_nothing_else(dev, new, width, lens, offsets):
    """lengths and offsets of any value: what lies around the operands and between them stays
    as it is, and of offsets that do not decrease, rows inside the inputs come out right"""
    rng = np.random.default_rng(27)
    kvh, H, hd, page = 16, 32, 64, 16
    p = Pair(dev, rng, [40, 10, 23], [new] * 3, page, kvh, hd, width=width)
    N, cap = 3 * new, p.o.table.shape[1] * page
    offsets = [int(x * new) if abs(x) < 100 else x for x in offsets]  # (given in sequences' rows)
    pools = [_guarded(t) for t in p.t[:4]]
    p.t = [t for t, _ in pools] + p.t[4:]
    lens_t, offsets_t = _i32(lens, dev), _i32(offsets, dev)
    p.c = K.PagedKV(*p.t, lens_t, offsets_t, hd)
    row = np.clip(offsets[:-1], 0, N)
    n = np.clip(offsets[1:], row, N) - row
    past = np.clip(lens, 0, cap)
    rising = list(offsets) == sorted(offsets)
    mine = sorted({i for a, m in zip(row, n) for i in range(a, a + m)})  # rows of a sequence

    wide, out = (torch.full((N + 64, H * hd + 16), x, device=dev) for x in (float("nan"), 5.0))
    q, o = wide[32:-32, 8:-8], out[32:-32, 8:-8]
    qv = _rows(rng, N, H, hd) / 64
    q.copy_(_cuda(qv.reshape(N, -1), dev))
    K.attn_paged(p.c, H, q, o)
    got = o.cpu().numpy().reshape(N, H, hd)
    o[mine] = 5.0
    assert (out == 5.0).all()
    held = np.clip(offsets, 0, N)
    if rising:
        want, tol = p.o.attend(qv.astype(np.float64), past, held, H)
        assert (np.abs(got - want) <= tol)[mine].all()

    k, v = _rows(rng, N, kvh, hd), _rows(rng, N, kvh, hd)
    turned = torch.full_like(wide, 5.0)
    K.kv_append(p.c, _cuda(k.reshape(N, -1), dev), _cuda(v.reshape(N, -1), dev), None, H=H, q=q,
                q_out=turned[32:-32, 8:-8])
    inside = turned[32:-32, 8:-8]
    if rising:
        assert torch.equal(inside[mine], q[mine])
    inside[mine] = 5.0
    assert (turned == 5.0).all()
    for t, big in pools:
        assert (big[:64] == 0xa5).all() and (big[-64:] == 0xa5).all()
    if rising:
        p.o.append(k, v, past, held)
        p.same()
