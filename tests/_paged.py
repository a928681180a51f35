"""Rotary positions, a paged e4m3 cache and the attention over it in float64, token by
token, for the tests of the kernels: numpy, no code shared with the library."""
import math

import numpy as np

CODES = np.zeros(256)
for _c in range(256):
    _e, _m = (_c >> 3) & 15, _c & 7
    CODES[_c] = (1 + _m / 8) * 2.0 ** (_e - 7) if _e else _m / 8 * 2.0 ** -6
    if _c & 127 == 127:
        CODES[_c] = np.nan
    if _c & 128:
        CODES[_c] = -CODES[_c]
FINITE = CODES[:127]  # 0 to 448, in order


def head_size(hd):
    return next(h for h in (32, 64, 96, 128, 256) if hd <= h)


def encode(x):
    """e4m3 codes of x, to nearest, ties to the even code; held to 448; NaN is 0x7f"""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(np.nan_to_num(x, nan=0.0, posinf=1e9, neginf=-1e9)), 448.0)
    hi = np.clip(np.searchsorted(FINITE, a), 1, 126)
    lo = hi - 1
    up = a - FINITE[lo]
    down = FINITE[hi] - a
    code = np.where((up > down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(np.isnan(x), 127, code | np.where(np.signbit(x), 128, 0))
    return code.astype(np.uint8)


def exponent(x):
    """the smallest e of -40 to 40 with every finite |x| <= 448 2^e"""
    a = np.abs(x[np.isfinite(x)])
    top = a.max() if a.size else 0.0
    e = -40
    while e < 40 and top > 448.0 * 2.0 ** e:
        e += 1
    return e


def freqs(rot, base=10000.0):
    return np.array([base ** (-2.0 * i / rot) for i in range(rot // 2)])


def turned(x, pos, f, interleaved=False, magnitude=1.0, back=False):
    """x [N, H, hd] with the first 2 len(f) values of every head turned by pos [N]"""
    y = np.array(x, np.float64)
    n = len(f)
    a = np.asarray(pos, np.float64)[:, None] * f
    c, s = magnitude * np.cos(a)[:, None], magnitude * np.sin(a)[:, None]
    if back:
        s = -s
    i1 = np.arange(n) * 2 if interleaved else np.arange(n)
    i2 = i1 + 1 if interleaved else i1 + n
    x1, x2 = y[..., i1].copy(), y[..., i2].copy()
    y[..., i1], y[..., i2] = x1 * c - x2 * s, x2 * c + x1 * s
    return y


class Cache:
    """the cache as numpy arrays, and what the calls do to it"""

    def __init__(self, pages, kv_heads, page, hd, table):
        self.hp, self.hd, self.page, self.kvh = head_size(hd), hd, page, kv_heads
        self.k = np.zeros((pages, kv_heads, page, self.hp), np.uint8)
        self.v = np.zeros((pages, kv_heads, self.hp, page), np.uint8)
        self.k_exp = np.full((pages, kv_heads), 127, np.uint8)
        self.v_exp = np.full((pages, kv_heads), 127, np.uint8)
        self.table = np.asarray(table)

    def _page(self, b, p):
        i = p // self.page
        pid = self.table[b, i] if i < self.table.shape[1] else -1
        return pid if 0 <= pid < self.k.shape[0] else -1

    def append(self, k, v, lens, offsets):
        """k (turned already), v [N, kv_heads, hd] at every sequence's next positions"""
        for b in range(len(lens)):
            start, n = offsets[b], offsets[b + 1] - offsets[b]
            p = lens[b]
            while p < lens[b] + n:
                to = min(lens[b] + n, (p // self.page + 1) * self.page)
                pid, s0, s1 = self._page(b, p), p % self.page, (to - 1) % self.page + 1
                rows = slice(start + p - lens[b], start + to - lens[b])
                p = to
                if pid < 0:
                    continue
                for h in range(self.kvh):
                    for x, pool, exps, turn in ((k, self.k, self.k_exp, False),
                                                (v, self.v, self.v_exp, True)):
                        new = np.asarray(x[rows, h], np.float64)
                        body = pool[pid, h].T if turn else pool[pid, h]  # [page, hp], a view
                        old = int(exps[pid, h]) - 127 if s0 else -40
                        e = max(old, exponent(new))
                        if s0 and e > old:
                            body[:s0, :self.hd] = encode(CODES[body[:s0, :self.hd]] * 2.0 ** (old - e))
                        body[s0:s1, :self.hd] = encode(new * 2.0 ** -e)
                        if not turn:
                            body[s0:s1, self.hd:] = 0
                        exps[pid, h] = e + 127

    def dense(self, b, length, h):
        """(keys, values, present, the values' scale) of one sequence's first `length` tokens
        of a head"""
        k, v, scale = np.zeros((length, self.hd)), np.zeros((length, self.hd)), np.zeros(length)
        here = np.zeros(length, bool)
        for p in range(length):
            pid = self._page(b, p)
            if pid < 0:
                continue
            here[p] = True
            scale[p] = 2.0 ** (int(self.v_exp[pid, h]) - 127)
            k[p] = CODES[self.k[pid, h, p % self.page, :self.hd]] * 2.0 ** (int(self.k_exp[pid, h]) - 127)
            v[p] = CODES[self.v[pid, h, :self.hd, p % self.page]] * scale[p]
        return k, v, here, scale

    def attend(self, q, lens, offsets, H, scale=None):
        """(o [N, H, hd], how far fp32 products of 22-bit operands may be off): a score is
        off by (2^-22 for q's two parts + (hd + 4) 2^-24 for the sum, its scale and its
        exponent) of scale sum |q k|; a probability by that and 2^-21 for its parts, the
        exponential and the ones it is relative to; and the weighted sum of L values by
        (L + 8) 2^-24 of sum p |v|, numerator and denominator alike.  A small probability's
        second part is rounded to a step of 2^-24 where the largest probability times its
        page's scale is at least 2^7: off by 2^-32 of that, times a code of up to 448, for
        each of the L"""
        group, scale = H // self.kvh, self.hd ** -0.5 if scale is None else scale
        cap = self.table.shape[1] * self.page
        o, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
        for b in range(len(lens)):
            n = offsets[b + 1] - offsets[b]
            if not n:
                continue
            length = min(lens[b] + n, cap)
            for h in range(self.kvh):
                k, v, here, vscale = self.dense(b, length, h)
                for j in range(h * group, (h + 1) * group):
                    for i in range(n):
                        r = offsets[b] + i
                        see = here & (np.arange(length) <= lens[b] + i)
                        if not see.any():
                            o[r, j] = 0.0
                            continue
                        ks, vs = k[see], v[see]
                        s = ks @ q[r, j] * scale
                        p = np.exp(s - s.max())
                        p /= p.sum()
                        o[r, j] = p @ vs
                        ds = np.abs(ks) @ np.abs(q[r, j]) * scale * (2.0 ** -22 + (self.hd + 4) * 2.0 ** -24)
                        rel = 2.0 * ds.max() + 2.0 ** -21 + 2.0 * (see.sum() + 8) * 2.0 ** -24
                        tol[r, j] = rel * (p @ np.abs(vs)) + see.sum() * 2.0 ** -32 * 448 * (p * vscale[see]).max()
        return o, tol


def layout(lens, new, page, pages, rng, extra=1):
    """(table [B, width] of distinct pages, -1 behind them; offsets)"""
    need = [-(-(a + n) // page) for a, n in zip(lens, new)]
    assert sum(need) <= pages
    ids = list(rng.permutation(pages)[:sum(need)])
    table = np.full((len(lens), max(need + [1]) + extra), -1, np.int32)
    for b, n in enumerate(need):
        table[b, :n] = ids[:n]
        ids = ids[n:]
    return table, np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
