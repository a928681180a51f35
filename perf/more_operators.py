"""Rotary positions, a paged 8-bit cache of keys and values, and the attention over it,
as cases to time and compare.

``run`` computes a case with elementary torch operations in float32 (the angles in
float64), or, where ``own`` is true, with the framework's calls over torch tensors
(``pico_amd.kernels``).  ``exact`` computes the same outputs in float64.  Sizes are those
of this repository's benchmark configurations (12 heads of 64, 8 sequences of 1024) or
generic ones.

The cache: ``k`` [pages, kv_heads, page, head] and ``v`` [pages, kv_heads, head, page] hold
e4m3 values (``head`` is the head size rounded up to 32, 64, 96, 128 or 256, with zeros
behind k's), ``k_exp`` and ``v_exp`` [pages, kv_heads] the powers of two that they are times,
as E8M0 bytes.  ``table`` [sequences, width] names each sequence's pages, ``lens`` the tokens
that it holds before the call, and rows ``offsets[b]`` to ``offsets[b + 1] - 1`` of the inputs
are its new tokens.
"""
import math
import random

import torch

DEV = "cuda:0"
E_MIN, E_MAX = -40, 40

own = False


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # positions, forward and backward: one token of each of 64 sequences
        {"name": "rope_token", "kind": "rope", "tokens": 64, "heads": 12, "hd": 64, "rot": 64,
         "interleaved": False, "scaling": "none", "far": 1024},
        # the benchmark model's training batch, queries and keys as one matrix
        {"name": "rope_train", "kind": "rope", "tokens": 8192, "heads": 24, "hd": 64, "rot": 64,
         "interleaved": False, "scaling": "none", "far": 1024},
        # a long document: half of each head turned, in neighbouring pairs, frequencies
        # scaled for a context 32 times the trained one
        {"name": "rope_long", "kind": "rope", "tokens": 16384, "heads": 32, "hd": 128, "rot": 64,
         "interleaved": True, "scaling": "parts", "far": 1 << 20},
        # cache: one token of each of 64 sequences being generated, with its queries turned
        {"name": "append_token", "kind": "append", "seqs": 64, "new": 1, "past": 2048,
         "heads": 32, "kv_heads": 8, "hd": 128, "rot": 128, "interleaved": False, "page": 64},
        # a few tokens each, of odd sizes, one sequence idle
        {"name": "append_odd", "kind": "append", "seqs": 13, "new": 9, "past": 700,
         "heads": 6, "kv_heads": 3, "hd": 80, "rot": 40, "interleaved": True, "page": 16},
        # four long prompts
        {"name": "append_prompt", "kind": "append", "seqs": 4, "new": 4096, "past": 100,
         "heads": 32, "kv_heads": 8, "hd": 128, "rot": 128, "interleaved": False, "page": 64},
        # attention: a token of each of 8 sequences of the benchmark model's length
        {"name": "attend_token", "kind": "attend", "seqs": 8, "new": 1, "past": 1023,
         "heads": 12, "kv_heads": 12, "hd": 64, "page": 64},
        # up to three tokens each, as a draft is verified, of odd sizes
        {"name": "attend_odd", "kind": "attend", "seqs": 13, "new": 3, "past": 1500,
         "heads": 20, "kv_heads": 4, "hd": 96, "page": 16},
        # a large serving batch: bound by the cache's bytes
        {"name": "attend_batch", "kind": "attend", "seqs": 64, "new": 1, "past": 8192,
         "heads": 32, "kv_heads": 8, "hd": 128, "page": 64},
        # one conversation with a very long past
        {"name": "attend_long", "kind": "attend", "seqs": 1, "new": 1, "past": 131071,
         "heads": 64, "kv_heads": 8, "hd": 128, "page": 128},
        # two prompts' chunks behind what the cache holds: bound by the products
        {"name": "attend_prompt", "kind": "attend", "seqs": 2, "new": 2048, "past": 6144,
         "heads": 32, "kv_heads": 8, "hd": 128, "page": 64},
        # a layer's step as a whole: the token goes into the cache and attends to it
        {"name": "step", "kind": "step", "seqs": 32, "new": 1, "past": 1024, "heads": 12,
         "kv_heads": 12, "hd": 64, "rot": 64, "interleaved": False, "page": 64},
    ]


def _log(rng, lo, hi):
    """a size between lo and hi, spread over the logarithm; odd as often as even"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend", "attend", "step"])
    hd = rng.choice([32, 64, 64, 96, 128, 128, 256, 2 * rng.randint(8, 128)])
    rot = hd if rng.random() < 0.6 else 2 * rng.randint(1, hd // 2)
    turn = {"rot": rot, "interleaved": rng.random() < 0.5}
    if kind == "rope":
        heads = _log(rng, 1, 64)
        return dict(turn, kind=kind, heads=heads, hd=hd, far=_log(rng, 16, 1 << 20),
                    tokens=_log(rng, 1, min(16384, (1 << 26) // (heads * hd))),
                    scaling=rng.choice(["none", "linear", "ntk", "parts"]))
    kv_heads = _log(rng, 1, 16)
    c = {"kind": kind, "kv_heads": kv_heads, "heads": kv_heads * _log(rng, 1, 8), "hd": hd,
         "page": rng.choice([16, 32, 64, 128])}
    if kind != "attend":
        c.update(turn)
    width = c["heads"] * hd
    c["seqs"] = _log(rng, 1, 64)
    if rng.random() < 0.6:
        c["new"] = rng.randint(1, 4)
    else:
        c["new"] = _log(rng, 1, max(1, min(4096, (1 << 24) // (width * c["seqs"]))))
    # the past within 2^28 values, and the products within the largest case's
    most = min(131072, (1 << 28) // (kv_heads * hd * c["seqs"]),
               (1 << 36) // (c["seqs"] * c["new"] * width))
    c["past"] = _log(rng, 1, max(1, most))
    return c


def _tokens(c):
    """(tokens held before, new tokens) of every sequence; the same for every seed"""
    r = random.Random(f"{c['seqs']} {c['new']} {c['past']}")
    n = c["seqs"]
    past = [c["past"] - (r.randrange(c["past"] // 2 + 1) if n > 1 else 0) for _ in range(n)]
    new = [c["new"] if c["new"] == 1 or c["new"] >= 64 else r.randint(1, c["new"])
           for _ in range(n)]
    if n >= 4 and c["new"] > 1:
        new[r.randrange(n)] = 0  # a sequence that waits
    return past, new


# ------------------------------------------------------------------- inputs
def _freqs(rot, scaling, far):
    """radians a position of the rot / 2 pairs; the scalings for a context of `far`
    tokens on frequencies made for 1/32 of it"""
    base, factor, length = 10000.0, 32.0, far / 32.0
    if scaling == "ntk" and rot > 2:
        base *= factor ** (rot / (rot - 2.0))
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "parts":
        # pairs that turn over 32 times in the trained length stay, those that turn less
        # than once are stretched
        keep = [min(1.0, max(0.0, (length * x / (2 * math.pi) - 1.0) / 31.0)) for x in f]
        f = [x * (g + (1.0 - g) / factor) for x, g in zip(f, keep)]
    return f


def _magnitude(scaling):
    return 0.1 * math.log(32.0) + 1.0 if scaling == "parts" else 1.0


def _head(hd):
    return next(h for h in (32, 64, 96, 128, 256) if hd <= h)


def _exponent(amax):
    """the smallest e with amax 2^-e <= 448, from -40 to 40"""
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8)
    return torch.where(amax > 0, e, E_MIN).clamp(E_MIN, E_MAX).to(torch.int32)


def _e4m3(x):
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    st = {"case": c}
    if c["kind"] == "rope":
        n, w = c["tokens"], c["heads"] * c["hd"]
        st.update(x=normal(n, w), dy=normal(n, w), y=torch.empty(n, w, device=DEV),
                  dx=torch.empty(n, w, device=DEV),
                  pos=torch.randint(0, c["far"], (n,), device=DEV, dtype=torch.int32, generator=g),
                  freqs=torch.tensor(_freqs(c["rot"], c["scaling"], c["far"]), device=DEV,
                                     dtype=torch.float64))
    else:
        past, new = _tokens(c)
        seqs, page, kvh, hd = c["seqs"], c["page"], c["kv_heads"], c["hd"]
        need = [-(-(p + n) // page) for p, n in zip(past, new)]
        total = sum(need) + 3
        free = torch.randperm(total, device=DEV, generator=g).to(torch.int32)
        width = max(need) + 1
        at = torch.cumsum(torch.tensor([0] + need), 0).to(DEV)
        col = torch.arange(width, device=DEV)
        used = col[None, :] < (at[1:] - at[:-1])[:, None]
        table = torch.where(used, free[(at[:-1, None] + col).clamp(max=total - 1)], -1)
        # some channels of the keys are larger than the rest, as they are in models
        gain = 1.0 + 3.0 * (torch.rand(kvh, hd, device=DEV, generator=g) > 0.95)
        k = torch.zeros(total, kvh, page, _head(hd), device=DEV, dtype=torch.uint8)
        v = torch.zeros(total, kvh, _head(hd), page, device=DEV, dtype=torch.uint8)
        x = normal(total, kvh, page, hd) * gain[:, None, :]
        ke = _exponent(x.abs().amax((2, 3)))
        k[..., :hd] = _e4m3(x * torch.exp2(-ke.float())[:, :, None, None])
        x = normal(total, kvh, hd, page)
        ve = _exponent(x.abs().amax((2, 3)))
        v[:, :, :hd] = _e4m3(x * torch.exp2(-ve.float())[:, :, None, None])
        del x
        n = sum(new)
        st.update(k_pool=k, v_pool=v, k_exp=(ke + 127).to(torch.uint8),
                  v_exp=(ve + 127).to(torch.uint8), table=table.contiguous(),
                  lens=torch.tensor(past, device=DEV, dtype=torch.int32),
                  offsets=torch.tensor([sum(new[:i]) for i in range(seqs + 1)], device=DEV,
                                       dtype=torch.int32),
                  q=normal(n, c["heads"] * hd), q_out=torch.empty(n, c["heads"] * hd, device=DEV),
                  o=torch.empty(n, c["heads"] * hd, device=DEV))
        if c["kind"] != "attend":
            st.update(k=(normal(n, kvh, hd) * gain).view(n, -1), v=normal(n, kvh * hd),
                      freqs=torch.tensor(_freqs(c["rot"], "none", 0), device=DEV,
                                         dtype=torch.float64))
    if own:
        _prepare_own(st)
    torch.cuda.synchronize()
    return st


# ----------------------------------------------------- plain torch operations
def _turned(x, hd, rot, interleaved, pos, freqs, magnitude=1.0, back=False):
    """x [n, heads * hd] with the first rot values of every head turned in pairs"""
    a = pos.double()[:, None] * freqs
    cos, sin = ((f(a) * magnitude).float()[:, None, :] for f in (torch.cos, torch.sin))
    if back:
        sin = -sin
    h = x.view(x.shape[0], -1, hd)
    r, rest = h[..., :rot], h[..., rot:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(2)
    else:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], 2)
    return torch.cat([r, rest], 2).view_as(x)


def _plain_rope(st):
    c = st["case"]
    args = c["hd"], c["rot"], c["interleaved"], st["pos"], st["freqs"], _magnitude(c["scaling"])
    return {"y": _turned(st["x"], *args), "dx": _turned(st["dy"], *args, back=True)}


def _rows(st):
    """(sequence, position) of every new token"""
    offsets = st["offsets"].long()
    row = torch.arange(st["q"].shape[0], device=DEV)
    seq = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
    return seq, st["lens"].long()[seq] + row - offsets[seq]


def _plain_put(pool, exps, x, pid, slot, transposed):
    """x [n, kv_heads, hd] into slots of pages: every page's exponent grows to what its
    new values need, and what it held already is rounded again where it does"""
    n, kvh, hd = x.shape
    pages = pool.shape[0]
    page = pool.shape[3 if transposed else 2]
    amax = torch.zeros(pages, kvh, device=DEV).scatter_reduce_(
        0, pid[:, None].expand(n, kvh), x.abs().amax(2), "amax")
    first = torch.full((pages,), page, device=DEV).scatter_reduce_(0, pid, slot, "amin")
    old = exps.to(torch.int32) - 127
    # a page whose first slot is written starts anew
    now = torch.maximum(torch.where(first[:, None] > 0, old, E_MIN), _exponent(amax))
    now = torch.where(first[:, None] < page, now, old)
    grown = torch.nonzero((first > 0) & (now > old).any(1)).view(-1)
    shift = torch.exp2((old - now)[grown].float())[:, :, None, None]
    held = torch.arange(page, device=DEV) < first[grown, None]
    held = held[:, None, None, :] if transposed else held[:, None, :, None]
    codes = pool[grown]
    again = _e4m3(codes.view(torch.float8_e4m3fn).float() * shift)
    pool[grown] = torch.where(held, again, codes)
    exps.copy_((now + 127).to(torch.uint8))
    codes = _e4m3(x * torch.exp2(-now[pid].float())[:, :, None])
    if transposed:
        pool[pid, :, :hd, slot] = codes
    else:
        pool[pid, :, slot, :hd] = codes


def _plain_append(st):
    c = st["case"]
    seq, pos = _rows(st)
    pid = st["table"].long()[seq, pos // c["page"]]
    slot = pos % c["page"]
    turn = c["hd"], c["rot"], c["interleaved"], pos, st["freqs"]
    shape = -1, c["kv_heads"], c["hd"]
    _plain_put(st["k_pool"], st["k_exp"], _turned(st["k"], *turn).view(shape), pid, slot, False)
    _plain_put(st["v_pool"], st["v_exp"], st["v"].view(shape), pid, slot, True)
    return _turned(st["q"], *turn)


def _pools(st):
    """the cache as the values that its bytes stand for"""
    return {"k": st["k_pool"].view(torch.float8_e4m3fn),
            "v": st["v_pool"].view(torch.float8_e4m3fn),
            "k_scale": st["k_exp"].view(torch.float8_e8m0fnu),
            "v_scale": st["v_exp"].view(torch.float8_e8m0fnu)}


def _plain_attend(st, q):
    c = st["case"]
    hd, kvh, group = c["hd"], c["kv_heads"], c["heads"] // c["kv_heads"]
    seqs, most = c["seqs"], max(_tokens(c)[1])
    pages = st["table"].long().clamp(min=0)
    width = pages.shape[1] * c["page"]

    def dense(pool, exps):  # [seqs, width / page, kv_heads, ., .]
        scale = torch.exp2(exps.float() - 127)[:, :, None, None]
        return pool[pages].view(torch.float8_e4m3fn).float() * scale[pages]

    k = dense(st["k_pool"][..., :hd], st["k_exp"]).transpose(1, 2).reshape(seqs, kvh, width, hd)
    v = dense(st["v_pool"][:, :, :hd], st["v_exp"]).permute(0, 2, 1, 4, 3)
    v = v.reshape(seqs, kvh, width, hd)
    # the new tokens of every sequence, padded to the most that one has
    i = torch.arange(most, device=DEV)
    offsets = st["offsets"].long()
    real = i < (offsets[1:] - offsets[:-1])[:, None]
    row = (offsets[:-1, None] + i).clamp(max=q.shape[0] - 1)
    rows = q[row].view(seqs, most, kvh, group, hd).permute(0, 2, 1, 3, 4)
    s = rows.reshape(seqs, kvh, most * group, hd) @ k.transpose(2, 3).contiguous()
    s *= hd ** -0.5
    reach = st["lens"].long()[:, None] + i  # the last key that a token sees
    seen = torch.arange(width, device=DEV) <= reach[:, :, None]
    seen = seen[:, None, :, None].expand(seqs, 1, most, group, width).flatten(2, 3)
    s.masked_fill_(~seen, -math.inf)
    p = s.sub_(s.amax(3, keepdim=True)).exp_()
    o = (p @ v) / p.sum(3, keepdim=True)
    o = o.view(seqs, kvh, most, group, hd).transpose(1, 2).reshape(seqs, most, -1)
    return o[real]


# ------------------------------------------------------ the framework's calls
def _prepare_own(st):
    from pico_amd import kernels as K

    c = st["case"]
    if c["kind"] == "rope":
        st["rope"] = K.Rope(K.rope_freqs(c["rot"], 10000.0, c["scaling"], factor=32.0,
                                         length=c["far"] / 32.0, low=1.0, high=32.0, device=DEV),
                            c["interleaved"], _magnitude(c["scaling"]))
        return
    st["cache"] = K.PagedKV(st["k_pool"], st["v_pool"], st["k_exp"], st["v_exp"], st["table"],
                            st["lens"], st["offsets"], c["hd"])
    if c["kind"] != "attend":
        st["rope"] = K.Rope(K.rope_freqs(c["rot"], 10000.0, device=DEV), c["interleaved"])
    if c["kind"] != "append":
        need = K.attn_paged_workspace(st["cache"], st["q"].shape[0], c["heads"])
        st["ws"] = torch.empty(max(1, need), device=DEV, dtype=torch.uint8)


def _run_own(st):
    from pico_amd import kernels as K

    c = st["case"]
    if c["kind"] == "rope":
        K.rope(st["rope"], c["heads"], st["x"], st["pos"], st["y"])
        K.rope(st["rope"], c["heads"], st["dy"], st["pos"], st["dx"], backward=True)
        return {"y": st["y"], "dx": st["dx"]}
    q = st["q"]
    if c["kind"] != "attend":
        K.kv_append(st["cache"], st["k"], st["v"], st["rope"], H=c["heads"], q=q,
                    q_out=st["q_out"])
        q = st["q_out"]
    if c["kind"] == "append":
        return dict(_pools(st), q=q)
    K.attn_paged(st["cache"], c["heads"], q, st["o"], ws=st["ws"])
    return {"o": st["o"]} if c["kind"] == "attend" else dict(_pools(st), o=st["o"])


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "rope":
        return _plain_rope(state)
    if kind == "attend":
        return {"o": _plain_attend(state, state["q"])}
    q = _plain_append(state)
    if kind == "append":
        return dict(_pools(state), q=q)
    return dict(_pools(state), o=_plain_attend(state, q))


# ------------------------------------------------------------- work and exact
def work(case):
    c = case
    if c["kind"] == "rope":
        n = c["tokens"] * c["heads"]
        # x and dy read, y and dx written; the positions
        return {"bytes": 4 * (4 * n * c["hd"] + 2 * c["tokens"]), "flops": 6 * n * c["rot"]}
    past, new = _tokens(c)
    n, hd, kvh, heads = sum(new), c["hd"], c["kv_heads"], c["heads"]
    put = n * hd * (2 * 4 * kvh + 2 * kvh + 8 * heads), 3 * n * c.get("rot", 0) * (heads + kvh)
    if c["kind"] == "append":
        return {"bytes": put[0], "flops": put[1]}
    # the cache's bytes up to every sequence's last token, q read and o written
    held = sum(p + m for p, m in zip(past, new) if m)
    bytes_ = 2 * held * kvh * hd + 8 * n * heads * hd
    flops = 4 * hd * heads * sum(p * m + m * (m + 1) // 2 for p, m in zip(past, new))
    if c["kind"] == "attend":
        return {"bytes": bytes_, "flops": flops}
    return {"bytes": bytes_ + put[0], "flops": flops + put[1]}


def _exact_turned(x, hd, rot, interleaved, pos, freqs, magnitude=1.0, back=False):
    """as a product of complex numbers"""
    a = pos.double()[:, None, None] * freqs
    w = torch.polar(torch.full_like(a, magnitude), -a if back else a)
    h = x.double().view(x.shape[0], -1, hd).clone()
    if interleaved:
        z = torch.view_as_complex(h[..., :rot].reshape(*h.shape[:2], rot // 2, 2).contiguous()) * w
        h[..., :rot] = torch.view_as_real(z).flatten(2)
    else:
        z = torch.complex(h[..., :rot // 2], h[..., rot // 2:rot]) * w
        h[..., :rot // 2], h[..., rot // 2:rot] = z.real, z.imag
    return h.view(x.shape)


def _exact_append(st):
    """page by page along every sequence; the values before their rounding to 8 bits have
    no other form, so k and v are rounded here too, from 64 bits"""
    c = st["case"]
    page, kvh, hd = c["page"], c["kv_heads"], c["hd"]
    past, new = _tokens(c)
    at = st["offsets"].tolist()
    pos = torch.cat([torch.arange(p, p + n) for p, n in zip(past, new)]).to(DEV)
    turn = hd, c["rot"], c["interleaved"], pos, st["freqs"]
    out = {"q": _exact_turned(st["q"], *turn)}
    src = {"k": _exact_turned(st["k"], *turn).view(-1, kvh, hd),
           "v": st["v"].double().view(-1, kvh, hd)}
    table = st["table"].tolist()
    for name, x in src.items():
        pool = st[name + "_pool"].view(torch.float8_e4m3fn).double()
        scale = torch.exp2(st[name + "_exp"].double() - 127)
        for b in range(c["seqs"]):
            p, end = past[b], past[b] + new[b]
            while p < end:
                to = min(end, (p // page + 1) * page)
                pid, s0, s1 = table[b][p // page], p % page, (to - 1) % page + 1
                rows = x[at[b] + p - past[b]:at[b] + to - past[b]].transpose(0, 1)
                top = torch.exp2(torch.ceil(torch.log2(
                    rows.abs().amax((1, 2)).clamp(min=2.0 ** -60) / 448))).clamp(2.0 ** E_MIN)
                if s0:
                    top = torch.maximum(top, scale[pid])
                    body = pool[pid, :, :s0] if name == "k" else pool[pid, :, :, :s0]
                    body.copy_(_round(body * (scale[pid] / top)[:, None, None]))
                scale[pid] = top
                codes = _round(rows / top[:, None, None])
                if name == "k":
                    pool[pid, :, s0:s1, :hd] = codes
                else:
                    pool[pid, :, :hd, s0:s1] = codes.transpose(1, 2)
                p = to
        out[name], out[name + "_scale"] = pool, scale
    return out


def _round(x):
    """to the nearest of e4m3's values, ties to even: 3 bits behind the first, down to 2^-9"""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_attend(st, q, k, v, k_scale, v_scale):
    c = st["case"]
    hd, kvh, group = c["hd"], c["kv_heads"], c["heads"] // c["kv_heads"]
    past, new = _tokens(c)
    at = st["offsets"].tolist()
    out = torch.empty(q.shape, device=DEV, dtype=torch.float64)
    for b in range(c["seqs"]):
        n, length = new[b], past[b] + new[b]
        if not n:
            continue
        pages = st["table"][b, :-(-length // c["page"])].long()
        mask = torch.arange(length, device=DEV) > torch.arange(past[b], length, device=DEV)[:, None]
        rows = q[at[b]:at[b] + n].view(n, kvh, group, hd)
        o = out[at[b]:at[b] + n].view(n, kvh, group, hd)
        for h in range(kvh):
            keys = (k(pages, h) * k_scale[pages, h, None, None]).flatten(0, 1)[:length, :hd]
            values = (v(pages, h) * v_scale[pages, h, None, None]).transpose(1, 2)
            values = values.flatten(0, 1)[:length, :hd]
            for j in range(group):
                s = (rows[:, h, j] @ keys.t()) / math.sqrt(hd)
                o[:, h, j] = torch.softmax(s.masked_fill_(mask, -math.inf), 1) @ values
    return out


def exact(case, seed):
    global own
    mine, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = mine
    c = case
    if c["kind"] == "rope":
        turn = c["hd"], c["rot"], c["interleaved"], st["pos"], st["freqs"], _magnitude(c["scaling"])
        return {"y": _exact_turned(st["x"], *turn), "dx": _exact_turned(st["dy"], *turn, back=True)}
    if c["kind"] != "attend":
        out = _exact_append(st)
        if c["kind"] == "append":
            return out
        q = out.pop("q")
        out["o"] = _exact_attend(st, q, lambda p, h: out["k"][p, h], lambda p, h: out["v"][p, h],
                                 out["k_scale"], out["v_scale"])
        return out

    def values(pool):
        return lambda p, h: pool[p, h].view(torch.float8_e4m3fn).double()

    return {"o": _exact_attend(st, st["q"].double(), values(st["k_pool"]), values(st["v_pool"]),
                               torch.exp2(st["k_exp"].double() - 127),
                               torch.exp2(st["v_exp"].double() - 127))}
