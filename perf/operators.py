"""The layer norm, gated recurrence and expert operators, as cases to time and compare.

``run`` computes a case with elementary torch operations in float32, or, where
``own`` is true, with the framework's calls: the launchers over torch tensors
(``pico_amd.kernels``) and pico's C API (``pico_amd.pico``).  ``exact`` computes
the same outputs in float64.  Sizes are those of this repository's benchmark
configurations (d_model 768, d_ff 2048, 8 sequences of 1024) or generic ones.
"""
import ctypes
import math

import torch

DEV = "cuda:0"
EPS = 1e-5

own = False


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # layer norm, forward and backward with the gain's and bias's gradients:
        # a small layer's batch, where launches count
        {"name": "layernorm_small", "kind": "layernorm", "rows": 64, "cols": 128},
        # sizes that are no multiple of anything
        {"name": "layernorm_odd", "kind": "layernorm", "rows": 2000, "cols": 1503},
        # a large model's activations
        {"name": "layernorm_large", "kind": "layernorm", "rows": 8192, "cols": 4096},
        # gated recurrence: one token of each of 64 sequences being generated
        {"name": "scan_token", "kind": "scan", "batch": 64, "seq": 1, "cols": 768,
         "backward": False},
        # the benchmark model's training batch, forward and backward
        {"name": "scan_train", "kind": "scan", "batch": 8, "seq": 1024, "cols": 768,
         "backward": True},
        # odd sizes
        {"name": "scan_odd", "kind": "scan", "batch": 3, "seq": 1001, "cols": 333,
         "backward": True},
        # one long document: few channels, all the work along the sequence
        {"name": "scan_long", "kind": "scan", "batch": 1, "seq": 65536, "cols": 512,
         "backward": True},
        # top-2 routing over many experts with its gradient, and the grouping of
        # the rows by expert
        {"name": "route", "kind": "route", "tokens": 8192, "experts": 64, "topk": 2},
        # a feed-forward of 8 experts on a few tokens being generated: bound by
        # the weights' bytes
        {"name": "experts_token", "kind": "experts", "tokens": 16, "d": 768, "ff": 2048,
         "experts": 8, "topk": 2},
        # products grouped by expert and both their gradients, odd sizes and one
        # expert without rows
        {"name": "product_odd", "kind": "product", "rows": 2000, "k": 333, "n": 517,
         "experts": 5, "precision": "fp32"},
        # the gate and up projection of 8 experts, bf16 multiplies
        {"name": "product_bf16", "kind": "product", "rows": 16384, "k": 768, "n": 4096,
         "experts": 8, "precision": "bf16"},
        # a training step's mixture-of-experts layer on the benchmark model's
        # batch, forward and backward through pico's API
        {"name": "moe_train", "kind": "moe", "tokens": 8192, "d": 768, "ff": 2048,
         "experts": 8, "topk": 2},
    ]


def _log(rng, lo, hi):
    """a size between lo and hi, spread over the logarithm; odd as often as even"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["layernorm", "scan", "scan", "route", "experts", "product", "product", "moe"])
    if kind == "layernorm":
        step = rng.choice([1, 4, 64])
        return {"kind": kind, "rows": _log(rng, 1, 8192),
                "cols": max(step, _log(rng, 64, 4096) // step * step)}
    if kind == "scan":
        if rng.random() < 0.25:
            return {"kind": kind, "batch": _log(rng, 1, 1024), "seq": rng.randint(1, 4),
                    "cols": _log(rng, 64, 4096), "backward": False}
        step = rng.choice([1, 4, 64])
        cols = max(step, _log(rng, 64, 2048) // step * step)
        seq = _log(rng, 2, min(65536, (1 << 25) // cols))
        return {"kind": kind, "batch": _log(rng, 1, max(1, min(64, (1 << 25) // (cols * seq)))),
                "seq": seq, "cols": cols, "backward": True}
    if kind == "route":
        experts = _log(rng, 2, 256)
        return {"kind": kind, "tokens": _log(rng, 1, 16384), "experts": experts,
                "topk": rng.randint(1, min(8, experts))}
    if kind == "product":
        step = rng.choice([1, 4, 64])
        return {"kind": kind, "rows": _log(rng, 1, 16384),
                "k": max(step, _log(rng, 32, 768) // step * step),
                "n": max(step, _log(rng, 32, 4096) // step * step), "experts": _log(rng, 1, 64),
                "precision": rng.choice(["fp32", "fp32", "bf16"])}
    experts = _log(rng, 2, 32)
    layer = {"kind": kind, "d": 4 * _log(rng, 16, 192), "ff": 4 * _log(rng, 16, 512),
             "experts": experts, "topk": rng.randint(1, min(4, experts))}
    most = 64 if kind == "experts" else 16384 // layer["topk"]
    return dict(layer, tokens=_log(rng, 1, most))


# ------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _logits(tokens, experts, topk, normal):
    """router logits with a preference among the experts, so that their loads are
    uneven; where experts are to spare some are masked for a token, and one token
    in 64 is padding (every expert masked)"""
    z = normal(tokens, experts, std=1.5) + normal(experts)
    t = torch.arange(tokens, device=DEV)
    z[t % 64 == 63] = -math.inf
    if experts >= 4 * topk:
        e = torch.arange(experts, device=DEV)
        z[(t[:, None] + 3 * e[None, :]) % 7 == 0] = -math.inf
    return z


def prepare(case, seed):
    c, g = case, _gen(seed)
    kind = c["kind"]
    st = {"case": c}

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, device=DEV, generator=g) * std + mean

    if kind == "layernorm":
        r, n = c["rows"], c["cols"]
        st.update(x=normal(r, n) + normal(r, 1, std=0.5), gain=normal(n, std=0.02, mean=1.0),
                  bias=normal(n, std=0.02), dy=normal(r, n))
    elif kind == "scan":
        b, t, n = c["batch"], c["seq"], c["cols"]
        # channels remember between a few and some hundred tokens
        rate = torch.rand(n, device=DEV, generator=g) * 5
        st.update(x=normal(b * t, n), f=normal(b * t, n) + rate, h0=normal(b, n, std=0.5))
        if c["backward"]:
            st["dh"] = normal(b * t, n)
    elif kind == "route":
        st.update(logits=_logits(c["tokens"], c["experts"], c["topk"], normal),
                  dgates=normal(c["tokens"], c["topk"]))
    elif kind == "product":
        n, e = c["rows"], c["experts"]
        share = torch.rand(e, device=DEV, generator=g) ** 2 + 1e-3
        if e > 2:
            share[e // 2] = 0.0  # an expert that no row chose
        edges = torch.round(torch.cumsum(share, 0) / share.sum() * n).to(torch.int32)
        edges[-1] = n
        st.update(offsets=torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), edges]),
                  x=normal(n, c["k"]), w=normal(e, c["k"], c["n"], std=c["k"] ** -0.5),
                  dy=normal(n, c["n"]))
    else:
        t, d, f, e = c["tokens"], c["d"], c["ff"], c["experts"]
        st.update(x=normal(t, d), logits=_logits(t, e, c["topk"], normal),
                  w13=normal(e, d, 2 * f, std=d ** -0.5), w2=normal(e, f, d, std=f ** -0.5))
    if own:
        _prepare_own(st)
    torch.cuda.synchronize()
    return st


# ----------------------------------------------------- plain torch operations
def _plain_layernorm(st):
    x, gain, dy = st["x"], st["gain"], st["dy"]
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + EPS)
    xh = xc * rstd
    y = xh * gain + st["bias"]
    gd = dy * gain
    dx = rstd * (gd - gd.mean(1, keepdim=True) - xh * (gd * xh).mean(1, keepdim=True))
    return {"y": y, "dx": dx, "dgain": (dy * xh).sum(0), "dbias": dy.sum(0)}


def _doubling(a, b):
    """y_t = a_t y_{t-1} + b_t along dim 1 with y_{-1} = 0, in log2(T) passes"""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _plain_scan(st):
    c = st["case"]
    shape = (c["batch"], c["seq"], c["cols"])
    x, f, h0 = st["x"].view(shape), st["f"].view(shape), st["h0"]
    s, r = 1.0 / (1.0 + torch.exp(-f)), 1.0 / (1.0 + torch.exp(f))
    b = r * x
    b[:, 0] += s[:, 0] * h0
    h = _doubling(s, b)
    out = {"h": h.view(-1, c["cols"])}
    if not c["backward"]:
        return out
    dh = st["dh"].view(shape)
    after = torch.cat([s[:, 1:], torch.zeros_like(s[:, :1])], 1)
    grad = _doubling(after.flip(1), dh.flip(1)).flip(1)
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    return dict(out, dx=(r * grad).reshape(-1, c["cols"]),
                df=(grad * (before - x) * s * r).reshape(-1, c["cols"]), dh0=s[:, 0] * grad[:, 0])


def _plain_topk(z, k):
    """(experts, gates): the k largest of each row, the lowest index first among
    equals, -inf never; and the softmax of the chosen"""
    z = z.clone()
    columns = torch.arange(z.shape[1], device=z.device)
    chosen, values = [], []
    for _ in range(k):
        top = z.amax(1, keepdim=True)
        at = torch.where(z == top, columns, z.shape[1]).amin(1)
        chosen.append(torch.where(top[:, 0] > -math.inf, at, -1))
        values.append(top[:, 0])
        z[columns == at[:, None]] = -math.inf
    values = torch.stack(values, 1)
    w = torch.where(values > -math.inf, torch.exp(values - values[:, :1]), 0.0)
    total = w.sum(1, keepdim=True)
    return torch.stack(chosen, 1).to(torch.int32), w / torch.where(total > 0, total, 1.0)


def _plain_plan(experts, count):
    """the slots in expert order: (offsets, order, place)"""
    flat = experts.reshape(-1).long()
    key = torch.where(flat < 0, count, flat)
    order = torch.sort(key, stable=True).indices
    edges = torch.cumsum((key[:, None] == torch.arange(count, device=key.device)).sum(0), 0)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    place = torch.where(flat < 0, -1, place)
    offsets = torch.cat([torch.zeros_like(edges[:1]), edges])
    return tuple(t.to(torch.int32) for t in (offsets, order, place))


def _plain_route(st):
    c = st["case"]
    experts, gates = _plain_topk(st["logits"], c["topk"])
    offsets, order, place = _plain_plan(experts, c["experts"])
    dg = st["dgates"]
    dz = gates * (dg - (gates * dg).sum(1, keepdim=True))
    dlogits = torch.zeros(c["tokens"], c["experts"] + 1, device=DEV)
    dlogits.scatter_add_(1, torch.where(experts < 0, c["experts"], experts).long(),
                         torch.where(experts < 0, 0.0, dz))
    return {"experts": experts, "gates": gates, "offsets": offsets, "order": order, "place": place,
            "dlogits": dlogits[:, :-1].contiguous()}


def _grouped(x, w, edges):
    return torch.cat([x[a:b] @ w[e] for e, (a, b) in enumerate(zip(edges, edges[1:]))])


def _plain_product(st):
    c = st["case"]
    x, w, dy = st["x"], st["w"], st["dy"]
    if c["precision"] == "bf16":
        x, w, dy = (t.bfloat16().float() for t in (x, w, dy))
    edges = st["offsets"].tolist()
    return {"y": _grouped(x, w, edges), "dx": _grouped(dy, w.transpose(1, 2), edges),
            "dw": torch.stack([x[a:b].t() @ dy[a:b] for a, b in zip(edges, edges[1:])])}


def _plain_layer(st, backward):
    c = st["case"]
    x, k, d = st["x"], c["topk"], c["d"]
    experts, gates = _plain_topk(st["logits"], k)
    offsets, order, place = _plain_plan(experts, c["experts"])
    edges = offsets.tolist()
    order, place = order.long()[:edges[-1]], place.long()
    xs = x[order // k]
    gu = _grouped(xs, st["w13"], edges)
    gate, up = gu[:, :c["ff"]], gu[:, c["ff"]:]
    s = 1.0 / (1.0 + torch.exp(-gate))
    h = gate * s * up
    ys = _grouped(h, st["w2"], edges)
    dropped = place.view(-1, k) < 0
    rows = torch.cat([ys, torch.zeros(1, d, device=DEV)])
    picked = rows[place].view(-1, k, d)  # (-1: the zero row)
    y = x + (picked * gates[:, :, None]).sum(1)
    if not backward:
        return {"y": y}
    # the gradient of sum(y)
    dys = gates.reshape(-1)[order][:, None].expand(-1, d)
    dgates = torch.where(dropped, 0.0, picked.sum(2))
    dz = gates * (dgates - (gates * dgates).sum(1, keepdim=True))
    dlogits = torch.zeros(c["tokens"], c["experts"] + 1, device=DEV)
    dlogits.scatter_add_(1, torch.where(experts < 0, c["experts"], experts).long(), dz)
    groups = list(zip(edges, edges[1:]))
    dw2 = torch.stack([h[a:b].t() @ dys[a:b] for a, b in groups])
    dh = _grouped(dys, st["w2"].transpose(1, 2), edges)
    dgu = torch.cat([dh * up * s * (1.0 + gate * (1.0 - s)), dh * gate * s], 1)
    dw13 = torch.stack([xs[a:b].t() @ dgu[a:b] for a, b in groups])
    dxs = torch.cat([_grouped(dgu, st["w13"].transpose(1, 2), edges),
                     torch.zeros(1, d, device=DEV)])
    dx = 1.0 + dxs[place].view(-1, k, d).sum(1)
    return {"y": y, "dx": dx, "dlogits": dlogits[:, :-1].contiguous(), "dw13": dw13, "dw2": dw2}


# ------------------------------------------------------ the framework's calls
class _Memory:
    """device memory of the library as torch sees it; keeps its owner alive"""

    def __init__(self, ptr, shape, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": "<f4",
                                         "data": (int(ptr), False), "version": 2}


class _Session:
    """the parameters and the arena of one pico program"""

    def __init__(self, work_bytes):
        from pico_amd.pico import Pico

        self.P = Pico()
        self.lib = self.P.lib
        self.params = []
        self.work = self.lib.arena_init(int(work_bytes))
        self.opt = self.lib.pico_optim_sgd_init(0.01)
        self.lib.pico_gpu_stream.restype = ctypes.c_void_p
        self.stream = torch.cuda.ExternalStream(self.lib.pico_gpu_stream(), device=DEV)

    def view(self, t, grad=False):
        ptr = t.contents.grad if grad else t.contents.data
        return torch.as_tensor(_Memory(ptr, self.P.shape(t), self), device=DEV)

    def param(self, values):
        t = self.P.param(list(values.shape))
        self.params.append(t)
        self.lib.pico_optim_sgd_add(self.opt, t)
        self.lib.pico_gpu_synchronize()
        self.view(t).copy_(values)
        torch.cuda.synchronize()
        return t

    def __del__(self):
        self.lib.pico_gpu_synchronize()
        self.lib.pico_optim_sgd_free(self.opt)
        for p in self.params:
            self.lib.pico_free(p)
        self.lib.arena_destroy(self.work)


def _empty(*shape, dtype=torch.float32):
    return torch.empty(*shape, device=DEV, dtype=dtype)


def _workspace(nbytes):
    return torch.empty(max(1, nbytes), device=DEV, dtype=torch.uint8)


def _prepare_own(st):
    from pico_amd import kernels as K

    c = st["case"]
    kind = c["kind"]
    if kind == "layernorm":
        r, n = c["rows"], c["cols"]
        st.update(y=_empty(r, n), mean=_empty(r), rstd=_empty(r), dx=_empty(r, n),
                  dgain=_empty(n), dbias=_empty(n), ws=_workspace(K.layernorm_bwd_workspace(r, n)))
    elif kind == "scan":
        b, t, n = c["batch"], c["seq"], c["cols"]
        st.update(h=_empty(b * t, n), ws=_workspace(K.gated_scan_workspace(b, t, n)))
        if c["backward"]:
            st.update(df=_empty(b * t, n), dx=_empty(b * t, n), dh0=_empty(b, n))
    elif kind == "product":
        st.update(y=torch.empty_like(st["dy"]), dx=torch.empty_like(st["x"]),
                  dw=torch.empty_like(st["w"]),
                  ws=_workspace(K.gemm_experts_dw_workspace(c["rows"], c["k"], c["n"],
                                                            c["experts"])))
    elif kind == "moe":
        n = c["tokens"] * c["topk"]
        s = _Session(8 * n * (3 * c["d"] + 3 * c["ff"]) + 16 * c["tokens"] * c["d"] + (1 << 24))
        st["leaves"] = {k: s.param(st.pop(k)) for k in ("x", "logits", "w13", "w2")}
        st["session"] = s
    else:
        n, e = c["tokens"] * c["topk"], c["experts"]
        st.update(experts=_empty(c["tokens"], c["topk"], dtype=torch.int32),
                  gates=_empty(c["tokens"], c["topk"]), offsets=_empty(e + 1, dtype=torch.int32),
                  order=_empty(n, dtype=torch.int32), place=_empty(n, dtype=torch.int32),
                  ws=_workspace(K.expert_plan_workspace(n, e)))
        if kind == "route":
            st["dlogits"] = torch.empty_like(st["logits"])
        else:
            d, f = c["d"], c["ff"]
            st.update(xs=_empty(n, d), gu=_empty(n, 2 * f), h=_empty(n, f), ys=_empty(n, d),
                      y=_empty(c["tokens"], d))


def _own_moe(st):
    c, s, v = st["case"], st["session"], st["leaves"]
    P, lib = s.P, s.lib
    # pico has a stream of its own, which nothing orders with torch's: it starts when
    # what torch has been given is done (it writes where that may still read), and
    # what torch is given from here on waits for it
    theirs, mine = s.stream, torch.cuda.current_stream()
    theirs.wait_stream(mine)
    lib.arena_ctx_push(s.work)
    try:
        lib.arena_reset(s.work)
        lib.pico_optim_sgd_zero_grad(s.opt)
        gates, route = P.route_topk(v["logits"], c["topk"])
        gu = P.expert_matmul(P.expert_gather(v["x"], route), v["w13"], route)
        h = P.swiglu(*P.split_cols(gu, 2))
        y = P.expert_combine(P.expert_matmul(h, v["w2"], route), gates, route, v["x"])
        P.backward(y)
    finally:
        lib.arena_ctx_pop()
        mine.wait_stream(theirs)
    return dict({"d" + n: s.view(t, grad=True) for n, t in v.items()}, y=s.view(y))


def _run_own(st):
    from pico_amd import kernels as K

    c = st["case"]
    kind = c["kind"]
    if kind == "moe":
        return _own_moe(st)
    if kind == "layernorm":
        K.layernorm_fwd(st["x"], st["gain"], st["bias"], st["y"], st["mean"], st["rstd"], EPS)
        K.layernorm_bwd(st["x"], st["gain"], st["mean"], st["rstd"], st["dy"], st["dx"],
                        st["dgain"], st["dbias"], ws=st["ws"])
        return {n: st[n] for n in ("y", "dx", "dgain", "dbias")}
    if kind == "scan":
        K.gated_scan_fwd(c["batch"], st["f"], st["x"], st["h"], h0=st["h0"], ws=st["ws"])
        if not c["backward"]:
            return {"h": st["h"]}
        K.gated_scan_bwd(c["batch"], st["f"], st["x"], st["h"], st["dh"], st["df"], st["dx"],
                         h0=st["h0"], dh0=st["dh0"], ws=st["ws"])
        return {n: st[n] for n in ("h", "dx", "df", "dh0")}
    if kind == "product":
        x, w, dy, offsets = st["x"], st["w"], st["dy"], st["offsets"]
        K.gemm_experts("N", x, w, offsets, st["y"], precision=c["precision"])
        K.gemm_experts("T", dy, w, offsets, st["dx"], precision=c["precision"])
        K.gemm_experts_dw(x, dy, offsets, st["dw"], precision=c["precision"], ws=st["ws"])
        return {n: st[n] for n in ("y", "dx", "dw")}
    K.route_topk(st["logits"], st["experts"], st["gates"])
    K.expert_plan(st["experts"], st["offsets"], st["order"], st["place"], ws=st["ws"])
    if kind == "route":
        K.route_topk_bwd(st["experts"], st["gates"], st["dgates"], st["dlogits"])
        return {n: st[n] for n in ("experts", "gates", "offsets", "order", "place", "dlogits")}
    offsets = st["offsets"]
    K.expert_gather(st["x"], c["topk"], offsets, st["order"], st["xs"])
    K.gemm_experts("N", st["xs"], st["w13"], offsets, st["gu"])
    K.swiglu_fwd(st["gu"][:, :c["ff"]], st["gu"][:, c["ff"]:], st["h"])
    K.gemm_experts("N", st["h"], st["w2"], offsets, st["ys"])
    K.expert_combine(st["place"], st["gates"], st["ys"], st["y"], c=st["x"])
    return {"y": st["y"]}


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "layernorm":
        return _plain_layernorm(state)
    if kind == "scan":
        return _plain_scan(state)
    if kind == "route":
        return _plain_route(state)
    if kind == "product":
        return _plain_product(state)
    return _plain_layer(state, kind == "moe")


# ------------------------------------------------------------- work and exact
def work(case):
    c = case
    kind = c["kind"]
    if kind == "layernorm":
        n = c["rows"] * c["cols"]
        # x and dy read, y and dx written; the vectors
        return {"bytes": 4 * (4 * n + 4 * c["cols"]), "flops": 22 * n}
    if kind == "scan":
        n, state = c["batch"] * c["seq"] * c["cols"], c["batch"] * c["cols"]
        if not c["backward"]:
            return {"bytes": 4 * (3 * n + state), "flops": 8 * n}
        return {"bytes": 4 * (6 * n + 2 * state), "flops": 20 * n}
    if kind == "route":
        n, slots = c["tokens"] * c["experts"], c["tokens"] * c["topk"]
        # logits read, their gradient written; experts, gates, order, place
        # written, the gates' gradient read
        return {"bytes": 4 * (2 * n + 5 * slots + c["experts"] + 1),
                "flops": n * c["topk"] + 10 * slots}
    if kind == "product":
        n, k, m, e = c["rows"], c["k"], c["n"], c["experts"]
        return {"bytes": 4 * (2 * n * (k + m) + 2 * e * k * m), "flops": 6 * n * k * m}
    n, d, f, e = c["tokens"] * c["topk"], c["d"], c["ff"], c["experts"]
    weights = 3 * min(e, n) * d * f
    flops = 6 * n * d * f
    if kind == "experts":
        return {"bytes": 4 * (weights + 2 * c["tokens"] * d + c["tokens"] * e), "flops": flops}
    return {"bytes": 4 * (weights + 3 * e * d * f + 3 * c["tokens"] * d + 2 * c["tokens"] * e),
            "flops": 3 * flops}


def _exact_scan(st):
    c = st["case"]
    b, t, n = c["batch"], c["seq"], c["cols"]
    x, f = (st[k].double().view(b, t, n).transpose(0, 1).contiguous() for k in ("x", "f"))
    s, q = torch.sigmoid(f), torch.sigmoid(-f)
    h = q * x
    prev = st["h0"].double()
    for i in range(t):
        prev = h[i].addcmul_(s[i], prev)

    def rows(a):
        return a.transpose(0, 1).reshape(b * t, n)

    out = {"h": rows(h)}
    if not c["backward"]:
        return out
    grad = st["dh"].double().view(b, t, n).transpose(0, 1).contiguous()
    for i in range(t - 2, -1, -1):
        grad[i].addcmul_(s[i + 1], grad[i + 1])
    prev = torch.cat([st["h0"].double()[None], h[:-1]])
    return dict(out, dx=rows(q * grad), df=rows(grad * (prev - x) * (s * q)), dh0=s[0] * grad[0])


def _exact_choice(z, k):
    """by sorting: (experts, gates as a differentiable function of z)"""
    experts = torch.sort(z.detach(), dim=1, descending=True, stable=True).indices[:, :k]
    picked = torch.gather(z, 1, experts)
    gone = torch.isinf(picked.detach()) & (picked.detach() < 0)
    gates = torch.softmax(torch.where(gone, -1e300, picked), 1)
    return torch.where(gone, -1, experts), torch.where(gone, 0.0, gates)


def _exact_layer(st, backward):
    c = st["case"]
    leaves = {k: st[k].double().requires_grad_(backward) for k in ("x", "logits", "w13", "w2")}
    x, w13, w2 = leaves["x"], leaves["w13"], leaves["w2"]
    experts, gates = _exact_choice(leaves["logits"], c["topk"])
    y = x
    for e in range(c["experts"]):
        token, slot = torch.nonzero(experts == e, as_tuple=True)
        gate, up = (x[token] @ w13[e]).split(c["ff"], 1)
        ys = (torch.nn.functional.silu(gate) * up) @ w2[e]
        y = y.index_add(0, token, ys * gates[token, slot][:, None])
    if not backward:
        return {"y": y}
    y.sum().backward()
    return dict({"d" + k: torch.zeros_like(t) if t.grad is None else t.grad
                 for k, t in leaves.items()}, y=y.detach())


def exact(case, seed):
    global own
    mine, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = mine
    c = case
    kind = c["kind"]
    if kind == "layernorm":
        x, gain, bias = (st[k].double().requires_grad_() for k in ("x", "gain", "bias"))
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + EPS) * gain + bias
        y.backward(st["dy"].double())
        return {"y": y.detach(), "dx": x.grad, "dgain": gain.grad, "dbias": bias.grad}
    if kind == "scan":
        return _exact_scan(st)
    if kind == "route":
        z = st["logits"].double().requires_grad_()
        experts, gates = _exact_choice(z, c["topk"])
        gates.backward(st["dgates"].double())
        kept = [[] for _ in range(c["experts"] + 1)]
        for slot, e in enumerate(experts.reshape(-1).tolist()):
            kept[e].append(slot)  # (-1: the last list)
        order = [slot for group in kept for slot in group]
        offsets = [0]
        for group in kept[:-1]:
            offsets.append(offsets[-1] + len(group))
        place = [-1] * len(order)
        for r, slot in enumerate(order[:offsets[-1]]):
            place[slot] = r

        def whole(v):
            return torch.tensor(v, dtype=torch.int32, device=DEV)

        return {"experts": experts.to(torch.int32), "gates": gates.detach(),
                "offsets": whole(offsets), "order": whole(order), "place": whole(place),
                "dlogits": torch.nan_to_num(z.grad, nan=0.0)}
    if kind == "product":
        x, w, dy = (st[k] for k in ("x", "w", "dy"))
        if c["precision"] == "bf16":
            x, w, dy = (t.to(torch.bfloat16) for t in (x, w, dy))
        x, w, dy = x.double(), w.double(), dy.double()
        y, dx = (torch.empty(c["rows"], m, device=DEV, dtype=torch.float64)
                 for m in (c["n"], c["k"]))
        dw = torch.zeros_like(w)
        at = st["offsets"].tolist()
        for e in range(c["experts"]):
            rows = slice(at[e], at[e + 1])
            y[rows] = x[rows] @ w[e]
            dx[rows] = dy[rows] @ w[e].t()
            dw[e] = x[rows].t() @ dy[rows]
        return {"y": y, "dx": dx, "dw": dw}
    return _exact_layer(st, kind == "moe")
