"""More operators around the experts whose speed is measured: the activation between an expert's two products with its
gradient, a whole MoE layer for the few tokens of a decode step, and low-rank adapters of many requests beside a
projection that they share, with their gradients.

A case is one operator as a program calls it: forward alone where a model answers, forward and gradients where it is
trained.  Sizes are those of the benchmark layers, of the cases in ``perf/operators.py`` and ``perf/cases.py``, and odd
ones in between.  With ``own`` false the operators are elementary torch operations in 32 bits (the choice of experts in
64), rounded once; with ``own`` true they are this library's.
"""
import math
import random

import torch

own = False  # whether run() calls this library

_TORCH = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _act(dtype, rows, I, act, gated, train, pad=0):
    return dict(op="activation", dtype=dtype, rows=rows, I=I, act=act, gated=gated, train=train, pad=pad)


def _moe(dtype, T, H, I, E, K, act="silu", gated=True, bias=False, off=0, pad=0):
    return dict(op="moe", dtype=dtype, T=T, H=H, I=I, E=E, K=K, act=act, gated=gated, bias=bias, off=off, pad=pad)


def _adapt(dtype, rows, requests, adapters, r, N, K, train, without=0.0, spare=0, pad=0):
    return dict(op="adapters", dtype=dtype, rows=rows, requests=requests, adapters=adapters, r=r, N=N, K=K, train=train,
                without=without, spare=spare, pad=pad)


def listed():
    return [
        # training: gated experts of the layer that the headline metric is quoted on, its 16384 sorted rows
        dict(_act("bf16", 16384, 2048, "silu", True, True), name="activation_train_bf16"),
        # training in 32 bits: odd rows and columns, a matrix inside a wider one, the reference's GELU without a gate
        dict(_act("fp32", 2943, 1087, "gelu", False, True, pad=5), name="activation_train_odd_fp32"),
        # serving: the next token of one sequence; nothing but the weights of its two experts
        dict(_moe("bf16", 1, 2048, 2048, 64, 2), name="moe_token_bf16"),
        # serving: a decode step of 16 sequences on the large FFN's experts
        dict(_moe("bf16", 16, 4096, 14336, 8, 2), name="moe_decode_large_bf16"),
        # serving: a decode step of 128 sequences, nearly every expert's weights for a few rows each
        dict(_moe("bf16", 128, 2048, 2048, 64, 2), name="moe_decode_bf16"),
        # serving: odd sizes, top-4, GELU with biases and without a gate, two experts out of service
        dict(_moe("fp16", 37, 1088, 2880, 24, 4, act="gelu", gated=False, bias=True, off=2, pad=8), name="moe_ragged_fp16"),
        # serving in 32 bits: the float benchmark layer's experts, as the reference activates them
        dict(_moe("fp32", 8, 2048, 2048, 16, 2, act="relu", gated=False, bias=True), name="moe_decode_fp32"),
        # serving: the next token of one request with an adapter of its own
        dict(_adapt("bf16", 1, 1, 8, 16, 2048, 2048, False), name="adapters_token_bf16"),
        # serving: a decode step of 128 requests, 32 adapters among them, an eighth of the requests without one
        dict(_adapt("bf16", 128, 128, 32, 16, 2048, 2048, False, without=0.125), name="adapters_decode_bf16"),
        # serving: prompts of uneven lengths, a batch padded behind the last one
        dict(_adapt("fp16", 7919, 23, 9, 32, 2880, 1088, False, without=0.2, spare=41), name="adapters_ragged_fp16"),
        # training: four adapters beside one projection of the large FFN's width, 16384 tokens
        dict(_adapt("bf16", 16384, 16, 4, 64, 4096, 4096, True), name="adapters_train_bf16"),
        # training in 32 bits: odd rank and sizes
        dict(_adapt("fp32", 2943, 7, 3, 12, 1087, 1090, True, without=0.1, spare=5, pad=3), name="adapters_train_odd_fp32"),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def _pick(rng):
    op = rng.choice(["activation", "moe", "moe", "adapters", "adapters"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    act = rng.choice(["silu", "silu", "gelu", "relu"])
    if op == "activation":
        return _act(dtype, _log(rng, 1, 32768), _log(rng, 64, 14336, rng.choice([1, 8, 64])), act, rng.random() < 0.7, rng.random() < 0.65,
                    pad=rng.choice([0, 0, 8, 5]))
    if op == "moe":
        E = rng.choice([4, 8, 16, 24, 32, 64, 128])
        off = rng.choice([0, 0, 0, 1, 2])
        step = rng.choice([8, 64, 64, 1])
        return _moe(dtype, _log(rng, 1, 128), _log(rng, 256, 4096, step), _log(rng, 256, 14336, step), E,
                    min(rng.choice([1, 2, 2, 4, 8]), E - off), act=act, gated=rng.random() < 0.7, bias=rng.random() < 0.3, off=off,
                    pad=rng.choice([0, 0, 8]))
    train = rng.random() < 0.5
    rows = _log(rng, 1, 16384)
    requests = rows if not train and rng.random() < 0.4 else _log(rng, 1, min(rows, 64))
    requests = min(requests, 512)
    step = rng.choice([8, 64, 64, 1])
    return _adapt(dtype, rows, requests, _log(rng, 1, 64), rng.choice([4, 8, 8, 16, 16, 32, 64, 12]), _log(rng, 256, 8192, step),
                  _log(rng, 256, 8192, step), train, without=rng.choice([0.0, 0.0, 0.2]), spare=rng.choice([0, 0, 37]), pad=rng.choice([0, 0, 8]))


def draw(rng):
    # no dearer than the dearest listed case of its kind
    while True:
        c = _pick(rng)
        w, most = work(c), 4.8e8
        if c["op"] == "moe":
            most = 1.7e9
            if c["E"] * c["H"] * c["I"] * (3 if c["gated"] else 2) > 1.4e9:
                continue
        if w["bytes"] <= most and w["flops"] <= (2.6e10 if c["op"] == "adapters" and c["dtype"] != "fp32" else 8e9):
            return c


# ---------------------------------------------------------------------------- inputs
def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    x = torch.randn(shape, generator=gen, device="cuda")
    return x.mul_(std).add_(mean).to(dtype)


def _inside(t, pad):
    """The same matrix, inside one that is `pad` columns wider."""
    if not pad:
        return t
    wide = torch.empty(t.shape[0], t.shape[1] + pad, dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _requests(case, seed):
    """Rows of every request and its adapter, -1 where it has none: every request has a row, lengths are uneven."""
    rng = random.Random(int(seed) * 7919 + 17)
    R = case["requests"]
    cuts = sorted(rng.sample(range(1, case["rows"]), R - 1))
    begin = [0] + cuts
    end = cuts + [case["rows"]]
    which = [-1 if rng.random() < case["without"] else rng.randrange(case["adapters"]) for _ in range(R)]
    return list(zip(begin, end, which))


def prepare(case, seed):
    gen, dt = torch.Generator(device="cuda").manual_seed(int(seed)), _TORCH[case["dtype"]]
    s = dict(case=case)
    empty = lambda shape, d=dt: torch.empty(shape, dtype=d, device="cuda")  # noqa: E731
    if case["op"] == "activation":
        R, I = case["rows"], case["I"]
        wide = 2 * I if case["gated"] else I
        s.update(z=_inside(_normal(gen, (R, wide), dt), case["pad"]), h=empty((R, I)))
        if case["train"]:
            s.update(dh=_normal(gen, (R, I), dt), dz=empty((R, wide)))
    elif case["op"] == "moe":
        T, H, I, E, K = (case[k] for k in "THIEK")
        up = 2 * I if case["gated"] else I
        gate_bias = None
        if case["off"]:  # experts out of service
            gate_bias = torch.zeros(E, device="cuda")
            gate_bias[torch.randperm(E, generator=gen, device="cuda")[:case["off"]]] = float("-inf")
        s.update(x=_inside(_normal(gen, (T, H), dt), case["pad"]), gate=_normal(gen, (E, H), dt, H ** -0.5), gate_bias=gate_bias,
                 w1=_normal(gen, (E, up, H), dt, H ** -0.5), w2=_normal(gen, (E, H, I), dt, I ** -0.5),
                 b1=_normal(gen, (E, up), dt, 0.1) if case["bias"] else None, b2=_normal(gen, (E, H), dt, 0.1) if case["bias"] else None,
                 out=empty((T, H)), topk=empty((T, K), torch.int32), weights=empty((T, K), torch.float32),
                 workspace=empty((_moe_workspace(T, I, K),), torch.uint8))
    else:
        rows, L, r, N, K = (case[k] for k in ("rows", "adapters", "r", "N", "K"))
        total = rows + case["spare"]  # rows behind the last request's belong to nobody
        plan = _requests(case, seed)
        s.update(plan=plan, offsets=torch.tensor([0] + [e for _, e, _ in plan], dtype=torch.int32, device="cuda"),
                 adapter=torch.tensor([w for _, _, w in plan], dtype=torch.int32, device="cuda"),
                 x=_inside(_normal(gen, (total, K), dt), case["pad"]), base=_inside(_normal(gen, (total, N), dt), case["pad"]),
                 a=_normal(gen, (L, r, K), dt, K ** -0.5), b=_normal(gen, (L, N, r), dt, 0.5 * r ** -0.5),
                 scale=torch.rand(L, generator=gen, device="cuda") * 1.5 + 0.5, y=empty((total, N)), u=empty((total, r), torch.float32))
        if case["train"]:
            s.update(dy=_normal(gen, (total, N), dt), dbase=_normal(gen, (total, K), dt), dx=empty((total, K)), da=empty((L, r, K)),
                     db=empty((L, N, r)), workspace=empty((4 * total * r + 256,), torch.uint8))
    return s


def _moe_workspace(T, I, K):
    """Bytes that a serving program sets aside: the activated rows of its tokens in 32 bits, and their experts."""
    return T * K * (4 * (I + 8) + 16) + 4096


# ---------------------------------------------------------------------------- one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from aristos_b200 import kleos
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream or None
    if case["op"] == "activation":
        kleos.activation(s["z"], case["act"], s["h"], stream)
        if not case["train"]:
            return dict(h=s["h"])
        kleos.activation_backward(s["dh"], s["z"], case["act"], s["dz"], stream)
        return dict(h=s["h"], dz=s["dz"])
    if case["op"] == "moe":
        kleos.moe_tokens(s["x"], s["gate"], s["gate_bias"], s["w1"], s["b1"], s["w2"], s["b2"], case["act"], s["out"], s["topk"],
                         s["weights"], s["workspace"], stream)
        return {k: s[k] for k in ("out", "topk", "weights")}
    # in 32 bits the plain form adds in place, into what the projection gave: so do the calls
    y = s["base"] if case["dtype"] == "fp32" else s["y"]
    kleos.adapter_products(s["x"], s["offsets"], s["adapter"], s["a"], s["b"], s["scale"], s["base"], y, s["u"], stream)
    if not case["train"]:
        return dict(y=y, u=s["u"])
    dx = s["dbase"] if case["dtype"] == "fp32" else s["dx"]
    kleos.adapter_products_backward(s["dy"], s["x"], s["u"], s["offsets"], s["adapter"], s["a"], s["b"], s["scale"], s["dbase"], dx,
                                    s["da"], s["db"], s["workspace"], stream)
    return dict(y=y, u=s["u"], dx=dx, da=s["da"], db=s["db"])


def _run_plain(s):
    return {"activation": _plain_activation, "moe": _plain_moe, "adapters": _plain_adapters}[s["case"]["op"]](s)


def _plain_act(g, act):
    """The activation and its slope."""
    if act == "relu":
        on = (g > 0).float()
        return torch.where(g > 0, g, torch.zeros_like(g)), on
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * 0.5 ** 0.5))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (2.0 * math.pi) ** -0.5
    p = 1.0 / (1.0 + torch.exp(-g))
    return g * p, p * (1.0 + g * (1.0 - p))


def _plain_activation(s):
    case, dt = s["case"], s["z"].dtype
    I, z = case["I"], s["z"].float()
    value, slope = _plain_act(z[:, :I], case["act"])
    got = dict(h=(value * z[:, I:] if case["gated"] else value).to(dt))
    if case["train"]:
        dh = s["dh"].float()
        got["dz"] = (torch.cat([dh * z[:, I:] * slope, dh * value], 1) if case["gated"] else dh * slope).to(dt)
    return got


def _plain_route(s):
    logits = s["x"].double() @ s["gate"].double().t()
    if s["gate_bias"] is not None:
        logits = logits + s["gate_bias"].double()
    order = torch.sort(logits, dim=1, descending=True, stable=True)
    top, ids = order.values[:, :s["case"]["K"]], order.indices[:, :s["case"]["K"]]
    p = torch.exp(top - top[:, :1])
    return ids, (p / p.sum(1, keepdim=True)).float()


def _plain_moe(s):
    case = s["case"]
    ids, weights = _plain_route(s)
    I, x = case["I"], s["x"].float()
    share = torch.zeros(case["T"], case["E"], device="cuda").scatter_(1, ids, weights)
    out = torch.zeros(case["T"], case["H"], device="cuda")
    for e in range(case["E"]):
        z = x @ s["w1"][e].float().t()
        if s["b1"] is not None:
            z = z + s["b1"][e].float()
        h = _plain_act(z[:, :I], case["act"])[0]
        if case["gated"]:
            h = h * z[:, I:]
        y = h @ s["w2"][e].float().t()
        if s["b2"] is not None:
            y = y + s["b2"][e].float()
        out = out + share[:, e:e + 1] * y
    return dict(out=out.to(s["x"].dtype), topk=ids.to(torch.int32), weights=weights)


def _plain_adapters(s):
    case, dt = s["case"], s["x"].dtype
    y, u = s["base"].float(), torch.zeros_like(s["u"])
    if case["train"]:
        dx, da, db = s["dbase"].float(), torch.zeros(s["a"].shape, device="cuda"), torch.zeros(s["b"].shape, device="cuda")
    for begin, end, which in s["plan"]:
        if which < 0:
            continue
        a, b, scale = s["a"][which].float(), s["b"][which].float(), s["scale"][which]
        x = s["x"][begin:end].float()
        one = x @ a.t()
        u[begin:end] = one
        y[begin:end] += scale * (one @ b.t())
        if case["train"]:
            dy = s["dy"][begin:end].float() * scale
            v = dy @ b
            dx[begin:end] += v @ a
            da[which] += v.t() @ x
            db[which] += dy.t() @ one
    got = dict(y=y.to(dt), u=u)
    if case["train"]:
        got.update(dx=dx.to(dt), da=da.to(dt), db=db.to(dt))
    return got


# ---------------------------------------------------------------------------- what a pass has to do
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "activation":
        n, wide = float(case["rows"]) * case["I"], 2 if case["gated"] else 1
        # z read, h written; trained: dh read, dz written (z is read once)
        return dict(bytes=size * n * (wide + 1 + (wide + 1 if case["train"] else 0)), flops=n * (25.0 if case["train"] else 10.0))
    if case["op"] == "moe":
        T, H, I, E, K = (case[k] for k in "THIEK")
        wide = 3 if case["gated"] else 2
        live = E - case["off"]
        used = live * (1.0 - (1.0 - K / live) ** T)  # experts that are expected to have a token
        weights = used * (wide * H * I + ((wide - 1) * I + H if case["bias"] else 0))
        return dict(bytes=size * (weights + 2.0 * T * H + E * H) + 8.0 * T * K, flops=2.0 * T * K * wide * H * I + 2.0 * T * E * H)
    rows, total, L, r, N, K = (case[k] for k in ("rows", "rows", "adapters", "r", "N", "K"))
    total += case["spare"]
    on = rows * (1.0 - case["without"])
    live = case["requests"] * (1.0 - case["without"])
    used = L * (1.0 - (1.0 - 1.0 / L) ** live)
    moved = on * K + 2.0 * total * N + used * r * (N + K)  # x, base, y, the adapters
    flops = 2.0 * on * r * (N + K)
    if case["train"]:
        moved += on * N + 2.0 * total * K + L * r * (N + K)  # dy, dbase, dx, the adapters' gradients
        flops *= 3.0
    return dict(bytes=size * moved + 4.0 * total * r + 8.0 * case["requests"], flops=flops)


# ---------------------------------------------------------------------------- 64-bit results
def exact(case, seed):
    s = prepare(case, seed)
    return {"activation": _exact_activation, "moe": _exact_moe, "adapters": _exact_adapters}[case["op"]](case, s)


def _exact_act(g, act):
    if act == "relu":
        return g.clamp(min=0.0)
    return g * (torch.special.ndtr(g) if act == "gelu" else torch.sigmoid(g))


def _exact_slope(g, act):
    if act == "relu":
        return torch.heaviside(g, torch.zeros_like(g))
    if act == "gelu":
        return torch.special.ndtr(g) + g * torch.exp(g.square() / -2.0) / math.sqrt(2.0 * math.pi)
    p = torch.sigmoid(g)
    return p + g * p * torch.sigmoid(-g)


def _exact_activation(case, s):
    I, act = case["I"], case["act"]
    g, up = s["z"][:, :I].double(), s["z"][:, I:].double()
    got = dict(h=_exact_act(g, act) * up if case["gated"] else _exact_act(g, act))
    if case["train"]:
        dh, dg = s["dh"].double(), _exact_slope(g, act)
        got["dz"] = torch.hstack([dh * up * dg, dh * _exact_act(g, act)]) if case["gated"] else dh * dg
    return got


def _exact_moe(case, s):
    T, K, I = case["T"], case["K"], case["I"]
    x = s["x"].double()
    logits = torch.einsum("th,eh->te", x, s["gate"].double())
    if s["gate_bias"] is not None:
        logits += s["gate_bias"].double()
    rows = logits.cpu().tolist()
    chosen = [sorted(range(case["E"]), key=lambda e: (-rows[t][e], e))[:K] for t in range(T)]
    ids = torch.tensor(chosen, device="cuda")
    weights = torch.softmax(logits.gather(1, ids), 1)
    out = torch.zeros(T, case["H"], dtype=torch.float64, device="cuda")
    for e in sorted({e for one in chosen for e in one}):
        places = [(t, one.index(e)) for t, one in enumerate(chosen) if e in one]
        t = torch.tensor([p[0] for p in places], device="cuda")
        k = torch.tensor([p[1] for p in places], device="cuda")
        z = torch.nn.functional.linear(x[t], s["w1"][e].double(), s["b1"][e].double() if case["bias"] else None)
        h = _exact_act(z[:, :I], case["act"])
        if case["gated"]:
            h = h * z[:, I:]
        y = torch.nn.functional.linear(h, s["w2"][e].double(), s["b2"][e].double() if case["bias"] else None)
        out.index_add_(0, t, y * weights[t, k, None])
    return dict(out=out, topk=None, weights=weights)


def _exact_adapters(case, s):
    rows, dt = s["x"].shape[0], torch.float64
    which = torch.full((rows,), -1, dtype=torch.long)
    for begin, end, w in s["plan"]:
        which[begin:end] = w
    which = which.cuda()
    y, u = s["base"].double(), torch.zeros(s["u"].shape, dtype=dt, device="cuda")
    if case["train"]:
        dx, da, db = s["dbase"].double(), torch.zeros(s["a"].shape, dtype=dt, device="cuda"), torch.zeros(s["b"].shape, dtype=dt, device="cuda")
    for w in range(case["adapters"]):  # all rows of an adapter at once
        mine = torch.nonzero(which == w)[:, 0]
        if not len(mine):
            continue
        a, b, scale = s["a"][w].double(), s["b"][w].double(), float(s["scale"][w])
        x = s["x"][mine].double()
        u[mine] = torch.einsum("tk,rk->tr", x, a)
        y[mine] += torch.einsum("tr,nr->tn", u[mine], b) * scale
        if case["train"]:
            dy = s["dy"][mine].double()
            v = torch.einsum("tn,nr->tr", dy, b) * scale
            dx[mine] += torch.einsum("tr,rk->tk", v, a)
            da[w] = torch.einsum("tr,tk->rk", v, x)
            db[w] = torch.einsum("tn,tr->nr", dy, u[mine]) * scale
    got = dict(y=y, u=u)
    if case["train"]:
        got.update(dx=dx, da=da, db=db)
    return got
