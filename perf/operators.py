"""The operators around the experts of an MoE block whose speed is measured: layer norm, the sort of
tokens by expert with the rows there and back, and the experts' products over the sorted rows, each
with its gradients.

A case is one operator as a program calls it: forward alone where a model answers, forward and
gradients where it is trained.  Sizes are those of the benchmark layers (``baseline_config``), the
layers beside them in ``perf/cases.py``, and odd ones in between.  With ``own`` false the operators
are elementary torch operations in 32 bits, rounded once at the end; with ``own`` true they are this
library's.
"""
import math
import random

import torch

own = False  # whether run() calls this library

_TORCH = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _norm(dtype, rows, H, train, params="fp32", pad=0, eps=1e-5):
    return dict(op="norm", dtype=dtype, rows=rows, H=H, train=train, params=params, pad=pad, eps=eps)


def _sort(dtype, T, K, E, H, train, zipf=0.0, drop=0.0):
    return dict(op="sort", dtype=dtype, T=T, K=K, E=E, H=H, train=train, zipf=zipf, drop=drop)


def _experts(dtype, rows, E, N, K, train, bias=False, skew=0.0, empty=0, spare=0):
    return dict(op="experts", dtype=dtype, rows=rows, E=E, N=N, K=K, train=train, bias=bias, skew=skew, empty=empty, spare=spare)


def listed():
    return [
        # serving: the norm in front of a layer for one token
        dict(_norm("bf16", 1, 2048, False), name="norm_token_bf16"),
        # training: the norm of a step of 16384 tokens, parameters kept in 32 bits
        dict(_norm("bf16", 16384, 4096, True), name="norm_train_bf16"),
        # training in 32 bits: odd rows and columns, rows that lie in a wider matrix
        dict(_norm("fp32", 2943, 1087, True, pad=5), name="norm_train_odd_fp32"),
        # serving: one token to its two experts and back
        dict(_sort("bf16", 1, 2, 64, 2048, False), name="sort_token_bf16"),
        # training: the hot-expert layer's tokens there, back, and both gradients
        dict(_sort("bf16", 16384, 2, 128, 2048, True, zipf=1.2), name="sort_train_zipf_bf16"),
        # training: top-4, an odd number of tokens, a tenth of the places without an expert
        dict(_sort("fp16", 2943, 4, 24, 1088, True, drop=0.1), name="sort_train_ragged_fp16"),
        # serving: the two experts of one token; nothing but the weights they read
        dict(_experts("bf16", 2, 64, 2048, 2048, False), name="experts_token_bf16"),
        # serving: a decode step of 128 sequences, nearly every expert's weights for a few rows each
        dict(_experts("bf16", 256, 64, 2048, 2048, False), name="experts_decode_bf16"),
        # training: the layer that the headline metric is quoted on
        dict(_experts("bf16", 16384, 64, 2048, 2048, True), name="experts_train_bf16"),
        # training: the large FFN's first product, the tensor pipe's own speed
        dict(_experts("bf16", 8192, 8, 14336, 4096, True), name="experts_train_large_bf16"),
        # training: fp16, biases, an odd number of rows, experts of very different popularity and one without any
        dict(_experts("fp16", 11771, 24, 2880, 1088, True, bias=True, skew=0.6, empty=1, spare=37), name="experts_train_ragged_fp16"),
        # training in 32 bits: the float benchmark layer's tokens
        dict(_experts("fp32", 4096, 16, 2048, 2048, True, bias=True), name="experts_train_fp32"),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, spread over the logarithm."""
    while True:
        v = max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))
        if v != 3 * 1024:
            return v


def _pick(rng):
    op = rng.choice(["norm", "sort", "experts", "experts"])
    train = rng.random() < 0.65
    if op == "norm":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return _norm(dtype, _log(rng, 1, 32768), _log(rng, 64, 8192, rng.choice([1, 8, 64])), train,
                     params=rng.choice(["fp32", dtype]), pad=rng.choice([0, 0, 8, 5]))
    if op == "sort":
        K = rng.choice([1, 2, 2, 4, 8])
        return _sort(rng.choice(["bf16", "bf16", "fp16", "fp32"]), _log(rng, 1, 16384), K, rng.choice([8, 12, 16, 24, 32, 64, 128, 256]),
                     _log(rng, 64, 8192, rng.choice([1, 8, 64])), train, zipf=rng.choice([0.0, 0.0, 1.2]), drop=rng.choice([0.0, 0.0, 0.1]))
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    rows, E = _log(rng, 1, 16384), rng.choice([1, 8, 12, 16, 24, 32, 64, 128])
    return _experts(dtype, rows, E, _log(rng, 256, 14336, rng.choice([8, 64])), _log(rng, 256, 8192, rng.choice([8, 64])), train,
                    bias=rng.random() < 0.3, skew=rng.choice([0.0, 0.0, 0.6]), empty=rng.choice([0, 0, 1]) if E > 1 else 0,
                    spare=rng.choice([0, 0, 37]))


def draw(rng):
    # no dearer than the dearest listed case of its kind
    while True:
        c = _pick(rng)
        w = work(c)
        if c["op"] == "experts":
            if w["flops"] <= (2.9e12 if c["dtype"] != "fp32" else 1.03e11) and c["E"] * c["N"] * c["K"] <= 4.8e8:
                return c
        elif w["bytes"] <= 6.8e8:
            return c


# ---------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    x = torch.randn(shape, generator=gen, device="cuda")
    return x.mul_(std).add_(mean).to(dtype)


def _counts(case, seed):
    """Rows of every expert: what a router of this skew gives it."""
    E, rng = case["E"], random.Random(int(seed) * 7919 + 13)
    weight = [0.0 if e < case["empty"] else (e + 1.0) ** -case["skew"] for e in range(E)]
    n = [0] * E
    for e in rng.choices(range(E), weight, k=case["rows"]):
        n[e] += 1
    return n


def _popularity(case):
    rank = list(range(case["E"]))
    random.Random(case["E"]).shuffle(rank)
    return torch.tensor([-case["zipf"] * math.log(r + 1.0) for r in rank], device="cuda")


def prepare(case, seed):
    gen, dt = _gen(seed), _TORCH[case["dtype"]]
    s = dict(case=case)
    empty = lambda shape, d=dt: torch.empty(shape, dtype=d, device="cuda")  # noqa: E731
    if case["op"] == "norm":
        R, H, pt = case["rows"], case["H"], _TORCH[case["params"]]
        # a residual stream: features of their own mean and size, rows of different size
        shape = torch.randn(2, H, generator=gen, device="cuda")
        size = torch.rand(R, 1, generator=gen, device="cuda") + 0.5
        x = torch.randn(R, H + case["pad"], generator=gen, device="cuda")[:, :H]
        x = (x * (0.5 + shape[0].abs()) + 0.5 * shape[1]) * size
        wide = empty((R, H + case["pad"]))
        wide[:, :H] = x.to(dt)
        s.update(x=wide[:, :H], weight=_normal(gen, (H,), pt, 0.1, 1.0), bias=_normal(gen, (H,), pt, 0.1),
                 y=empty((R, H)), mean=empty((R,), torch.float32), rstd=empty((R,), torch.float32))
        if case["train"]:
            s.update(dy=_normal(gen, (R, H), dt), dx=empty((R, H)), dweight=empty((H,), pt), dbias=empty((H,), pt))
            s["workspace"] = empty((_norm_workspace(R, H),), torch.uint8)
    elif case["op"] == "sort":
        T, K, E, H = case["T"], case["K"], case["E"], case["H"]
        logits = torch.randn(T, E, generator=gen, device="cuda") + _popularity(case)
        top = torch.topk(logits, K, dim=1)
        ids = top.indices.to(torch.int32)
        if case["drop"]:  # places that lost their expert to its capacity
            ids = torch.where(torch.rand(T, K, generator=gen, device="cuda") < case["drop"], torch.full_like(ids, -1), ids)
        s.update(topk=ids.contiguous(), weights=torch.softmax(top.values, 1).contiguous(), x=_normal(gen, (T, H), dt),
                 results=_normal(gen, (T * K, H), dt), offsets=empty((E + 1,), torch.int32), row_of=empty((T, K), torch.int32),
                 source=empty((T * K,), torch.int32), rows=empty((T * K, H)), out=empty((T, H)))
        if case["train"]:
            s.update(dout=_normal(gen, (T, H), dt), drows=_normal(gen, (T * K, H), dt), dresults=empty((T * K, H)),
                     dweights=empty((T, K), torch.float32), dx=empty((T, H)))
    else:
        R, E, N, K = case["rows"], case["E"], case["N"], case["K"]
        n = _counts(case, seed)
        total = R + case["spare"]  # rows past the last expert's belong to nobody
        at = [0]
        for v in n:
            at.append(at[-1] + v)
        s.update(offsets=torch.tensor(at, dtype=torch.int32, device="cuda"), most=max(n), x=_normal(gen, (total, K), dt),
                 w=_normal(gen, (E, N, K), dt, K ** -0.5), bias=_normal(gen, (E, N), dt, 0.1) if case["bias"] else None,
                 y=empty((total, N)))
        if case["train"]:
            s.update(dy=_normal(gen, (total, N), dt), dx=empty((total, K)), dw=empty((E, N, K)),
                     dbias=empty((E, N)) if case["bias"] else None)
    return s


def _norm_workspace(rows, H):
    """Bytes that a training program sets aside for the sums over rows: 296 partial sums of two rows at most."""
    return 296 * 2 * 4 * H


# ---------------------------------------------------------------------------- one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from aristos_b200 import kleos
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream or None
    if case["op"] == "norm":
        kleos.layer_norm(s["x"], s["weight"], s["bias"], case["eps"], s["y"], s["mean"], s["rstd"], stream)
        if not case["train"]:
            return dict(y=s["y"], mean=s["mean"], rstd=s["rstd"])
        kleos.layer_norm_backward(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"], s["dx"], s["dweight"], s["dbias"],
                                  s["workspace"], stream)
        return {k: s[k] for k in ("y", "mean", "rstd", "dx", "dweight", "dbias")}
    if case["op"] == "sort":
        kleos.sort_tokens(s["topk"], case["E"], s["offsets"], s["row_of"], s["source"], stream)
        kleos.gather_tokens(s["x"], s["row_of"], s["offsets"], s["rows"], stream)
        kleos.combine_tokens(s["results"], s["row_of"], s["weights"], s["out"], stream)
        if not case["train"]:
            return {k: s[k] for k in ("offsets", "row_of", "source", "rows", "out")}
        kleos.combine_tokens_backward(s["dout"], s["results"], s["row_of"], s["weights"], s["offsets"], s["dresults"],
                                      s["dweights"], stream)
        kleos.gather_tokens_backward(s["drows"], s["row_of"], s["dx"], stream)
        return {k: s[k] for k in ("offsets", "row_of", "source", "rows", "out", "dresults", "dweights", "dx")}
    kleos.expert_products(s["x"], s["offsets"], s["w"], s["bias"], s["y"], stream)
    if not case["train"]:
        return dict(y=s["y"])
    kleos.expert_products_dx(s["dy"], s["offsets"], s["w"], s["dx"], stream)
    kleos.expert_products_dw(s["dy"], s["x"], s["offsets"], s["dw"], s["dbias"], stream)
    return {k: s[k] for k in ("y", "dx", "dw", "dbias") if s[k] is not None}


def _run_plain(s):
    return {"norm": _plain_norm, "sort": _plain_sort, "experts": _plain_experts}[s["case"]["op"]](s)


def _plain_norm(s):
    case = s["case"]
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + case["eps"])
    h = c * rstd
    got = dict(y=(h * w + b).to(s["x"].dtype), mean=mean[:, 0], rstd=rstd[:, 0])
    if case["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
        got.update(dx=dx.to(s["x"].dtype), dweight=(dy * h).sum(0).to(s["weight"].dtype), dbias=dy.sum(0).to(s["bias"].dtype))
    return got


def _plain_sort(s):
    case, dt = s["case"], s["x"].dtype
    T, K, E, H = case["T"], case["K"], case["E"], case["H"]
    ids = s["topk"].reshape(-1).long()
    ids = torch.where((ids < 0) | (ids >= E), torch.full_like(ids, E), ids)  # those without an expert come last
    order = torch.sort(ids, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(T * K, device=ids.device)
    offsets = torch.searchsorted(ids[order], torch.arange(E + 1, device=ids.device))
    has = (ids < E).view(T, K, 1)
    filled = (torch.arange(T * K, device=ids.device) < offsets[E])
    row_of = torch.where(ids < E, place, -1).view(T, K)
    source = torch.where(filled, order, -1)
    token = order // K
    rows = torch.where(filled[:, None], s["x"][token], torch.zeros((), dtype=dt, device=ids.device))
    w = s["weights"]
    results = torch.where(has, s["results"][place].view(T, K, H).float(), 0.0)
    out = (results * w[:, :, None]).sum(1).to(dt)
    got = dict(offsets=offsets.to(torch.int32), row_of=row_of.to(torch.int32), source=source.to(torch.int32), rows=rows, out=out)
    if case["train"]:
        dout = s["dout"].float()
        dresults = torch.where(filled[:, None], dout[token] * w.reshape(-1)[order][:, None], 0.0).to(dt)
        dweights = (results * dout[:, None, :]).sum(2)
        dx = torch.where(has, s["drows"][place].view(T, K, H).float(), 0.0).sum(1).to(dt)
        got.update(dresults=dresults, dweights=dweights, dx=dx)
    return got


def _plain_experts(s):
    # each expert's rows as one matrix of a batch, as high as the fullest
    case, dt, off, most = s["case"], s["x"].dtype, s["offsets"].long(), max(1, s["most"])
    R, E, N, K = s["x"].shape[0], case["E"], case["N"], case["K"]
    row = torch.arange(R, device=off.device)
    expert = torch.searchsorted(off[1:].contiguous(), row, right=True)
    mine = expert < E
    place = torch.where(mine, expert * most + row - off[torch.clamp(expert, max=E)], E * most)  # one more row for those of nobody

    def batch(a):
        wide = torch.zeros(E * most + 1, a.shape[1], device=a.device)
        wide[place] = a.float()
        return wide[:-1].view(E, most, a.shape[1])

    def back(a):
        return torch.where(mine[:, None], a.reshape(E * most, -1)[torch.clamp(place, max=E * most - 1)], 0.0).to(dt)

    w, x = s["w"].float(), batch(s["x"])
    y = torch.bmm(x, w.transpose(1, 2))
    if s["bias"] is not None:
        y = y + s["bias"].float()[:, None, :]
    got = dict(y=back(y))
    if case["train"]:
        dy = batch(s["dy"])
        got.update(dx=back(torch.bmm(dy, w)), dw=torch.bmm(dy.transpose(1, 2), x).to(dt))
        if s["bias"] is not None:
            got["dbias"] = dy.sum(1).to(dt)
    return got


# ---------------------------------------------------------------------------- what a pass has to do
def _used(case):
    """Experts that are expected to have a row at all."""
    E, weight = case["E"], [0.0 if e < case["empty"] else (e + 1.0) ** -case["skew"] for e in range(case["E"])]
    return sum(1.0 - (1.0 - w / sum(weight)) ** case["rows"] for w in weight) if E > 1 else 1.0


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        R, H, p = case["rows"], case["H"], 4 if case["params"] == "fp32" else 2
        back = case["train"]
        return dict(bytes=size * R * H * (4.0 if back else 2.0) + 8.0 * R + p * H * (4.0 if back else 2.0),
                    flops=R * H * (19.0 if back else 7.0))
    if case["op"] == "sort":
        T, K, E, H = case["T"], case["K"], case["E"], case["H"]
        n, filled = T * K, T * K * (1.0 - case["drop"])
        moved = T * H + n * H + filled * H + T * H  # x, rows, results, out
        if case["train"]:
            moved += T * H + n * H + filled * H + T * H  # dout, dresults, drows, dx
        return dict(bytes=size * moved + 4.0 * (3 * n + E + 1) + 4.0 * n * (2 if case["train"] else 1),
                    flops=filled * H * (6.0 if case["train"] else 2.0))
    R, E, N, K = case["rows"], case["E"], case["N"], case["K"]
    total, weights = R + case["spare"], _used(case) * N * K
    moved = R * K + weights + total * N
    if case["train"]:
        moved += R * N + total * K + E * N * K
    if case["bias"]:
        moved += E * N * (2 if case["train"] else 1)
    return dict(bytes=float(size * moved), flops=2.0 * R * N * K * (3 if case["train"] else 1))


# ---------------------------------------------------------------------------- 64-bit results
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "sort": _exact_sort, "experts": _exact_experts}[case["op"]](case, s)


def _exact_norm(case, s):
    x, w, b = (s[k].double() for k in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x, dim=1, correction=0)
    rstd = (var + case["eps"]).rsqrt()
    h = (x - mean[:, None]) * rstd[:, None]
    got = dict(y=torch.addcmul(b, h, w), mean=mean, rstd=rstd)
    if case["train"]:
        dy = s["dy"].double()
        g, H = dy * w, case["H"]
        dx = (g * H - g.sum(1)[:, None] - h * torch.einsum("ij,ij->i", g, h)[:, None]) * (rstd / H)[:, None]
        got.update(dx=dx, dweight=torch.einsum("ij,ij->j", dy, h), dbias=torch.einsum("ij->j", dy))
    return got


def _exact_sort(case, s):
    T, K, E, H = case["T"], case["K"], case["E"], case["H"]
    ids = s["topk"].reshape(-1).cpu().tolist()
    lists = [[] for _ in range(E)]
    for i, e in enumerate(ids):
        if 0 <= e < E:
            lists[e].append(i)
    source = torch.tensor([i for one in lists for i in one], dtype=torch.long, device="cuda")  # place in topk of every row
    n, w = len(source), s["weights"].double().reshape(-1)
    token = source // K
    rows = torch.zeros(T * K, H, dtype=torch.float64, device="cuda")
    rows[:n] = s["x"].double()[token]
    results = s["results"][:n].double()
    out = torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add_(0, token, results * w[source, None])
    got = dict(offsets=None, row_of=None, source=None, rows=rows, out=out)
    if case["train"]:
        dout = s["dout"].double()[token]
        dresults, dweights = torch.zeros_like(rows), torch.zeros(T * K, dtype=torch.float64, device="cuda")
        dresults[:n] = dout * w[source, None]
        dweights[source] = torch.einsum("ij,ij->i", dout, results)
        dx = torch.zeros_like(out).index_add_(0, token, s["drows"][:n].double())
        got.update(dresults=dresults, dweights=dweights.view(T, K), dx=dx)
    return got


def _exact_experts(case, s):
    at = s["offsets"].cpu().tolist()
    total, E, N, K = s["x"].shape[0], case["E"], case["N"], case["K"]
    new = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")  # noqa: E731
    got = dict(y=new(total, N))
    if case["train"]:
        got.update(dx=new(total, K), dw=new(E, N, K))
        if case["bias"]:
            got["dbias"] = new(E, N)
    for e in range(E):
        r, w = slice(at[e], at[e + 1]), s["w"][e].double()
        x = s["x"][r].double()
        got["y"][r] = torch.nn.functional.linear(x, w, s["bias"][e].double() if case["bias"] else None)
        if case["train"]:
            dy = s["dy"][r].double()
            got["dx"][r], got["dw"][e] = dy @ w, dy.t() @ x
            if case["bias"]:
                got["dbias"][e] = dy.sum(0)
    return got
