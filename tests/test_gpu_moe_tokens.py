"""A whole layer for a few tokens against 64 bits."""
import pytest
import torch

from aristos_b200 import kleos
from tests.operator_util import DT, EPS, HALF_UNIT, LEAST, check, gen, randn, stream, wide
from tests.test_gpu_activation import reference

pytestmark = pytest.mark.gpu


class Layer:
    def __init__(self, T, H, I, E, K, dtype="bf16", act="silu", gated=True, bias=False, pad=0, seed=0):
        g, dt, up = gen(T + H + I + seed), DT[dtype], I * (2 if gated else 1)
        self.T, self.H, self.I, self.E, self.K, self.act, self.gated = T, H, I, E, K, act, gated
        self.x, self.gate, self.gate_bias = randn(g, (T, H), dt), randn(g, (E, H), dt, H ** -0.5), None
        self.w1, self.w2 = randn(g, (E, up, H), dt, H ** -0.5), randn(g, (E, H, I), dt, I ** -0.5)
        self.b1, self.b2 = (randn(g, (E, up), dt, 0.1), randn(g, (E, H), dt, 0.1)) if bias else (None, None)
        self.out = torch.full((T, H), float("nan"), dtype=dt, device="cuda")
        if pad:
            self.x, self.out = wide(self.x, pad, 0), wide(self.out, 0, pad)
        self.topk = torch.full((T, K), 7777, dtype=torch.int32, device="cuda")
        self.weights = torch.full((T, K), float("nan"), device="cuda")
        self.workspace = torch.full((kleos.moe_tokens_workspace(T, I, K),), 0xFF, dtype=torch.uint8, device="cuda")

    def run(self, gate=True):
        kleos.moe_tokens(self.x, self.gate if gate else None, self.gate_bias if gate else None, self.w1, self.b1, self.w2, self.b2, self.act,
                         self.out, self.topk, self.weights, self.workspace, stream())
        return self

    def choice(self):
        """Experts and weights in 64 bits; -1 where only experts that are out are left."""
        logits = self.x.double() @ self.gate.double().t()
        if self.gate_bias is not None:
            logits = logits + self.gate_bias.double()
        top = torch.sort(logits, dim=1, descending=True, stable=True)
        values, ids = top.values[:, :self.K], top.indices[:, :self.K].to(torch.int32)
        there = values > float("-inf")
        p = torch.where(there, torch.exp(values - values[:, :1]), 0.0)
        return torch.where(there, ids, -1), torch.where(there, p / p.sum(1, keepdim=True), 0.0)

    def result(self, ids, weights):
        """out in 64 bits and a bound on its error before the last rounding: chains of H and I additions, the activation's bound,
        the hidden value's rounding to two parts of the element type (2^-16 relative, which is what two bf16 parts keep)."""
        x, T, I = self.x.double(), self.T, self.I
        fast = self.x.dtype != torch.float32
        out, off = (torch.zeros(T, self.H, dtype=torch.float64, device="cuda") for _ in range(2))
        for e in set(ids[(ids >= 0) & (ids < self.E)].tolist()):
            share = torch.where(ids == e, weights.double(), 0.0).sum(1, keepdim=True)
            mine = (ids == e).any(1, keepdim=True)
            w1, w2 = self.w1[e].double(), self.w2[e].double()
            b1 = self.b1[e].double() if self.b1 is not None else torch.zeros(w1.shape[0], dtype=torch.float64, device="cuda")
            z = x @ w1.t() + b1
            dz = (self.H + 1) * EPS * (x.abs() @ w1.abs().t() + b1.abs())
            f, _, df, _ = reference(z[:, :I], self.act, fast)
            df = df + 1.2 * dz[:, :I]  # (no slope is above 1.13)
            h, dh = f, df
            if self.gated:
                u, du = z[:, I:], dz[:, I:]
                h, dh = f * u, df * (u.abs() + du) + f.abs() * du + EPS * (f * u).abs()
            dh = dh + (HALF_UNIT[self.x.dtype] * (h.abs() + dh) + LEAST[self.x.dtype] if fast else 0.0)
            y, dy = h @ w2.t(), dh @ w2.abs().t() + (I + 1) * EPS * (h.abs() @ w2.abs().t())
            if self.b2 is not None:
                y = y + self.b2[e].double()
            out += torch.where(mine, share * y, 0.0)
            off += torch.where(mine, share * (dy + 10 * EPS * y.abs()), 0.0)
        return out, off

    def verify(self):
        ids, weights = self.choice()
        assert torch.equal(self.topk, ids), "experts"
        check(self.weights, weights, 2 * EPS * weights, "weights")
        out, off = self.result(ids, weights)
        check(self.out, out, off, "out")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,H,I,E,K", [(1, 256, 512, 8, 2), (1, 8, 8, 1, 1), (2, 2048, 264, 64, 2), (7, 264, 1096, 12, 4), (16, 512, 256, 4, 3), (37, 1088, 136, 24, 8),
                                       (64, 128, 640, 128, 2), (127, 320, 328, 5, 5), (128, 512, 520, 16, 8), (128, 256, 64, 1, 1), (9, 64, 2048, 1024, 8), (33, 1024, 1024, 8, 2)])
def test_layers(T, H, I, E, K, dtype):
    Layer(T, H, I, E, K, dtype).run().verify()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", list(kleos.ACTIVATIONS))
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("pad", [0, 8, 3])
def test_forms(pad, gated, act, dtype):
    Layer(19, 264, 200, 6, 2, dtype, act, gated, bias=True, pad=pad).run().verify()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,H,I,E,K", [(1, 1, 1, 1, 1), (3, 77, 99, 5, 2), (30, 1087, 131, 9, 4), (11, 264, 131, 4, 2), (11, 131, 264, 4, 2), (128, 100, 60, 3, 3)])
def test_odd_sizes(T, H, I, E, K, dtype):
    Layer(T, H, I, E, K, dtype, bias=True).run().verify()


@pytest.mark.parametrize("dtype", list(DT))
def test_ties_go_to_the_lower_expert(dtype):
    layer = Layer(40, 128, 64, 16, 4, dtype)
    layer.gate[5:11] = layer.gate[2]
    layer.gate[15] = layer.gate[0]
    layer.run().verify()
    zeros = Layer(3, 128, 64, 16, 4, dtype)
    zeros.gate.zero_()
    zeros.run().verify()
    assert zeros.topk.tolist() == [[0, 1, 2, 3]] * 3


@pytest.mark.parametrize("dtype", list(DT))
def test_experts_out_of_service(dtype):
    for out in ([3], [0, 1, 2, 3, 4, 5], list(range(7)), list(range(8))):
        layer = Layer(21, 128, 72, 8, 3, dtype, bias=True)
        layer.gate_bias = randn(gen(5), (8,), torch.float32)
        layer.gate_bias[out] = float("-inf")
        layer.w1[out], layer.w2[out] = float("nan"), float("nan")
        layer.run().verify()
    assert bool((layer.topk == -1).all()) and bool((layer.out == 0).all()) and bool((layer.weights == 0).all())


def test_gate_bias_of_the_lowest_value():
    layer = Layer(21, 128, 72, 8, 3)
    layer.gate_bias = torch.zeros(8, device="cuda")
    layer.gate_bias[[1, 4]] = torch.finfo(torch.float32).min
    layer.run().verify()
    layer.gate_bias.fill_(torch.finfo(torch.float32).min)  # the logits are lost in it: ties
    layer.run()
    assert bool(torch.isfinite(layer.out).all()) and bool((layer.topk >= 0).all())


@pytest.mark.parametrize("dtype", list(DT))
def test_a_token_that_is_not_a_number(dtype):
    layer = Layer(9, 128, 72, 8, 2, dtype).run()
    before, ids = layer.out.clone(), layer.topk.clone()
    layer.x[4, 17] = float("nan")
    layer.run()
    keep = torch.arange(9, device="cuda") != 4
    assert torch.equal(layer.out[keep], before[keep]) and torch.equal(layer.topk[keep], ids[keep])
    assert bool(torch.isnan(layer.out[4]).all()) and bool(torch.isnan(layer.weights[4]).all())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,K", [(6, 3), (128, 8), (1, 1), (100, 2)])
def test_the_callers_own_choice(T, K, dtype):
    """Places without an expert, one expert twice and three times for a token, weights that do not add up to one."""
    E = 5
    layer, g = Layer(T, 136, 72, E, K, dtype), gen(T)
    layer.topk = torch.randint(-2, E + 2, (T, K), generator=g, device="cuda", dtype=torch.int32)
    layer.topk[0] = 1
    layer.weights = torch.randn(T, K, generator=g, device="cuda")
    layer.weights[(layer.topk < 0) | (layer.topk >= E)] = float("nan")
    layer.gate = torch.full_like(layer.gate, float("nan"))
    ids, weights = layer.topk.clone(), layer.weights.clone()
    layer.run(gate=False)
    assert torch.equal(layer.topk, ids) and bool(((layer.weights == weights) | weights.isnan()).all())
    out, off = layer.result(ids, weights)
    absolute = layer.result(ids, weights.abs())[1]  # (weights of both signs)
    check(layer.out, out, absolute, "out")


def test_all_tokens_of_one_expert():
    for dtype in DT:
        layer = Layer(128, 136, 264, 6, 1, dtype)
        layer.gate_bias = torch.zeros(6, device="cuda")
        layer.gate_bias[4] = 100.0
        layer.run().verify()
        assert bool((layer.topk == 4).all())


@pytest.mark.parametrize("dtype", list(DT))
def test_the_same_bits(dtype):
    layer = Layer(50, 264, 328, 8, 2, dtype).run()
    first = layer.out.clone()
    for _ in range(3):
        layer.workspace.fill_(0x7F)
        assert torch.equal(layer.run().out, first)


def test_no_tokens():
    layer = Layer(0, 64, 32, 4, 2)
    layer.run()
