"""Hidden values of a layer for a few tokens past fp16's range (65504): they are values like others, as long as the results are."""
import pytest
import torch

from tests.operator_util import check, gen
from tests.test_gpu_moe_tokens import Layer

pytestmark = pytest.mark.gpu


def large(*size, up=8, down=13, **form):
    layer = Layer(*size, dtype="fp16", **form)
    layer.x *= 2.0 ** 4
    layer.gate *= 2.0 ** -4
    layer.w1 *= 2.0 ** up
    layer.w2 *= 2.0 ** -down
    return layer


@pytest.mark.parametrize("T,H,I,E,K", [(1, 256, 512, 8, 2), (1, 8, 8, 1, 1), (7, 264, 1096, 12, 4), (37, 1088, 136, 24, 8), (128, 512, 520, 16, 8), (128, 100, 60, 3, 3),
                                       (30, 1087, 131, 9, 4), (11, 264, 131, 4, 2), (9, 64, 2048, 64, 8)])
@pytest.mark.parametrize("act", ["silu", "relu"])
def test_hidden_values_past_the_range(T, H, I, E, K, act):
    layer = large(T, H, I, E, K, act=act)  # z about 2^12, its products 2^24
    layer.run().verify()
    plain = large(T, H, I, E, K, up=12, down=4, act=act, gated=False, bias=True, pad=3)  # z about 2^16
    plain.run().verify()
    assert bool((plain.out != 0).any())


def test_a_few_of_them():
    """One expert's rows of W1 are large, in two columns: most places have none, and are the same bits as without."""
    layer = Layer(40, 264, 200, 6, 2, "fp16", "relu", False, bias=True).run()
    before = layer.out.clone()
    layer.w1[2, [5, 77]] *= 2.0 ** 11
    layer.w1[2, [5, 77]] = layer.w1[2, [5, 77]] * 64
    layer.w2[2, :, [5, 77]] *= 2.0 ** -11
    layer.run().verify()
    without = (layer.topk != 2).all(1)
    assert bool(without.any()) and torch.equal(layer.out[without], before[without])


def test_far_past_it():
    """Products of z and z' up to 2^60: fp16 weights of 2^-24 bring them back where they are small enough."""
    layer = Layer(3, 64, 40, 2, 1, "fp16", "relu", True)
    layer.x.fill_(2.0 ** 12)
    layer.w1.fill_(2.0 ** 12)
    layer.w2.zero_()
    layer.w2[:, :, 3] = 2.0 ** -24
    layer.weights = torch.full((3, 1), 2.0 ** -40, device="cuda")
    layer.topk = torch.tensor([[0], [1], [0]], dtype=torch.int32, device="cuda")
    layer.run(gate=False)
    # z = 64 2^24 = 2^30, h = 2^60, out = 2^60 2^-24 2^-40
    assert bool((layer.out == 2.0 ** -4).all())


def test_an_expert_twice():
    layer, g = large(20, 136, 72, 5, 3), gen(3)
    layer.topk = torch.randint(-1, 6, (20, 3), generator=g, device="cuda", dtype=torch.int32)
    layer.topk[0] = 1
    layer.weights = torch.randn(20, 3, generator=g, device="cuda")
    layer.run(gate=False)
    out, _ = layer.result(layer.topk, layer.weights)
    check(layer.out, out, layer.result(layer.topk, layer.weights.abs())[1], "out")


def test_infinities_and_nan_stay():
    layer = large(9, 128, 72, 8, 2).run()
    before = layer.out.clone()
    layer.b1 = torch.zeros(8, 144, dtype=torch.float16, device="cuda")
    layer.b1[:, 7] = float("inf")
    layer.b1[:, 72:] = 0
    layer.run()
    assert not bool(torch.isfinite(layer.out).any()) and bool(torch.isfinite(before).all())
    layer.b1.zero_()
    assert torch.equal(layer.run().out, before)
    layer.x[4, 17] = float("nan")
    layer.run()
    keep = torch.arange(9, device="cuda") != 4
    assert torch.equal(layer.out[keep], before[keep]) and bool(torch.isnan(layer.out[4]).all())
