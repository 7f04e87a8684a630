"""The router of a layer for a few tokens where products or logits pass the floats' range: the choice is that of 64 bits."""
import pytest
import torch

from tests.operator_util import DT, EPS, check, gen
from tests.test_gpu_moe_tokens import Layer

pytestmark = pytest.mark.gpu
INF = float("inf")


def same_choice(layer):
    ids, weights = layer.choice()
    assert torch.equal(layer.topk, ids)
    assert torch.equal(layer.weights.isnan(), weights.isnan())
    there = ~weights.isnan()
    check(layer.weights[there], weights[there], 2 * EPS * weights[there], "weights")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,H", [(1, 64), (21, 264), (9, 77), (128, 2048)])
def test_a_gate_row_that_takes_its_expert_out(T, H, dtype):
    layer = Layer(T, H, 72, 16, 3, dtype)
    layer.x[:, 5] = layer.x[:, 5].abs() + 0.5
    layer.gate[[2, 11], 5] = -INF
    layer.run()
    same_choice(layer)
    assert not bool(((layer.topk == 2) | (layer.topk == 11)).any())
    layer.verify()
    # all of them: nothing is chosen
    layer.gate[:, 5] = -INF
    layer.run()
    assert bool((layer.topk == -1).all()) and bool((layer.weights == 0).all()) and bool((layer.out == 0).all())


@pytest.mark.parametrize("dtype", list(DT))
def test_a_token_with_one_infinity(dtype):
    """Its logits are infinities of the gate's signs there: experts of minus infinity are out, as many as there are are chosen."""
    layer = Layer(9, 128, 72, 8, 4, dtype)
    layer.x[4, 17] = -INF
    layer.gate[:, 17] = layer.gate[:, 17].abs() + 0.01  # all experts out
    layer.x[[0, 1, 2, 3, 5, 6, 7, 8], 17] = 0
    layer.run()
    same_choice(layer)
    assert layer.topk[4].tolist() == [-1] * 4 and bool((layer.out[4] == 0).all())
    layer.gate[3, 17] *= -1  # one is of plus infinity, and its weight (infinity less infinity) no number
    layer.run()
    same_choice(layer)
    assert layer.topk[4].tolist() == [3, -1, -1, -1]
    assert bool(torch.isfinite(layer.out[[0, 1, 2, 3, 5, 6, 7, 8]]).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("H", [64, 264, 77])
def test_products_past_the_range_of_floats(H, dtype):
    """Products of 2^100 to 2^126 each: the logits, of 2^200 and more, differ in their first bits, in 64 bits."""
    layer = Layer(7, H, 40, 12, 2, dtype)
    layer.x.zero_()
    layer.gate.zero_()
    layer.x[:, 3] = torch.tensor([2.0 ** 100, -2.0 ** 110, 2.0 ** 120, 1.0, 0.0, -2.0 ** 90, 3.0 * 2.0 ** 100], device="cuda").to(layer.x.dtype)
    layer.gate[:, 3] = (torch.arange(12, device="cuda") * 5 % 12 - 6.0).to(layer.x.dtype) * 2.0 ** 120
    layer.gate[:, 6] = torch.randn(12, generator=gen(2), device="cuda").to(layer.x.dtype)
    layer.x[:, 6] = 1
    layer.run()
    same_choice(layer)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_sums_past_the_range_of_floats_on_the_way(dtype):
    """2^127 and 2^127 and as much of the other sign later: the sum is what is left of it, exactly."""
    layer = Layer(3, 512, 40, 8, 2, dtype)
    layer.x[:, :256], layer.x[:, 256:] = 2.0 ** 127, -2.0 ** 127
    layer.gate.fill_(1)
    layer.gate[:, 0] = torch.tensor([1.0, 1.5, 0.5, 1.25, 0.75, 1.0, 1.75, 0.25], device="cuda").to(layer.x.dtype)
    layer.run()
    same_choice(layer)
