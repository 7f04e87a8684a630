"""The layer for few tokens in 16 bits is off by its two roundings and no more: h between the products, and the result.

A rounding of evenly spread values to a step of twice HALF_UNIT (of values just above a power of two, where it is largest) is off by HALF_UNIT / sqrt(3) of the
2-norm.  h's comes out of the second product as it went in, as its errors are independent of the weights: together sqrt(2 / 3) HALF_UNIT at most, 0.0032 in
bf16, where values spread over all of a binade give 0.0024.  Sums of 32 bits are nothing beside that."""
import pytest
import torch

from tests.operator_util import HALF_UNIT
from tests.test_gpu_moe_tokens import Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("gated,act", [(True, "silu"), (False, "gelu"), (True, "relu")])
@pytest.mark.parametrize("T,H,I,E,K", [(1, 2048, 2048, 8, 2), (16, 1024, 3584, 8, 2), (128, 512, 520, 16, 8), (37, 1088, 1337, 24, 4)])
def test_two_roundings(T, H, I, E, K, gated, act, dtype):
    layer = Layer(T, H, I, E, K, dtype, act, gated).run()
    out, _ = layer.result(*layer.choice())
    off = float((layer.out.double() - out).norm() / out.norm())
    assert off <= (2 / 3) ** 0.5 * HALF_UNIT[layer.x.dtype]
