"""A layer for a few tokens over very long rows: sums of 16-bit products are as good as 32-bit sums are, and a result is rounded once.

The other product of each layer here is exact (one value a row), so that a result is one long sum of terms of one sign and its rounding.  The matrix
unit cuts its running sums off, by about half a unit in 2^23 a step of sixteen terms; sums that leave it every 8192 terms at most lose 512 such halves of
what is half as large on the way, 2^-16, and what it cuts off the terms when it lines them up may be as much again.  The additions of the parts, 2^7 a warp
and eight warps, are off by 2^-24 of half the sum each at most: 2^-18.  2^-14 is allowed beside half a unit of the result.
"""
import pytest
import torch

from tests.operator_util import HALF_UNIT, gen
from tests.test_gpu_moe_tokens import Layer

pytestmark = pytest.mark.gpu


def near(got, want, dt):
    return float(((got.double() - want) / want).abs().max()) <= HALF_UNIT[dt] * (1 + 2.0 ** -14) + 2.0 ** -14


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,I", [(1, 1 << 22), (1, (1 << 22) - 4), (1, (1 << 22) - 1), (9, 1 << 22), (9, 65536), (9, 65544), (9, 131072), (1, 73731)])
def test_long_rows_of_the_second_product(T, I, dtype):
    """Rows that are not a multiple of 16 or of 4 bytes too, and as long as stays on the unit and a little longer."""
    layer, g = Layer(T, 16, I, 1, 1, dtype, act="relu", gated=False), gen(1)
    layer.w1.zero_()
    layer.w1[0, :, 0] = torch.rand(I, generator=g, device="cuda").add_(0.5).to(layer.x.dtype)
    layer.x.zero_()
    layer.x[:, 0] = (torch.arange(T, device="cuda") % 2 + 1).to(layer.x.dtype)
    layer.w2.copy_(layer.w2.abs() * 4)
    layer.run()
    want = layer.x[:, :1].double() * (layer.w2[0].double() @ layer.w1[0, :, 0].double())[None]
    assert near(layer.out, want, layer.x.dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T", [1, 9])
def test_long_rows_of_the_first_product(T, gated, dtype):
    H = 1 << 22
    layer = Layer(T, H, 16, 1, 1, dtype, act="relu", gated=gated)
    layer.x.copy_(layer.x.abs())
    layer.w1.copy_(layer.w1.abs() * 4)
    if gated:  # the second factor is one
        layer.w1[0, 16:] = 0
        layer.x[:, 7] = 1
        layer.w1[0, 16:, 7] = 1
    layer.w2.zero_()
    layer.w2[0, :16] = torch.eye(16, device="cuda").to(layer.x.dtype)
    layer.run()
    want = layer.x.double() @ layer.w1[0, :16].double().t()
    assert near(layer.out[:, :16], want, layer.x.dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,H,I,E,K,gated", [(16, 40, 70000, 8, 2, True), (40, 72, 20001, 64, 4, False), (128, 33, 34000, 9, 8, True), (5, 140002, 24, 6, 3, True),
                                             (40, 40008, 56, 32, 2, True), (21, 50001, 40, 16, 2, False)])
def test_layers_of_long_rows(T, H, I, E, K, gated, dtype):
    """Several experts, tokens and blocks to a column, every alignment; the same bits again."""
    layer = Layer(T, H, I, E, K, dtype, gated=gated, bias=True).run()
    layer.verify()
    first = layer.out.clone()
    layer.workspace.fill_(0x7F)
    assert torch.equal(layer.run().out, first)
