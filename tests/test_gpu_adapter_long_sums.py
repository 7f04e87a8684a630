"""Gradients of adapters with many rows: sums of 16-bit products are as good as 32-bit sums are.

The factors are exact here (a row of A and a column of B have one value each, a power of two, so u and v are values of x and dy moved
by it), and so are their products in 32 bits: what is off is the sums.  The matrix unit cuts its running sums off instead of rounding them, by
about half a unit in 2^23 a step of sixteen rows.  Sums that leave it after two steps at most lose two such units of a part of the
whole (2.4e-7), and what it cuts off the terms when it lines them up may be as much again; the additions of the parts in 32 bits, rounded to nearest,
are n / 32 of at most 2^-24 each, of either sign: sqrt(n / 32) 2^-24 in the 2-norm, 2.8e-6 for 70000 rows in one block.  3e-6 of
the 2-norm is allowed.
"""
import pytest
import torch

from aristos_b200 import kleos
from tests.operator_util import HALF_UNIT, gen, stream
from tests.test_gpu_adapters import Case

pytestmark = pytest.mark.gpu


def exact_factors(lengths, which, L, r, N, K, dtype, grads):
    c = Case(lengths, which, L, r, N, K, dtype, grads=grads)
    g = gen(r)
    at_k, at_n = (torch.randint(0, n, (L, r), generator=g, device="cuda") for n in (K, N))
    power = lambda: torch.randint(-2, 3, (L, r), generator=g, device="cuda").float().exp2().to(c.dt)  # noqa: E731
    c.a.zero_().scatter_(2, at_k[..., None], power()[..., None])
    c.b.zero_().scatter_(1, at_n[:, None, :], power()[:, None, :])
    c.scale = torch.tensor([0.5, 2.0, 1.0], device="cuda")[:L].contiguous()
    return c


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", ["both signs", "one sign"])
@pytest.mark.parametrize("lengths", [[257, 0, 31], [20011, 1, 300], [70000]])
@pytest.mark.parametrize("r,N,K", [(16, 264, 136), (64, 136, 520), (128, 264, 264)])
def test_float_gradients_of_many_rows(r, N, K, lengths, kind, dtype):
    c = exact_factors(lengths, list(range(len(lengths))), len(lengths), r, N, K, dtype, torch.float32)
    if kind == "one sign":
        c.x.copy_(c.x.abs())
        c.dy.copy_(c.dy.abs())
    c.all()
    begin = 0
    for l, n in enumerate(lengths):
        x, dy = c.x[begin:begin + n].double(), c.dy[begin:begin + n].double()
        a, b, s = c.a[l].double(), c.b[l].double(), float(c.scale[l])
        for name, got, want in (("da", c.da[l], s * (dy @ b).t() @ x), ("db", c.db[l], s * dy.t() @ (x @ a.t()))):
            assert float((got.double() - want).norm()) <= 3e-6 * float(want.norm()), (name, l)
        begin += n


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_gradients_of_many_rows_in_16_bits(dtype):
    """Half a unit of the result, and what the unit cuts off of sums that stay there: 200000 rows in eight blocks are 1563 steps of half a unit in 2^23 each, of
    a sum that is half as large on the way, 2^-14.4; what it cuts off the terms may be as much again.  2^-13 is allowed beside the rounding."""
    c = exact_factors([200000], [0], 1, 16, 72, 80, dtype, None)
    c.x.copy_(c.x.abs() * 0.25)
    c.dy.copy_(c.dy.abs() * 0.25)
    c.all()
    x, dy, a, b, s = c.x.double(), c.dy.double(), c.a[0].double(), c.b[0].double(), float(c.scale[0])
    for name, got, want in (("da", c.da[0], s * (dy @ b).t() @ x), ("db", c.db[0], s * dy.t() @ (x @ a.t()))):
        assert bool((want < 60000).all())
        assert float(((got.double() - want) / want).abs().max()) <= HALF_UNIT[c.dt] * (1 + 2.0 ** -13) + 2.0 ** -13, name
    again = c.da.clone(), c.db.clone()
    kleos.adapter_products_backward(c.dy, c.x, c.u, c.offsets, c.adapter, c.a, c.b, c.scale, c.dbase, c.dx, c.da, c.db, c.workspace, stream())
    assert torch.equal(c.da, again[0]) and torch.equal(c.db, again[1])
