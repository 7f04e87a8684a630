"""Weight gradients in floats from 16-bit operands: long sums are as good as 32-bit sums are.

The matrix unit cuts its running sums off instead of rounding them, so a sum that stays there for long drifts: by about half a
unit in 2^23 a step of sixteen terms.  Sums that are read back every 256 terms and added in registers, rounded to nearest, lose 16
such halves of a sum that is half as large on the way, 5e-7 to 1e-6 whatever the number of terms; what the unit cuts off the
terms themselves when it lines them up may be as much again, and the additions of the parts stay below 1e-6.  3e-6 of the 2-norm is
allowed for any number of rows.
"""
import pytest
import torch

from aristos_b200 import kleos
from tests.operator_util import DT, gen, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", ["both signs", "one sign"])
@pytest.mark.parametrize("counts", [[255], [257, 0, 300], [4096, 31, 4097], [20011, 1, 256], [70000]])
@pytest.mark.parametrize("N,K", [(264, 136), (128, 520)])
def test_float_gradients_of_many_rows(N, K, counts, kind, dtype):
    g, rows = gen(sum(counts) + N), sum(counts)
    x, dy = (torch.randn(rows, n, generator=g, device="cuda") for n in (K, N))
    if kind == "one sign":
        x, dy = x.abs(), dy.abs()
    x, dy = x.to(DT[dtype]), dy.to(DT[dtype])
    at = [sum(counts[:e]) for e in range(len(counts) + 1)]
    offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
    dw = torch.full((len(counts), N, K), 9.0, device="cuda")
    kleos.expert_products_dw(dy, x, offsets, dw, None, stream())
    for e, n in enumerate(counts):
        r = slice(at[e], at[e + 1])
        want = dy[r].double().t() @ x[r].double()
        assert float((dw[e].double() - want).norm()) <= 3e-6 * float(want.norm()), e
    again = torch.empty_like(dw)
    kleos.expert_products_dw(dy, x, offsets, again, None, stream())
    assert torch.equal(dw, again)
