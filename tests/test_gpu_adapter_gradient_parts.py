"""Gradients of adapters in floats are as good as u and v are, which are 32-bit values: they are no 16-bit factors there.

3e-6 of the 2-norm for the sums, as for factors that are exact; u and v as factors of two parts are off by HALF_UNIT squared at most, 2^-16 in bf16 and
2^-22 in fp16.

Results in 16 bits of few rows are off by their own rounding alone: HALF_UNIT / sqrt(3) of the 2-norm at most (of values just above a power of two)."""
import pytest
import torch

from tests.operator_util import HALF_UNIT
from tests.test_gpu_adapters import Case

pytestmark = pytest.mark.gpu


def off_by(c, lengths, most):
    begin = 0
    for l, n in enumerate(lengths):
        x, dy, u = c.x[begin:begin + n].double(), c.dy[begin:begin + n].double(), c.u[begin:begin + n].double()
        s, b = float(c.scale[l]), c.b[l].double()
        for name, got, want in (("da", c.da[l], s * (dy @ b).t() @ x), ("db", c.db[l], s * dy.t() @ u)):
            off = float((got.double() - want).norm())
            assert off <= most * float(want.norm()), (name, l, off / float(want.norm()))
        begin += n


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("r", [2, 8, 12, 16, 32, 48, 64, 66, 128])
@pytest.mark.parametrize("lengths", [[1], [5, 31, 0, 33], [300, 2000, 17, 700]])
def test_factors_of_two_parts(lengths, r, dtype):
    c = Case(lengths, list(range(len(lengths))), len(lengths), r, 264, 328, dtype, grads=torch.float32)
    c.all()
    half = HALF_UNIT[c.dt]
    off_by(c, lengths, 3e-6 + half * half)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("r", [2, 8, 12, 16, 32, 48, 64, 66, 128])
@pytest.mark.parametrize("lengths", [[1], [4], [5, 31, 0, 33], [300, 17, 195]])
def test_few_rows_in_16_bits(lengths, r, dtype):
    c = Case(lengths, list(range(len(lengths))), len(lengths), r, 264, 328, dtype)
    c.all()
    half = HALF_UNIT[c.dt]
    off_by(c, lengths, half / 3 ** 0.5 + half * half + 3e-6)
