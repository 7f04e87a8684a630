"""fp16 adapters whose u (v) has values of very different sizes in a row: a rank that is large does not lose the others, where the
adapter's second factor leaves it out.

Bound: the chains of K (N) and r additions, half a unit of each value as a factor, and 2^-38 of its row's largest (half the smallest fp16 value,
after a division that leaves the largest at 2^14 at least)."""
import pytest
import torch

from aristos_b200 import kleos
from tests.operator_util import EPS, HALF_UNIT, check, stream
from tests.test_gpu_adapters import Case

pytestmark = pytest.mark.gpu
HALF = HALF_UNIT[torch.float16]


def bound(inner, chain, outer, r):
    """Of inner @ outer; chain: error of inner."""
    whole = inner.abs() + chain
    return (chain + HALF * whole + 2.0 ** -38 * whole.amax(1, keepdim=True)) @ outer.abs() + (r + 4) * EPS * (whole @ outer.abs())


@pytest.mark.parametrize("lengths,r", [([1] * 20, 16), ([1] * 20, 4), ([1] * 20, 64), ([5, 70, 17], 16), ([5, 70, 17], 32), ([300, 200], 64), ([300, 200], 128),
                                       ([12000, 9000], 16), ([12000, 9000], 32), ([12000, 9000], 64)])
def test_a_rank_that_the_second_factor_leaves_out(lengths, r):
    c = Case(lengths, [i % 2 for i in range(len(lengths))], 2, r, 136, 264, "fp16")
    large = r // 2
    c.x *= 2.0 ** 2
    c.dy *= 2.0 ** 2
    a, b = c.a.clone(), c.b * 2.0 ** -9
    # forward: u of that rank about 2^17, of the others 2^-7; B leaves it out.  base is not there: it would hide what is lost
    c.a *= 2.0 ** -9
    c.a[:, large], c.b[:, :, large] = 2.0 ** 11, 0
    kleos.adapter_products(c.x, c.offsets, c.adapter, c.a, c.b, c.scale, None, c.y, c.u, stream())
    # backward: the same for v, which A leaves out then
    a[:, large], b[:, :, large] = 0, 2.0 ** 11
    kleos.adapter_products_backward(c.dy, c.x, c.u, c.offsets, c.adapter, a, b, c.scale, None, c.dx, stream=stream())
    for l in range(2):
        mine = c.of == l
        s, x, dy = float(c.scale[l]), c.x[mine].double(), c.dy[mine].double()
        u, u1 = x @ c.a[l].double().t(), c.K * EPS * (x.abs() @ c.a[l].double().abs().t())
        y, q = s * (u @ c.b[l].double().t()), c.b[l].double().t()
        assert float(u[:, large].abs().max() / y.abs().max()) > 2.0 ** 18
        check(c.y[mine], y, abs(s) * bound(u, u1, q, r) + EPS * y.abs(), "y")
        v, v1 = s * (dy @ b[l].double()), abs(s) * (c.N + 1) * EPS * (dy.abs() @ b[l].double().abs())
        dx = v @ a[l].double()
        check(c.dx[mine], dx, bound(v, v1, a[l].double(), r) + EPS * dx.abs(), "dx")
        assert float((c.y[mine].double() - y).norm() / y.norm()) <= 3 * HALF and float((c.dx[mine].double() - dx).norm() / dx.norm()) <= 3 * HALF


@pytest.mark.parametrize("lengths", [[1] * 20, [300, 200], [12000, 9000]])
def test_a_rank_that_is_infinite(lengths):
    """The others, past 65504, stay numbers: what comes out is the infinity times B, and nothing that is not a number."""
    c = Case(lengths, [i % 2 for i in range(len(lengths))], 2, 16, 136, 264, "fp16")
    c.x.copy_(c.x.abs() + 1)
    c.a.copy_(c.a.abs() * 2.0 ** 14)
    c.a[:, 3, 9] = float("inf")
    c.b[:, :, 4] = -c.b[:, :, 3]
    c.scale = None
    kleos.adapter_products(c.x, c.offsets, c.adapter, c.a, c.b, None, None, c.y, c.u, stream())
    assert bool((c.u[:, 3] == float("inf")).all()) and float(c.u[:, 4].min()) > 65504
    for l in range(2):
        mine = c.of == l
        want = torch.where(c.b[l, :, 3] > 0, float("inf"), float("-inf")).expand(int(mine.sum()), -1)
        assert torch.equal(c.y[mine].float(), want.float())
