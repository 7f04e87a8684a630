"""fp16 gradients of adapters whose ranks, and whose rows, are of very different sizes: a row of dA (a column of dB) is made of its own
rank's u (v) alone, and is as good as if there were no other."""
import pytest
import torch

from aristos_b200 import kleos
from tests.operator_util import EPS, HALF_UNIT, check, gen, stream
from tests.test_gpu_adapters import Case

pytestmark = pytest.mark.gpu
HALF = HALF_UNIT[torch.float16]


def expected(c):
    """dA and dB from the u and v that the call has (u is an input; v is made of dy, B and scale), and bounds: the chains of N additions for v,
    half a unit of each factor and 2^-38 of its rank's largest (half the smallest fp16 value, a power of two of at least 2^-14 of that largest later),
    the sums over the rows."""
    da, db = torch.zeros(c.a.shape, dtype=torch.float64, device="cuda"), torch.zeros(c.b.shape, dtype=torch.float64, device="cuda")
    oda, odb = torch.zeros_like(da), torch.zeros_like(db)
    for l in range(c.L):
        mine = torch.nonzero(c.of == l)[:, 0]
        n, s = len(mine), float(c.scale[l])
        x, dy, u, b = c.x[mine].double(), c.dy[mine].double(), c.u[mine].double(), c.b[l].double()
        v = s * (dy @ b)
        v1 = abs(s) * (c.N + 1) * EPS * (dy.abs() @ b.abs())
        vv = v.abs() + v1
        rounded = lambda t: HALF * t + 2.0 ** -38 * t.amax(0, keepdim=True)  # noqa: E731
        da[l], db[l] = v.t() @ x, s * (dy.t() @ u)
        oda[l] = (v1 + rounded(vv)).t() @ x.abs() + (n + 2) * EPS * (vv.t() @ x.abs())
        odb[l] = abs(s) * (dy.abs().t() @ rounded(u.abs()) + (n + 3) * EPS * (dy.abs().t() @ u.abs()))
    return da, oda, db, odb


def backward(c):
    kleos.adapter_products_backward(c.dy, c.x, c.u, c.offsets, c.adapter, c.a, c.b, c.scale, None, c.dx, c.da, c.db, c.workspace, stream())


@pytest.mark.parametrize("r", [2, 4, 16, 32, 48, 64, 66, 128])
@pytest.mark.parametrize("lengths", [[40, 3, 0, 90], [700, 300, 9, 2000]])
def test_ranks_of_different_sizes(lengths, r):
    """Ranks from 2^-12 to 2^9 of one another, and of their own order: the largest is neither the first nor the last."""
    c = Case(lengths, [0, 2, 1, 1], 3, r, 136, 264, "fp16", grads=torch.float32)
    power = (torch.arange(r, device="cuda") * 7 % 22 - 12).float().exp2()
    c.a.copy_((c.a.float() * power[:, None]))
    c.b.copy_((c.b.float() * power[None, :]))
    c.forward()
    backward(c)
    da, oda, db, odb = expected(c)
    check(c.da, da, oda, "da")
    check(c.db, db, odb, "db")


@pytest.mark.parametrize("r", [16, 64])
@pytest.mark.parametrize("at", [0, 33, 999])
def test_one_row_far_above_the_others(at, r):
    """It is the largest of its column of x alone: elsewhere x (dy) is zero there, so the other rows' sums stand by themselves."""
    c = Case([1000], [0], 1, r, 136, 264, "fp16", grads=torch.float32)
    c.x *= 2.0 ** -9
    c.dy *= 2.0 ** -9
    c.x[at], c.dy[at] = 0, 0
    c.x[at, 0], c.dy[at, 0] = 2.0 ** 15, 2.0 ** 15
    c.forward()
    backward(c)
    da, oda, db, odb = expected(c)
    check(c.da, da, oda, "da")
    check(c.db, db, odb, "db")
    # (the bound has the large row's share in column 0 and the other rows' in the others)
    assert float((c.da[0, :, 1:].double() - da[0, :, 1:]).norm() / da[0, :, 1:].norm()) <= 2 * HALF
    assert float((c.db[0, 1:].double() - db[0, 1:]).norm() / db[0, 1:].norm()) <= 2 * HALF


@pytest.mark.parametrize("at", [0, 70, 999])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_one_rank_that_is_not_a_number(value, at):
    """The other ranks, far above 65504 here, are what they would be without it."""
    c = Case([1000], [0], 1, 16, 136, 264, "fp16", grads=torch.float32)
    c.dy.copy_(c.dy.abs() + 2.0 ** -10)
    c.forward()
    c.u *= 2.0 ** 20
    backward(c)
    db = c.db.clone()
    c.u[at, 5] = value
    backward(c)
    others = torch.arange(16, device="cuda") != 5
    assert torch.equal(c.db[:, :, others], db[:, :, others])
    bad = c.db[0, :, 5]
    # (dy is positive, so the sum is that infinity times the scale's sign)
    want = value * float(c.scale[0])
    assert bool((bad == want).all()) if value == value else bool(bad.isnan().all())


@pytest.mark.parametrize("size", [2.0 ** 127, 2.0 ** 100, 2.0 ** -120])
def test_ends_of_the_range(size):
    """u near the largest and the smallest float: dy makes the results floats again."""
    c = Case([300], [0], 1, 16, 136, 264, "fp16", grads=torch.float32)
    c.forward()
    c.u.copy_(torch.rand(c.u.shape, generator=gen(1), device="cuda") * size)
    c.dy *= 2.0 ** -13 if size > 1 else 2.0 ** 8
    backward(c)
    _, _, db, odb = expected(c)
    check(c.db, db, odb, "db")
