"""Adapters of many requests, and their gradients, against 64 bits."""
import pytest
import torch

from aristos_b200 import kleos
from tests.operator_util import DT, EPS, HALF_UNIT, check, gen, randn, stream, wide

pytestmark = pytest.mark.gpu
NAN = float("nan")


class Case:
    """`lengths`: rows of every request; `first` and `spare`: rows before the first and behind the last."""

    def __init__(self, lengths, which, L, r, N, K, dtype="bf16", first=0, spare=0, pad=0, grads=None, seed=0):
        g, dt = gen(sum(lengths) + r + N + K + seed), DT[dtype]
        cuts = [first]
        for n in lengths:
            cuts.append(cuts[-1] + n)
        rows = cuts[-1] + spare
        self.rows, self.R, self.L, self.r, self.N, self.K, self.dt = rows, len(lengths), L, r, N, K, dt
        self.offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
        self.adapter = torch.tensor(which, dtype=torch.int32, device="cuda")
        of = torch.full((rows,), -1, dtype=torch.long)
        for i, l in enumerate(which):
            of[cuts[i]:cuts[i + 1]] = l if 0 <= l < L else -1
        self.of = of.cuda()
        put = (lambda t, left, right: wide(t, left, right)) if pad else (lambda t, left, right: t)
        full = lambda *shape, dtype=dt: torch.full(shape, NAN, dtype=dtype, device="cuda")  # noqa: E731
        self.x, self.dy = put(randn(g, (rows, K), dt), pad, 0), put(randn(g, (rows, N), dt), 0, pad)
        self.base, self.dbase = put(randn(g, (rows, N), dt), pad, pad), put(randn(g, (rows, K), dt), 0, pad)
        self.a, self.b = randn(g, (L, r, K), dt, K ** -0.5), randn(g, (L, N, r), dt, r ** -0.5)
        self.scale = torch.rand(L, generator=g, device="cuda") * 2 - 0.5
        self.y, self.dx, self.u = put(full(rows, N), pad, 0), put(full(rows, K), pad, pad), full(rows, r, dtype=torch.float32)
        gt = grads or dt
        self.da, self.db = full(L, r, K, dtype=gt), full(L, N, r, dtype=gt)
        self.workspace = torch.full((kleos.adapter_products_workspace(rows, r),), 0xFF, dtype=torch.uint8, device="cuda")

    def forward(self):
        kleos.adapter_products(self.x, self.offsets, self.adapter, self.a, self.b, self.scale, self.base, self.y, self.u, stream())

    def backward(self):
        kleos.adapter_products_backward(self.dy, self.x, self.u, self.offsets, self.adapter, self.a, self.b, self.scale, self.dbase, self.dx,
                                        self.da, self.db, self.workspace, stream())

    def verify(self):
        """Bounds: chains of K, N, r and rows additions; u and v, as factors of the second products, rounded to the element type:
        half a unit of each value, and in fp16, where they are divided by a power of two up to their largest first, at least half the
        smallest value of fp16 times that."""
        half, least = (0.0, 0.0) if self.dt == torch.float32 else (HALF_UNIT[self.dt], 2.0 ** -24 if self.dt == torch.float16 else 0.0)
        rounded = lambda t, most: half * t + least * most  # noqa: E731
        y, dx = (t.double() if t is not None else 0.0 for t in (self.base, self.dbase))
        y, dx = y + torch.zeros(self.rows, self.N, dtype=torch.float64, device="cuda"), dx + torch.zeros(self.rows, self.K, dtype=torch.float64, device="cuda")
        u, da, db = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (self.u, self.a, self.b))
        oy, odx, ou, oda, odb = (torch.zeros_like(t) for t in (y, dx, u, da, db))
        row = lambda t: t.amax(1, keepdim=True).expand_as(t)  # noqa: E731
        for l in range(self.L):
            mine = torch.nonzero(self.of == l)[:, 0]
            if not len(mine):
                continue
            n, s = len(mine), float(self.scale[l]) if self.scale is not None else 1.0
            a, b, x, dy = self.a[l].double(), self.b[l].double(), self.x[mine].double(), self.dy[mine].double()
            one = x @ a.t()
            u1 = self.K * EPS * (x.abs() @ a.abs().t())
            u[mine], ou[mine] = one, u1
            uu = one.abs() + u1
            y[mine] += s * (one @ b.t())
            oy[mine] = abs(s) * ((u1 + rounded(uu, row(uu))) @ b.abs().t() + (self.r + 4) * EPS * (uu @ b.abs().t())) + EPS * y[mine].abs()
            v = s * (dy @ b)
            v1 = abs(s) * (self.N + 1) * EPS * (dy.abs() @ b.abs())
            vv = v.abs() + v1
            dx[mine] += v @ a
            odx[mine] = (v1 + rounded(vv, row(vv))) @ a.abs() + (self.r + 4) * EPS * (vv @ a.abs()) + EPS * dx[mine].abs()
            da[l], db[l] = v.t() @ x, s * (dy.t() @ one)
            oda[l] = (v1 + rounded(vv, vv.amax())).t() @ x.abs() + (n + 2) * EPS * (vv.t() @ x.abs())
            odb[l] = abs(s) * (dy.abs().t() @ (u1 + rounded(uu, uu.amax())) + (n + 3) * EPS * (dy.abs().t() @ uu))
        check(self.u, u, ou, "u")
        check(self.y, y, oy, "y")
        check(self.dx, dx, odx, "dx")
        if self.da is not None:
            check(self.da, da, oda, "da")
        if self.db is not None:
            check(self.db, db, odb, "db")

    def all(self):
        self.forward()
        self.backward()
        return self


def _uneven(rows, R, seed):
    import random
    rng = random.Random(seed)
    cuts = [0] + sorted(rng.randrange(rows + 1) for _ in range(R - 1)) + [rows]
    return [b - a for a, b in zip(cuts, cuts[1:])], [rng.randrange(-1, 4) for _ in range(R)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("r", [1, 2, 4, 6, 8, 12, 16, 20, 24, 32, 48, 64, 66, 128])
def test_ranks(r, dtype):
    Case([5, 70, 0, 17, 1], [1, 0, 2, -1, 1], 3, r, 264, 328, dtype, first=2, spare=3).all().verify()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,R,r,N,K", [(1, 1, 16, 2048, 2048), (1, 1, 8, 8, 8), (64, 64, 16, 512, 256), (500, 7, 32, 264, 1096), (1500, 300, 16, 136, 520),
                                          (4096, 3, 16, 512, 640), (300, 2, 64, 2048, 264), (33, 33, 16, 40, 2888), (129, 2, 16, 1032, 24),
                                          (20000, 5, 64, 136, 72), (20000, 5, 32, 72, 136), (12000, 30, 16, 8, 200), (20000, 3, 12, 136, 72), (700, 2, 4, 264, 136)])
def test_shapes(rows, R, r, N, K, dtype):
    lengths, which = _uneven(rows, R, rows) if R != rows else ([1] * R, [i % 5 - 1 for i in range(R)])
    Case(lengths, which if rows > 1 else [0], 4, r, N, K, dtype, spare=5).all().verify()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("pad", [0, 8, 3])
@pytest.mark.parametrize("r,N,K", [(3, 77, 99), (12, 1087, 131), (16, 131, 264), (16, 264, 131), (1, 1, 1), (20, 250, 254)])
def test_odd_sizes(r, N, K, pad, dtype):
    Case([40, 3, 0, 90], [0, 2, 1, 1], 3, r, N, K, dtype, spare=4, pad=pad).all().verify()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("pad", [8, 3])
def test_strides_and_gradients_in_floats(pad, dtype):
    Case([40, 3, 0, 90], [0, 2, 1, 1], 3, 16, 264, 136, dtype, spare=4, pad=pad, grads=torch.float32).all().verify()


@pytest.mark.parametrize("dtype", list(DT))
def test_forms(dtype):
    """No scale, no base, in place, no u, no gradients of the adapters; an adapter's requests apart from one another."""
    c = Case([20, 30, 7, 64, 1], [1, 0, 1, 5, 1], 3, 16, 136, 264, dtype, spare=2)
    c.scale = None
    c.all().verify()
    y, dx = c.y.clone(), c.dx.clone()
    kleos.adapter_products(c.x, c.offsets, c.adapter, c.a, c.b, None, c.base, c.y, None, stream())
    kleos.adapter_products_backward(c.dy, c.x, c.u, c.offsets, c.adapter, c.a, c.b, None, c.dbase, c.dx, stream=stream())
    assert torch.equal(c.y, y) and torch.equal(c.dx, dx)
    kleos.adapter_products(c.x, c.offsets, c.adapter, c.a, c.b, None, c.base, c.base, None, stream())
    kleos.adapter_products_backward(c.dy, c.x, c.u, c.offsets, c.adapter, c.a, c.b, None, c.dbase, c.dbase, stream=stream())
    assert torch.equal(c.base, y) and torch.equal(c.dbase, dx)
    c.base, c.dbase = None, None
    c.all().verify()


@pytest.mark.parametrize("dtype", list(DT))
def test_what_lies_in_rows_of_others(dtype):
    """NaN in the rows of nobody and of requests without an adapter, infinities in adapters that no request has: neither is
    multiplied in."""
    c = Case([20, 33, 7, 64], [1, -1, 1, 0], 3, 16, 136, 264, dtype, first=3, spare=6)
    out = c.of < 0
    c.x[out], c.dy[out] = NAN, NAN
    c.a[2], c.b[2] = float("inf"), NAN
    c.all()
    assert torch.equal(c.y[out], c.base[out]) and torch.equal(c.dx[out], c.dbase[out]) and bool((c.u[out] == 0).all())
    assert bool((c.da[2] == 0).all()) and bool((c.db[2] == 0).all())
    for t in (c.y, c.dx, c.u, c.da, c.db):
        assert bool(torch.isfinite(t).all())


@pytest.mark.parametrize("dtype", list(DT))
def test_one_row_that_is_not_a_number(dtype):
    c = Case([20, 33], [1, 0], 2, 16, 136, 264, dtype).all()
    y, dx = c.y.clone(), c.dx.clone()
    c.x[5, 100], c.dy[5, 100] = NAN, float("inf")
    c.all()
    keep = torch.arange(53, device="cuda") != 5
    assert torch.equal(c.y[keep], y[keep]) and torch.equal(c.dx[keep], dx[keep])
    assert bool(torch.isnan(c.y[5]).all()) and not bool(torch.isfinite(c.dx[5]).any())
    assert bool(torch.isfinite(c.da[0]).all()) and bool(torch.isfinite(c.db[0]).all())


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_inner_values_past_the_element_types_range(dtype):
    """u far above 65504 (or far below the smallest fp16 value) is no infinity (or zero) on its way."""
    for x, a, b in ((5, 11, -14), (-5, -10, 12)):  # u is about 2^(x + a)
        c = Case([20, 33], [1, 0], 2, 16, 136, 264, dtype)
        c.x *= 2.0 ** x
        c.a *= 2.0 ** a
        c.b *= 2.0 ** b
        c.forward()
        c.da = c.db = None
        c.dy.zero_()
        kleos.adapter_products_backward(c.dy, c.x, c.u, c.offsets, c.adapter, c.a, c.b, c.scale, c.dbase, c.dx, stream=stream())
        c.verify()


def test_nothing_to_do():
    c = Case([0, 0], [0, 1], 2, 16, 24, 40)
    c.all()
    assert bool((c.da == 0).all()) and bool((c.db == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_differences(dtype):
    """dA and dB are the slopes of the sum of dy y: central differences, which are exact up to rounding as y is linear in each."""
    c = Case([40, 25], [1, 0], 2, 16, 72, 80, dtype, grads=torch.float32)
    c.all()
    c2 = Case([40, 25], [1, 0], 2, 16, 72, 80, "fp32")
    for n in ("x", "dy", "base", "a", "b", "scale"):
        getattr(c2, n).copy_(getattr(c, n).float())
    g = gen(3)
    for name, grad in (("a", c.da), ("b", c.db)):
        way = torch.randn(grad.shape, generator=g, device="cuda")
        sums = []
        for sign in (1, -1):
            at = getattr(c2, name).clone()
            getattr(c2, name).add_(way, alpha=sign)
            c2.forward()
            sums.append(float((c2.dy.double() * c2.y.double()).sum()))
            setattr(c2, name, at)
        got, want = (sums[0] - sums[1]) / 2, float((grad.double() * way.double()).sum())
        # y of both signs is rounded to 2^-24 of up to about 40 each, summed at random over 65 x 72 values; in bf16 u and v are rounded
        # to 2^-9 of themselves, so that the gradients are off by that part of their 2-norm at most, in a direction of their own
        part = 1e-4 if dtype == "fp32" else 2.0 ** -8
        assert abs(got - want) <= part * float(grad.double().norm() * way.double().norm())


@pytest.mark.parametrize("dtype", list(DT))
def test_the_same_bits(dtype):
    lengths, which = _uneven(3000, 9, 4)
    c = Case(lengths, which, 4, 16, 264, 328, dtype).all()
    first = [t.clone() for t in (c.y, c.u, c.dx, c.da, c.db)]
    for _ in range(3):
        c.all()
        assert all(torch.equal(a, b) for a, b in zip(first, (c.y, c.u, c.dx, c.da, c.db)))


def test_offsets_that_say_too_much():
    """What offsets say outside the matrices is not read or written: neighbours keep what was there."""
    c = Case([20, 33], [1, 0], 2, 16, 136, 264, spare=10)
    c.offsets.copy_(torch.tensor([-5, 30, 10 ** 9], dtype=torch.int32))
    c.of = torch.tensor([1] * 30 + [0] * 33, device="cuda")
    c.all().verify()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lengths", [[1] * 20, [300, 200], [12000, 9000]])
def test_long_sums(lengths, dtype):
    """u is a 32-bit result: the matrix unit's running sums, which it cuts off (up to about 2^-27 of the sum of magnitudes a term), are
    of at most 256 terms each, and of a warp's share of 8192 that are added up in 32 bits: 2^-19 of terms of one sign at worst."""
    c = Case(lengths, [i % 2 for i in range(len(lengths))], 2, 16, 64, 8192, dtype)
    c.x.copy_(c.x.abs())
    c.a.copy_(c.a.abs())
    c.forward()
    for l in range(2):
        mine = c.of == l
        want = c.x[mine].double() @ c.a[l].double().t()
        assert float(((c.u[mine].double() - want) / want).abs().max()) <= 2.0 ** -19
