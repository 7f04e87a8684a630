"""What the float products promise beside the general bounds: the precision of fp32 multiply-adds for long sums, the
infinities and NaNs of 32-bit arithmetic, and what is left of operands near the ends of the exponents' range."""
import pytest
import torch

from aristos_b200 import kleos
from tests.operator_util import EPS, gen, stream
from tests.test_gpu_expert_products import _case, _dw, _dx, _forward

pytestmark = pytest.mark.gpu

# The h h sums are cut off at each of the eight steps of sixteen terms between two read-backs, by half a unit in 2^23 on average of
# a sum that is half as large on the way: 2.4e-7 for terms of one sign.  The parts' additions, rounded to nearest, add
# sqrt(terms / 128) halves of 2^-24, 1.2e-7 for 8192 terms; the products that are left out and the small sums' own cuts (2^-6 of 32
# steps) about as much again.  6e-7 of the 2-norm is allowed, for terms of both signs too; operands of two parts are
# 1.7e-5 away, TF32's 2.9e-4.
LONG = 6e-7


def _inputs(counts, N, K, kind):
    c = _case(counts, N, K, "fp32", bias=False)
    if kind == "one sign":
        for name in ("x", "dy", "w"):
            c[name].abs_()
    return c


def _off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("kind", ["both signs", "one sign"])
@pytest.mark.parametrize("counts,N,K", [([300], 512, 520), ([257, 0, 64, 129], 264, 2048), ([400], 2048, 1088), ([129, 200], 136, 8192),
                                        ([300, 31], 8192, 136), ([513], 5000, 4096)])
def test_products_of_long_sums(counts, N, K, kind):
    c = _inputs(counts, N, K, kind)
    y, dx = _forward(c), _dx(c)
    for e in range(c["E"]):
        r = slice(c["at"][e], c["at"][e + 1])
        if counts[e]:
            w = c["w"][e].double()
            assert _off(y[r], c["x"][r].double() @ w.t()) <= LONG, ("y", e)
            assert _off(dx[r], c["dy"][r].double() @ w) <= LONG, ("dx", e)


@pytest.mark.parametrize("kind", ["both signs", "one sign"])
@pytest.mark.parametrize("counts", [[512], [1500, 33], [4097, 0, 300], [8192]])
def test_weight_gradients_of_long_sums(counts, kind):
    c = _inputs(counts, 264, 200, kind)
    dw, _ = _dw(c, bias=False)
    for e in range(c["E"]):
        r = slice(c["at"][e], c["at"][e + 1])
        if counts[e]:
            assert _off(dw[e], c["dy"][r].double().t() @ c["x"][r].double()) <= LONG, e


def _same_pattern(got, want, what):
    for name, f in (("+inf", torch.isposinf), ("-inf", torch.isneginf), ("NaN", torch.isnan)):
        assert torch.equal(f(got), f(want)), f"{name} of {what}"


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("counts,N,K", [([300, 45], 264, 520), ([2, 1], 264, 520), ([40], 39, 50), ([3, 60], 256, 2048)])
def test_lone_infinities(counts, N, K, dtype):
    """One infinite operand among finite ones makes infinities of the products' signs, NaN where it meets a zero or an infinity of
    the other sign."""
    c = _case(counts, N, K, dtype)
    inf = float("inf")
    x, dy, w = c["x"], c["dy"], c["w"]
    x[0, 7], x[1, 3], dy[0, 5], dy[1, 0] = inf, -inf, -inf, inf
    x[2, K - 1], x[2, 0], dy[2, N - 1], dy[2, 2] = inf, -inf, inf, inf
    w[0, 4, 9], w[-1, N - 1, K - 1], w[0, 11, 7] = -inf, inf, 0.0
    got = _forward(c), _dx(c), _dw(c, bias=False)[0]
    for e in range(c["E"]):
        r = slice(c["at"][e], c["at"][e + 1])
        xe, de, we = x[r].double(), dy[r].double(), w[e].double()
        _same_pattern(got[0][r], xe @ we.t() + c["bias"][e].double(), "y")
        _same_pattern(got[1][r], de @ we, "dx")
        _same_pattern(got[2][e], de.t() @ xe, "dw")


@pytest.mark.parametrize("size", [2.0 ** -118, 2.0 ** -126, 2.0 ** -131])
def test_operands_near_the_least(size):
    """The parts of an operand are multiples of 2^-133, so that is what it is held to below 2^-110; the other operand is as large as
    makes the products ordinary."""
    c = _case([300], 264, 136, "fp32", bias=False)
    x, dy, w = c["x"].double() * size, c["dy"].double() * size, c["w"].double()
    c["x"], c["dy"], c["w"] = x.float(), dy.float(), (w * 2.0 ** 100).float()
    for got, a, b in ((_forward(c), c["x"], c["w"][0].t()), (_dx(c), c["dy"], c["w"][0])):
        a, b = a.double(), b.double()
        bound = 2.0 ** -133 * b.abs().sum(0) + (2 * b.shape[0] + 8) * EPS * (a.abs() @ b.abs())
        assert bool(((got.double() - a @ b).abs() <= bound).all())
    big = _case([300], 264, 136, "fp32", bias=False)
    small, big["x"] = big["dy"], big["x"] * 2.0 ** 100
    big["dy"] = small * size
    dw = _dw(big, bias=False)[0][0].double()
    a, b = big["dy"].double().t(), big["x"].double()
    assert bool(((dw - a @ b).abs() <= 2.0 ** -133 * b.abs().sum(0) + (2 * 300 + 8) * EPS * (a.abs() @ b.abs())).all())


def test_operands_near_the_greatest():
    c = _case([300], 264, 136, "fp32", bias=False)
    c["x"] = (c["x"].double().clamp(-3, 3) * 2.0 ** 126).float()
    c["w"] *= 2.0 ** -9
    a, b = c["x"].double(), c["w"][0].double().t()
    got = _forward(c).double()
    assert bool(torch.isfinite(got).all())
    assert bool(((got - a @ b).abs() <= (2 * 136 + 8) * EPS * (a.abs() @ b.abs())).all())
