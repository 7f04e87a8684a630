"""Layer norm and its gradients against 64-bit arithmetic."""
import pytest
import torch

from aristos_b200 import kleos
from tests.operator_util import DT, EPS, check, gen, randn, refused, stream, wide

pytestmark = pytest.mark.gpu

CHAIN = 64 * EPS  # additions of a row one after the other: at most 32 of a thread, then the tree's ten


def _run(x, w, b, eps, dy, param, pad=(0, 0)):
    R, H = x.shape
    y, dx = (wide(torch.zeros_like(x), *pad) for _ in range(2))
    mean, rstd = (torch.full((R,), 9.0, device="cuda") for _ in range(2))
    dw, db = (torch.full((H,), 9.0, dtype=param, device="cuda") for _ in range(2))
    ws = torch.full((kleos.layer_norm_workspace(H),), 255, dtype=torch.uint8, device="cuda")
    kleos.layer_norm(x, w, b, eps, y, mean, rstd, stream())
    kleos.layer_norm_backward(dy, x, w, mean, rstd, dx, dw, db, ws, stream())
    return y, mean, rstd, dx, dw, db


def _reference(x, w, b, eps, dy):
    x, dy = x.double(), dy.double()
    w = torch.ones(x.shape[1], device="cuda").double() if w is None else w.double()
    b = torch.zeros(x.shape[1], device="cuda").double() if b is None else b.double()
    m = x.mean(1, keepdim=True)
    r = ((x - m).square().mean(1, keepdim=True) + eps).rsqrt()
    h, g = (x - m) * r, dy * w
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    values = (h * w + b, m[:, 0], r[:, 0], dx, (dy * h).sum(0), dy.sum(0))
    # bounds on the errors before rounding
    size = r * x.abs().amax(1, keepdim=True)
    eh = CHAIN * (size + h.abs() * (1 + size))
    em = eh.amax(1, keepdim=True)
    mg, mgh = g.abs().mean(1, keepdim=True), (g * h).abs().mean(1, keepdim=True)
    n = (x.shape[0] + 64) * EPS
    bounds = (w.abs() * eh + 4 * EPS * ((h * w).abs() + b.abs()), CHAIN * x.abs().mean(1), r[:, 0] * CHAIN * (1 + size[:, 0]),
              r * (2 * CHAIN * (g.abs() + mg + h.abs() * mgh) + em * (mgh + (h.abs() + em) * mg)) + CHAIN * (1 + size) * dx.abs(),
              n * (dy * h).abs().sum(0) + (dy.abs() * eh).sum(0), n * dy.abs().sum(0))
    return values, bounds


NAMES = ("y", "mean", "rstd", "dx", "dweight", "dbias")


def _compare(x, w, b, eps, dy, param, pad=(0, 0)):
    for name, got, ref, bound in zip(NAMES, _run(x, w, b, eps, dy, param, pad), *_reference(x, w, b, eps, dy)):
        check(got, ref, bound, name)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("R,H", [(1, 1), (3, 2), (2, 31), (1, 64), (700, 64), (5, 100), (33, 255), (9, 256), (300, 512), (17, 1000), (8, 1087),
                                 (1, 2048), (601, 2048), (40, 4096), (3, 5000), (6, 8192), (5, 8193), (4, 16384), (7, 20001), (600, 16392)])
def test_rows_and_columns(dtype, R, H):
    g = gen(R * 31 + H)
    dt = DT[dtype]
    param = torch.float32 if (R + H) % 2 else dt
    x = randn(g, (R, H), dt, 2.0, 0.5)
    _compare(x, randn(g, (H,), param, 0.3, 1.0), randn(g, (H,), param), 1e-5, randn(g, (R, H), dt), param)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("H,left,right", [(512, 8, 0), (512, 1, 0), (1087, 0, 5), (96, 3, 2), (2048, 0, 7)])
def test_rows_inside_a_wider_matrix(dtype, H, left, right):
    g = gen(H + left)
    dt = DT[dtype]
    x, dy = (wide(randn(g, (37, H), dt), left, right) for _ in range(2))
    _compare(x, randn(g, (H,), dt, 0.3, 1.0), randn(g, (H,), dt), 1e-5, dy, dt, (left, right))


@pytest.mark.parametrize("dtype", list(DT))
def test_without_parameters_or_statistics(dtype):
    g = gen(3)
    x, dy = (randn(g, (19, 768), DT[dtype]) for _ in range(2))
    _compare(x, None, None, 1e-6, dy, torch.float32)
    y, z = torch.empty_like(x), torch.empty_like(x)
    kleos.layer_norm(x, None, None, 1e-6, y, stream=stream())
    mean, rstd = torch.empty(19, device="cuda"), torch.empty(19, device="cuda")
    kleos.layer_norm(x, None, None, 1e-6, z, mean, rstd, stream())
    assert torch.equal(y, z)
    dx, full = torch.empty_like(x), torch.empty_like(x)
    kleos.layer_norm_backward(dy, x, None, mean, rstd, dx, stream=stream())  # no parameters' gradients, no workspace
    db = torch.empty(768, device="cuda")
    ws = torch.empty(kleos.layer_norm_workspace(768), dtype=torch.uint8, device="cuda")
    kleos.layer_norm_backward(dy, x, None, mean, rstd, full, None, db, ws, stream())
    assert torch.equal(dx, full)
    check(db, dy.double().sum(0), (19 + 64) * EPS * dy.double().abs().sum(0), "dbias alone")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_constant_rows_and_large_means(dtype):
    """A variance of zero, and rows whose mean is a thousand times their spread."""
    g = gen(4)
    dt = DT[dtype]
    x = randn(g, (6, 1024), dt)
    x[0], x[1], x[2] = 0.0, 3.0, -7.5
    x[3] = (x[3].float() + 1000.0).to(dt)
    _compare(x, randn(g, (1024,), dt, 0.3, 1.0), randn(g, (1024,), dt), 1e-5, randn(g, (6, 1024), dt), dt)


def test_infinite_and_nan_values_stay_in_their_rows():
    g = gen(5)
    x = randn(g, (40, 2048), torch.bfloat16)
    y, z = torch.empty_like(x), torch.empty_like(x)
    kleos.layer_norm(x, None, None, 1e-5, y, stream=stream())
    x[7, 100], x[20, 3] = float("inf"), float("nan")
    kleos.layer_norm(x, None, None, 1e-5, z, stream=stream())
    others = [r for r in range(40) if r not in (7, 20)]
    assert torch.equal(y[others], z[others]) and bool(z[7].isnan().any()) and bool(z[20].isnan().all())


def test_no_rows():
    x = torch.empty(0, 64, device="cuda")
    dw, db = torch.ones(64, device="cuda"), torch.ones(64, device="cuda")
    e = torch.empty(0, device="cuda")
    kleos.layer_norm(x, None, None, 1e-5, x, stream=stream())
    ws = torch.empty(kleos.layer_norm_workspace(64), dtype=torch.uint8, device="cuda")
    kleos.layer_norm_backward(x, x, None, e, e, x, dw, db, ws, stream())
    assert not bool(dw.any()) and not bool(db.any())


def test_same_bits_every_time_and_on_another_stream():
    g = gen(6)
    x, dy = (randn(g, (3001, 1536), torch.bfloat16) for _ in range(2))
    w = randn(g, (1536,), torch.float32)
    one = _run(x, w, None, 1e-5, dy, torch.float32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        two = _run(x, w, None, 1e-5, dy, torch.float32)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(one, two):
        assert torch.equal(a, b)


def test_gradients_against_differences():
    """Central differences of the forward pass along random directions; the loss is <y, dy>.  With a step of 2^-5
    the third derivative (about ten for values, directions and gradients of size one) adds 2^-10 / 6 * 10 = 1.6e-3 of the
    gradient's norm, the forward's rounding 1e-6 of it; six times that is allowed."""
    g = gen(7)
    R, H = 24, 320
    x, dy = (randn(g, (R, H), torch.float32) for _ in range(2))
    w, b = randn(g, (H,), torch.float32, 0.3, 1.0), randn(g, (H,), torch.float32)
    _, _, _, dx, dw, db = _run(x, w, b, 1e-5, dy, torch.float32)

    def loss(x, w, b):
        y = torch.empty_like(x)
        kleos.layer_norm(x, w, b, 1e-5, y, stream=stream())
        return float((y.double() * dy.double()).sum())

    step = 2.0 ** -5
    for i, (grad, at) in enumerate(((dx, x), (dw, w), (db, b))):
        for seed in range(3):
            d = randn(gen(100 + seed), at.shape, torch.float32)
            ends = [[x, w, b], [x, w, b]]
            ends[0][i], ends[1][i] = at + step * d, at - step * d
            slope = (loss(*ends[0]) - loss(*ends[1])) / (2 * step)
            want = float((grad.double() * d.double()).sum())
            assert abs(slope - want) <= 1e-2 * float(grad.norm()) * float(d.norm()) / at.numel() ** 0.5, (i, seed, slope, want)


def test_refusals():
    x = torch.zeros(4, 64, device="cuda")
    y, m = torch.empty_like(x), torch.empty(4, device="cuda")
    w = torch.ones(64, device="cuda")
    ln, back = kleos.layer_norm, kleos.layer_norm_backward
    refused(-7, ln, x.double(), None, None, 1e-5, y.double())
    refused(-8, ln, x, w[:63], None, 1e-5, y)
    refused(-8, ln, x, w.bfloat16(), None, 1e-5, y)
    refused(-8, ln, x, w, w.bfloat16(), 1e-5, y)
    refused(-8, ln, x, w, None, -1.0, y)
    refused(-8, ln, x, w, None, float("nan"), y)
    refused(-8, ln, x, w, None, 1e-5, y[:3])
    refused(-8, ln, x, w, None, 1e-5, y.bfloat16())
    refused(-8, ln, x.t(), w[:4], None, 1e-5, y.t())
    refused(-8, ln, x, w, None, 1e-5, y, m[:3], m)
    refused(-8, ln, x.cpu(), None, None, 1e-5, y)
    refused(-8, ln, x[:1].expand(4, 64), None, None, 1e-5, y)
    refused(-8, back, x, x, w, m, m, y, w, w)                                                     # no workspace
    refused(-8, back, x, x, w, m, m, y, w, w, torch.empty(100, device="cuda"))                    # too small a one
    refused(-8, back, x, x, w, m.double(), m, y)


def test_rows_past_two_to_the_31_elements():
    R, H = 1100000, 2048
    g = gen(12)
    x = torch.ones(R, H, dtype=torch.bfloat16, device="cuda")
    dy = torch.zeros_like(x)
    x[-40:], dy[-40:] = randn(g, (40, H), x.dtype), randn(g, (40, H), x.dtype)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    w, b = randn(g, (H,), torch.float32, 0.3, 1.0), randn(g, (H,), torch.float32)
    dw, db = torch.empty(H, device="cuda"), torch.empty(H, device="cuda")
    ws = torch.empty(kleos.layer_norm_workspace(H), dtype=torch.uint8, device="cuda")
    kleos.layer_norm(x, w, b, 1e-5, y, mean, rstd, stream())
    kleos.layer_norm_backward(dy, x, w, mean, rstd, dx, dw, db, ws, stream())
    got = y[-40:], mean[-40:], rstd[-40:], dx[-40:], dw, db
    for name, v, ref, bound in zip(NAMES, got, *_reference(x[-40:], w, b, 1e-5, dy[-40:])):
        check(v, ref, bound, name)
    assert bool((y[:-40] == b.bfloat16()).all()) and not bool(dx[:-40].any())
