"""The activation between an expert's products and its gradient against 64 bits."""
import math

import pytest
import torch

from aristos_b200 import kleos
from tests.operator_util import DT, EPS, check, gen, randn, stream, wide

pytestmark = pytest.mark.gpu


def reference(g, act, fast):
    """Value, slope and bounds on their 32-bit errors.

    SiLU: expf is within 2 ulp (2^-22), its sum, quotient and products round 2^-24 each; 16-bit types use __expf, within 2 + 1.173 |z|
    ulp, and __fdividef, within 2 ulp: 2^-17 in all up to |z| = 40.  GELU: erfcf is within 4 ulp, its argument carries two
    roundings, which the tail multiplies by z^2; the same for the slope's exponential."""
    if act == "relu":
        return g.clamp(min=0), (g > 0).double(), torch.zeros_like(g), torch.zeros_like(g)
    if act == "gelu":
        n = 0.5 * torch.special.erfc(-g * 0.5 ** 0.5)  # (torch.special.ndtr is 0.5 (1 + erf) on the GPU: zero below -8.3)
        d = torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
        rel = (12 + 2 * g * g) * EPS
        return g * n, n + g * d, rel * (g * n).abs(), rel * (n + (g * d).abs())
    p, q = torch.sigmoid(g), torch.sigmoid(-g)
    rel = 2.0 ** -17 if fast else 12 * EPS
    return g * p, p * (1 + g * q), rel * (g * p).abs(), rel * p * (1 + g.abs() * q)


def _run(z, dh, act, gated, h, dz):
    kleos.activation(z, act, h, stream())
    kleos.activation_backward(dh, z, act, dz, stream())
    I = h.shape[1]
    g, u, d = z[:, :I].double(), z[:, I:].double() if gated else torch.ones_like(h, dtype=torch.float64), dh.double()
    f, slope, df, ds = reference(g, act, z.dtype != torch.float32)
    check(h, f * u, (df + EPS * f.abs()) * u.abs(), "h")
    first = (ds + 2 * EPS * slope.abs()) * (d * u).abs()
    check(dz[:, :I], d * u * slope, first, "dz")
    if gated:
        check(dz[:, I:], d * f, (df + EPS * f.abs()) * d.abs(), "dz of the other half")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", list(kleos.ACTIVATIONS))
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("R,I,pad", [(1, 1, 0), (1, 2048, 0), (3, 7, 0), (37, 100, 3), (301, 264, 8), (5, 1087, 5), (700, 512, 2), (2, 9000, 0), (4097, 40, 0)])
def test_values_and_gradients(R, I, pad, gated, act, dtype):
    g, dt, cols = gen(R + I), DT[dtype], I * (2 if gated else 1)
    z, dh = randn(g, (R, cols), dt, 2.0), randn(g, (R, I), dt)
    h, dz = torch.full((R, I), float("nan"), dtype=dt, device="cuda"), torch.full((R, cols), float("nan"), dtype=dt, device="cuda")
    if pad:
        z, dh, h, dz = wide(z, pad, 0), wide(dh, 0, pad), wide(h, pad, pad), wide(dz, 0, pad)
    _run(z, dh, act, gated, h, dz)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", list(kleos.ACTIVATIONS))
def test_range(act, dtype):
    """From far below to far above, zero and the smallest values among them."""
    one = torch.cat([torch.linspace(-9, 9, 1001), torch.tensor([0.0, -0.0, 6e-5, -6e-5, 40.0, 30.5])]).to("cuda").to(DT[dtype])
    z = torch.stack([one, one.flip(0)])
    ones = torch.ones_like(z)
    _run(z, ones, act, False, torch.empty_like(z), torch.empty_like(z))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", list(kleos.ACTIVATIONS))
def test_infinities_and_nan(act, dtype):
    z = torch.tensor([[float("inf"), float("nan"), -60000.0, 60000.0]], device="cuda").to(DT[dtype])
    h, dz = torch.zeros_like(z), torch.zeros_like(z)
    kleos.activation(z, act, h, stream())
    kleos.activation_backward(torch.ones_like(z), z, act, dz, stream())
    assert h[0, 0] == float("inf") and bool(torch.isnan(h[0, 1])) and h[0, 2] == 0 and h[0, 3] == z[0, 3]
    assert bool(torch.isnan(dz[0, 1])) == (act != "relu") and dz[0, 2] == 0 and dz[0, 3] == 1


def test_differences():
    """The slopes are those of the values: central differences in floats."""
    z = torch.linspace(-4, 4, 801, device="cuda")[None].contiguous()
    step = 2.0 ** -8
    for act in ("gelu", "silu"):
        up, down, dz = (torch.empty_like(z) for _ in range(3))
        kleos.activation(z + step, act, up, stream())
        kleos.activation(z - step, act, down, stream())
        kleos.activation_backward(torch.ones_like(z), z, act, dz, stream())
        # third derivatives up to 2, times step^2 / 6; rounding of values up to 4 over 2 step
        assert float(((up - down) / (2 * step) - dz).abs().max()) <= 2 * step ** 2 / 6 + 8 * 4 * EPS / step
