"""Matrices past 2^31 elements: what lies behind is read and written where it lies."""
import pytest
import torch

from aristos_b200 import kleos
from tests.operator_util import EPS, HALF_UNIT, check, gen, randn, stream
from tests.test_gpu_activation import reference
from tests.test_gpu_moe_tokens import Layer

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_activation():
    R, I = 300000, 4096  # z has 2.46e9 elements
    z, h = torch.zeros(R, 2 * I, dtype=BF16, device="cuda"), torch.empty(R, I, dtype=BF16, device="cuda")
    last = randn(gen(1), (50, 2 * I), BF16)
    z[-50:] = last
    kleos.activation(z, "silu", h, stream())
    g, u = last[:, :I].double(), last[:, I:].double()
    f, _, df, _ = reference(g, "silu", True)
    check(h[-50:], f * u, (df + EPS * f.abs()) * u.abs(), "h")
    assert bool((h[:1000] == 0).all())
    dz = torch.empty_like(z)
    kleos.activation_backward(h, z, "silu", dz, stream())
    check(dz[-50:, I:], h[-50:].double() * f, (df + EPS * f.abs()) * h[-50:].double().abs(), "dz")


@pytest.mark.parametrize("requests", [1, 65600])
def test_adapters(requests):
    """One prompt, and a request a row."""
    rows, K, N, r = 65600, 32768, 72, 16
    g = gen(2)
    x, dx = torch.zeros(rows, K, dtype=BF16, device="cuda"), torch.empty(rows, K, dtype=BF16, device="cuda")
    x[-50:], dy = randn(g, (50, K), BF16), torch.zeros(rows, N, dtype=BF16, device="cuda")
    dy[-50:] = randn(g, (50, N), BF16)
    a, b = randn(g, (2, r, K), BF16, K ** -0.5), randn(g, (2, N, r), BF16, r ** -0.5)
    requests = min(requests, 65536)
    offsets = torch.linspace(0, rows, requests + 1, device="cuda").to(torch.int32) if requests == 1 else torch.cat([torch.arange(requests, device="cuda"), torch.tensor([rows], device="cuda")]).to(torch.int32)
    adapter = torch.ones(requests, dtype=torch.int32, device="cuda")
    y, u = torch.empty(rows, N, dtype=BF16, device="cuda"), torch.empty(rows, r, device="cuda")
    kleos.adapter_products(x, offsets, adapter, a, b, None, None, y, u, stream())
    ws = torch.empty(kleos.adapter_products_workspace(rows, r), dtype=torch.uint8, device="cuda")
    da, db = torch.empty_like(a), torch.empty_like(b)
    kleos.adapter_products_backward(dy, x, u, offsets, adapter, a, b, None, None, dx, da, db, ws, stream())
    xx, yy, A, B = x[-50:].double(), dy[-50:].double(), a[1].double(), b[1].double()
    uu, v, half = xx @ A.t(), yy @ B, HALF_UNIT[BF16]
    du, dv = K * EPS * (xx.abs() @ A.abs().t()), N * EPS * (yy.abs() @ B.abs())
    check(u[-50:], uu, du, "u")
    check(y[-50:], uu @ B.t(), (du + half * (uu.abs() + du)) @ B.abs().t() + 20 * EPS * (uu.abs() @ B.abs().t()), "y")
    check(dx[-50:], v @ A, (dv + half * (v.abs() + dv)) @ A.abs() + 20 * EPS * (v.abs() @ A.abs()), "dx")
    check(da[1], v.t() @ xx, (dv + half * (v.abs() + dv)).t() @ xx.abs() + 100 * EPS * (v.abs().t() @ xx.abs()), "da")
    check(db[1], yy.t() @ uu, yy.abs().t() @ (du + half * (uu.abs() + du)) + 100 * EPS * (yy.abs().t() @ uu.abs()), "db")
    assert bool((y[:-50] == 0).all()) and bool((da[0] == 0).all())


def test_experts():
    layer = Layer(3, 4608, 4096, 2, 1)  # grown to 64 experts: W1 has 2.4e9 elements
    one, two = layer.w1[0].clone(), layer.w2[0].clone()
    layer.E = 64
    layer.gate = randn(gen(3), (64, 4608), BF16, 4608 ** -0.5)
    layer.w1, layer.w2 = torch.zeros(64, 8192, 4608, dtype=BF16, device="cuda"), torch.zeros(64, 4608, 4096, dtype=BF16, device="cuda")
    layer.w1[63], layer.w2[63] = one, two
    layer.gate_bias = torch.zeros(64, device="cuda")
    layer.gate_bias[63] = 50.0
    layer.run().verify()
    assert bool((layer.topk == 63).all()) and bool((layer.out != 0).any())
