"""The activation, the layer for a few tokens and the adapters as they are used together and beside the other operators: chains,
several streams, graphs, elements around the outputs."""
import pytest
import torch

from aristos_b200 import kleos
from examples.moe_block import MoEBlock
from tests.operator_util import DT, HALF_UNIT, gen, randn, stream
from tests.test_gpu_adapters import Case
from tests.test_gpu_moe_tokens import Layer
from tests.test_gpu_operator_bounds import Outputs

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- chains
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act,gated", [("silu", True), ("gelu", False)])
@pytest.mark.parametrize("T", [1, 7, 128])
def test_layer_is_the_chain_of_its_operators(T, act, gated, dtype):
    """moe_tokens against sort, gather, products, activation, products and combine with the experts that it chose: each way rounds its
    results, the chain its hidden and expert results before them; 2-norm."""
    layer = Layer(T, 264, 328, 12, 3, dtype, act, gated, bias=True).run()
    dt, E, K, I, H = layer.x.dtype, layer.E, layer.K, layer.I, layer.H
    new = lambda *shape, dtype=dt: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    offsets, row_of, s = new(E + 1, dtype=torch.int32), new(T, K, dtype=torch.int32), stream()
    kleos.sort_tokens(layer.topk, E, offsets, row_of, None, s)
    rows, z, h, y, out = new(T * K, H), new(T * K, layer.w1.shape[1]), new(T * K, I), new(T * K, H), new(T, H)
    kleos.gather_tokens(layer.x, row_of, offsets, rows, s)
    kleos.expert_products(rows, offsets, layer.w1, layer.b1, z, s)
    kleos.activation(z, act, h, s)
    kleos.expert_products(h, offsets, layer.w2, layer.b2, y, s)
    kleos.combine_tokens(y, row_of, layer.weights, out, s)
    off = float((out.double() - layer.out.double()).norm() / layer.out.double().norm())
    assert off <= max(5 * HALF_UNIT[dt], 4e-6)  # (roundings of z, h, y and two of out; floats: sums in another order)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_adapters_beside_a_projection(dtype):
    """A shared projection (one expert's products), the adapters onto it in place, and the gradients of both onto each other."""
    c = Case([37, 1, 90], [1, 0, 1], 2, 16, 264, 328, dtype)
    g = gen(9)
    w = randn(g, (1, c.N, c.K), c.dt, c.K ** -0.5)
    one = torch.tensor([0, c.rows], dtype=torch.int32, device="cuda")
    y, dx, s = torch.empty_like(c.y), torch.empty_like(c.dx), stream()
    kleos.expert_products(c.x, one, w, None, y, s)
    c.base = y.clone()
    kleos.adapter_products(c.x, c.offsets, c.adapter, c.a, c.b, c.scale, y, y, c.u, s)
    kleos.expert_products_dx(c.dy, one, w, dx, s)
    c.dbase = dx.clone()
    kleos.adapter_products_backward(c.dy, c.x, c.u, c.offsets, c.adapter, c.a, c.b, c.scale, dx, dx, c.da, c.db, c.workspace, s)
    c.y, c.dx = y, dx
    c.verify()


# 2-norm errors: each of the about ten roundings to the element type on the longest way is half a unit, 2^-9 or 2^-12 of the
# 2-norm on average.
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-6), (torch.bfloat16, 2e-2), (torch.float16, 2.5e-3)])
@pytest.mark.parametrize("act,gated", [("silu", True), ("gelu", True), ("silu", False)])
def test_block_with_gated_experts(act, gated, dtype, tol):
    T, H, inner, E, K = 150, 128, 192, 6, 2
    block = MoEBlock(H, inner, E, K, dtype, seed=3, act=act, gated=gated)
    g = gen(11)
    x, dout = (torch.randn(T, H, generator=g, device="cuda").to(dtype) for _ in range(2))
    block.params["b1"] += (torch.randn(block.params["b1"].shape, generator=g, device="cuda") * 0.1).to(dtype)
    y, grads = block.forward(x), block.backward(dout)
    ids = block.kept["ids"].long()
    p = {n: v.double().requires_grad_() for n, v in block.params.items()}
    xx = x.double().requires_grad_()
    h = torch.nn.functional.layer_norm(xx, (H,), p["norm_w"], p["norm_b"], block.eps)
    weights = torch.softmax((h @ p["gate"].t()).gather(1, ids), 1)
    want = xx
    f = torch.nn.functional.silu if act == "silu" else torch.nn.functional.gelu
    for k in range(K):
        e = ids[:, k]
        u = torch.einsum("th,tih->ti", h, p["w1"][e]) + p["b1"][e]
        a = f(u[:, :inner]) * u[:, inner:] if gated else f(u)
        want = want + weights[:, k, None] * torch.einsum("ti,thi->th", a, p["w2"][e])
    want.backward(dout.double())
    assert float((y.double() - want.detach()).norm() / want.detach().norm()) <= tol
    for name, grad in grads.items():
        ref = xx.grad if name == "x" else p[name].grad
        assert float((grad.double() - ref).norm()) <= tol * float(ref.norm()), name
    few = x[:9].contiguous()
    assert float((block.answer(few).double() - want.detach()[:9]).norm() / want.detach()[:9].norm()) <= tol


# ---------------------------------------------------------------- streams and graphs
SIZES = {"layer": lambda: Layer(40, 264, 328, 8, 2, "bf16"), "token": lambda: Layer(1, 512, 520, 16, 2, "fp16", bias=True), "few columns": lambda: Layer(33, 256, 64, 64, 4, "bf16"),
         "float layer": lambda: Layer(9, 264, 72, 8, 2, "fp32"), "odd layer": lambda: Layer(17, 77, 99, 5, 2, "bf16"), "decode": lambda: Case([1] * 30, [i % 4 - 1 for i in range(30)], 3, 16, 264, 520),
         "prompts": lambda: Case([300, 77, 1], [1, 0, 1], 2, 32, 264, 328, "fp16", spare=5), "many": lambda: Case([6000, 4000], [0, 1], 2, 16, 136, 200),
         "odd adapters": lambda: Case([40, 9], [1, 0], 2, 12, 99, 77, "fp32")}


def _run(c):
    if isinstance(c, Layer):
        c.run()
        return [c.out, c.topk, c.weights]
    c.all()
    return [c.y, c.u, c.dx, c.da, c.db]


def _renew(c, seed):
    g = gen(seed)
    for t in (c.x,) if isinstance(c, Layer) else (c.x, c.dy, c.base, c.dbase):
        t.copy_(torch.randn(t.shape, generator=g, device="cuda"))


def test_all_at_once():
    cases = {n: make() for n, make in SIZES.items()}
    want = {n: [t.clone() for t in _run(c)] for n, c in cases.items()}
    side = {n: torch.cuda.Stream() for n in cases}
    for s in side.values():
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for n, c in cases.items():
            with torch.cuda.stream(side[n]):
                _run(c)
    torch.cuda.synchronize()
    for n, c in cases.items():
        outs = [c.out, c.topk, c.weights] if isinstance(c, Layer) else [c.y, c.u, c.dx, c.da, c.db]
        assert all(torch.equal(a, b) for a, b in zip(want[n], outs)), n


@pytest.mark.parametrize("name", list(SIZES))
def test_in_a_graph(name):
    c, s = SIZES[name](), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _run(c)
    torch.cuda.synchronize()
    graph, twice = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    for g, n in ((graph, 1), (twice, 2)):  # (two graphs that share the workspace, one after the other)
        with torch.cuda.graph(g, stream=s):
            for _ in range(n):
                outs = _run(c)
    for seed in (2, 3):
        _renew(c, seed)
        want = [t.clone() for t in _run(c)]
        for g in (graph, twice):
            c.workspace.fill_(0xFF)
            for t in outs:
                t.fill_(-1)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, outs)), name


def test_activation_in_a_graph():
    g = gen(1)
    z, dh, h, dz = randn(g, (300, 200), torch.bfloat16), randn(g, (300, 100), torch.bfloat16), torch.empty(300, 100, dtype=torch.bfloat16, device="cuda"), torch.empty(300, 200, dtype=torch.bfloat16, device="cuda")

    def both():
        kleos.activation(z, "silu", h, stream())
        kleos.activation_backward(dh, z, "silu", dz, stream())

    both()
    torch.cuda.synchronize()
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=s):
        both()
    z.copy_(torch.randn(z.shape, generator=g, device="cuda"))
    both()
    want = h.clone(), dz.clone()
    h.zero_(), dz.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(h, want[0]) and torch.equal(dz, want[1])


def test_a_call_after_what_it_reads_was_written():
    """Weights, tokens and h of one call come from kernels right before it, time and again."""
    layer, s = Layer(20, 512, 264, 8, 2, "bf16"), torch.cuda.Stream()
    other = Layer(20, 512, 264, 8, 2, "bf16", seed=7)
    want = [layer.run().out.clone(), other.run().out.clone()]
    one = Layer(20, 512, 264, 8, 2, "bf16")
    with torch.cuda.stream(s):
        for i in range(20):
            src = (layer, other)[i % 2]
            for n in ("x", "gate", "w1", "w2"):
                getattr(one, n).copy_(getattr(src, n))
            one.run()
            assert torch.equal(one.out, want[i % 2])


# ---------------------------------------------------------------- elements around the outputs
PADS = [(0, 0), (8, 8), (16, 0), (3, 0), (0, 5), (2, 2)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("pads", PADS)
@pytest.mark.parametrize("R,I,gated", [(5, 8, True), (37, 100, False), (301, 264, True), (9, 1087, True)])
def test_around_activations(R, I, gated, pads, dtype):
    g, dt, out = gen(R + I), DT[dtype], Outputs()
    wide = I * (2 if gated else 1)
    z, dh, h, dz = randn(g, (R, wide), dt), randn(g, (R, I), dt), out.rows(R, I, dt, *pads), out.rows(R, wide, dt, *pads)
    kleos.activation(z, "silu", h, stream())
    kleos.activation_backward(dh, z, "silu", dz, stream())
    out.check()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("pads", PADS)
@pytest.mark.parametrize("T,H,I,E,K,gated", [(1, 264, 328, 8, 2, True), (40, 136, 264, 6, 3, False), (128, 77, 99, 5, 2, True), (9, 2048, 64, 32, 2, True)])
def test_around_layers(T, H, I, E, K, gated, pads, dtype):
    layer, out = Layer(T, H, I, E, K, dtype, gated=gated), Outputs()
    layer.out, layer.topk, layer.weights = out.rows(T, H, layer.x.dtype, *pads), out.flat((T, K), torch.int32), out.flat((T, K), torch.float32)
    n = kleos.moe_tokens_workspace(T, I, K)
    whole = torch.full((n + 512,), 0xA5, dtype=torch.uint8, device="cuda")
    layer.workspace = whole[256:256 + n]
    layer.run()
    out.check()
    assert bool((whole[:256] == 0xA5).all()) and bool((whole[256 + n:] == 0xA5).all())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("pads", PADS)
@pytest.mark.parametrize("lengths,r,N,K", [([1] * 20, 16, 264, 328), ([100, 3, 0, 70], 32, 136, 264), ([5000, 4800], 16, 72, 136), ([40, 9], 12, 99, 77), ([30, 64], 128, 264, 136)])
def test_around_adapters(lengths, r, N, K, pads, dtype):
    c, out = Case(lengths, [i % 3 - 1 for i in range(len(lengths))], 2, r, N, K, dtype, first=1, spare=3), Outputs()
    f32, n = torch.float32, kleos.adapter_products_workspace(c.rows, r)
    c.y, c.dx, c.u = out.rows(c.rows, N, c.dt, *pads), out.rows(c.rows, K, c.dt, *pads), out.flat((c.rows, r), f32)
    c.da, c.db = out.flat((2, r, K), c.dt), out.flat((2, N, r), c.dt)
    whole = torch.full((n + 512,), 0xA5, dtype=torch.uint8, device="cuda")
    c.workspace = whole[256:256 + n]
    c.all()
    out.check()
    assert bool((whole[:256] == 0xA5).all()) and bool((whole[256 + n:] == 0xA5).all())
