"""The operators on several streams at once and in graphs: the bits are those of the same calls one after the other."""
import pytest
import torch

from aristos_b200 import kleos
from tests.operator_util import DT, gen, randn, stream
from tests.test_gpu_expert_products import _case, _dw, _dx, _forward

pytestmark = pytest.mark.gpu

# (counts, N, K, type): sums split over a cluster, streamed weights, tiles of floats, many tiles, FP32 pipes
KINDS = {"split": ([31, 1, 96], 520, 2048, "bf16"), "streamed": ([1, 1], 2048, 2048, "bf16"), "few floats": ([8, 0, 9], 1024, 1024, "fp32"),
         "floats": ([300, 77], 512, 520, "fp32"), "many": ([300, 50, 0, 700], 512, 320, "fp16"), "odd": ([130, 9], 99, 77, "bf16")}


def _all(c):
    return (_forward(c), _dx(c), *_dw(c), *_dw(c, torch.float32))


def test_every_kind_of_product_at_once():
    cases = {name: _case(*kind, spare=3) for name, kind in KINDS.items()}
    want = {name: _all(c) for name, c in cases.items()}
    side = {name: torch.cuda.Stream() for name in cases}
    got = {name: [] for name in cases}
    for s in side.values():
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for name, c in cases.items():
            with torch.cuda.stream(side[name]):
                got[name].append(_all(c))
    torch.cuda.synchronize()
    for name, runs in got.items():
        for run in runs:
            assert all(torch.equal(a, b) for a, b in zip(want[name], run)), name


class Block:
    """Everything around one product of an MoE block and back, on buffers of its own."""

    def __init__(self, T, H, inner, E, K, dtype, seed):
        g, dt = gen(seed), DT[dtype]
        new = lambda *shape, dtype=dt: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
        f32, i32 = torch.float32, torch.int32
        self.E, self.x, self.dout = E, randn(g, (T, H), dt), randn(g, (T, inner), dt)
        self.w, self.bias = randn(g, (E, inner, H), dt, H ** -0.5), randn(g, (E, inner), dt)
        self.nw, self.nb = randn(g, (H,), f32, 0.1, 1.0), randn(g, (H,), f32)
        self.topk = torch.randint(-1, E, (T, K), generator=g, device="cuda", dtype=i32)
        self.p = torch.rand(T, K, generator=g, device="cuda")
        self.h, self.mean, self.rstd = new(T, H), new(T, dtype=f32), new(T, dtype=f32)
        self.offsets, self.row_of, self.source = new(E + 1, dtype=i32), new(T, K, dtype=i32), new(T * K, dtype=i32)
        self.rows, self.z, self.out = new(T * K, H), new(T * K, inner), new(T, inner)
        self.dz, self.dp, self.drows, self.dh, self.dx = new(T * K, inner), new(T, K, dtype=f32), new(T * K, H), new(T, H), new(T, H)
        self.dw, self.db, self.dnw, self.dnb = new(E, inner, H, dtype=f32), new(E, inner, dtype=f32), new(H, dtype=f32), new(H, dtype=f32)
        self.space = torch.empty(kleos.layer_norm_workspace(H), dtype=torch.uint8, device="cuda")

    def run(self):
        s = stream()
        kleos.layer_norm(self.x, self.nw, self.nb, 1e-5, self.h, self.mean, self.rstd, s)
        kleos.sort_tokens(self.topk, self.E, self.offsets, self.row_of, self.source, s)
        kleos.gather_tokens(self.h, self.row_of, self.offsets, self.rows, s)
        kleos.expert_products(self.rows, self.offsets, self.w, self.bias, self.z, s)
        kleos.combine_tokens(self.z, self.row_of, self.p, self.out, s)
        kleos.combine_tokens_backward(self.dout, self.z, self.row_of, self.p, self.offsets, self.dz, self.dp, s)
        kleos.expert_products_dw(self.dz, self.rows, self.offsets, self.dw, self.db, s)
        kleos.expert_products_dx(self.dz, self.offsets, self.w, self.drows, s)
        kleos.gather_tokens_backward(self.drows, self.row_of, self.dh, s)
        kleos.layer_norm_backward(self.dh, self.x, self.nw, self.mean, self.rstd, self.dx, self.dnw, self.dnb, self.space, s)

    def results(self):
        names = ("h", "mean", "rstd", "offsets", "row_of", "source", "rows", "z", "out", "dz", "dp", "drows", "dh", "dx", "dw", "db", "dnw", "dnb")
        return {n: getattr(self, n).clone() for n in names}

    def renew(self, seed):
        g = gen(seed)
        for t in (self.x, self.dout, self.p):
            t.copy_(torch.rand(t.shape, generator=g, device="cuda") - 0.5)
        self.topk.copy_(torch.randint(-1, self.E, self.topk.shape, generator=g, device="cuda", dtype=torch.int32))


SIZES = [(1, 264, 520, 8, 2, "bf16"), (60, 512, 1024, 6, 2, "fp32"), (500, 264, 136, 16, 4, "fp16"), (3000, 1024, 512, 8, 2, "bf16"), (40, 99, 77, 3, 3, "bf16")]


@pytest.mark.parametrize("size", SIZES)
def test_a_chain_in_a_graph(size):
    b = Block(*size, seed=1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        b.run()
        b.run()
    for seed in (2, 3):
        b.renew(seed)
        b.run()
        want = b.results()
        for t in (b.h, b.rows, b.z, b.out, b.dz, b.drows, b.dh, b.dx, b.dw):
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for name, got in b.results().items():
            assert torch.equal(got, want[name]), name


def test_chains_on_several_streams():
    blocks = [Block(*size, seed=i) for i, size in enumerate(SIZES)]
    want = []
    for b in blocks:
        b.run()
        want.append(b.results())
    streams = [torch.cuda.Stream() for _ in blocks]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for b, s in zip(blocks, streams):
            with torch.cuda.stream(s):
                b.run()
    torch.cuda.synchronize()
    for b, w in zip(blocks, want):
        for name, got in b.results().items():
            assert torch.equal(got, w[name]), name
