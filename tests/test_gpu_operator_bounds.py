"""The operators write what they say and nothing beside it: elements around every output keep what was there."""
import pytest
import torch

from aristos_b200 import kleos
from tests.operator_util import DT, gen, randn, stream

pytestmark = pytest.mark.gpu
GUARD = 64  # elements in front of an output and behind it: every alignment that a kernel asks for is kept


class Outputs:
    """Outputs inside larger buffers of one byte over and over: a NaN that no kernel stores, or a number that no index is."""

    def __init__(self):
        self.all = []

    @staticmethod
    def _byte(dtype):
        return 0xFF if dtype.is_floating_point else 0xA5

    def _bytes(self, n, dtype):
        return torch.full((n * dtype.itemsize,), self._byte(dtype), dtype=torch.uint8, device="cuda").view(dtype)

    def flat(self, shape, dtype):
        n = 1
        for s in shape:
            n *= s
        whole = self._bytes(n + 2 * GUARD, dtype)
        mine = torch.zeros(n + 2 * GUARD, dtype=torch.bool, device="cuda")
        mine[GUARD:GUARD + n] = True
        self.all.append((whole, mine))
        return whole[GUARD:GUARD + n].view(shape)

    def rows(self, R, C, dtype, left, right):
        whole = self._bytes((R + 2) * (left + C + right), dtype).view(R + 2, -1)
        mine = torch.zeros(whole.shape, dtype=torch.bool, device="cuda")
        mine[1:-1, left:left + C] = True
        self.all.append((whole, mine))
        return whole[1:-1, left:left + C]

    def check(self):
        for i, (whole, mine) in enumerate(self.all):
            bytes_ = whole.contiguous().view(torch.uint8).view(*whole.shape, whole.dtype.itemsize)
            byte = self._byte(whole.dtype)
            assert bool((bytes_[~mine] == byte).all()), f"output {i}: written outside"
            assert whole.dtype.itemsize == 1 or not bool((bytes_[mine] == byte).all(-1).any()), f"output {i}: not written"


PADS = [(0, 0), (8, 8), (16, 0), (3, 0), (0, 5), (2, 2)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("pads", PADS)
@pytest.mark.parametrize("R,H", [(5, 8), (37, 100), (3, 264), (301, 512), (9, 1087), (40, 1096), (5, 2880), (700, 2047), (3, 4100), (2, 9000), (2, 16392), (2, 9001)])
def test_layer_norm(R, H, pads, dtype):
    g, dt, out = gen(R + H), DT[dtype], Outputs()
    x, dy, w = randn(g, (R, H), dt), randn(g, (R, H), dt), randn(g, (H,), dt, 0.3, 1.0)
    y, dx = (out.rows(R, H, dt, *pads) for _ in range(2))
    mean, rstd = (out.flat((R,), torch.float32) for _ in range(2))
    dw, db = (out.flat((H,), dt) for _ in range(2))
    room = Outputs()  # (its bytes need not all be written)
    space = room.flat((kleos.layer_norm_workspace(H),), torch.uint8)
    kleos.layer_norm(x, w, w, 1e-5, y, mean, rstd, stream())
    kleos.layer_norm_backward(dy, x, w, mean, rstd, dx, dw, db, space, stream())
    out.check()
    room.check()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("pads", PADS)
@pytest.mark.parametrize("T,K,E,H", [(1, 2, 8, 264), (7, 8, 16, 33), (600, 2, 32, 1024), (130, 4, 24, 1000), (40, 3, 5, 2050), (3, 1, 1024, 7001), (5000, 2, 16, 72)])
def test_sort_and_moves(T, K, E, H, pads, dtype):
    g, dt, out = gen(T + H), DT[dtype], Outputs()
    topk = torch.randint(-1, E, (T, K), generator=g, device="cuda", dtype=torch.int32)
    i32 = torch.int32
    offsets, row_of, source = out.flat((E + 1,), i32), out.flat((T, K), i32), out.flat((T * K,), i32)
    kleos.sort_tokens(topk, E, offsets, row_of, source, stream())
    x, dout, results = randn(g, (T, H), dt), randn(g, (T, H), dt), randn(g, (T * K, H), dt)
    w = torch.rand(T, K, generator=g, device="cuda")
    rows, drows, dw = out.flat((T * K, H), dt), out.flat((T * K, H), dt), out.flat((T, K), torch.float32)
    o, dx = (out.rows(T, H, dt, *pads) for _ in range(2))
    kleos.gather_tokens(x, row_of, offsets, rows, stream())
    kleos.combine_tokens(results, row_of, w, o, stream())
    kleos.combine_tokens_backward(dout, results, row_of, w, offsets, drows, dw, stream())
    kleos.gather_tokens_backward(results, row_of, dx, stream())
    out.check()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("pads", PADS)
@pytest.mark.parametrize("counts,N,K", [([1], 264, 136), ([2, 0, 1], 40, 2056), ([40, 0, 61], 192, 136), ([300, 17], 264, 1096), ([33], 39, 50),
                                        ([70, 0, 1], 520, 1032), ([700, 250, 9], 1000, 328)])
def test_products(counts, N, K, pads, dtype):
    g, dt, out = gen(N + K), DT[dtype], Outputs()
    at = [sum(counts[:e]) for e in range(len(counts) + 1)]
    R, E = at[-1] + 3, len(counts)
    offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
    x, dy, w, bias = randn(g, (R, K), dt), randn(g, (R, N), dt), randn(g, (E, N, K), dt), randn(g, (E, N), dt)
    y, dx = out.rows(R, N, dt, *pads), out.rows(R, K, dt, *pads)
    kleos.expert_products(x, offsets, w, bias, y, stream())
    kleos.expert_products_dx(dy, offsets, w, dx, stream())
    for grad in {dt, torch.float32}:
        dw, db = out.flat((E, N, K), grad), out.flat((E, N), grad)
        kleos.expert_products_dw(dy, x, offsets, dw, db, stream())
    out.check()
