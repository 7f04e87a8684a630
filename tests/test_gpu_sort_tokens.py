"""Tokens sorted by expert, their rows there and back, and the gradients of both."""
import pytest
import torch

from aristos_b200 import kleos
from tests.operator_util import DT, EPS, check, gen, randn, refused, stream, wide

pytestmark = pytest.mark.gpu


def _sort(topk, E):
    T, K = topk.shape
    offsets = torch.full((E + 1,), -7, dtype=torch.int32, device="cuda")
    row_of = torch.full((T, K), -7, dtype=torch.int32, device="cuda")
    source = torch.full((T * K,), -7, dtype=torch.int32, device="cuda")
    kleos.sort_tokens(topk, E, offsets, row_of, source, stream())
    return offsets, row_of, source


def _expected(topk, E):
    ids = topk.reshape(-1).tolist()
    lists = [[] for _ in range(E)]
    for i, e in enumerate(ids):
        if 0 <= e < E:
            lists[e].append(i)
    offsets, source = [0], []
    for one in lists:
        source += one
        offsets.append(len(source))
    row_of = [-1] * len(ids)
    for r, i in enumerate(source):
        row_of[i] = r
    return offsets, row_of, source + [-1] * (len(ids) - len(source))


def _topk(g, T, K, E, kind):
    ids = torch.randint(0, E, (T, K), generator=g, device="cuda", dtype=torch.int32)
    if kind == "dropped":
        ids[torch.rand(T, K, generator=g, device="cuda") < 0.3] = -1
    elif kind == "outside":
        odd = torch.tensor([-1, E, E + 1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
        mask = torch.rand(T, K, generator=g, device="cuda") < 0.5
        ids = torch.where(mask, odd[torch.randint(0, 5, (T, K), generator=g, device="cuda")], ids)
    elif kind == "one":
        ids[:] = E - 1
    elif kind == "none":
        ids[:] = -1
    return ids.contiguous()


@pytest.mark.parametrize("kind", ["all", "dropped", "outside", "one", "none"])
@pytest.mark.parametrize("T,K,E", [(1, 1, 1), (1, 2, 64), (5, 8, 7), (31, 1, 2), (33, 3, 255), (1000, 2, 16), (2048, 2, 1024), (4097, 1, 64),
                                   (4096, 8, 128), (40001, 2, 1000), (1025, 4, 1)])
def test_order(T, K, E, kind):
    topk = _topk(gen(T + K), T, K, E, kind)
    for got, want in zip(_sort(topk, E), _expected(topk, E)):
        assert got.reshape(-1).tolist() == want


def test_large_and_without_source():
    topk = _topk(gen(2), 300007, 4, 256, "dropped")
    offsets, row_of, source = _sort(topk, 256)
    ids = torch.where(topk.reshape(-1) < 0, 256, topk.reshape(-1))
    order = torch.sort(ids, stable=True).indices
    n = int((ids < 256).sum())
    assert int(offsets[-1]) == n and torch.equal(source[:n].long(), order[:n]) and bool((source[n:] == -1).all())
    assert torch.equal(row_of.reshape(-1)[order[:n]].long(), torch.arange(n, device="cuda"))
    again = torch.empty_like(row_of)
    kleos.sort_tokens(topk, 256, offsets, again, None, stream())
    assert torch.equal(again, row_of)


def test_no_tokens():
    topk = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    offsets, row_of, _ = _sort(topk, 5)
    assert offsets.tolist() == [0] * 6
    x = torch.empty(0, 64, device="cuda")
    kleos.gather_tokens(x, row_of, offsets, x, stream())
    kleos.combine_tokens(x, row_of, None, x, stream())
    kleos.combine_tokens_backward(x, x, row_of, None, offsets, x, None, stream())


MOVES = [(1, 2, 64, 2048, "all"), (7, 8, 16, 64, "dropped"), (300, 2, 8, 1088, "all"), (129, 4, 24, 1000, "dropped"), (65, 1, 4, 1, "all"),
         (50, 3, 5, 33, "outside"), (20, 2, 4, 96, "none"), (600, 2, 32, 4096, "all"), (9, 5, 3, 9000, "dropped"), (5000, 2, 16, 72, "dropped")]


def _case(T, K, E, H, kind, dtype):
    g = gen(T * 3 + H)
    topk = _topk(g, T, K, E, kind)
    offsets, row_of, source = _sort(topk, E)
    n = int(offsets[-1])
    place = row_of.reshape(-1).long()
    return g, DT[dtype], offsets, row_of, source.long(), n, place


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,K,E,H,kind", MOVES)
@pytest.mark.parametrize("pad", [(0, 0), (0, 3), (8, 0), (1, 0)])
def test_gather_and_its_gradient(T, K, E, H, kind, dtype, pad):
    g, dt, offsets, row_of, source, n, place = _case(T, K, E, H, kind, dtype)
    x = wide(randn(g, (T, H), dt), *pad)
    rows = torch.full((T * K, H), float("nan"), dtype=dt, device="cuda")
    kleos.gather_tokens(x, row_of, offsets, rows, stream())
    assert torch.equal(rows[:n], x[source[:n] // K]) and not bool(rows[n:].any())
    drows = randn(g, (T * K, H), dt)
    drows[n:] = float("nan")  # rows of nobody
    dx = wide(torch.full((T, H), 9.0, dtype=dt, device="cuda"), *pad)
    kleos.gather_tokens_backward(drows, row_of, dx, stream())
    terms = torch.where(place[:, None] >= 0, drows[place.clamp_min(0)].double(), 0.0).view(T, K, H)
    check(dx, terms.sum(1), (K + 1) * EPS * terms.abs().sum(1), "dx")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,K,E,H,kind", MOVES)
@pytest.mark.parametrize("pad", [(0, 0), (8, 5)])
def test_combine_and_its_gradients(T, K, E, H, kind, dtype, pad):
    g, dt, offsets, row_of, source, n, place = _case(T, K, E, H, kind, dtype)
    has = (place >= 0).view(T, K)
    rows = randn(g, (T * K, H), dt)
    rows[n:] = float("nan")
    w = torch.rand(T, K, generator=g, device="cuda")
    w[~has] = float("nan")  # the weight of a place without an expert counts for nothing
    out = wide(torch.full((T, H), 9.0, dtype=dt, device="cuda"), *pad)
    kleos.combine_tokens(rows, row_of, w, out, stream())
    mine = torch.where(place[:, None] >= 0, rows[place.clamp_min(0)].double(), 0.0).view(T, K, H)
    wd = torch.where(has, w.double(), 0.0)[:, :, None]
    check(out, (mine * wd).sum(1), (K + 1) * EPS * (mine * wd).abs().sum(1), "out")
    dout = wide(randn(g, (T, H), dt), *pad)
    drows = torch.full((T * K, H), float("nan"), dtype=dt, device="cuda")
    dw = torch.full((T, K), float("nan"), device="cuda")
    kleos.combine_tokens_backward(dout, rows, row_of, w, offsets, drows, dw, stream())
    want = torch.zeros(T * K, H, dtype=torch.float64, device="cuda")
    want[:n] = dout.double()[source[:n] // K] * w.double().reshape(-1)[source[:n], None]
    check(drows, want, 2 * EPS * want.abs(), "drows")
    products = mine * dout.double()[:, None, :]
    check(dw, products.sum(2), (H / 32 + 32) * EPS * products.abs().sum(2), "dweights")
    again = torch.empty_like(drows)
    kleos.combine_tokens_backward(dout, rows, row_of, w, offsets, again, None, stream())
    assert torch.equal(again, drows)


def test_gradients_against_differences():
    """combine is linear in the rows and in the weights, so a difference over any step is the slope: what is left is the
    rounding of both losses."""
    g, dt, offsets, row_of, source, n, place = _case(70, 3, 6, 320, "dropped", "fp32")
    rows, dout = randn(g, (210, 320), dt), randn(g, (70, 320), dt)
    rows[n:] = 0.0
    w = torch.rand(70, 3, generator=g, device="cuda")
    drows, dw = torch.empty_like(rows), torch.empty_like(w)
    kleos.combine_tokens_backward(dout, rows, row_of, w, offsets, drows, dw, stream())

    def loss(rows, w):
        out = torch.empty(70, 320, device="cuda")
        kleos.combine_tokens(rows, row_of, w, out, stream())
        return float((out.double() * dout.double()).sum())

    d, v = randn(g, rows.shape, dt), randn(g, w.shape, dt)
    size = float(rows.norm() + d.norm()) * float(dout.norm())
    assert abs(loss(rows + d, w) - loss(rows, w) - float((drows.double() * d.double()).sum())) <= 8 * EPS * size
    assert abs(loss(rows, w + v) - loss(rows, w) - float((dw.double() * v.double()).sum())) <= 64 * EPS * size


def test_rows_outside_the_matrix_are_not_touched():
    """A row_of that leads past the rows: those places count as without an expert."""
    row_of = torch.tensor([[0, 2], [4, -3]], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 99], dtype=torch.int32, device="cuda")  # and offsets past the end
    x = torch.arange(1.0, 17.0, device="cuda").view(2, 8)
    both = torch.full((6, 8), 5.0, device="cuda")
    rows = both[:4]
    kleos.gather_tokens(x, row_of, offsets, rows, stream())
    assert torch.equal(both[4:], torch.full((2, 8), 5.0, device="cuda")) and torch.equal(rows[0], x[0]) and torch.equal(rows[2], x[0])
    out = torch.empty(2, 8, device="cuda")
    kleos.combine_tokens(rows, row_of, None, out, stream())
    assert torch.equal(out, torch.stack([2 * x[0], torch.zeros(8, device="cuda")]))


def test_refusals():
    topk = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    off, row_of, src = _sort(topk, 8)
    x, rows = torch.zeros(4, 64, device="cuda"), torch.zeros(8, 64, device="cuda")
    w = torch.ones(4, 2, device="cuda")
    refused(-8, kleos.sort_tokens, topk.long(), 8, off, row_of)
    refused(-8, kleos.sort_tokens, topk, 9, off, row_of)
    refused(-8, kleos.sort_tokens, topk, 0, off[:1], row_of)
    refused(-8, kleos.sort_tokens, topk, 8, off, row_of[:3])
    refused(-8, kleos.sort_tokens, topk, 8, off, row_of, src[:7])
    big = torch.zeros(1026, dtype=torch.int32, device="cuda")
    refused(-8, kleos.sort_tokens, topk, 1025, big, row_of)
    nine = torch.zeros(4, 9, dtype=torch.int32, device="cuda")
    refused(-8, kleos.sort_tokens, nine, 8, off, torch.zeros_like(nine))
    refused(-8, kleos.gather_tokens, x[:3], row_of, off, rows)
    refused(-8, kleos.gather_tokens, x, row_of, off, rows[:7])
    refused(-8, kleos.gather_tokens, x, row_of, off.long(), rows)
    refused(-8, kleos.gather_tokens, x, row_of, off, rows.half())
    refused(-7, kleos.gather_tokens, x.int(), row_of, off, rows.int())
    refused(-8, kleos.combine_tokens, rows, row_of, w.bfloat16(), x)
    refused(-8, kleos.combine_tokens, rows, row_of, w[:, :1], x)
    refused(-8, kleos.combine_tokens, rows, row_of, w, x[:, :63])
    refused(-8, kleos.combine_tokens, rows[:, :63], row_of, w, x[:, :63])
    refused(-8, kleos.combine_tokens_backward, x, rows, row_of, w, off, rows[:5])
    refused(-8, kleos.combine_tokens_backward, x, rows, row_of, w, off, torch.zeros_like(rows), w.t())


def test_rows_past_two_to_the_31_elements():
    T, K, E, H = 550000, 2, 4, 2048
    topk = torch.zeros(T, K, dtype=torch.int32, device="cuda")
    topk[:, 1] = 3
    offsets, row_of, _ = _sort(topk, E)
    g = gen(8)
    x = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
    x[-50:] = randn(g, (50, H), x.dtype)
    rows = torch.empty(T * K, H, dtype=torch.bfloat16, device="cuda")
    kleos.gather_tokens(x, row_of, offsets, rows, stream())
    assert torch.equal(rows[-50:], x[-50:]) and not bool(rows[T:-50].any())
    w = torch.rand(T, K, generator=g, device="cuda")
    out = torch.empty_like(x)
    kleos.combine_tokens(rows, row_of, w, out, stream())
    want = x[-50:].double() * w[-50:].double().sum(1, keepdim=True)
    check(out[-50:], want, 3 * EPS * want.abs(), "out")
    dw = torch.empty_like(w)
    drows = torch.empty_like(rows)
    kleos.combine_tokens_backward(x, rows, row_of, w, offsets, drows, dw, stream())
    want = x[-50:].double() * w[-50:, 1:].double()
    check(drows[-50:], want, 2 * EPS * want.abs(), "drows")
    squares = x[-50:].double().square().sum(1, keepdim=True).expand(50, 2)
    check(dw[-50:], squares, (H / 32 + 32) * EPS * squares, "dweights")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,K,E,H", [(1, 8, 12, 8190), (3, 8, 9, 7271), (2, 3, 4, 4098), (40, 1, 4, 2050), (2400, 3, 8, 66), (1300, 8, 16, 322)])
def test_pairs_of_elements_and_several_blocks_a_token(T, K, E, H, dtype):
    for pad in ((0, 0), (2, 0), (1, 0)):
        test_gather_and_its_gradient(T, K, E, H, "dropped", dtype, pad)
        test_combine_and_its_gradients(T, K, E, H, "dropped", dtype, pad)
