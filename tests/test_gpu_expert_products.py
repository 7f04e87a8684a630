"""The experts' products over sorted rows and their gradients against 64-bit products."""
import pytest
import torch

from aristos_b200 import kleos
from tests.operator_util import DT, EPS, check, gen, randn, refused, stream, wide

pytestmark = pytest.mark.gpu

# The matrix unit adds sixteen products of a step to the running sum without rounding to nearest: four units of the
# larger ones a step are granted, beside the half unit of an ordinary addition for every term.
def _bound(n, terms):
    return (2 * n + 8) * EPS * terms


def _offsets(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda"), at


def _case(counts, N, K, dtype, spare=0, bias=True, pads=(0, 0), seed=0):
    g = gen(N * 7 + K + sum(counts) + seed)
    dt = DT[dtype]
    offsets, at = _offsets(counts)
    R, E = at[-1] + spare, len(counts)
    x, dy = randn(g, (R, K), dt), randn(g, (R, N), dt)
    x[at[-1]:], dy[at[-1]:] = float("nan"), float("nan")  # rows of nobody
    return dict(offsets=offsets, at=at, x=wide(x, *pads), dy=wide(dy, *pads), w=randn(g, (E, N, K), dt, K ** -0.5),
                bias=randn(g, (E, N), dt) if bias else None, R=R, E=E, N=N, K=K, dt=dt, pads=pads)


def _out(c, cols):
    return wide(torch.full((c["R"], cols), 9.0, dtype=c["dt"], device="cuda"), *c["pads"])


def _forward(c):
    y = _out(c, c["N"])
    kleos.expert_products(c["x"], c["offsets"], c["w"], c["bias"], y, stream())
    return y


def _dx(c):
    dx = _out(c, c["K"])
    kleos.expert_products_dx(c["dy"], c["offsets"], c["w"], dx, stream())
    return dx


def _dw(c, grad=None, bias=True):
    grad = grad or c["dt"]
    dw = torch.full((c["E"], c["N"], c["K"]), 9.0, dtype=grad, device="cuda")
    db = torch.full((c["E"], c["N"]), 9.0, dtype=grad, device="cuda") if bias else None
    kleos.expert_products_dw(c["dy"], c["x"], c["offsets"], dw, db, stream())
    return dw, db


def _verify(c, grad=None):
    y, dx = _forward(c), _dx(c)
    dw, db = _dw(c, grad)
    for e in range(c["E"]):
        r = slice(c["at"][e], c["at"][e + 1])
        n = c["at"][e + 1] - c["at"][e]
        x, dy, w = c["x"][r].double(), c["dy"][r].double(), c["w"][e].double()
        b = c["bias"][e].double() if c["bias"] is not None else torch.zeros(c["N"], device="cuda").double()
        check(y[r], x @ w.t() + b, _bound(c["K"], x.abs() @ w.abs().t() + b.abs()), f"y of expert {e}")
        check(dx[r], dy @ w, _bound(c["N"], dy.abs() @ w.abs()), f"dx of expert {e}")
        check(dw[e], dy.t() @ x, _bound(n, dy.abs().t() @ x.abs()), f"dw of expert {e}")
        check(db[e], dy.sum(0), _bound(n, dy.abs().sum(0)), f"dbias of expert {e}")
    assert not bool(y[c["at"][-1]:].any()) and not bool(dx[c["at"][-1]:].any())


GROUPS = {"one": [1], "pair": [1, 0, 1], "few": [0, 3, 15, 16, 17, 0, 33, 1], "tiles": [256, 255, 257, 0, 128, 31, 288, 289],
          "skewed": [700, 5, 0, 64, 130], "single": [517], "empty": [0, 0, 0]}


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("N,K", [(64, 64), (256, 128), (320, 72), (8, 8), (136, 520), (264, 1088), (33, 21), (1, 5), (515, 130)])
@pytest.mark.parametrize("groups", list(GROUPS))
def test_groups_and_sizes(groups, N, K, dtype):
    _verify(_case(GROUPS[groups], N, K, dtype, spare=3 if groups in ("few", "skewed", "empty") else 0))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("counts,N,K", [([130, 0, 400, 77], 2048, 512), ([1, 1], 2048, 2048), ([9, 300], 512, 2880), ([40] * 33, 256, 256),
                                        ([1] * 300, 64, 128)])
def test_larger(counts, N, K, dtype):
    _verify(_case(counts, N, K, dtype, spare=5))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("pads", [(8, 0), (0, 8), (1, 0), (0, 3)])
def test_rows_inside_a_wider_matrix(dtype, pads):
    _verify(_case([100, 0, 61], 192, 136, dtype, spare=4, pads=pads))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("N,K", [(256, 192), (40, 264), (33, 40)])
def test_weight_gradients_in_floats(dtype, N, K):
    _verify(_case([300, 0, 7, 64], N, K, dtype), torch.float32)


@pytest.mark.parametrize("dtype", list(DT))
def test_without_bias(dtype):
    c = _case([40, 3], 128, 64, dtype, bias=False)
    _verify(c)
    assert torch.equal(_dw(c, bias=False)[0], _dw(c)[0])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("N,K", [(192, 136), (33, 21)])
def test_infinite_values_stay_with_their_expert(dtype, N, K):
    c = _case([50, 20, 70], N, K, dtype)
    before = _forward(c), _dx(c), *_dw(c)
    c["w"][1] = float("nan")
    c["x"][50:70], c["dy"][50:70] = float("inf"), float("nan")
    after = _forward(c), _dx(c), *_dw(c)
    keep = torch.tensor([r for r in range(140) if not 50 <= r < 70], device="cuda")
    for a, b in zip(before[:2], after[:2]):
        assert torch.equal(a[keep], b[keep]) and not bool(torch.isfinite(b[50:70]).any())
    for a, b in zip(before[2:], after[2:]):
        assert torch.equal(a[[0, 2]], b[[0, 2]]) and not bool(torch.isfinite(b[1]).any())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_offsets_that_lie(dtype):
    """Offsets past the rows, and descending ones, read and write nothing outside."""
    c = _case([60, 40], 64, 72, dtype)
    c["offsets"] = torch.tensor([-5, 70, 400], dtype=torch.int32, device="cuda")
    y = _forward(c)
    x, w = c["x"].double(), c["w"].double()
    for e, r in ((0, slice(0, 70)), (1, slice(70, 100))):
        want = x[r] @ w[e].t() + c["bias"][e].double()
        check(y[r], want, _bound(72, x[r].abs() @ w[e].abs().t() + c["bias"][e].double().abs()), "y")
    c["offsets"] = torch.tensor([0, 90, 30], dtype=torch.int32, device="cuda")
    _forward(c), _dx(c), _dw(c)
    torch.cuda.synchronize()


def test_no_rows():
    for dtype in DT:
        c = _case([0, 0], 64, 72, dtype)
        _forward(c), _dx(c)
        dw, db = _dw(c)
        assert not bool(dw.any()) and not bool(db.any())


def test_same_bits_every_time_and_on_two_streams():
    c = _case([300, 50, 0, 700], 512, 320, "bf16")
    want = _forward(c), _dx(c), *_dw(c)
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([(_forward(c), _dx(c), *_dw(c)) for _ in range(3)])
    torch.cuda.synchronize()
    for runs in got:
        for run in runs:
            assert all(torch.equal(a, b) for a, b in zip(want, run))


def test_captured():
    c = _case([64, 200], 256, 128, "bf16")
    y = _forward(c)
    z = torch.empty_like(y)
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=s):
        kleos.expert_products(c["x"], c["offsets"], c["w"], c["bias"], z, stream())
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, z)


def test_gradients_against_differences():
    """y is linear in x, W and the bias, so a difference over any step is the slope up to rounding."""
    c = _case([30, 0, 55, 9], 96, 40, "fp32")
    dx = _dx(c)
    dw, db = _dw(c)

    def loss(**changed):
        return float((_forward({**c, **changed}).double() * c["dy"].double()).sum())

    at = loss()
    g = gen(9)
    for name, grad in (("x", dx), ("w", dw), ("bias", db)):
        d = randn(g, c[name].shape, torch.float32)
        size = float(c["x"].norm() * c["w"].norm() + d.norm() * (c["x"].norm() + c["w"].norm())) * float(c["dy"].norm())
        assert abs(loss(**{name: c[name] + d}) - at - float((grad.double() * d.double()).sum())) <= 16 * EPS * size, name


def test_refusals():
    c = _case([4, 4], 16, 24, "bf16")
    y = torch.empty(8, 16, dtype=torch.bfloat16, device="cuda")
    fwd, dx, dw = kleos.expert_products, kleos.expert_products_dx, kleos.expert_products_dw
    refused(-7, fwd, c["x"].double(), c["offsets"], c["w"].double(), None, y.double())
    refused(-8, fwd, c["x"], c["offsets"].long(), c["w"], None, y)
    refused(-8, fwd, c["x"], c["offsets"][:2], c["w"], None, y)
    refused(-8, fwd, c["x"], c["offsets"], c["w"][:, :, :16], None, y)
    refused(-8, fwd, c["x"], c["offsets"], c["w"].transpose(1, 2), None, y)
    refused(-8, fwd, c["x"], c["offsets"], c["w"].half(), None, y)
    refused(-8, fwd, c["x"], c["offsets"], c["w"], c["bias"].float(), y)
    refused(-8, fwd, c["x"], c["offsets"], c["w"], None, y[:7])
    refused(-8, fwd, c["x"], c["offsets"], c["w"], None, y[:, :8])
    refused(-8, fwd, c["x"], c["offsets"][:1], c["w"][:0], None, y)
    refused(-8, dx, c["dy"], c["offsets"], c["w"], torch.empty(8, 16, dtype=torch.bfloat16, device="cuda"))
    refused(-8, dw, c["dy"], c["x"][:7], c["offsets"], torch.empty_like(c["w"]))
    refused(-8, dw, c["dy"], c["x"], c["offsets"], torch.empty_like(c["w"]).half())
    refused(-8, dw, c["dy"], c["x"], c["offsets"], torch.empty_like(c["w"]), torch.empty(2, 16, device="cuda"))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("counts", [[1], [2], [1, 1], [3], [2, 2], [32], [33], [16, 0, 16], [16, 1, 16], [1] * 32, [1] * 33])
@pytest.mark.parametrize("N,K", [(272, 160), (2304, 200), (8448, 64), (39, 50)])
def test_as_many_rows_as_another_kernel_takes(dtype, counts, N, K):
    """Row counts on both sides of where a few rows become many, sizes on both sides of where one or two are streamed."""
    _verify(_case(counts, N, K, dtype, spare=1))


@pytest.mark.parametrize("dtype", list(DT))
def test_most_experts(dtype):
    counts = [(e * 7919) % 5 if e % 3 else 0 for e in range(1024)]
    _verify(_case(counts, 72, 40, dtype, spare=2))


@pytest.mark.parametrize("dtype", list(DT))
def test_many_tiles_of_every_height(dtype):
    """More tiles than block pairs, row counts whose last tile ends everywhere in its steps of 16, 32 and 64."""
    _verify(_case([n for n in range(1, 130, 7)] + [250, 300, 511, 513, 1025], 1056, 328, dtype))


def test_rows_past_two_to_the_31_elements():
    R, K, N = 1100000, 2048, 64
    g = gen(11)
    last = 300
    offsets = torch.tensor([0, R - last, R], dtype=torch.int32, device="cuda")
    x = torch.zeros(R, K, dtype=torch.bfloat16, device="cuda")
    dy = torch.zeros(R, N, dtype=torch.bfloat16, device="cuda")
    x[-last:], dy[-last:] = randn(g, (last, K), x.dtype), randn(g, (last, N), x.dtype)
    w = randn(g, (2, N, K), x.dtype, K ** -0.5)
    y, dx, dw = torch.empty_like(dy), torch.empty_like(x), torch.empty_like(w)
    kleos.expert_products(x, offsets, w, None, y, stream())
    kleos.expert_products_dx(dy, offsets, w, dx, stream())
    kleos.expert_products_dw(dy, x, offsets, dw, None, stream())
    xs, ds, ws = x[-last:].double(), dy[-last:].double(), w[1].double()
    check(y[-last:], xs @ ws.t(), _bound(K, xs.abs() @ ws.abs().t()), "y")
    check(dx[-last:], ds @ ws, _bound(N, ds.abs() @ ws.abs()), "dx")
    check(dw[1], ds.t() @ xs, _bound(last, ds.abs().t() @ xs.abs()), "dw")
    assert not bool(y[:-last].any()) and not bool(dx[:-last].any()) and not bool(dw[0].any())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("counts,N", [([2500], 136), ([2500], 37), ([1300, 0, 71], 264), ([129], 2048), ([1025], 8)])
def test_bias_gradient_of_many_rows(counts, N, dtype):
    c = _case(counts, N, 16, dtype, spare=3)
    for grad in (c["dt"], torch.float32):
        _, db = _dw(c, grad)
        for e, n in enumerate(counts):
            dy = c["dy"][c["at"][e]:c["at"][e + 1]].double()
            check(db[e], dy.sum(0), _bound(n, dy.abs().sum(0)), f"dbias of expert {e}")
        assert torch.equal(_dw(c, grad)[1], db)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("counts,N,K", [([1], 264, 2056), ([3], 1088, 4104), ([70, 0, 1], 520, 1032), ([64, 65], 256, 4096), ([2, 0, 33, 0], 4096, 264),
                                        ([538], 728, 1544), ([31, 1, 96], 8, 2048), ([17], 1024, 1024), ([150, 150], 512, 512)])
def test_few_tiles_with_long_sums(counts, N, K, dtype):
    for pads in ((0, 0), (8, 16)):
        c = _case(counts, N, K, dtype, spare=3, pads=pads)
        _verify(c)
        y, dx = _forward(c), _dx(c)
        for _ in range(3):
            assert torch.equal(_forward(c), y) and torch.equal(_dx(c), dx)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("N,K", [(520, 1032), (264, 2056)])
def test_infinite_values_stay_with_their_expert_in_split_sums(dtype, N, K):
    test_infinite_values_stay_with_their_expert(dtype, N, K)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_split_sums_with_offsets_that_lie(dtype):
    c = _case([60, 40], 256, 2048, dtype)
    c["offsets"] = torch.tensor([-5, 70, 400], dtype=torch.int32, device="cuda")
    y = _forward(c)
    x, w = c["x"].double(), c["w"].double()
    for e, r in ((0, slice(0, 70)), (1, slice(70, 100))):
        b = c["bias"][e].double()
        check(y[r], x[r] @ w[e].t() + b, _bound(2048, x[r].abs() @ w[e].abs().t() + b.abs()), "y")
    c["offsets"] = torch.tensor([0, 90, 30], dtype=torch.int32, device="cuda")
    _forward(c), _dx(c)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("counts,N,K", [([1000], 1024, 136), ([300, 0, 900], 512, 192), ([2000], 520, 264), ([64] * 20, 256, 128)])
def test_tiles_of_fewer_rows(counts, N, K, dtype):
    _verify(_case(counts, N, K, dtype, spare=2))
