"""What the Python calls of the operators around the experts refuse before anything is launched; needs no GPU.

The tensors are stand-ins that say what a tensor on GPU 0 would say, with an aligned address that nothing reads: every
call here has to be refused, by the checks of arguments or by the C entry point's.
"""
import pytest
import torch

from aristos_b200 import kleos

ARG, UNSUPPORTED = -8, -7


class Stand:
    """A contiguous tensor on GPU 0 as far as the checks can tell."""
    is_cuda = True

    def __init__(self, shape, dtype):
        self.shape, self.dtype = torch.Size(shape), dtype

    def dim(self):
        return len(self.shape)

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 4096

    @property
    def nbytes(self):
        return self.shape.numel() * self.dtype.itemsize


@pytest.fixture
def launched(monkeypatch):
    """The calls that pass the checks.  Those of an element type without a code go on to the entry point, which refuses it
    before it looks at anything else; the others are only recorded."""
    calls = []

    def launch(call, dev, *args):
        calls.append(call)
        if -1 in args:
            kleos._check(kleos._entry[call](*args), call)

    monkeypatch.setattr(kleos, "_launch", launch)
    kleos._bind()
    return calls


def _refused(code, call, *args):
    with pytest.raises(kleos.KleosError) as e:
        call(*args)
    assert e.value.code == code, str(e.value)


@pytest.mark.parametrize("dtype", [torch.float64, torch.int32, torch.float8_e4m3fn])
@pytest.mark.parametrize("params", ["weight", "bias", "both"])
def test_norm_of_a_type_with_parameters_of_the_same(launched, dtype, params):
    x, y, m = Stand((4, 64), dtype), Stand((4, 64), dtype), Stand((4,), torch.float32)
    w = Stand((64,), dtype) if params != "bias" else None
    b = Stand((64,), dtype) if params != "weight" else None
    _refused(UNSUPPORTED, kleos.layer_norm, x, w, b, 1e-5, y)
    _refused(UNSUPPORTED, kleos.layer_norm_backward, x, x, w, m, m, y, w, b, Stand((1 << 20,), torch.uint8))


PAST = 2 ** 32  # a C int takes the sizes below from PAST + 4 for 4


def test_sizes_that_a_c_int_does_not_hold(launched):
    i32, f32 = torch.int32, torch.float32
    offsets = Stand((9,), i32)
    for T, K in ((PAST + 4, 2), (4, PAST + 2), (2 ** 31, 1)):
        _refused(ARG, kleos.sort_tokens, Stand((T, K), i32), 8, offsets, Stand((T, K), i32))
    x, many = Stand((4, 64), f32), Stand((PAST + 9,), i32)
    topk, row_of, w = Stand((4, 2), i32), Stand((4, 2), i32), Stand((PAST + 8, 16, 64), f32)
    rows, y = Stand((8, 64), f32), Stand((4, 16), f32)
    _refused(ARG, kleos.sort_tokens, topk, PAST + 8, many, row_of)
    _refused(ARG, kleos.gather_tokens, x, row_of, many, rows)
    _refused(ARG, kleos.combine_tokens_backward, x, rows, row_of, None, many, rows)
    _refused(ARG, kleos.expert_products, x, many, w, None, y)
    _refused(ARG, kleos.expert_products_dx, y, many, w, x)
    _refused(ARG, kleos.expert_products_dw, y, x, many, w)
    wide, all_rows = Stand((4, PAST + 2), i32), Stand((4 * (PAST + 2), 64), f32)
    _refused(ARG, kleos.gather_tokens, x, wide, offsets, all_rows)
    _refused(ARG, kleos.combine_tokens, all_rows, wide, None, x)
    _refused(ARG, kleos.combine_tokens_backward, x, all_rows, wide, None, offsets, all_rows)
    _refused(ARG, kleos.layer_norm_workspace, PAST + 64)
    assert not launched
