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
