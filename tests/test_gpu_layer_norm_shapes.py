"""Layer norm at every number of threads and vectors that a row may have, and with more rows than are on their way at once, so
that every stage of a ring is filled several times; against 64-bit arithmetic."""
import pytest
import torch

from tests.operator_util import DT, gen, randn
from tests.test_gpu_layer_norm import _compare

pytestmark = pytest.mark.gpu

WHOLE = [8, 248, 256, 264, 504, 512, 520, 760, 768, 776, 1016, 1024, 1032, 1088, 1536, 1544, 2040, 2056, 2560, 2880, 3064, 3080, 4088, 4104,
         6144, 6152, 8184, 8200, 16376]
ODD = [7, 255, 257, 511, 513, 777, 1023, 1025, 1999, 2047, 2049, 3001, 4095, 4097, 6001, 8191]


def _rows(R, H, dtype, pad=(0, 0)):
    g, dt = gen(R + 3 * H), DT[dtype]
    param = torch.float32 if H % 3 else dt
    _compare(randn(g, (R, H), dt, 2.0, 0.5), randn(g, (H,), param, 0.3, 1.0), randn(g, (H,), param), 1e-5, randn(g, (R, H), dt), param, pad)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("H", WHOLE + ODD)
def test_every_shape(dtype, H):
    _rows(3, H, dtype)
    _rows(467, H, dtype)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("R,H", [(100003, 256), (60001, 512), (40001, 760), (20001, 1000), (15001, 1088), (12001, 1536), (12007, 2040), (9001, 2880),
                                 (6001, 4096), (4001, 6144), (3001, 8192), (1201, 16384), (50001, 255), (20001, 777), (9001, 2047), (5003, 3001), (3001, 6001)])
def test_more_rows_than_on_their_way(dtype, R, H):
    _rows(R, H, dtype)
