"""What the C entry points of the operators around the experts refuse before any device work; needs no GPU."""
import ctypes

import pytest

from aristos_b200 import kleos

ONE = 4096  # a non-null, aligned stand-in for a device pointer
ARG, UNSUPPORTED = -8, -7


def _call(name, *args):
    return getattr(kleos.load_library(), name)(*args)


def _changed(args, at, value):
    return [value if i == at else a for i, a in enumerate(args)]


NORM = [ONE, 64, ONE, ONE, 4, 64, 1e-5, 2, 2, ONE, 64, ONE, ONE, None]
BACK = [ONE, 64, ONE, 64, ONE, ONE, ONE, 4, 64, 2, 2, ONE, 64, ONE, ONE, ONE, 1 << 30, None]
SORT = [ONE, 4, 2, 8, ONE, ONE, ONE, None]
GATHER = [ONE, 64, ONE, ONE, 4, 2, 8, 64, 2, ONE, None]
COMBINE = [ONE, ONE, ONE, 4, 2, 64, 2, ONE, 64, None]
COMBINE_BACK = [ONE, 64, ONE, ONE, ONE, ONE, 4, 2, 8, 64, 2, ONE, ONE, None]
PRODUCTS = [ONE, 64, ONE, ONE, ONE, 4, 2, 32, 64, 2, ONE, 32, None]
DX = [ONE, 32, ONE, ONE, 4, 2, 32, 64, 2, ONE, 64, None]
DW = [ONE, 32, ONE, 64, ONE, 4, 2, 32, 64, 2, 2, ONE, ONE, None]


@pytest.mark.parametrize("name,args,at,value,code", [
    ("kleos_layer_norm", NORM, 7, 1, UNSUPPORTED), ("kleos_layer_norm", NORM, 7, 7, UNSUPPORTED), ("kleos_layer_norm", NORM, 8, 3, UNSUPPORTED),
    ("kleos_layer_norm", NORM, 0, None, ARG), ("kleos_layer_norm", NORM, 9, None, ARG), ("kleos_layer_norm", NORM, 4, -1, ARG),
    ("kleos_layer_norm", NORM, 5, 0, ARG), ("kleos_layer_norm", NORM, 1, 63, ARG), ("kleos_layer_norm", NORM, 10, 63, ARG),
    ("kleos_layer_norm", NORM, 6, -1e-5, ARG), ("kleos_layer_norm", NORM, 6, float("nan"), ARG), ("kleos_layer_norm", NORM, 0, ONE + 1, ARG),
    ("kleos_layer_norm", NORM, 2, ONE + 1, ARG), ("kleos_layer_norm", NORM, 11, ONE + 2, ARG),
    ("kleos_layer_norm", _changed(_changed(NORM, 1, 1 << 40), 10, 1 << 40), 5, (1 << 28) + 1, ARG),
    ("kleos_gather_tokens", _changed(GATHER, 1, 1 << 40), 7, (1 << 28) + 1, ARG),
    ("kleos_expert_products", PRODUCTS, 7, (1 << 22) + 1, ARG),
    ("kleos_expert_products", _changed(_changed(PRODUCTS, 5, 0x7fff0000), 11, 1 << 22), 7, 1 << 22, ARG),   # tiles past 2^31
    ("kleos_expert_products_dw", _changed(_changed(_changed(DW, 1, 1 << 22), 3, 1 << 22), 7, 1 << 22), 8, 1 << 22, ARG),
    ("kleos_layer_norm_backward", BACK, 15, None, ARG), ("kleos_layer_norm_backward", BACK, 16, 296 * 2 * 4 * 64 - 1, ARG),
    ("kleos_layer_norm_backward", BACK, 15, ONE + 8, ARG), ("kleos_layer_norm_backward", BACK, 5, None, ARG),
    ("kleos_layer_norm_backward", BACK, 11, None, ARG), ("kleos_layer_norm_backward", BACK, 12, 32, ARG),
    ("kleos_layer_norm_backward", BACK, 9, 1, UNSUPPORTED),
    ("kleos_sort_tokens", SORT, 0, None, ARG), ("kleos_sort_tokens", SORT, 1, -1, ARG), ("kleos_sort_tokens", SORT, 2, 0, ARG),
    ("kleos_sort_tokens", SORT, 2, 9, ARG), ("kleos_sort_tokens", SORT, 1, 1 << 30, ARG), ("kleos_sort_tokens", SORT, 3, 0, ARG),
    ("kleos_sort_tokens", SORT, 3, 1025, ARG), ("kleos_sort_tokens", SORT, 4, None, ARG), ("kleos_sort_tokens", SORT, 6, ONE + 2, ARG),
    ("kleos_gather_tokens", GATHER, 8, 1, UNSUPPORTED), ("kleos_gather_tokens", GATHER, 1, 63, ARG), ("kleos_gather_tokens", GATHER, 3, None, ARG),
    ("kleos_gather_tokens", GATHER, 9, ONE + 1, ARG), ("kleos_gather_tokens", GATHER, 7, 0, ARG), ("kleos_gather_tokens", GATHER, 6, 1025, ARG),
    ("kleos_combine_tokens", COMBINE, 0, None, ARG), ("kleos_combine_tokens", COMBINE, 6, 4, UNSUPPORTED), ("kleos_combine_tokens", COMBINE, 8, 63, ARG),
    ("kleos_combine_tokens", COMBINE, 2, ONE + 1, ARG),
    ("kleos_combine_tokens_backward", COMBINE_BACK, 5, None, ARG), ("kleos_combine_tokens_backward", COMBINE_BACK, 11, None, ARG),
    ("kleos_combine_tokens_backward", COMBINE_BACK, 7, 9, ARG), ("kleos_combine_tokens_backward", COMBINE_BACK, 10, 1, UNSUPPORTED),
    ("kleos_expert_products", PRODUCTS, 9, 1, UNSUPPORTED), ("kleos_expert_products", PRODUCTS, 6, 0, ARG), ("kleos_expert_products", PRODUCTS, 6, 1025, ARG),
    ("kleos_expert_products", PRODUCTS, 5, -1, ARG), ("kleos_expert_products", PRODUCTS, 1, 63, ARG), ("kleos_expert_products", PRODUCTS, 11, 31, ARG),
    ("kleos_expert_products", PRODUCTS, 3, None, ARG), ("kleos_expert_products", PRODUCTS, 7, 0, ARG), ("kleos_expert_products", PRODUCTS, 4, ONE + 1, ARG),
    ("kleos_expert_products_dx", DX, 8, 9, UNSUPPORTED), ("kleos_expert_products_dx", DX, 9, None, ARG), ("kleos_expert_products_dx", DX, 1, 31, ARG),
    ("kleos_expert_products_dx", DX, 2, ONE + 1, ARG),
    ("kleos_expert_products_dw", DW, 10, 3, UNSUPPORTED), ("kleos_expert_products_dw", DW, 11, None, ARG), ("kleos_expert_products_dw", DW, 2, None, ARG),
    ("kleos_expert_products_dw", DW, 3, 63, ARG), ("kleos_expert_products_dw", DW, 12, ONE + 1, ARG),
])
def test_refused(name, args, at, value, code):
    assert _call(name, *_changed(args, at, value)) == code


def test_nothing_to_do():
    """Calls over no rows or tokens, which write nothing, succeed without a launch."""
    assert _call("kleos_layer_norm", *_changed(NORM, 4, 0)) == 0
    assert _call("kleos_gather_tokens", *_changed(GATHER, 4, 0)) == 0
    assert _call("kleos_combine_tokens", *_changed(COMBINE, 3, 0)) == 0
    assert _call("kleos_combine_tokens_backward", *_changed(COMBINE_BACK, 6, 0)) == 0
    assert _call("kleos_expert_products", *_changed(PRODUCTS, 5, 0)) == 0
    assert _call("kleos_expert_products_dx", *_changed(DX, 4, 0)) == 0


def test_workspace():
    assert kleos.layer_norm_workspace(4096) == 296 * 2 * 4 * 4096
    with pytest.raises(kleos.KleosError) as e:
        kleos.layer_norm_workspace(0)
    assert e.value.code == ARG
    assert kleos.load_library().kleos_layer_norm_workspace.restype is ctypes.c_longlong
