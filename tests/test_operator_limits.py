"""Sizes at the ends of what the C entry points of the operators take; needs no GPU: what is past the end is refused before
any device work, and what is not reaches the question which device is current."""
import pytest

from tests.test_operator_abi import ARG, BACK, NORM, _call, _changed

MOST_ROWS = 0x7fff0000


@pytest.mark.parametrize("name,args,at", [("kleos_layer_norm", NORM, 4), ("kleos_layer_norm_backward", BACK, 7)])
@pytest.mark.parametrize("rows", [MOST_ROWS + 1, 2 ** 31 - 1])
def test_norm_of_more_rows_than_launches_are_counted_in(name, args, at, rows):
    assert _call(name, *_changed(args, at, rows)) == ARG
