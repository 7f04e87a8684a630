"""What the calls of the activation, the layer for a few tokens and the adapters refuse before anything is launched; needs no GPU."""
import pytest
import torch

from aristos_b200 import kleos
from tests.test_operator_abi import ARG, ONE, UNSUPPORTED, _call, _changed
from tests.test_operator_checks import PAST, Stand, _refused, launched  # noqa: F401

ACT = [ONE, 64, 4, 32, 2, 1, 2, ONE, 32, None]
ACT_BACK = [ONE, 32, ONE, 64, 4, 32, 2, 1, 2, ONE, 64, None]
MOE = [ONE, 64, ONE, ONE, ONE, ONE, ONE, ONE, 4, 64, 32, 8, 2, 2, 1, 2, ONE, 64, ONE, ONE, ONE, 4 * 2 * 4 * 32, None]
ADAPT = [ONE, 64, ONE, ONE, ONE, ONE, ONE, ONE, 32, 10, 3, 2, 8, 32, 64, 2, ONE, 32, ONE, None]
ADAPT_BACK = [ONE, 32, ONE, 64, ONE, ONE, ONE, ONE, ONE, ONE, ONE, 64, 10, 3, 2, 8, 32, 64, 2, 2, ONE, 64, ONE, ONE, ONE, 4 * 10 * 8, None]


@pytest.mark.parametrize("name,args,at,value,code", [
    ("kleos_activation", ACT, 6, 1, UNSUPPORTED), ("kleos_activation", ACT, 4, 3, ARG), ("kleos_activation", ACT, 4, -1, ARG), ("kleos_activation", ACT, 2, -1, ARG),
    ("kleos_activation", ACT, 3, 0, ARG), ("kleos_activation", ACT, 1, 63, ARG), ("kleos_activation", ACT, 8, 31, ARG), ("kleos_activation", ACT, 0, None, ARG),
    ("kleos_activation", ACT, 7, None, ARG), ("kleos_activation", ACT, 0, ONE + 1, ARG), ("kleos_activation", ACT, 2, 0x7fff0001, ARG),
    ("kleos_activation", _changed(_changed(ACT, 1, 1 << 40), 8, 1 << 40), 3, (1 << 22) + 1, ARG),
    ("kleos_activation_backward", ACT_BACK, 8, 9, UNSUPPORTED), ("kleos_activation_backward", ACT_BACK, 6, 3, ARG), ("kleos_activation_backward", ACT_BACK, 1, 31, ARG),
    ("kleos_activation_backward", ACT_BACK, 3, 63, ARG), ("kleos_activation_backward", ACT_BACK, 10, 63, ARG), ("kleos_activation_backward", ACT_BACK, 9, None, ARG),
    ("kleos_activation_backward", ACT_BACK, 2, ONE + 1, ARG), ("kleos_activation_backward", ACT_BACK, 0, None, ARG),
    ("kleos_moe_tokens", MOE, 15, 1, UNSUPPORTED), ("kleos_moe_tokens", MOE, 13, 3, ARG), ("kleos_moe_tokens", MOE, 8, 129, ARG), ("kleos_moe_tokens", MOE, 8, -1, ARG),
    ("kleos_moe_tokens", MOE, 12, 0, ARG), ("kleos_moe_tokens", MOE, 12, 9, ARG), ("kleos_moe_tokens", MOE, 11, 1, ARG), ("kleos_moe_tokens", MOE, 11, 1025, ARG),
    ("kleos_moe_tokens", MOE, 9, 0, ARG), ("kleos_moe_tokens", MOE, 10, 0, ARG), ("kleos_moe_tokens", MOE, 1, 63, ARG), ("kleos_moe_tokens", MOE, 17, 63, ARG),
    ("kleos_moe_tokens", MOE, 2, None, ARG), ("kleos_moe_tokens", MOE, 0, None, ARG), ("kleos_moe_tokens", MOE, 4, None, ARG), ("kleos_moe_tokens", MOE, 6, None, ARG),
    ("kleos_moe_tokens", MOE, 18, None, ARG), ("kleos_moe_tokens", MOE, 19, None, ARG), ("kleos_moe_tokens", MOE, 20, None, ARG), ("kleos_moe_tokens", MOE, 20, ONE + 8, ARG),
    ("kleos_moe_tokens", MOE, 21, 4 * 2 * 4 * 32 - 1, ARG), ("kleos_moe_tokens", MOE, 4, ONE + 1, ARG), ("kleos_moe_tokens", MOE, 18, ONE + 2, ARG),
    ("kleos_adapter_products", ADAPT, 15, 1, UNSUPPORTED), ("kleos_adapter_products", ADAPT, 9, -1, ARG), ("kleos_adapter_products", ADAPT, 10, 0, ARG),
    ("kleos_adapter_products", ADAPT, 10, 65537, ARG), ("kleos_adapter_products", ADAPT, 11, 0, ARG), ("kleos_adapter_products", ADAPT, 11, 65536, ARG),
    ("kleos_adapter_products", ADAPT, 12, 0, ARG), ("kleos_adapter_products", ADAPT, 12, 129, ARG), ("kleos_adapter_products", ADAPT, 13, 0, ARG),
    ("kleos_adapter_products", ADAPT, 14, (1 << 22) + 1, ARG), ("kleos_adapter_products", ADAPT, 1, 63, ARG), ("kleos_adapter_products", ADAPT, 8, 31, ARG),
    ("kleos_adapter_products", ADAPT, 17, 31, ARG), ("kleos_adapter_products", ADAPT, 17, 33, ARG),  # (base is y here, and has another stride then)
    ("kleos_adapter_products", ADAPT, 2, None, ARG), ("kleos_adapter_products", ADAPT, 3, None, ARG), ("kleos_adapter_products", ADAPT, 16, None, ARG),
    ("kleos_adapter_products", ADAPT, 18, ONE + 2, ARG), ("kleos_adapter_products", ADAPT, 5, ONE + 1, ARG),
    ("kleos_adapter_products_backward", ADAPT_BACK, 18, 1, UNSUPPORTED), ("kleos_adapter_products_backward", ADAPT_BACK, 19, 3, UNSUPPORTED),
    ("kleos_adapter_products_backward", ADAPT_BACK, 24, None, ARG), ("kleos_adapter_products_backward", ADAPT_BACK, 24, ONE + 8, ARG),
    ("kleos_adapter_products_backward", ADAPT_BACK, 25, 4 * 10 * 8 - 1, ARG), ("kleos_adapter_products_backward", ADAPT_BACK, 4, None, ARG),
    ("kleos_adapter_products_backward", ADAPT_BACK, 21, 63, ARG), ("kleos_adapter_products_backward", ADAPT_BACK, 21, 65, ARG),
    ("kleos_adapter_products_backward", ADAPT_BACK, 1, 31, ARG), ("kleos_adapter_products_backward", ADAPT_BACK, 20, None, ARG),
    ("kleos_adapter_products_backward", ADAPT_BACK, 22, ONE + 1, ARG), ("kleos_adapter_products_backward", ADAPT_BACK, 15, 129, ARG),
])
def test_refused(name, args, at, value, code):
    assert _call(name, *_changed(args, at, value)) == code


def test_nothing_to_do():
    assert _call("kleos_activation", *_changed(ACT, 2, 0)) == 0
    assert _call("kleos_activation_backward", *_changed(ACT_BACK, 4, 0)) == 0
    assert _call("kleos_moe_tokens", *_changed(MOE, 8, 0)) == 0
    assert _call("kleos_adapter_products", *_changed(ADAPT, 9, 0)) == 0


def test_workspaces():
    assert kleos.moe_tokens_workspace(128, 2047, 8) == 128 * 8 * 4 * 2048
    assert kleos.adapter_products_workspace(1000, 12) == 48000
    for bad in ((129, 64, 2), (1, 0, 2), (1, 64, 9), (-1, 64, 2), (PAST + 1, 64, 2)):
        _refused(ARG, kleos.moe_tokens_workspace, *bad)
    for bad in ((-1, 8), (10, 0), (10, 129), (PAST + 1, 8)):
        _refused(ARG, kleos.adapter_products_workspace, *bad)


def _layer(T=4, H=64, I=32, E=8, K=2, dtype=torch.bfloat16, gated=True):
    s = lambda *shape, dtype=dtype: Stand(shape, dtype)  # noqa: E731
    up = I * (2 if gated else 1)
    return dict(x=s(T, H), gate=s(E, H), gate_bias=s(E, dtype=torch.float32), w1=s(E, up, H), b1=s(E, up), w2=s(E, H, I), b2=s(E, H), act="silu", out=s(T, H),
                topk=s(T, K, dtype=torch.int32), weights=s(T, K, dtype=torch.float32), workspace=s(1 << 20, dtype=torch.uint8))


def _adapt(rows=10, R=3, L=2, r=8, N=32, K=64, dtype=torch.bfloat16):
    s = lambda *shape, dtype=dtype: Stand(shape, dtype)  # noqa: E731
    return dict(dy=s(rows, N), x=s(rows, K), u=s(rows, r, dtype=torch.float32), offsets=s(R + 1, dtype=torch.int32), adapter=s(R, dtype=torch.int32), a=s(L, r, K),
                b=s(L, N, r), scale=s(L, dtype=torch.float32), base=s(rows, N), y=s(rows, N), dbase=s(rows, K), dx=s(rows, K), da=s(L, r, K), db=s(L, N, r),
                workspace=s(4 * rows * r, dtype=torch.uint8))


FORWARD = ("x", "offsets", "adapter", "a", "b", "scale", "base", "y", "u")
BACKWARD = ("dy", "x", "u", "offsets", "adapter", "a", "b", "scale", "dbase", "dx", "da", "db", "workspace")


def test_python_passes_what_fits(launched):  # noqa: F811
    kleos.moe_tokens(*_layer().values())
    kleos.moe_tokens(*_layer(gated=False).values())
    c = _adapt()
    kleos.adapter_products(*[c[n] for n in FORWARD])
    kleos.adapter_products_backward(*[c[n] for n in BACKWARD])
    kleos.activation(Stand((4, 64), torch.float16), "gelu", Stand((4, 32), torch.float16))
    kleos.activation_backward(Stand((4, 32), torch.float32), Stand((4, 32), torch.float32), "relu", Stand((4, 32), torch.float32))
    assert len(launched) == 6


@pytest.mark.parametrize("name,shape", [("gate", (8, 63)), ("gate", (7, 64)), ("gate_bias", (7,)), ("w1", (8, 65, 64)), ("w1", (8, 64, 63)), ("w1", (8, 64)), ("w2", (7, 64, 32)),
                                        ("w2", (8, 63, 32)), ("b1", (8, 32)), ("b2", (8, 32)), ("out", (4, 63)), ("out", (5, 64)), ("topk", (5, 2)), ("topk", (8,)),
                                        ("weights", (4, 3)), ("x", (4,))])
def test_layers_that_do_not_fit(launched, name, shape):  # noqa: F811
    c = _layer()
    c[name] = Stand(shape, c[name].dtype)
    _refused(ARG, kleos.moe_tokens, *c.values())
    assert not launched


@pytest.mark.parametrize("name", ["gate", "w1", "w2", "b1", "out", "gate_bias", "topk", "weights"])
def test_layers_of_mixed_types(launched, name):  # noqa: F811
    c = _layer()
    c[name] = Stand(c[name].shape, torch.float64)
    _refused(ARG, kleos.moe_tokens, *c.values())
    c = _layer()
    c["act"] = "tanh"
    _refused(ARG, kleos.moe_tokens, *c.values())
    assert not launched


@pytest.mark.parametrize("name,shape", [("offsets", (3,)), ("offsets", (5,)), ("adapter", (4,)), ("adapter", (3, 1)), ("a", (2, 8, 63)), ("a", (2, 64)), ("b", (2, 31, 8)), ("b", (3, 32, 8)),
                                        ("b", (2, 32, 7)), ("scale", (3,)), ("base", (10, 31)), ("y", (9, 32)), ("y", (10,)), ("u", (10, 7)), ("x", (10,))])
def test_adapters_that_do_not_fit(launched, name, shape):  # noqa: F811
    c = _adapt()
    c[name] = Stand(shape, c[name].dtype)
    _refused(ARG, kleos.adapter_products, *[c[n] for n in FORWARD])
    assert not launched


@pytest.mark.parametrize("name,shape", [("dy", (10, 31)), ("dy", (9, 32)), ("x", (10, 63)), ("u", (10, 7)), ("dbase", (10, 63)), ("dx", (9, 64)), ("da", (2, 8, 63)), ("db", (2, 31, 8)), ("adapter", (4,))])
def test_gradients_of_adapters_that_do_not_fit(launched, name, shape):  # noqa: F811
    c = _adapt()
    c[name] = Stand(shape, c[name].dtype)
    _refused(ARG, kleos.adapter_products_backward, *[c[n] for n in BACKWARD])
    assert not launched


def test_gradients_of_two_types(launched):  # noqa: F811
    c = _adapt()
    c["da"] = Stand((2, 8, 64), torch.float32)
    _refused(ARG, kleos.adapter_products_backward, *[c[n] for n in BACKWARD])
    assert not launched


def test_activations_that_do_not_fit(launched):  # noqa: F811
    s = lambda *shape, dtype=torch.float16: Stand(shape, dtype)  # noqa: E731
    for z, h in ((s(4, 65), s(4, 32)), (s(4, 48), s(4, 32)), (s(5, 64), s(4, 32)), (s(4, 64, dtype=torch.float32), s(4, 32)), (s(64), s(4, 32)), (s(4, 64), s(32))):
        _refused(ARG, kleos.activation, z, "silu", h)
    _refused(ARG, kleos.activation, s(4, 64), "swish", s(4, 32))
    _refused(ARG, kleos.activation_backward, s(4, 32), s(4, 64), "silu", s(4, 32))
    assert not launched


@pytest.mark.parametrize("dtype", [torch.float64, torch.int32, torch.float8_e4m3fn])
def test_element_types(launched, dtype):  # noqa: F811
    _refused(UNSUPPORTED, kleos.activation, Stand((4, 64), dtype), "silu", Stand((4, 32), dtype))
    _refused(UNSUPPORTED, kleos.moe_tokens, *_layer(dtype=dtype).values())
    c = _adapt(dtype=dtype)
    _refused(UNSUPPORTED, kleos.adapter_products, *[c[n] for n in FORWARD])


def test_sizes_that_a_c_int_does_not_hold(launched):  # noqa: F811
    _refused(ARG, kleos.moe_tokens, *_layer(E=PAST + 8).values())
    _refused(ARG, kleos.moe_tokens, *_layer(K=PAST + 2).values())
    _refused(ARG, kleos.moe_tokens, *_layer(I=PAST + 32).values())
    _refused(ARG, kleos.moe_tokens, *_layer(T=PAST + 4).values())
    for size in (dict(R=PAST + 3), dict(L=PAST + 2), dict(r=PAST + 8), dict(rows=PAST + 10), dict(N=PAST + 32), dict(K=PAST + 64)):
        c = _adapt(**size)
        _refused(ARG, kleos.adapter_products, *[c[n] for n in FORWARD])
        _refused(ARG, kleos.adapter_products_backward, *[c[n] for n in BACKWARD])
    _refused(ARG, kleos.activation, Stand((4, PAST + 64), torch.float16), "silu", Stand((4, PAST // 2 + 32), torch.float16))
    assert not launched
