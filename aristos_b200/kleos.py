"""Host-side mirror of the reference's API for the MoE forward path, on top of the C ABI.

Function names and argument meaning follow the reference's host functions:
``initialize`` / ``finalize`` / ``get_rank`` (csrc/include/kleos/bootstrap.cuh:532-588) and
``moe::forwardHost`` / ``forwardHostBench`` (csrc/include/kleos/moe/moe.cuh:146-205).  The
packed device buffers are the reference's (moe.cuh:92-98).  Errors raise ``KleosError``
instead of terminating the process (reference: debug.cuh:19-43).

There is no CPU path: loading fails loudly if ``libkleos_b200.so`` has not been built, and
``initialize`` fails if no sm_100 GPU is present.
"""
from __future__ import annotations

import ctypes
import json
import os
import tempfile
from dataclasses import asdict

from .config import KleosConfig

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libkleos_b200.so")

EXPORTS = (
    "kleos_get_unique_id", "kleos_config_probe", "kleos_set_device", "kleos_initialize", "kleos_set_gate_bias",
    "kleos_forward", "kleos_forward_bench", "kleos_forward_host", "kleos_forward_host_async",
    "kleos_host_sync", "kleos_get_rank",
    "kleos_local_experts", "kleos_get_info", "kleos_last_status", "kleos_clear_status", "kleos_debug_routing",
    "kleos_phase_times", "kleos_flow_timeline", "kleos_debug_flow_stamps", "kleos_debug_flow_stalls", "kleos_debug_tile_order", "kleos_launch_count", "kleos_debug_gemm_stats", "kleos_debug_suppress_return_flag", "kleos_gate_stats", "kleos_plan_placement", "kleos_placement_model", "kleos_route_static",
    "kleos_layer_norm", "kleos_layer_norm_workspace", "kleos_layer_norm_backward", "kleos_sort_tokens", "kleos_gather_tokens",
    "kleos_combine_tokens", "kleos_combine_tokens_backward", "kleos_expert_products", "kleos_expert_products_dx",
    "kleos_expert_products_dw", "kleos_activation", "kleos_activation_backward", "kleos_moe_tokens_workspace", "kleos_moe_tokens",
    "kleos_adapter_products", "kleos_adapter_products_workspace", "kleos_adapter_products_backward", "kleos_finalize", "kleos_error_string",
)

PHASE_NAMES = ("route", "slots", "dispatch", "plan", "gemm1", "gemm2", "combine", "total")


class KleosError(RuntimeError):
    def __init__(self, code: int, what: str):
        super().__init__(f"{what}: {code}")
        self.code = code


class Status(ctypes.Structure):
    _fields_ = [("code", ctypes.c_int32), ("where", ctypes.c_int32),
                ("detail", ctypes.c_int32), ("epoch", ctypes.c_int32)]


class LayerInfo(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in
                ("rank", "world", "local_experts", "S", "H", "I", "E", "K", "EC", "pEC", "PX",
                 "torch_dtype", "hidden_act", "elem_bytes")] + \
               [("input_elems", ctypes.c_int64), ("output_elems", ctypes.c_int64)]


# argument types of the operators around the experts: p pointer, l long long, i int, f float
_C = dict(p=ctypes.c_void_p, l=ctypes.c_longlong, i=ctypes.c_int, f=ctypes.c_float)
_OPERATOR_ARGS = {
    "kleos_layer_norm_workspace": "i", "kleos_layer_norm": "plppiifiiplppp", "kleos_layer_norm_backward": "plplpppiiiiplppplp",
    "kleos_sort_tokens": "piiipppp", "kleos_gather_tokens": "plppiiiiipp", "kleos_combine_tokens": "pppiiiiplp",
    "kleos_combine_tokens_backward": "plppppiiiiippp", "kleos_expert_products": "plpppiiiiiplp",
    "kleos_expert_products_dx": "plppiiiiiplp", "kleos_expert_products_dw": "plplpiiiiiippp",
    "kleos_activation": "plliiiiplp", "kleos_activation_backward": "plplliiiiplp",
    "kleos_moe_tokens_workspace": "iii", "kleos_moe_tokens": "plppppppiiiiiiiiplppplp",
    "kleos_adapter_products": "plppppppliiiiiiiplpp", "kleos_adapter_products_workspace": "ii",
    "kleos_adapter_products_backward": "plplpppppppliiiiiiiiplppplp",
}

_lib = None


def load_library() -> ctypes.CDLL:
    """dlopen the in-tree CUDA library.  Raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(
                f"{LIB_PATH} is missing: build it with `python -m aristos_b200.build` "
                "(this package has no CPU fallback)")
        lib = ctypes.CDLL(LIB_PATH)
        lib.kleos_error_string.restype = ctypes.c_char_p
        lib.kleos_initialize.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
        lib.kleos_forward.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
        lib.kleos_forward_bench.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int,
                                            ctypes.c_int, ctypes.POINTER(ctypes.c_float)]
        lib.kleos_forward_host.argtypes = [ctypes.c_void_p] * 4
        lib.kleos_forward_host_async.argtypes = [ctypes.c_void_p] * 4
        lib.kleos_set_gate_bias.argtypes = [ctypes.c_void_p, ctypes.c_int]
        lib.kleos_debug_routing.argtypes = [ctypes.c_void_p] * 4
        lib.kleos_gate_stats.argtypes = [ctypes.c_void_p] * 3
        lib.kleos_phase_times.argtypes = [ctypes.POINTER(ctypes.c_float), ctypes.c_int]
        lib.kleos_get_unique_id.argtypes = [ctypes.c_void_p]
        for name in ("kleos_layer_norm_workspace", "kleos_moe_tokens_workspace", "kleos_adapter_products_workspace"):
            getattr(lib, name).restype = ctypes.c_longlong
        for name, args in _OPERATOR_ARGS.items():
            getattr(lib, name).argtypes = [_C[c] for c in args]
        _lib = lib
    return _lib


def _check(rc: int, what: str) -> None:
    if rc != 0:
        msg = load_library().kleos_error_string(rc).decode()
        raise KleosError(rc, f"{what}: {msg}")


def get_unique_id() -> bytes:
    """128-byte bootstrap id created on rank 0 and handed to every rank's ``initialize``."""
    buf = ctypes.create_string_buffer(128)
    _check(load_library().kleos_get_unique_id(buf), "kleos_get_unique_id")
    return buf.raw


def set_device(device: int) -> None:
    _check(load_library().kleos_set_device(device), "kleos_set_device")


def initialize(config, rank: int = 0, world: int = 1, unique_id: bytes | None = None) -> LayerInfo:
    """``config`` is a path to a kleos_config.json or a KleosConfig (written to a temp file,
    since the C ABI reads the same JSON file the reference's build reads)."""
    lib = load_library()
    tmp = None
    if isinstance(config, KleosConfig):
        tmp = tempfile.NamedTemporaryFile("w", suffix=".json", delete=False)
        json.dump(asdict(config), tmp)
        tmp.close()
        path = tmp.name
    else:
        path = str(config)
    try:
        idbuf = ctypes.create_string_buffer(unique_id, 128) if unique_id is not None else None
        _check(lib.kleos_initialize(path.encode(), rank, world, idbuf), "kleos_initialize")
    finally:
        if tmp is not None:
            os.unlink(tmp.name)
    return get_info()


def config_probe(path: str, world: int = 1) -> LayerInfo:
    """Sizes the C++ host layer derives from a kleos_config.json; needs no GPU."""
    info = LayerInfo()
    _check(load_library().kleos_config_probe(str(path).encode(), world, ctypes.byref(info)),
           "kleos_config_probe")
    return info


def get_info() -> LayerInfo:
    info = LayerInfo()
    _check(load_library().kleos_get_info(ctypes.byref(info)), "kleos_get_info")
    return info


def get_rank() -> int:
    return load_library().kleos_get_rank()


def local_experts() -> int:
    return load_library().kleos_local_experts()


def set_gate_bias(bias) -> None:
    lib = load_library()
    if bias is None:
        _check(lib.kleos_set_gate_bias(None, 0), "kleos_set_gate_bias")
        return
    import numpy as np
    b = np.ascontiguousarray(bias, dtype=np.float32)
    _check(lib.kleos_set_gate_bias(b.ctypes.data, b.size), "kleos_set_gate_bias")


def forward_host(iP, oP, stream=None) -> None:
    """Asynchronous layer forward on packed DEVICE buffers (torch tensors or raw pointers)."""
    _check(load_library().kleos_forward(_ptr(iP), _ptr(oP), stream), "kleos_forward")


def forward_host_bench(iP, oP, skip: int = 32, trials: int = 32) -> float:
    """Mean milliseconds per forward over ``trials`` launches after ``skip`` warm-ups."""
    ms = ctypes.c_float(0)
    _check(load_library().kleos_forward_bench(_ptr(iP), _ptr(oP), skip, trials, ctypes.byref(ms)),
           "kleos_forward_bench")
    return ms.value


def forward_from_host(host_activations, iP, oP, host_output) -> None:
    """End-to-end step with host buffers: H2D activations, forward, D2H layer output, sync."""
    _check(load_library().kleos_forward_host(_ptr(host_activations), _ptr(iP), _ptr(oP),
                                             _ptr(host_output)), "kleos_forward_host")


def forward_from_host_async(host_activations, iP, oP, host_output) -> None:
    """Queue one end-to-end step (H2D, forward, D2H on three streams); see host_sync()."""
    _check(load_library().kleos_forward_host_async(_ptr(host_activations), _ptr(iP), _ptr(oP),
                                                   _ptr(host_output)), "kleos_forward_host_async")


def host_sync() -> None:
    """Wait for every queued end-to-end step and raise on a device-side error."""
    _check(load_library().kleos_host_sync(), "kleos_host_sync")


def phase_times() -> dict:
    arr = (ctypes.c_float * 8)()
    _check(load_library().kleos_phase_times(arr, 8), "kleos_phase_times")
    return dict(zip(PHASE_NAMES, [float(v) for v in arr]))


def gemm_stats():
    """Per-block stall counters of the last two GEMM launches (needs KLEOS_GEMM_STATS=1)."""
    import numpy as np
    buf = np.zeros(2 * 256 * 12, dtype=np.int64)
    n = load_library().kleos_debug_gemm_stats(buf.ctypes.data_as(ctypes.c_void_p), buf.size)
    if n < 0:
        _check(n, "kleos_debug_gemm_stats")
    return buf[:n].reshape(2, -1, 12)


def route_static(A, Wg, gate_bias, S, H, E, K, torch_dtype, probs, topk, mcw, stream=None) -> None:
    """Router without any device allocation (fixed scratch inside the library): see
    kleos_route_static in include/kleos_b200.h for limits, the float calls' no-overlap rule and what a
    wait that runs out leaves in topk and mcw."""
    lib = load_library()
    lib.kleos_route_static.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p] + \
        [ctypes.c_int] * 5 + [ctypes.c_void_p] * 4
    _check(lib.kleos_route_static(_ptr(A), _ptr(Wg), _ptr(gate_bias), S, H, E, K, torch_dtype,
                                  _ptr(probs), _ptr(topk), _ptr(mcw), stream),
           "kleos_route_static")


# ---------------------------------------------------------------------------- operators around the experts
# Arguments are torch tensors on one GPU; sizes and row strides are read from them, and what does not fit together raises
# KleosError (KLEOS_E_ARG, or KLEOS_E_UNSUPPORTED for an element type) before anything is launched.  They run on
# `stream` (a cudaStream_t; None is the per-thread default stream, which other streams of the program do not wait for:
# pass the stream that the tensors are used on).  See include/kleos_b200.h for what each computes.
_ARG = -8
_MOST_ROWS = 0x7fff0000  # sizes are C ints
_entry = {}              # entry points by name
_torch = None


def _bind():
    """torch and the entry points, at the first call (a small call is as fast as its checks)."""
    global _torch, _codes
    import torch
    lib = load_library()
    _entry.update({name: getattr(lib, name) for name in _OPERATOR_ARGS})
    _codes = {torch.float32: 0, torch.bfloat16: 2, torch.float16: 3}
    _torch = torch
    return torch


def _refuse(call: str, what: str):
    raise KleosError(_ARG, f"{call}: {what}")


def _first(call, name, t):
    """Shape, row stride, element type and device of the matrix that the others go by."""
    if t.dim() != 2 or not t.is_cuda:
        _refuse(call, f"{name} must be a matrix on the GPU")
    return t.shape, _rows(call, name, t, t.shape[0], t.shape[1], t.dtype, t.get_device()), t.dtype, t.get_device()


def _rows(call, name, t, rows, cols, dtype, dev) -> int:
    """Row stride of a matrix whose rows are contiguous."""
    if t.shape != (rows, cols) or t.dtype is not dtype or t.get_device() != dev:
        _refuse(call, f"{name} must be {rows} x {cols}, {dtype}, on GPU {dev}")
    if t.is_contiguous():
        if rows > _MOST_ROWS or cols > _MOST_ROWS:
            _refuse(call, f"{name} is too large")
        return cols or 1
    ld, one = t.stride()
    if (cols > 1 and one != 1) or (rows > 1 and ld < cols) or rows > _MOST_ROWS or cols > _MOST_ROWS:
        _refuse(call, f"the rows of {name} must be contiguous, and must not overlap")
    return ld if rows > 1 else cols or 1


def _whole(call, name, t, shape, dtype, dev) -> int:
    """Address of a contiguous tensor of this shape, type and device."""
    if t.shape != shape or t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
        _refuse(call, f"{name} must be contiguous, of shape {tuple(shape)}, {dtype}, on GPU {dev}")
    return t.data_ptr()


def _maybe(call, name, t, shape, dtype, dev):
    return None if t is None else _whole(call, name, t, shape, dtype, dev)


def _launch(call, dev, *args) -> None:
    """Calls the entry point with the tensors' device as the current one."""
    if dev == _torch.cuda.current_device():
        rc = _entry[call](*args)
    else:
        with _torch.cuda.device(dev):
            rc = _entry[call](*args)
    if rc:
        _check(rc, call)


def layer_norm_workspace(H: int) -> int:
    """Bytes of workspace that layer_norm_backward needs for dweight and dbias."""
    n = load_library().kleos_layer_norm_workspace(H) if H <= _MOST_ROWS else _ARG
    if n < 0:
        _check(n, "kleos_layer_norm_workspace")
    return n


def _param_type(call, dtype, *params):
    """The one type of the parameters that are given: floats, or the element type."""
    kind = None
    for p in params:
        if p is not None:
            if kind is None:
                kind = p.dtype
                if kind is not dtype and kind is not _torch.float32:
                    _refuse(call, f"the parameters must be floats or {dtype}")
            elif p.dtype is not kind:
                _refuse(call, "the parameters and their gradients must have one type")
    return kind or _torch.float32


def layer_norm(x, weight, bias, eps, y, mean=None, rstd=None, stream=None) -> None:
    """y = layer norm of the rows of x; weight and bias may be None; mean and rstd (floats, one a row) are for the
    backward pass."""
    call, torch = "kleos_layer_norm", _torch or _bind()
    (R, H), ldx, dt, dev = _first(call, "x", x)
    ldy = _rows(call, "y", y, R, H, dt, dev)
    pt = _param_type(call, dt, weight, bias)
    _launch(call, dev, x.data_ptr(), ldx, _maybe(call, "weight", weight, (H,), pt, dev), _maybe(call, "bias", bias, (H,), pt, dev), R, H, eps,
            _codes.get(dt, -1), _codes.get(pt, -1), y.data_ptr(), ldy, _maybe(call, "mean", mean, (R,), torch.float32, dev),
            _maybe(call, "rstd", rstd, (R,), torch.float32, dev), stream)


def layer_norm_backward(dy, x, weight, mean, rstd, dx, dweight=None, dbias=None, workspace=None, stream=None) -> None:
    """Gradients of layer_norm.  dweight and dbias need a workspace of layer_norm_workspace(H) bytes."""
    call, torch = "kleos_layer_norm_backward", _torch or _bind()
    (R, H), ldx, dt, dev = _first(call, "x", x)
    lddy, lddx = _rows(call, "dy", dy, R, H, dt, dev), _rows(call, "dx", dx, R, H, dt, dev)
    pt = _param_type(call, dt, weight, dweight, dbias)
    space, room = None, 0
    if workspace is not None:
        space, room = _whole(call, "workspace", workspace, workspace.shape, workspace.dtype, dev), workspace.nbytes
    _launch(call, dev, dy.data_ptr(), lddy, x.data_ptr(), ldx, _maybe(call, "weight", weight, (H,), pt, dev),
            _whole(call, "mean", mean, (R,), torch.float32, dev), _whole(call, "rstd", rstd, (R,), torch.float32, dev), R, H,
            _codes.get(dt, -1), _codes.get(pt, -1), dx.data_ptr(), lddx, _maybe(call, "dweight", dweight, (H,), pt, dev),
            _maybe(call, "dbias", dbias, (H,), pt, dev), space, room, stream)


def _offsets(call, offsets, dev):
    """Number of experts and address."""
    if offsets.dim() != 1 or not 2 <= offsets.shape[0] <= _MOST_ROWS:
        _refuse(call, "offsets must have an entry per expert and one more")
    return offsets.shape[0] - 1, _whole(call, "offsets", offsets, offsets.shape, _torch.int32, dev)


def _places(call, row_of, T, dev):
    """Experts of a token and address."""
    if row_of.dim() != 2 or row_of.shape[0] != T or row_of.shape[1] > _MOST_ROWS:
        _refuse(call, "row_of must have a row per token and a column per expert of it")
    return row_of.shape[1], _whole(call, "row_of", row_of, row_of.shape, _torch.int32, dev)


def sort_tokens(topk, num_experts, offsets, row_of, source=None, stream=None) -> None:
    """Rows of the tokens' experts, sorted by expert: offsets [E + 1], row_of [T, K], source [T * K], all int32."""
    call, torch = "kleos_sort_tokens", _torch or _bind()
    if topk.dim() != 2 or not topk.is_cuda:
        _refuse(call, "topk must be a matrix on the GPU")
    (T, K), i32, dev = topk.shape, torch.int32, topk.get_device()
    if max(T, K, num_experts) > 0x7fffffff:  # (the entry point refuses what else is too large)
        _refuse(call, "too many tokens, places or experts")
    _launch(call, dev, _whole(call, "topk", topk, (T, K), i32, dev), T, K, num_experts,
            _whole(call, "offsets", offsets, (num_experts + 1,), i32, dev), _whole(call, "row_of", row_of, (T, K), i32, dev),
            _maybe(call, "source", source, (T * K,), i32, dev), stream)


def gather_tokens(x, row_of, offsets, rows, stream=None) -> None:
    """rows[row_of[t, k]] = x[t], zeros from offsets[E] on."""
    call = "kleos_gather_tokens"
    _torch or _bind()
    (T, H), ldx, dt, dev = _first(call, "x", x)
    K, at = _places(call, row_of, T, dev)
    E, off = _offsets(call, offsets, dev)
    _launch(call, dev, x.data_ptr(), ldx, at, off, T, K, E, H, _codes.get(dt, -1), _whole(call, "rows", rows, (T * K, H), dt, dev), stream)


def combine_tokens(rows, row_of, weights, out, stream=None) -> None:
    """out[t] = sum over k of weights[t, k] * rows[row_of[t, k]]; weights None: ones."""
    call, torch = "kleos_combine_tokens", _torch or _bind()
    (T, H), ldo, dt, dev = _first(call, "out", out)
    K, at = _places(call, row_of, T, dev)
    _launch(call, dev, _whole(call, "rows", rows, (T * K, H), dt, dev), at, _maybe(call, "weights", weights, (T, K), torch.float32, dev), T, K, H,
            _codes.get(dt, -1), out.data_ptr(), ldo, stream)


def gather_tokens_backward(drows, row_of, dx, stream=None) -> None:
    """Gradient of gather_tokens: dx[t] = sum over k of drows[row_of[t, k]]."""
    combine_tokens(drows, row_of, None, dx, stream)


def combine_tokens_backward(dout, rows, row_of, weights, offsets, drows, dweights=None, stream=None) -> None:
    """Gradients of combine_tokens for the rows (zeros from offsets[E] on) and the weights."""
    call, torch = "kleos_combine_tokens_backward", _torch or _bind()
    (T, H), ldd, dt, dev = _first(call, "dout", dout)
    K, at = _places(call, row_of, T, dev)
    E, off = _offsets(call, offsets, dev)
    _launch(call, dev, dout.data_ptr(), ldd, _whole(call, "rows", rows, (T * K, H), dt, dev), at,
            _maybe(call, "weights", weights, (T, K), torch.float32, dev), off, T, K, E, H, _codes.get(dt, -1),
            _whole(call, "drows", drows, (T * K, H), dt, dev), _maybe(call, "dweights", dweights, (T, K), torch.float32, dev), stream)


def expert_products(x, offsets, w, bias, y, stream=None) -> None:
    """y[r] = x[r] W[e]^T + bias[e] for the rows of every expert, zeros from offsets[E] on; bias may be None."""
    call = "kleos_expert_products"
    _torch or _bind()
    (R, K), ldx, dt, dev = _first(call, "x", x)
    E, off = _offsets(call, offsets, dev)
    N = w.shape[1] if w.dim() == 3 else _refuse(call, "w must be [experts, N, K]")
    ldy = _rows(call, "y", y, R, N, dt, dev)
    _launch(call, dev, x.data_ptr(), ldx, off, _whole(call, "w", w, (E, N, K), dt, dev), _maybe(call, "bias", bias, (E, N), dt, dev), R, E, N, K,
            _codes.get(dt, -1), y.data_ptr(), ldy, stream)


def expert_products_dx(dy, offsets, w, dx, stream=None) -> None:
    """dx[r] = dy[r] W[e] for the rows of every expert, zeros from offsets[E] on."""
    call = "kleos_expert_products_dx"
    _torch or _bind()
    (R, N), lddy, dt, dev = _first(call, "dy", dy)
    E, off = _offsets(call, offsets, dev)
    K = w.shape[2] if w.dim() == 3 else _refuse(call, "w must be [experts, N, K]")
    lddx = _rows(call, "dx", dx, R, K, dt, dev)
    _launch(call, dev, dy.data_ptr(), lddy, off, _whole(call, "w", w, (E, N, K), dt, dev), R, E, N, K, _codes.get(dt, -1), dx.data_ptr(), lddx, stream)


def expert_products_dw(dy, x, offsets, dw, dbias=None, stream=None) -> None:
    """dw[e] = sum over the rows of expert e of dy[r]^T x[r], dbias[e] = sum of dy[r]; in the element type or floats."""
    call, torch = "kleos_expert_products_dw", _torch or _bind()
    (R, N), lddy, dt, dev = _first(call, "dy", dy)
    K = x.shape[1] if x.dim() == 2 else _refuse(call, "x must be a matrix")
    ldx = _rows(call, "x", x, R, K, dt, dev)
    E, off = _offsets(call, offsets, dev)
    gt = torch.float32 if dw.dtype is torch.float32 else dt
    _launch(call, dev, dy.data_ptr(), lddy, x.data_ptr(), ldx, off, R, E, N, K, _codes.get(dt, -1), _codes.get(gt, -1),
            _whole(call, "dw", dw, (E, N, K), gt, dev), _maybe(call, "dbias", dbias, (E, N), gt, dev), stream)


ACTIVATIONS = {"relu": 0, "gelu": 1, "silu": 2}


def _activation_code(call, act) -> int:
    code = ACTIVATIONS.get(act)
    return _refuse(call, f"act must be one of {', '.join(ACTIVATIONS)}") if code is None else code


def _gated(call, name, wide, I) -> int:
    """Whether the first product has a second half that the activated one is multiplied with."""
    if wide not in (I, 2 * I):
        _refuse(call, f"{name} must have {I} columns, or gated {2 * I}")
    return int(wide != I)


def activation(z, act, h, stream=None) -> None:
    """h = f(z), or f(z[:, :I]) * z[:, I:] where z has twice the columns of h; act is "relu", "gelu" (erf form) or "silu"."""
    call = "kleos_activation"
    _torch or _bind()
    (R, I), ldh, dt, dev = _first(call, "h", h)
    gated = _gated(call, "z", z.shape[1] if z.dim() == 2 else _refuse(call, "z must be a matrix"), I)
    ldz = _rows(call, "z", z, R, I << gated, dt, dev)
    _launch(call, dev, z.data_ptr(), ldz, R, I, _activation_code(call, act), gated, _codes.get(dt, -1), h.data_ptr(), ldh, stream)


def activation_backward(dh, z, act, dz, stream=None) -> None:
    """Gradient of activation: dz from dh and z."""
    call = "kleos_activation_backward"
    _torch or _bind()
    (R, I), lddh, dt, dev = _first(call, "dh", dh)
    gated = _gated(call, "z", z.shape[1] if z.dim() == 2 else _refuse(call, "z must be a matrix"), I)
    ldz, lddz = _rows(call, "z", z, R, I << gated, dt, dev), _rows(call, "dz", dz, R, I << gated, dt, dev)
    _launch(call, dev, dh.data_ptr(), lddh, z.data_ptr(), ldz, R, I, _activation_code(call, act), gated, _codes.get(dt, -1), dz.data_ptr(), lddz, stream)


def moe_tokens_workspace(tokens: int, inner: int, top_k: int) -> int:
    """Bytes of workspace that moe_tokens needs."""
    n = load_library().kleos_moe_tokens_workspace(tokens, inner, top_k) if max(tokens, inner, top_k) <= _MOST_ROWS else _ARG
    if n < 0:
        _check(n, "kleos_moe_tokens_workspace")
    return n


def moe_tokens(x, gate, gate_bias, w1, b1, w2, b2, act, out, topk, weights, workspace, stream=None) -> None:
    """A whole MoE layer for up to 128 tokens: the router (gate [E, H], gate_bias [E] floats or None), the experts that it chose
    (w1 [E, I, H], gated [E, 2 I, H], w2 [E, H, I], biases or None) and the weighted sum of their results.

    topk and weights [T, K] are written; without a gate they are read, as the caller's own router chose.  workspace has
    moe_tokens_workspace(T, I, K) bytes."""
    call, torch = "kleos_moe_tokens", _torch or _bind()
    (T, H), ldx, dt, dev = _first(call, "x", x)
    if w1.dim() != 3 or w2.dim() != 3 or topk.dim() != 2:
        _refuse(call, "w1 and w2 must have three dimensions, topk two")
    E, _, I = w2.shape
    K = topk.shape[1]
    gated = _gated(call, "w1", w1.shape[1], I)
    if max(T, E, I, K) > _MOST_ROWS:
        _refuse(call, "too many experts, columns or places")
    ldo = _rows(call, "out", out, T, H, dt, dev)
    space = _whole(call, "workspace", workspace, workspace.shape, workspace.dtype, dev)
    _launch(call, dev, x.data_ptr(), ldx, _maybe(call, "gate", gate, (E, H), dt, dev), _maybe(call, "gate_bias", gate_bias, (E,), torch.float32, dev),
            _whole(call, "w1", w1, (E, I << gated, H), dt, dev), _maybe(call, "b1", b1, (E, I << gated), dt, dev),
            _whole(call, "w2", w2, (E, H, I), dt, dev), _maybe(call, "b2", b2, (E, H), dt, dev), T, H, I, E, K, _activation_code(call, act), gated,
            _codes.get(dt, -1), out.data_ptr(), ldo, _whole(call, "topk", topk, (T, K), torch.int32, dev),
            _whole(call, "weights", weights, (T, K), torch.float32, dev), space, workspace.nbytes, stream)


def _adapters(call, offsets, adapter, a, b, scale, K, N, dt, dev):
    """Requests, adapters and rank, and the addresses that both passes take."""
    if adapter.dim() != 1 or a.dim() != 3:
        _refuse(call, "adapter must be a vector and a [adapters, rank, K]")
    R, (L, r, _) = adapter.shape[0], a.shape
    if max(R, L, r) > _MOST_ROWS or R < 1:
        _refuse(call, "there must be a request, and not more requests, adapters or ranks than an int holds")
    return (R, L, r), (_whole(call, "offsets", offsets, (R + 1,), _torch.int32, dev), _whole(call, "adapter", adapter, (R,), _torch.int32, dev),
                       _whole(call, "a", a, (L, r, K), dt, dev), _whole(call, "b", b, (L, N, r), dt, dev),
                       _maybe(call, "scale", scale, (L,), _torch.float32, dev))


def adapter_products(x, offsets, adapter, a, b, scale, base, y, u=None, stream=None) -> None:
    """y = base + scale[l] u b[l]^T, u = x a[l]^T, for the rows of every request (offsets [R + 1]) and its adapter l (adapter [R],
    -1 without one).  a [L, r, K], b [L, N, r]; scale may be None; base may be y itself or None; u [rows, r] floats, for the
    backward pass, may be None."""
    call, torch = "kleos_adapter_products", _torch or _bind()
    (rows, K), ldx, dt, dev = _first(call, "x", x)
    N = y.shape[1] if y.dim() == 2 else _refuse(call, "y must be a matrix")
    ldy = _rows(call, "y", y, rows, N, dt, dev)
    ldb = ldy if base is None else _rows(call, "base", base, rows, N, dt, dev)
    (R, L, r), at = _adapters(call, offsets, adapter, a, b, scale, K, N, dt, dev)
    _launch(call, dev, x.data_ptr(), ldx, *at, None if base is None else base.data_ptr(), ldb, rows, R, L, r, N, K, _codes.get(dt, -1), y.data_ptr(),
            ldy, _maybe(call, "u", u, (rows, r), torch.float32, dev), stream)


def adapter_products_workspace(rows: int, rank: int) -> int:
    """Bytes of workspace that adapter_products_backward needs for da."""
    n = load_library().kleos_adapter_products_workspace(rows, rank) if max(rows, rank) <= _MOST_ROWS else _ARG
    if n < 0:
        _check(n, "kleos_adapter_products_workspace")
    return n


def adapter_products_backward(dy, x, u, offsets, adapter, a, b, scale, dbase, dx, da=None, db=None, workspace=None, stream=None) -> None:
    """Gradients of adapter_products: dx = dbase + scale[l] dy b[l] a[l] (dbase may be dx itself or None), da and db [as a and b, in
    the element type or floats], summed over each adapter's rows.  da needs a workspace of adapter_products_workspace(rows, r) bytes."""
    call, torch = "kleos_adapter_products_backward", _torch or _bind()
    (rows, N), lddy, dt, dev = _first(call, "dy", dy)
    K = x.shape[1] if x.dim() == 2 else _refuse(call, "x must be a matrix")
    ldx, lddx = _rows(call, "x", x, rows, K, dt, dev), _rows(call, "dx", dx, rows, K, dt, dev)
    ldb = lddx if dbase is None else _rows(call, "dbase", dbase, rows, K, dt, dev)
    (R, L, r), at = _adapters(call, offsets, adapter, a, b, scale, K, N, dt, dev)
    one = da if da is not None else db
    gt = torch.float32 if one is not None and one.dtype is torch.float32 else dt
    space, room = None, 0
    if workspace is not None:
        space, room = _whole(call, "workspace", workspace, workspace.shape, workspace.dtype, dev), workspace.nbytes
    _launch(call, dev, dy.data_ptr(), lddy, x.data_ptr(), ldx, _whole(call, "u", u, (rows, r), torch.float32, dev), *at,
            None if dbase is None else dbase.data_ptr(), ldb, rows, R, L, r, N, K, _codes.get(dt, -1), _codes.get(gt, -1), dx.data_ptr(), lddx,
            _maybe(call, "da", da, (L, r, K), gt, dev), _maybe(call, "db", db, (L, N, r), gt, dev), space, room, stream)


FLOW_MILESTONES = ("start", "planned", "first_tile", "last_gemm1_tile", "last_tile", "dispatched",
                   "combined", "end", "routed", "slotted", "gate_logits", "gate_done", "topk_done",
                   "probs_done", "slot_base", "slots_done", "route_begin", "first_operands", "topk_pass1")


def flow_timeline() -> dict:
    """Milestones of the persistent kernel in the most recent forward_host_bench, in milliseconds
    after the kernel's start (see kleos_flow_timeline in include/kleos_b200.h)."""
    buf = (ctypes.c_float * len(FLOW_MILESTONES))()
    lib = load_library()
    lib.kleos_flow_timeline.argtypes = [ctypes.POINTER(ctypes.c_float), ctypes.c_int]
    _check(lib.kleos_flow_timeline(buf, len(FLOW_MILESTONES)), "kleos_flow_timeline")
    return {n: float(buf[i]) for i, n in enumerate(FLOW_MILESTONES)}


def flow_stamps():
    """Milestones of every block of the persistent kernel in the last timed forward of
    forward_host_bench: int64 array [blocks, milestones] of global-timer nanoseconds, 0 where a
    block never passed the milestone (kleos_debug_flow_stamps)."""
    import numpy as np
    lib = load_library()
    lib.kleos_debug_flow_stamps.argtypes = [ctypes.POINTER(ctypes.c_longlong), ctypes.c_int,
                                            ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_int)]
    nb, per = ctypes.c_int(0), ctypes.c_int(0)
    _check(lib.kleos_debug_flow_stamps(None, 0, ctypes.byref(nb), ctypes.byref(per)), "kleos_debug_flow_stamps")
    out = np.zeros((nb.value, per.value), dtype=np.int64)
    _check(lib.kleos_debug_flow_stamps(out.ctypes.data_as(ctypes.POINTER(ctypes.c_longlong)), out.size,
                                       ctypes.byref(nb), ctypes.byref(per)), "kleos_debug_flow_stamps")
    return out


FLOW_STALLS = ("producer_wait_stage", "producer_wait_data", "producer_total", "mma_wait_accumulator",
               "mma_wait_operands", "mma_wait_task", "mma_total", "readback_wait_accumulator",
               "readback_publish", "readback_store", "readback_total", "producer_proxy_fence")


def flow_stalls() -> dict:
    """Where the tile-stream roles of the persistent kernel waited in the last timed forward
    (kleos_debug_flow_stalls), milliseconds averaged over blocks."""
    buf = (ctypes.c_float * len(FLOW_STALLS))()
    lib = load_library()
    lib.kleos_debug_flow_stalls.argtypes = [ctypes.POINTER(ctypes.c_float), ctypes.c_int]
    _check(lib.kleos_debug_flow_stalls(buf, len(FLOW_STALLS)), "kleos_debug_flow_stalls")
    return {n: float(buf[i]) for i, n in enumerate(FLOW_STALLS) if n != "unused"}


def launch_count() -> int:
    """Kernels the library has launched for forward calls since initialize()."""
    lib = load_library()
    lib.kleos_launch_count.restype = ctypes.c_longlong
    n = lib.kleos_launch_count()
    if n < 0:
        raise KleosError(int(n), "kleos_launch_count")
    return int(n)


def last_status() -> Status:
    st = Status()
    _check(load_library().kleos_last_status(ctypes.byref(st)), "kleos_last_status")
    return st


def debug_routing(info: LayerInfo) -> dict:
    import numpy as np
    topk = np.empty((info.S, info.K), dtype=np.int32)
    slots = np.empty((info.S, info.K), dtype=np.int32)
    counts = np.empty(info.E, dtype=np.uint32)
    mcw = np.empty(info.S, dtype=np.float32)
    _check(load_library().kleos_debug_routing(topk.ctypes.data, slots.ctypes.data,
                                              counts.ctypes.data, mcw.ctypes.data),
           "kleos_debug_routing")
    return dict(topk=topk, slots=slots, counts=counts, mcw=mcw)


class PlacementRequest(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("world", "rank", "num_experts", "expert_cost", "is_training")] + \
               [(n, ctypes.c_uint32) for n in ("moe_stages", "p2p_buffer_mb", "grad_buffer_mb")] + \
               [(n, ctypes.c_void_p) for n in ("alpha", "beta", "rate", "mem")]


class PlacementResult(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("feasible", "group_size", "group_rank", "local_experts",
                                              "expert_slots", "widest_group", "matches_data_path")]


def placement_model(config) -> dict:
    """Cost-model constants of the placement planner for a layer (needs no GPU)."""
    import tempfile
    lib = load_library()
    vals = [ctypes.c_uint32() for _ in range(3)]
    with tempfile.TemporaryDirectory() as d:
        path = config if isinstance(config, str) else os.path.join(d, "kleos_config.json")
        if not isinstance(config, str):
            config.to_json(path)
        _check(lib.kleos_placement_model(path.encode(), *[ctypes.byref(v) for v in vals]),
               "kleos_placement_model")
    return dict(moe_stages=vals[0].value, p2p_buffer=vals[1].value, grad_buffer=vals[2].value)


def plan_placement(alpha, beta, rate, mem, num_experts, model: dict, rank: int = 0,
                   expert_cost: int = 1, training: bool = False) -> dict:
    """Device groups and expert placement from a measured topology (host only)."""
    import numpy as np
    a = np.ascontiguousarray(alpha, dtype=np.float32)
    b = np.ascontiguousarray(beta, dtype=np.float32)
    r = np.ascontiguousarray(rate, dtype=np.float32)
    m = np.ascontiguousarray(mem, dtype=np.uint32)
    world = r.size
    assert a.shape == (world, world) and b.shape == (world, world) and m.size == world
    rq = PlacementRequest(world, rank, num_experts, expert_cost, int(training), model["moe_stages"],
                          model["p2p_buffer"], model["grad_buffer"], a.ctypes.data, b.ctypes.data,
                          r.ctypes.data, m.ctypes.data)
    res = PlacementResult()
    d2g = np.zeros(world, dtype=np.uint32)
    ranks = np.zeros(world, dtype=np.uint32)
    e2m = np.zeros(num_experts, dtype=np.uint32)
    lib = load_library()
    lib.kleos_plan_placement.argtypes = [ctypes.c_void_p] * 5
    _check(lib.kleos_plan_placement(ctypes.byref(rq), ctypes.byref(res), d2g.ctypes.data,
                                    ranks.ctypes.data, e2m.ctypes.data), "kleos_plan_placement")
    out = dict(feasible=bool(res.feasible), device_to_group=d2g.tolist())
    if res.feasible:
        out.update(group_ranks=ranks[:res.group_size].tolist(), group_rank=res.group_rank,
                   expert_to_member=e2m.tolist(), local_experts=res.local_experts,
                   expert_slots=res.expert_slots, widest_group=res.widest_group,
                   matches_data_path=bool(res.matches_data_path))
    return out


def gate_stats(info: LayerInfo) -> dict:
    """Training-mode gate statistics of the last forward: mean probability and mean (unclamped)
    selection count per expert, and the auxiliary loss (needs is_training = 1)."""
    import numpy as np
    mean_prob = np.empty(info.E, dtype=np.float32)
    mean_count = np.empty(info.E, dtype=np.float32)
    loss = np.empty(1, dtype=np.float32)
    _check(load_library().kleos_gate_stats(mean_prob.ctypes.data, mean_count.ctypes.data,
                                           loss.ctypes.data), "kleos_gate_stats")
    return dict(mean_prob=mean_prob, mean_count=mean_count, loss=float(loss[0]))


def finalize() -> None:
    _check(load_library().kleos_finalize(), "kleos_finalize")


def _ptr(x):
    if x is None or isinstance(x, int):
        return x
    if hasattr(x, "data_ptr"):
        return x.data_ptr()
    if hasattr(x, "ctypes"):
        return x.ctypes.data
    raise TypeError(type(x))
