"""What the tests of the operators around the experts share.

Tolerances are per value: half a unit of the type that a result is rounded to, and for the 32-bit sums before that the
bound n * 2^-24 * sum of |terms| of a chain of n additions.
"""
import torch

from aristos_b200 import kleos

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}  # half the smallest fp16 value
EPS = 2.0 ** -24


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)


def wide(t, left, right):
    """The same matrix inside a wider one, whose other columns are NaN."""
    w = torch.full((t.shape[0], left + t.shape[1] + right), float("nan"), dtype=t.dtype, device=t.device)
    v = w[:, left:left + t.shape[1]]
    v.copy_(t)
    return v


def stream():
    return torch.cuda.current_stream().cuda_stream or None


def check(got, ref, before, what):
    """`before`: bound on the error before the result is rounded to its type."""
    assert got.shape == ref.shape, what
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    dt, got, ref = got.dtype, got.double(), ref.double()
    tol = HALF_UNIT[dt] * (ref.abs() + before) + LEAST[dt] + before
    off = (got - ref).abs()
    worst = float((off / tol.clamp_min(1e-300)).max()) if off.numel() else 0.0
    assert bool((off <= tol).all()), f"{what}: {int((off > tol).sum())} of {off.numel()} values off, worst {worst:.3g} times the bound"


def refused(code, call, *args):
    try:
        call(*args)
    except kleos.KleosError as e:
        assert e.code == code, f"{e} instead of {code}"
        return
    raise AssertionError("not refused")
