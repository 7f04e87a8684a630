"""The example block: all operators together against torch's differentiation of the same block in 64 bits."""
import pytest
import torch

from examples.moe_block import MoEBlock, train

pytestmark = pytest.mark.gpu


def _reference(block, x, ids, on, dout):
    """Outputs and gradients in 64 bits, for the experts that the block chose and the inner units that it left on: where an
    inner value is within a rounding of zero its ReLU may go either way, and the gradient with it."""
    p = {n: v.double().requires_grad_() for n, v in block.params.items()}
    x = x.double().requires_grad_()
    h = torch.nn.functional.layer_norm(x, (x.shape[1],), p["norm_w"], p["norm_b"], block.eps)
    weights = torch.softmax((h @ p["gate"].t()).gather(1, ids), 1)
    y = x
    for k in range(ids.shape[1]):
        e = ids[:, k]
        a = (torch.einsum("th,tih->ti", h, p["w1"][e]) + p["b1"][e]) * on[:, k]
        y = y + weights[:, k, None] * torch.einsum("ti,thi->th", a, p["w2"][e])
    y.backward(dout.double())
    return y.detach(), dict({n: v.grad for n, v in p.items()}, x=x.grad)


# 2-norm errors: each of the about ten roundings to the element type on the longest way (norm, rows, three products, sums) is
# half a unit, 2^-9 or 2^-12 of the 2-norm on average.
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-6), (torch.bfloat16, 2e-2), (torch.float16, 2.5e-3)])
@pytest.mark.parametrize("T,H,inner,E,K", [(300, 128, 192, 6, 2), (7, 64, 96, 16, 2), (129, 264, 136, 3, 3)])
def test_outputs_and_gradients(T, H, inner, E, K, dtype, tol):
    block = MoEBlock(H, inner, E, K, dtype, seed=T)
    gen = torch.Generator(device="cuda").manual_seed(T + H)
    x, dout = (torch.randn(T, H, generator=gen, device="cuda").to(dtype) for _ in range(2))
    block.params["norm_w"] += torch.randn(H, generator=gen, device="cuda") * 0.1
    block.params["b1"] += (torch.randn(E, inner, generator=gen, device="cuda") * 0.1).to(dtype)
    y = block.forward(x)
    grads = block.backward(dout)
    on = (block.kept["a"] > 0)[block.kept["row_of"].long()]  # [T, K, inner]
    want, wanted = _reference(block, x, block.kept["ids"].long(), on, dout)
    assert float((y.double() - want).norm() / want.norm()) <= tol
    for name, grad in grads.items():
        off, size = float((grad.double() - wanted[name]).norm()), float(wanted[name].norm())
        assert off <= tol * size, (name, off / size)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_block_learns(dtype):
    losses = train(512, 128, 256, 8, 60, dtype)
    assert losses[-1] < 0.5 * losses[0] and all(b == b for b in losses)
