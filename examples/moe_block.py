"""An MoE block that is trained with this library's operators: layer norm, sort by expert, rows there, two products
with an activation between them, rows back, residual, and the gradients of all of it.

    python examples/moe_block.py [--tokens 2048 --hidden 512 --inner 1024 --experts 16 --steps 50 --dtype bf16 --act silu --gated]

trains one block to reproduce another's outputs on random tokens and prints the loss, and what the trained block answers for
a few tokens in one call.  ``MoEBlock`` keeps what its backward pass needs between the two calls and returns the gradients by
parameter name; ``answer`` is the forward pass of a decode step.  Every kernel runs on the current torch stream.  The router's own
product and softmax are plain torch: they are a few values a token.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from aristos_b200 import kleos  # noqa: E402


class MoEBlock:
    """y = x + sum over the k chosen experts e of p_e W2[e] f(W1[e] norm(x) + b1[e]); gated, f(z) stands for f(z[:inner]) z[inner:]."""

    def __init__(self, hidden, inner, experts, top_k=2, dtype=torch.bfloat16, seed=0, eps=1e-5, act="relu", gated=False):
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def normal(shape, std, dtype):
            return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)

        self.experts, self.top_k, self.eps, self.act, self.inner = experts, top_k, eps, act, inner
        up = 2 * inner if gated else inner
        self.params = dict(
            norm_w=torch.ones(hidden, device="cuda"), norm_b=torch.zeros(hidden, device="cuda"),
            gate=normal((experts, hidden), hidden ** -0.5, torch.float32),
            w1=normal((experts, up, hidden), hidden ** -0.5, dtype), b1=torch.zeros(experts, up, dtype=dtype, device="cuda"),
            w2=normal((experts, hidden, inner), inner ** -0.5, dtype))
        self.workspace = torch.empty(kleos.layer_norm_workspace(hidden), dtype=torch.uint8, device="cuda")

    def forward(self, x):
        p, (T, H), K, E = self.params, x.shape, self.top_k, self.experts
        stream = torch.cuda.current_stream().cuda_stream or None
        new = lambda *shape, dtype=x.dtype: torch.empty(shape, dtype=dtype, device=x.device)  # noqa: E731
        h, mean, rstd = new(T, H), new(T, dtype=torch.float32), new(T, dtype=torch.float32)
        kleos.layer_norm(x, p["norm_w"], p["norm_b"], self.eps, h, mean, rstd, stream)
        top = torch.topk(h.float() @ p["gate"].t(), K, dim=1)
        weights, ids = torch.softmax(top.values, 1), top.indices.to(torch.int32)
        offsets, row_of = new(E + 1, dtype=torch.int32), new(T, K, dtype=torch.int32)
        kleos.sort_tokens(ids, E, offsets, row_of, stream=stream)
        rows, u, a, z = new(T * K, H), new(T * K, p["w1"].shape[1]), new(T * K, self.inner), new(T * K, H)
        kleos.gather_tokens(h, row_of, offsets, rows, stream)
        kleos.expert_products(rows, offsets, p["w1"], p["b1"], u, stream)
        kleos.activation(u, self.act, a, stream)
        kleos.expert_products(a, offsets, p["w2"], None, z, stream)
        out = new(T, H)
        kleos.combine_tokens(z, row_of, weights, out, stream)
        self.kept = dict(x=x, h=h, mean=mean, rstd=rstd, weights=weights, ids=ids, offsets=offsets, row_of=row_of, rows=rows, u=u, a=a, z=z)
        return out.add_(x)

    def answer(self, x):
        """The same for up to 128 tokens, whose experts' weights are read once and whose rows are not moved."""
        p, (T, H), K = self.params, x.shape, self.top_k
        stream = torch.cuda.current_stream().cuda_stream or None
        h, out = torch.empty_like(x), torch.empty_like(x)
        kleos.layer_norm(x, p["norm_w"], p["norm_b"], self.eps, h, stream=stream)
        top = torch.topk(h.float() @ p["gate"].t(), K, dim=1)
        workspace = torch.empty(kleos.moe_tokens_workspace(T, self.inner, K), dtype=torch.uint8, device=x.device)
        kleos.moe_tokens(h, None, None, p["w1"], p["b1"], p["w2"], None, self.act, out, top.indices.to(torch.int32), torch.softmax(top.values, 1), workspace, stream)
        return out.add_(x)

    def backward(self, dout):
        """Gradients of the parameters, and of x under "x"."""
        p, k, stream = self.params, self.kept, torch.cuda.current_stream().cuda_stream or None
        dz, dw = torch.empty_like(k["z"]), torch.empty_like(k["weights"])
        kleos.combine_tokens_backward(dout, k["z"], k["row_of"], k["weights"], k["offsets"], dz, dw, stream)
        grads = {n: torch.empty_like(p[n]) for n in ("norm_w", "norm_b", "w1", "b1", "w2")}
        da = torch.empty_like(k["a"])
        kleos.expert_products_dw(dz, k["a"], k["offsets"], grads["w2"], None, stream)
        kleos.expert_products_dx(dz, k["offsets"], p["w2"], da, stream)
        du = torch.empty_like(k["u"])
        kleos.activation_backward(da, k["u"], self.act, du, stream)
        drows = torch.empty_like(k["rows"])
        kleos.expert_products_dw(du, k["rows"], k["offsets"], grads["w1"], grads["b1"], stream)
        kleos.expert_products_dx(du, k["offsets"], p["w1"], drows, stream)
        dh = torch.empty_like(k["h"])
        kleos.gather_tokens_backward(drows, k["row_of"], dh, stream)
        # the router: softmax over the chosen logits, then its product
        dtop = k["weights"] * (dw - (dw * k["weights"]).sum(1, keepdim=True))
        dlogits = torch.zeros(dout.shape[0], self.experts, device=dout.device).scatter_(1, k["ids"].long(), dtop)
        grads["gate"] = dlogits.t() @ k["h"].float()
        dh = (dh.float() + dlogits @ p["gate"]).to(dh.dtype)
        dx = torch.empty_like(dh)
        kleos.layer_norm_backward(dh, k["x"], p["norm_w"], k["mean"], k["rstd"], dx, grads["norm_w"], grads["norm_b"], self.workspace, stream)
        grads["x"] = dx.add_(dout)
        return grads


def train(tokens, hidden, inner, experts, steps, dtype, rate=0.1, act="relu", gated=False, trained=None):
    """Losses of a block that learns another's outputs, one a step; `trained` is called with the block and its tokens at the end."""
    teacher, student = (MoEBlock(hidden, inner, experts, dtype=dtype, seed=s, act=act, gated=gated) for s in (1, 2))
    student.params["gate"].copy_(teacher.params["gate"])
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(tokens, hidden, generator=gen, device="cuda").to(dtype)
    want = teacher.forward(x)
    losses = []
    for _ in range(steps):
        diff = student.forward(x).float() - want.float()
        losses.append((diff * diff).sum(1).mean())
        grads = student.backward((diff * (2.0 / tokens)).to(dtype))
        for name, param in student.params.items():
            param.add_(grads[name], alpha=-rate)
    if trained:
        trained(student, x)
    return [float(v) for v in losses]


def answers(block, x):
    """How far the answers for the first tokens, in one call, are from the block's forward pass."""
    few = x[:8].contiguous()
    want = block.forward(few).float()
    off = (block.answer(few).float() - want).norm() / want.norm()
    print(f"8 tokens in one call: {float(off):.1e} from the forward pass")


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("tokens", 2048), ("hidden", 512), ("inner", 1024), ("experts", 16), ("steps", 50)):
        ap.add_argument("--" + name, type=int, default=default)
    ap.add_argument("--dtype", choices=("fp32", "bf16", "fp16"), default="bf16")
    ap.add_argument("--act", choices=tuple(kleos.ACTIVATIONS), default="relu")
    ap.add_argument("--gated", action="store_true")
    a = ap.parse_args()
    dtype = dict(fp32=torch.float32, bf16=torch.bfloat16, fp16=torch.float16)[a.dtype]
    losses = train(a.tokens, a.hidden, a.inner, a.experts, a.steps, dtype, act=a.act, gated=a.gated, trained=answers)
    for i in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {i:4d}  loss {losses[i]:.4f}")
    print(f"step {len(losses) - 1:4d}  loss {losses[-1]:.4f}")


if __name__ == "__main__":
    main()
