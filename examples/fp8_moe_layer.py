"""A decoder layer's linears and experts on FP8 weights, as a rollout runs them.

    python examples/fp8_moe_layer.py [tokens]

Weights are quantized once into 128x128 tiles, the layout a synced FP8 checkpoint has.
Then the layer's products run on them: one quantization of the activations serves q, k
and v (``fp8_matmul``), o_proj quantizes its own (``fp8_block_linear``), and the MLP is
routed (``route_experts``) to experts (``fp8_experts``).  The trainer's side routes the
same way and takes the gradient of the router's weight through the choice.
"""

from __future__ import annotations

import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "lumen-rl_amd"))
from lumenrl_amd.quantization import (  # noqa: E402
    fp8_block_linear,
    fp8_block_quant,
    fp8_experts,
    fp8_matmul,
    quantize_fp8_blockwise,
    route_experts,
)


class MoeLayer:
    def __init__(self, hidden=1024, inter=384, experts=32, top_k=4, kv=256, device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)

        def weight(*shape):
            return (torch.randn(shape, generator=g, device=device) * shape[-1] ** -0.5).bfloat16()

        self.top_k = top_k
        self.dense = {"q": weight(hidden, hidden), "k": weight(kv, hidden), "v": weight(kv, hidden), "o": weight(hidden, hidden),
                      "gate_up": weight(experts, 2 * inter, hidden), "down": weight(experts, hidden, inter)}
        self.router = weight(experts, hidden)  # stays in bf16, as FP8 checkpoints keep it
        self.fp8 = {name: quantize_fp8_blockwise(w) for name, w in self.dense.items()}

    def projections(self, x):
        """q, k and v of x [T, H] from one quantization of it, and o_proj of q."""
        codes, scales = fp8_block_quant(x, (1, 128))
        q, k, v = (fp8_matmul(codes, scales, *self.fp8[name]) for name in "qkv")
        return q, k, v, fp8_block_linear(q, *self.fp8["o"])

    def mlp(self, x):
        """The routed experts of x [..., H]."""
        weights, ids = route_experts(F.linear(x, self.router), self.top_k)
        return fp8_experts(x, ids, weights, *self.fp8["gate_up"], *self.fp8["down"])

    def router_gradient(self, x, grad):
        """The router weight's gradient, where ``grad`` [T, top_k] is that of the experts' weights."""
        router = self.router.detach().requires_grad_()
        weights, _ = route_experts(F.linear(x, router), self.top_k)
        return torch.autograd.grad(weights, router, grad)[0]

    def reference_mlp(self, x):
        """The same experts on the bf16 weights, in float32."""
        p = F.linear(x, self.router).float()
        top = torch.topk(p, self.top_k)
        w = torch.softmax(top.values, -1)
        out = torch.zeros_like(x, dtype=torch.float32)
        for e in range(self.router.shape[0]):
            tok, slot = (top.indices == e).nonzero(as_tuple=True)
            g, u = F.linear(x[tok].float(), self.dense["gate_up"][e].float()).chunk(2, -1)
            out.index_add_(0, tok, F.linear(F.silu(g) * u, self.dense["down"][e].float()) * w[tok, slot][:, None])
        return out


def main(tokens: int = 64) -> dict:
    layer = MoeLayer()
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(tokens, 1024, generator=g, device="cuda").bfloat16()
    q, k, v, o = layer.projections(x)
    errors = {}
    for name, y, a in (("q", q, x), ("k", k, x), ("v", v, x), ("o", o, q)):
        want = F.linear(a.float(), layer.dense[name].float())
        errors[name] = float((y.float() - want).norm() / want.norm())
    want = layer.reference_mlp(x)
    errors["experts"] = float((layer.mlp(x).float() - want).norm() / want.norm())
    grad = layer.router_gradient(x, torch.randn(tokens, layer.top_k, generator=g, device="cuda"))
    errors["router gradient finite"] = bool(grad.isfinite().all())
    return errors


if __name__ == "__main__":
    for name, err in main(int(sys.argv[1]) if len(sys.argv) > 1 else 64).items():
        print(f"{name}: {err if isinstance(err, bool) else f'{err:.4f} of the bf16 weights result'}")
