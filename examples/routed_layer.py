"""A routed layer, trained and then served: the routed operators as they work together.

Every token goes through its best experts, each a gated pair of products:

    y[t] = sum over the token's experts e of  w[t, e] * (silu(x W_gate[e]) * (x W_up[e])) W_out[e]

Training keeps of a layer only its input, the routing and the gated activation's input in 8 bits.  Serving takes the
experts' weights in 4 bits, one token or a few at a time.

    python examples/routed_layer.py            # a few training steps on a synthetic task, then single tokens
"""

from __future__ import annotations

import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from tensor0_b200 import routed  # noqa: E402


class RoutedLayer:
    """Weights of a routed layer of ``experts`` gated experts of ``width``, each token through ``top_k`` of them."""

    def __init__(self, size: int, width: int, experts: int, top_k: int, *, dtype=torch.bfloat16, seed: int = 0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def normal(*shape, scale):
            return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)
        self.top_k = top_k
        self.router = normal(size, experts, scale=size ** -0.5)
        self.w_in = normal(experts, size, 2 * width, scale=size ** -0.5)     # [gate | up]
        self.w_out = normal(experts, width, size, scale=width ** -0.5)
        self.balance = torch.zeros(experts, device="cuda")                    # enters the choice only

    def parameters(self) -> tuple[torch.Tensor, ...]:
        return self.router, self.w_in, self.w_out

    def forward(self, x: torch.Tensor, mask: torch.Tensor | None = None) -> tuple[torch.Tensor, tuple]:
        """The layer's result for token rows ``x``, and what its gradient needs.  ``mask``: False for padding."""
        logits = x @ self.router
        r = routed.route(logits, self.top_k, score="sigmoid", bias=self.balance, mask=mask)
        h = routed.routed_matmul(x, self.w_in, r, gather=True)
        a, kept = routed.gated_save(h, routing=r)
        y = routed.routed_sum(routed.routed_matmul(a, self.w_out, r), r)
        return y, (x, logits, r, kept)

    def backward(self, saved: tuple, y_grad: torch.Tensor) -> tuple[torch.Tensor, tuple[torch.Tensor, ...]]:
        """Gradients of the input and of ``parameters()``."""
        x, logits, r, kept = saved
        a_grad = routed.routed_matmul(y_grad, self.w_out, r, gather=True, transpose=True)
        h_grad, a, weights_grad = routed.gated_backward(kept, a_grad, routing=r)
        out_grad = routed.routed_weight_grad(a, y_grad, r, gather_y=True)
        in_grad = routed.routed_weight_grad(x, h_grad, r, gather_x=True)
        logits_grad = routed.route_backward(logits, r, weights_grad, score="sigmoid")
        x_grad = routed.routed_sum(routed.routed_matmul(h_grad, self.w_in, r, transpose=True), r)
        return x_grad + logits_grad @ self.router.T, (x.T @ logits_grad, in_grad, out_grad)

    def rebalance(self, r: routed.Routing, rate: float = 0.01) -> None:
        """Raise the choice value of experts with fewer rows than the mean, lower the others'."""
        rows = (r.offsets[1:] - r.offsets[:-1]).float()
        self.balance += rate * torch.sign(rows.mean() - rows)


class ServedLayer:
    """A trained layer with its experts' weights in 4 bits."""

    def __init__(self, layer: RoutedLayer, group: int = 32):
        self.top_k, self.router, self.balance = layer.top_k, layer.router, layer.balance
        self.w_in, self.w_out = routed.pack_int4(layer.w_in, group), routed.pack_int4(layer.w_out, group)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        r = routed.route(x @ self.router, self.top_k, score="sigmoid", bias=self.balance)
        h = routed.routed_matvec(x, self.w_in, r, gather=True)
        return routed.routed_sum(routed.routed_matvec(routed.gated(h, routing=r), self.w_out, r), r)


def train(layer: RoutedLayer, steps: int, tokens: int, rate: float = 0.2, seed: int = 1) -> list[float]:
    """Fit the layer to another layer's results by plain gradient descent; the loss of every step."""
    size = layer.router.shape[0]
    teacher = RoutedLayer(size, layer.w_out.shape[1], layer.router.shape[1], layer.top_k, seed=seed + 100)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    mask = torch.arange(tokens, device="cuda") < tokens - tokens // 16        # the end of the batch is padding
    master = [p.float() for p in layer.parameters()]
    losses = []
    for _ in range(steps):
        x = torch.randn(tokens, size, generator=g, device="cuda").to(layer.router.dtype)
        target, _ = teacher.forward(x, mask)
        y, saved = layer.forward(x, mask)
        error = (y - target).float()
        losses.append(float(error.square().mean()))
        _, grads = layer.backward(saved, (error / tokens).to(x.dtype))
        for weight, copy, grad in zip(layer.parameters(), master, grads):
            copy -= rate * grad.float()
            weight.copy_(copy)
        layer.rebalance(saved[2])
    return losses


def main() -> None:
    layer = RoutedLayer(512, 384, 16, 4)
    losses = train(layer, 60, 2048)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {len(losses)} steps")
    served = ServedLayer(layer)
    x = torch.randn(1, 512, device="cuda").bfloat16()
    y, _ = layer.forward(x)
    z = served(x)
    print(f"4-bit weights: off by {float((z - y).float().norm() / y.float().norm()):.3f} of a token's result")
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(200):
        served(x)
    torch.cuda.synchronize()
    print(f"one token: {(time.perf_counter() - start) / 200 * 1e6:.0f} us")


if __name__ == "__main__":
    main()
