"""The routed operators together: a layer's result and gradients against 64-bit autograd on the same routing, a
training run that learns, and the served form against the dequantised weights."""

import sys
from pathlib import Path

import pytest
import torch

from tensor0_b200 import routed

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
import routed_layer  # noqa: E402

pytestmark = pytest.mark.gpu


def relative(got, expected):
    return float((got.double().cpu() - expected).norm() / expected.norm())


def plain_layer(x, router, w_in, w_out, r, top_k):
    """The layer by a loop over the experts; differentiable."""
    width = w_out.shape[1]
    chosen = r.experts.cpu().long()
    scores = torch.sigmoid(x @ router)
    picked = torch.where(chosen >= 0, scores.gather(1, chosen.clamp(min=0)), torch.zeros((), dtype=x.dtype))
    weights = picked / (picked.sum(1, keepdim=True) + 1e-20)
    y = torch.zeros_like(x)
    for e in range(router.shape[1]):
        for slot in range(top_k):
            t = torch.nonzero(chosen[:, slot] == e)[:, 0]
            h = x[t] @ w_in[e]
            a = torch.nn.functional.silu(h[:, :width]) * h[:, width:]
            y = y.index_add(0, t, weights[t, slot][:, None] * (a @ w_out[e]))
    return y


@pytest.mark.parametrize("tokens, size, width, experts, top_k, dtype",
                         [(40, 64, 48, 4, 2, torch.bfloat16), (333, 136, 200, 10, 3, torch.float16)])
def test_layer_against_autograd(tokens, size, width, experts, top_k, dtype):
    layer = routed_layer.RoutedLayer(size, width, experts, top_k, dtype=dtype, seed=3)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(tokens, size, generator=g).to(dtype).cuda()
    mask = (torch.rand(tokens, generator=g) < 0.9).cuda()
    y_grad = torch.randn(tokens, size, generator=g).to(dtype).cuda()
    y, saved = layer.forward(x, mask)
    x_grad, grads = layer.backward(saved, y_grad)
    leaves = [v.double().cpu().requires_grad_() for v in (x, *layer.parameters())]
    expected = plain_layer(*leaves, saved[2], top_k)
    expected.backward(y_grad.double().cpu())
    # A 16-bit value is off by 2^-9 (BF16) at most, four roundings on the way to y.  The backward pass has the
    # activation's input in 8 bits: half a step of 1/127 of a group's largest value, 0.3 steps in the mean, is about
    # 0.8 % of a value of a normal distribution, which enters each gradient at most twice.
    assert relative(y, expected.detach()) < 4 * 2.0 ** -9
    for got, leaf in zip((x_grad, *grads), leaves):
        assert relative(got, leaf.grad) < 0.03
    assert float(y[~mask].abs().max()) == 0.0 and float(x_grad[~mask].abs().max()) == 0.0


def test_training_learns_and_repeats_its_bits():
    runs = [routed_layer.train(routed_layer.RoutedLayer(128, 64, 8, 2), 20, 512) for _ in range(2)]
    assert runs[0] == runs[1]
    assert runs[0][-1] < 0.9 * runs[0][0]


@pytest.mark.parametrize("tokens", [1, 7])
def test_served_layer(tokens):
    layer = routed_layer.RoutedLayer(256, 128, 8, 3, seed=5)
    served = routed_layer.ServedLayer(layer)
    x = torch.randn(tokens, 256, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    got = served(x)

    def values(weights):
        codes = weights.codes.long()
        q = torch.stack([codes & 15, codes >> 4], 3).flatten(2) - 8
        return (q.double() * weights.scales.double().repeat_interleave(weights.group, dim=2)).transpose(1, 2).cpu()

    r = routed.route(x @ layer.router, 3, score="sigmoid", bias=layer.balance)
    expected = plain_layer(x.double().cpu(), layer.router.double().cpu(), values(served.w_in), values(served.w_out), r, 3)
    assert relative(got, expected) < 4 * 2.0 ** -9
