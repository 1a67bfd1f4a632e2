"""Routed operators at inputs that are not finite, at the limits that they accept, on strided operands, and from more
than one thread.  Tolerances are those of ``test_routed``: they follow from the arithmetic."""

import math
import subprocess
import sys
import threading
from pathlib import Path

import numpy as np
import pytest
import torch

from tensor0_b200 import _native, build, routed
from test_routed import (A, B, C, D, E, F, G, H, HALF, TYPES, call, make_routing, near, plain_choice, plain_product,
                         wide)

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
import routed_layer  # noqa: E402

gpu = pytest.mark.gpu


# ----------------------------------------------------------------------------------------------------------------
# Router


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [6, 300])                  # one block, and several
@pytest.mark.parametrize("experts, groups, top_groups, best, bias",
                         [(16, 1, 1, 1, True), (40, 1, 1, 2, False), (64, 4, 2, 1, True), (256, 8, 4, 2, True)])
def test_a_choice_by_scores_surfaces_numbers_that_are_not(experts, groups, top_groups, best, bias, tokens, dtype):
    """A NaN logit takes no expert and the others stay; +inf takes the score 1, shared if there are several.  The
    weights and the gradient of such a row are NaN, other rows are as without it."""
    g = torch.Generator().manual_seed(experts + tokens)
    logits = torch.randn(tokens, experts, generator=g).to(TYPES[dtype])
    b = 0.3 * torch.randn(experts, generator=g) if bias else None
    plain = {"groups": groups, "top_groups": top_groups, "group_best": best, "bias": None if b is None else b.cuda()}
    fine = routed.route(logits.cuda(), 4, **plain)
    logits[0, 5] = math.nan
    logits[1, 5] = math.inf
    logits[2, 3], logits[2, 7] = math.nan, math.inf
    logits[3, 2] = logits[3, 11] = math.inf
    logits[4] = math.nan
    r = routed.route(logits.cuda(), 4, **plain)
    # The definition on the same rows: without the NaN logits, and at +inf the scores' limits.
    x = logits[:5].double().numpy()
    infinite = np.isinf(x).any(1, keepdims=True)
    limit = np.where(infinite, np.where(np.isinf(x), 0.0, -1e30), x)
    limit[np.isnan(x)] = -np.inf
    with np.errstate(all="ignore"):
        chosen, scores = plain_choice(limit, 4, groups, top_groups, best, True, None if b is None else wide(b), None)
    got = r.experts[:5].cpu().numpy()
    for t in np.unique(np.nonzero(got != chosen)[0]):         # closer than 32-bit choice values are rounded
        value = scores[t] + (0 if b is None else wide(b))
        assert (got[t] >= 0).all() and (chosen[t] >= 0).all(), t
        assert np.max(np.abs(np.sort(value[got[t]]) - np.sort(value[chosen[t]]))) < 2.0 ** -20, t
    assert (chosen[:4] >= 0).all() and (chosen[4] < 0).all()
    assert torch.isnan(r.weights[:4]).all() and (r.weights[4] == 0).all()
    assert torch.equal(r.experts[5:], fine.experts[5:]) and torch.equal(r.weights[5:], fine.weights[5:])
    grad = routed.route_backward(logits.cuda(), r, torch.ones(tokens, 4).cuda())
    assert torch.isnan(grad[:4]).any(1).all() and (grad[4] == 0).all() and torch.isfinite(grad[5:]).all()


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("best", [1, 2])
def test_a_bias_excludes_experts(best, score):
    """An expert whose bias is -inf or NaN is not chosen; the others are as if its score were out of the choice."""
    g = torch.Generator().manual_seed(8)
    logits, bias = torch.randn(90, 32, generator=g), 0.3 * torch.randn(32, generator=g)
    bias[3], bias[17] = math.nan, -math.inf
    plain = {"groups": 4, "top_groups": 2, "group_best": best, "score": score}
    r = routed.route(logits.cuda(), 4, bias=bias.cuda(), **plain)
    low = bias.clone()
    low[[3, 17]] = -1e30                                  # below every other
    expected = routed.route(logits.cuda(), 4, bias=low.cuda(), **plain)
    assert not torch.isin(r.experts.cpu(), torch.tensor([3, 17])).any() and torch.isfinite(r.weights).all()
    assert all(torch.equal(a, b) for a, b in zip(r, expected))


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient_of_choices_far_below_the_largest(renormalize, score):
    """A bias picks experts whose scores are small: their gradient is as exact as any other's."""
    g = torch.Generator().manual_seed(5)
    logits = -torch.randint(8 * 20, 8 * 70, (100, 32), generator=g).float() / 8      # differences are exact
    logits[:, 0] = 0.0
    bias = torch.zeros(32)
    bias[1:4] = 8.0
    r = routed.route(logits.cuda(), 3, score=score, renormalize=renormalize, bias=bias.cuda())
    assert (r.experts.sort(1).values.cpu() == torch.tensor([1, 2, 3])).all()
    up = torch.randn(100, 3, generator=g).cuda()
    got = wide(routed.route_backward(logits.cuda(), r, up, score=score, renormalize=renormalize))
    x, chosen, grad = wide(logits), r.experts.long().cpu().numpy(), wide(up)
    e = np.exp(x)
    s = e / e.sum(1, keepdims=True) if score == "softmax" else 1 / (1 + np.exp(-x))
    p = np.take_along_axis(s, chosen, 1)
    size = np.abs(grad)
    if renormalize:
        total = p.sum(1, keepdims=True) + 1e-20
        mean = (grad * p / total).sum(1, keepdims=True)
        size = (size + (size * p / total).sum(1, keepdims=True)) / total
        grad = (grad - mean) / total
    ds, ds_size = np.zeros_like(s), np.zeros_like(s)
    np.put_along_axis(ds, chosen, grad, 1)
    np.put_along_axis(ds_size, chosen, size, 1)
    if score == "softmax":
        expected = s * (ds - (grad * p).sum(1, keepdims=True))
        magnitude = s * (ds_size + (size * p).sum(1, keepdims=True))
    else:
        expected, magnitude = ds * s * (1 - s), ds_size * s
    # Two exponentials of 2 units of 2^-23, their sums, three divisions of 2 and about five roundings: 16 units.
    near(torch.from_numpy(got), expected, 16 * 2.0 ** -23 * magnitude + 1e-37, "logits")


# ----------------------------------------------------------------------------------------------------------------
# Gated activation and its checkpoint


@gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("width, group", [(64, 32), (128, 64), (256, 128), (61, 32), (77, 64), (130, 128)])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_checkpoint_of_an_infinity_is_not_a_number(value, width, group, dtype):
    """The whole group of an infinite value loads as NaN, and its gradient is NaN: no infinity of the other sign."""
    h = torch.randn(3, 2 * width, generator=torch.Generator().manual_seed(width)).to(HALF[dtype][0])
    gate, up = 5, width + width - 1                       # the gate's first group, the up's last
    h[1, gate] = h[2, up] = value
    _, kept = routed.gated_save(h.cuda(), group=group)
    column = np.arange(2 * width)
    of = np.where(column < width, column // group, 1000 + (column - width) // group)
    values = wide(routed.checkpoint_load(kept))
    for row, at in ((1, gate), (2, up)):
        assert np.array_equal(np.isnan(values[row]), of == of[at])
        assert np.isfinite(values[row][of != of[at]]).all()
    assert np.isfinite(values[0]).all()
    h_grad, a, weights_grad = routed.gated_backward(kept, torch.ones(3, width).to(HALF[dtype][0]).cuda())
    assert torch.isnan(h_grad[1, gate]) and torch.isnan(h_grad[2, up - width]) and torch.isnan(a[2, up - width])
    assert torch.isnan(weights_grad[1:]).all() and torch.isfinite(weights_grad[0]) and torch.isfinite(h_grad[0]).all()


@gpu
def test_gates_far_below_zero_keep_bf16_range():
    """silu(-88) is -5e-37, a normal number of BF16: down to the smallest subnormal, 2^-133."""
    gates = -torch.linspace(80, 99, 96).bfloat16()
    h = torch.cat([gates, torch.ones(96).bfloat16()])[None].cuda()
    a, kept = routed.gated_save(h, group=32)
    g = wide(h)[0, :96]
    silu = g / (1 + np.exp(-g))
    # exp's argument is rounded: 1.2 |gate| + 2 units of 2^-23; the sigmoid may be a subnormal of 2^-149.
    slack = 125 * 2.0 ** -23
    near(a[0], silu, (1.01 * 2.0 ** -8 + slack) * np.abs(silu) + 2.0 ** -134 + 100 * 2.0 ** -149, "activation")
    assert float(a[0, 0]) < 0
    da = torch.ones(1, 96).bfloat16().cuda()
    h_grad, again, weights_grad = routed.gated_backward(kept, da)
    x = wide(routed.checkpoint_load(kept))[0]
    g, u = x[:96], x[96:]
    s = 1 / (1 + np.exp(-g))
    near(again[0], g * s * u, (1.01 * 2.0 ** -8 + slack) * np.abs(g * s * u) + 2.0 ** -134 + 100 * 2.0 ** -149, "again")
    both = np.concatenate([u * (s + g * s * (1 - s)), g * s])
    size = np.concatenate([np.abs(u) * (s + np.abs(g * s)), np.abs(g * s)])
    near(h_grad[0], both, 1.01 * 2.0 ** -8 * np.abs(both) + slack * size + 2.0 ** -134 + 200 * 2.0 ** -149, "gradient")


# ----------------------------------------------------------------------------------------------------------------
# 4-bit products


def plain_four(codes, scales, group):
    q = np.stack([codes.numpy() & 15, codes.numpy() >> 4], 3).reshape(codes.shape[0], codes.shape[1], -1)
    return (q.astype(np.float64) - 8) * np.repeat(wide(scales), group, axis=2)


@gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("tokens, experts, top_k, inner, outer, group",
                         [(1, 4, 2, 64, 24, 32), (5, 3, 2, 1152, 40, 64), (20, 2, 2, 2176, 300, 128),
                          (3, 7, 2, 96, 33, 32)])
def test_infinite_rows_through_4_bit_weights(tokens, experts, top_k, inner, outer, group, dtype):
    """An infinity times a weight is an infinity of the product's sign (NaN times a weight of zero, and NaN where
    infinities of both signs meet), in its own row only."""
    kind, unit, tiny = HALF[dtype]
    host, r = make_routing(tokens, experts, top_k, 31)
    g = torch.Generator().manual_seed(inner)
    x = torch.randn(tokens, inner, generator=g).to(kind)
    x[0, inner - 3] = math.inf
    if tokens > 2:
        x[1, 7], x[2, 1], x[2, inner // 2] = -math.inf, math.inf, math.nan
    if tokens > 4:
        x[4, 5], x[4, inner - 1] = math.inf, math.inf
    codes = torch.randint(0, 256, (experts, outer, inner // 2), generator=g, dtype=torch.uint8)
    codes[:, 0] = 0x88                                    # a row of zero weights
    scales = ((0.1 + torch.rand(experts, outer, inner // group, generator=g)) / math.sqrt(inner)).to(kind)
    got = routed.routed_matvec(x.cuda(), routed.Int4Weights(codes.cuda(), scales.cuda(), group), r, gather=True)
    w = plain_four(codes, scales, group)
    with np.errstate(all="ignore"):
        y, size = plain_product(host, wide(x), w.transpose(0, 2, 1), True, top_k)
        spread = np.broadcast_to(np.repeat(wide(scales), group, axis=2), w.shape)
        excess, _ = plain_product(host, np.abs(wide(x)), spread.transpose(0, 2, 1), True, top_k)
    assert np.isinf(y).any() and np.isnan(y).any()
    # A group's sum is one of (16 + q) x from -24 x on, whatever its weights are; the groups' sums are added.
    error = group * 2.0 ** -23 * 55 * excess + inner // group * 2.0 ** -23 * size
    near(got, y, np.where(np.isfinite(y), 1.01 * unit * np.abs(y) + tiny + error, 0.0), "rows")


@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
def test_large_rows_through_4_bit_weights(group):
    """BF16 values whose products fit 32 bits, though 16 times them, or their sum, would not."""
    inner, outer = 256, 40
    host, r = make_routing(4, 2, 1, 32)
    g = torch.Generator().manual_seed(group)
    x = torch.randn(4, inner, generator=g).bfloat16()
    x[0, 3], x[0, 9] = 2e37, 2e37
    x[1, 3], x[1, 200] = 2e37, -2e37
    x[2] = 1e36
    codes = torch.randint(0, 256, (2, outer, inner // 2), generator=g, dtype=torch.uint8)
    scales = torch.full((2, outer, inner // group), 2.0 ** -6).bfloat16()
    got = routed.routed_matvec(x.cuda(), routed.Int4Weights(codes.cuda(), scales.cuda(), group), r, gather=True)
    y, size = plain_product(host, wide(x), plain_four(codes, scales, group).transpose(0, 2, 1), True, 1)
    near(got, y, 1.01 * 2.0 ** -8 * np.abs(y) + inner * 2.0 ** -23 * size, "rows")


@gpu
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_packed_weights_that_are_not_finite_stay_so(value):
    """A weight that has no 4-bit code makes its group NaN, and no infinity of the other sign or finite value."""
    w = torch.randn(2, 128, 6, generator=torch.Generator().manual_seed(3)).bfloat16()
    w[1, 40, 2] = value
    _, r = make_routing(8, 2, 2, 33)
    got = routed.routed_matvec(torch.ones(8, 128).bfloat16().cuda(), routed.pack_int4(w.cuda(), 32), r, gather=True)
    bad = torch.zeros(16, 6, dtype=torch.bool)
    bad[int(r.offsets[1]):, 2] = True                     # expert 1's rows
    assert torch.equal(torch.isnan(got).cpu(), bad) and torch.isfinite(got.cpu()[~bad]).all()


# ----------------------------------------------------------------------------------------------------------------
# Strides and graphs


@gpu
@pytest.mark.parametrize("begin", [0, 3, 8])
def test_rows_of_wider_tensors(begin):
    """Every row operand as columns of a wider tensor, on 16-byte boundaries and off them: the bits of a copy."""
    host, r = make_routing(60, 6, 3, 41)
    g = torch.Generator().manual_seed(begin)
    store = torch.randn(180, 320, generator=g).half().cuda()
    wider = torch.randn(60, 320, generator=g).half().cuda()

    def part(rows, width):
        return rows[:, begin:begin + width]
    y = part(store, 136)
    assert torch.equal(routed.routed_sum(y, r), routed.routed_sum(y.contiguous(), r))
    h = part(store, 272)
    a, kept = routed.gated_save(h, routing=r)
    copied, copied_kept = routed.gated_save(h.contiguous(), routing=r)
    assert all(torch.equal(one, other) for one, other in zip((a, *kept[:2]), (copied, *copied_kept[:2])))
    assert torch.equal(routed.gated(h, routing=r), a)
    da = part(store, 136)
    strided = routed.gated_backward(kept, da, routing=r)
    for one, other in zip(strided, routed.gated_backward(kept, da.contiguous(), routing=r)):
        # Off the boundaries a lane has other columns: the weight's gradient is summed in another order.
        if one.dtype == torch.float16:
            assert torch.equal(one, other)
        else:
            assert torch.allclose(one, other, rtol=0, atol=136 * 2.0 ** -23 * 60)
    x = part(wider, 64)
    for gather_y in (False, True):
        dy = part(wider if gather_y else store, 136)
        got = routed.routed_weight_grad(x, dy, r, gather_x=True, gather_y=gather_y)
        expected, size = np.zeros((6, 64, 136)), np.zeros((6, 64, 136))
        for e in range(6):
            p = np.arange(host[4][e], host[4][e + 1])
            left, right = wide(x)[host[2][p] // 3], wide(dy)[host[2][p] // 3 if gather_y else p]
            expected[e], size[e] = left.T @ right, np.abs(left).T @ np.abs(right)
        near(got, expected, 1.01 * 2.0 ** -11 * np.abs(expected) + 2.0 ** -25 + 180 * 2.0 ** -23 * size)
    codes = torch.randint(0, 256, (6, 40, 32), generator=g, dtype=torch.uint8).cuda()
    four = routed.Int4Weights(codes, torch.rand(6, 40, 2, generator=g).half().cuda(), 32)
    assert torch.equal(routed.routed_matvec(x, four, r, gather=True),
                       routed.routed_matvec(x.contiguous(), four, r, gather=True))
    rows = part(store, 64)
    assert torch.equal(routed.routed_matvec(rows, four, r), routed.routed_matvec(rows.contiguous(), four, r))


@gpu
@pytest.mark.parametrize("tokens", [3, 200])
def test_a_captured_layer_repeats_its_results(tokens):
    layer = routed_layer.RoutedLayer(128, 64, 8, 2, seed=7)
    served = routed_layer.ServedLayer(layer)
    x = torch.randn(tokens, 128, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    y_grad = torch.randn(tokens, 128, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()

    def step():
        y, saved = layer.forward(x)
        x_grad, grads = layer.backward(saved, y_grad)
        return (y, x_grad, *grads, served(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (3, 4):
        x.copy_(torch.randn(tokens, 128, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        for one, other in zip(captured, step()):
            assert torch.equal(one, other)


# ----------------------------------------------------------------------------------------------------------------
# Threads


@gpu
@pytest.mark.parametrize("name", ["routed_matmul", "routed_weight_grad", "routed_matvec"])
def test_a_threads_first_call(name):
    """A thread that has not used the device yet, as autograd's are: the same result as on the main thread."""
    _, r = make_routing(12, 4, 2, 17)
    x, w = torch.randn(12, 64).bfloat16().cuda(), torch.randn(4, 64, 32).bfloat16().cuda()
    y = torch.randn(24, 32).bfloat16().cuda()
    call = {"routed_matmul": lambda: routed.routed_matmul(x, w, r, gather=True),
            "routed_weight_grad": lambda: routed.routed_weight_grad(x, y, r, gather_x=True),
            "routed_matvec": lambda: routed.routed_matvec(x, routed.Int4Weights(*four), r, gather=True)}[name]
    four = routed.pack_int4(w, 32)
    expected = call()
    found = []

    def work():
        try:
            found.append(call())
        except Exception as error:
            found.append(error)
    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    assert isinstance(found[0], torch.Tensor), found[0]
    assert torch.equal(found[0], expected)


# ----------------------------------------------------------------------------------------------------------------
# Autograd


@gpu
def test_autograd_is_refused_and_not_ignored():
    _, r = make_routing(6, 4, 2, 1)
    x, w = torch.randn(6, 32).half().cuda(), torch.randn(4, 32, 16).half().cuda()
    h, logits = torch.randn(12, 32).half().cuda(), torch.randn(6, 4).cuda()
    a, kept = routed.gated_save(h)
    four = routed.pack_int4(w, 32)
    calls = [
        (lambda t: routed.route(t, 2), logits),
        (lambda t: routed.route_backward(t, r, torch.ones(6, 2).cuda()), logits),
        (lambda t: routed.route_backward(logits, r, t), torch.ones(6, 2).cuda()),
        (lambda t: routed.routed_matmul(t, w, r, gather=True), x),
        (lambda t: routed.routed_matmul(x, t, r, gather=True), w),
        (lambda t: routed.routed_matmul(x, w, r, gather=True, out=t), torch.empty(12, 16).half().cuda()),
        (lambda t: routed.routed_weight_grad(t, h, r, gather_x=True), x),
        (lambda t: routed.routed_weight_grad(x, t, r, gather_x=True), h),
        (lambda t: routed.routed_sum(t, r), h),
        (lambda t: routed.gated_save(t), h),
        (lambda t: routed.gated(t), h),
        (lambda t: routed.gated_save(h, routing=r._replace(weights=t)), r.weights.clone()),
        (lambda t: routed.gated_backward(kept, t), a.clone()),
        (lambda t: routed.checkpoint_load(kept._replace(scales=t)), kept.scales.clone()),
        (lambda t: routed.routed_matvec(t, four, r, gather=True), x),
        (lambda t: routed.routed_matvec(x, four._replace(scales=t), r, gather=True), four.scales.clone()),
    ]
    for number, (call, tensor) in enumerate(calls):
        leaf = tensor.detach().clone().requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            call(leaf)
            raise AssertionError(f"call {number} was taken")
        with torch.no_grad():
            call(leaf)
        call(leaf.detach())


@gpu
def test_weights_that_train_are_packed_without_a_graph():
    w = torch.randn(2, 64, 8).bfloat16().cuda().requires_grad_()
    packed = routed.pack_int4(w, 32)
    assert not packed.scales.requires_grad
    plain = routed.pack_int4(w.detach(), 32)
    assert torch.equal(packed.codes, plain.codes) and torch.equal(packed.scales, plain.scales)


@gpu
def test_a_bias_has_no_gradient_and_is_taken():
    logits, bias = torch.randn(9, 8).cuda(), torch.randn(8).cuda()
    r = routed.route(logits, 2, bias=bias.clone().requires_grad_())
    assert all(torch.equal(a, b) for a, b in zip(r, routed.route(logits, 2, bias=bias)))


class Product(torch.autograd.Function):
    """How a user joins the operators to autograd: each backward operator in its own Function."""
    @staticmethod
    def forward(ctx, x, w, *routing):
        r = routed.Routing(*routing)
        ctx.save_for_backward(x, w, *routing)
        return routed.routed_sum(routed.routed_matmul(x, w, r, gather=True), r)

    @staticmethod
    def backward(ctx, y_grad):
        x, w, *routing = ctx.saved_tensors
        r = routed.Routing(*routing)
        rows = routed.routed_matmul(y_grad, w, r, gather=True, transpose=True)
        w_grad = routed.routed_weight_grad(x, y_grad, r, gather_x=True, gather_y=True)
        return routed.routed_sum(rows, r), w_grad, *[None] * 5


@gpu
def test_operators_inside_a_function():
    host, r = make_routing(40, 4, 2, 21)
    g = torch.Generator().manual_seed(2)
    x = torch.randint(-2, 3, (40, 64), generator=g).bfloat16().cuda().requires_grad_()
    w = torch.randint(-2, 3, (4, 64, 8), generator=g).bfloat16().cuda().requires_grad_()
    y = Product.apply(x, w, *r)
    y.backward(torch.ones_like(y))
    xd, wd = x.detach().double().cpu().requires_grad_(), w.detach().double().cpu().requires_grad_()
    chosen = torch.from_numpy(host[0]).long()
    expected = torch.einsum("ti,tkio->to", xd, wd[chosen])
    expected.backward(torch.ones_like(expected))
    # sums of whole numbers: exact up to 256, beyond that one rounding of each row and of the sum
    assert torch.allclose(y.detach().double().cpu(), expected.detach(), rtol=2 * 2.0 ** -8, atol=2.0)
    assert torch.allclose(x.grad.double().cpu(), xd.grad, rtol=2 * 2.0 ** -8, atol=0.5)
    assert torch.allclose(w.grad.double().cpu(), wd.grad, rtol=2.0 ** -8, atol=0.5)


SHARED_LIMIT = r"""
// AllowShared with the runtime's calls replaced: the limit that a kernel has, as two threads raise it.
#include <cuda_runtime.h>

#include <chrono>
#include <condition_variable>
#include <mutex>
#include <thread>

std::mutex g_mutex;
std::condition_variable g_changed;
int g_limit = 0;
bool g_shrunk = false, g_large_set = false, g_small_done = false;

cudaError_t FakeDevice(int* device) { return *device = 0, cudaSuccess; }

template <typename Kernel>
cudaError_t FakeAttribute(Kernel*, cudaFuncAttribute, int bytes) {
  std::unique_lock<std::mutex> lock(g_mutex);
  g_shrunk = g_shrunk || bytes < g_limit;
  g_limit = bytes;
  if (bytes == 200000) {   // the other thread's call comes before this one returns, if it can
    g_large_set = true;
    g_changed.notify_all();
    g_changed.wait_for(lock, std::chrono::milliseconds(500), [] { return g_small_done; });
  }
  return cudaSuccess;
}
#define cudaGetDevice FakeDevice
#define cudaFuncSetAttribute FakeAttribute
#include "routed.cuh"

namespace t0b {
void Check(cudaError_t, const char*) {}
}

__global__ void Nothing() {}

int main() {
  std::thread large([] { t0b::AllowShared<Nothing>(200000); });
  std::thread small([] {
    {
      std::unique_lock<std::mutex> lock(g_mutex);
      g_changed.wait(lock, [] { return g_large_set; });
    }
    t0b::AllowShared<Nothing>(60000);
    const std::lock_guard<std::mutex> lock(g_mutex);
    g_small_done = true;
    g_changed.notify_all();
  });
  large.join();
  small.join();
  t0b::AllowShared<Nothing>(200000);
  return g_shrunk || g_limit != 200000;
}
"""


def test_a_kernels_shared_memory_limit_only_grows(tmp_path):
    source, program = tmp_path / "limit.cu", tmp_path / "limit"
    source.write_text(SHARED_LIMIT)
    subprocess.run([build.nvcc(), *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr", "-I", str(build.CSRC),
                    str(source), "-o", str(program)], check=True)
    assert subprocess.run([str(program)], timeout=60).returncode == 0


# ----------------------------------------------------------------------------------------------------------------
# Refusals

MOST = (1 << 31) - 256          # entries


@pytest.mark.parametrize("entries", [MOST + 1, (1 << 31) - 1])
def test_more_entries_than_the_indices_hold_are_refused(entries):
    """Kernels form indices of up to a tile past the last entry in 32 bits.  (The missing operand is refused later.)"""
    for name, arguments in [
            ("t0b_route", (11, entries, 8, 1, 1, 1, 1, 0, 1, 1.0, None, 8, None, None, A, B, C, D, E, F, 1 << 40)),
            ("t0b_route_backward", (11, entries, 8, 1, 0, 1, 1.0, None, 8, B, C, D)),
            ("t0b_routed_product", (10, 0, entries, 2, 1, 16, 32, 0, None, entries, 16, B, C, D, E)),
            ("t0b_routed_product", (10, 1, entries, 2, 1, 16, 32, 1, None, entries, 32, B, C, D, E)),
            ("t0b_routed_weight_grad", (10, entries, 2, 1, 16, 32, 0, None, entries, 16, 0, B, entries, 32, C, D, E)),
            ("t0b_routed_sum", (10, entries, 1, 8, None, 8, B, C)),
            ("t0b_routed_matvec4", (10, entries, 2, 1, 64, 32, 32, 1, None, entries, 64, B, C, D, E, F))]:
        status, text = call(name, *arguments)
        assert status == 1 and "2^31 - 256" in text, (name, text)


@pytest.mark.parametrize("name, arguments", [
    ("t0b_gated_save", (10, 4, 8, 32, A, 16, B, C, D, 2, D, E, F)),                     # a
    ("t0b_gated_save", (10, 4, 8, 32, A, 16, B, C, D + 8, 2, E, D, F)),                 # codes, from 8 bytes before on
    ("t0b_gated_save", (10, 4, 8, 32, A, 16, B, C, D, 2, E, F, D)),                     # scales
    ("t0b_gated_backward", (10, 4, 8, 32, A, B, C, 8, E, F, D, 2, D, G, H)),            # h_grad
    ("t0b_gated_backward", (10, 4, 8, 32, A, B, C, 8, E, F, D, 2, G, D, H)),            # a
    ("t0b_gated_backward", (10, 4, 8, 32, A, B, C, 8, E, F, D, 2, G, H, D)),            # weights_grad
])
def test_gated_results_over_the_routings_offsets_are_refused(name, arguments):
    """Every block reads the offsets while others write."""
    status, text = call(name, *arguments)
    assert status == 1 and "overlap" in text, text


@pytest.mark.parametrize("tokens, experts", [(1000, 513), (1000, 1 << 30), (MOST + 1, 8), (1 << 60, 8), (-1, 8),
                                             (1000, 0)])
def test_a_route_that_is_refused_needs_no_workspace(tokens, experts):
    """The binding asks for the size before the router checks its arguments: no memory for what it refuses."""
    build.build()
    assert _native.lib().t0b_route_workspace(tokens, experts) == 0
    assert _native.lib().t0b_route_workspace(1000, 512) > 0


@gpu
@pytest.mark.parametrize("experts", [4, 16])
def test_router_gradient_refuses_another_routers_routing(experts):
    logits = torch.randn(10, 8).cuda()
    r = routed.route(torch.randn(10, experts).cuda(), 2)
    with pytest.raises(ValueError, match="experts"):
        routed.route_backward(logits, r, torch.ones(10, 2).cuda())
