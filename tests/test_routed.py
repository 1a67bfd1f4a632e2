"""Routed operators against plain implementations in 64 bits: router, products, sums, gated activations with 8-bit
checkpoints and 4-bit products, at the sizes and masks where they can go wrong.

Tolerances follow from the arithmetic and were set before the first run.  A value rounded once to F16 or BF16 is off
by at most u = 2^-11 or 2^-8 of its magnitude (half a unit in the last place), plus half the smallest subnormal of
F16.  A sum of n products in 32 bits is off by at most n 2^-23 of the sum of the products' magnitudes: 2^-24 per
rounded addition, twice that for the tensor cores' truncated additions.
"""

import math

import numpy as np
import pytest
import torch

from tensor0_b200 import _native, build, routed

gpu = pytest.mark.gpu

HALF = {"f16": (torch.float16, 2.0 ** -11, 2.0 ** -25), "bf16": (torch.bfloat16, 2.0 ** -8, 0.0)}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def wide(tensor):
    return tensor.detach().to("cpu", torch.float64).numpy()


# ----------------------------------------------------------------------------------------------------------------
# Plain implementations


def plain_choice(x, top_k, groups, top_groups, best, softmax, bias, mask):
    """(experts [tokens, top_k], scores [tokens, experts]): the choice by values of 32 bits, as the router defines
    it, token by token; the scores in 64 bits."""
    tokens, experts = x.shape
    chosen = np.full((tokens, top_k), -1, np.int32)
    scores = np.zeros((tokens, experts))
    for t in range(tokens):
        if mask is not None and not mask[t]:
            continue
        row = x[t].astype(np.float64)
        with np.errstate(all="ignore"):
            if softmax:
                e = np.exp(row - row.max())
                scores[t] = e / e.sum()
            else:
                scores[t] = 1 / (1 + np.exp(-row))
        value = row if bias is None and best == 1 else scores[t] + (0 if bias is None else bias)
        value = np.where(row > -np.inf, value, -np.inf)
        value = np.where(np.isnan(value), -np.inf, value)
        size = experts // groups
        ranked = []
        for g in range(groups):
            part = np.sort(value[g * size:(g + 1) * size])[::-1]
            total = part[0] + (part[1] if best == 2 and size > 1 and part[1] > -np.inf else 0)
            ranked.append((-total, g))
        kept = {g for _, g in sorted(ranked)[:top_groups]}
        order = sorted((-value[e], e) for e in range(experts) if e // size in kept and value[e] > -np.inf)
        for n, (_, e) in enumerate(order[:top_k]):
            chosen[t, n] = e
    return chosen, scores


def plain_weights(chosen, scores, renormalize, scale):
    picked = np.where(chosen >= 0, np.take_along_axis(scores, np.maximum(chosen, 0), 1), 0.0)
    return scale * (picked / (picked.sum(1, keepdims=True) + 1e-20) if renormalize else picked)


def plain_order(chosen, experts):
    """rows, positions, offsets by a loop over the entries."""
    flat = chosen.reshape(-1)
    rows = [i for e in [*range(experts), -1] for i in range(flat.size) if flat[i] == e]
    positions = np.full(flat.size, -1, np.int32)
    for p, i in enumerate(rows):
        if flat[i] >= 0:
            positions[i] = p
    offsets = np.cumsum([0] + [int((flat == e).sum()) for e in range(experts)])
    return np.array(rows, np.int32), positions.reshape(chosen.shape), offsets.astype(np.int32)


def make_routing(tokens, experts, top_k, seed, absent=0.0, only=None):
    """A routing (host arrays, device Routing): random experts, `absent` of the entries without one, or all entries
    among the experts `only`."""
    rng = np.random.default_rng(seed)
    pool = np.arange(experts) if only is None else np.array(only)
    chosen = np.stack([rng.permutation(pool)[:top_k] if len(pool) >= top_k else rng.choice(pool, top_k)
                       for _ in range(tokens)]) if tokens else np.zeros((0, top_k))
    chosen = np.where(rng.random((tokens, top_k)) < absent, -1, chosen).astype(np.int32)
    weights = rng.uniform(0.05, 1.0, (tokens, top_k)).astype(np.float32) * (chosen >= 0)
    rows, positions, offsets = plain_order(chosen, experts)
    host = (chosen, weights.astype(np.float32), rows, positions, offsets)
    return host, routed.Routing(*(torch.from_numpy(np.ascontiguousarray(v)).cuda() for v in host))


def near(got, expected, bound, what=""):
    """Every value within its bound; values that are not finite in the same places."""
    got = wide(got)
    assert got.shape == expected.shape, what
    assert np.array_equal(np.isnan(got), np.isnan(expected)), what
    fine = np.isfinite(expected)
    assert np.array_equal(got[~fine & ~np.isnan(expected)], expected[~fine & ~np.isnan(expected)]), what
    worst = np.max(np.abs(got - expected)[fine] - np.broadcast_to(bound, expected.shape)[fine], initial=-np.inf)
    assert worst <= 0, f"{what}: off by {worst} more than the bound"


# ----------------------------------------------------------------------------------------------------------------
# Router

ROUTES = [
    # tokens, experts, top_k, groups, top_groups, best, score, bias, renormalize, dtype, mask
    (1, 1, 1, 1, 1, 1, "softmax", False, True, "f32", None),
    (1, 8, 2, 1, 1, 1, "softmax", False, False, "bf16", None),
    (3, 33, 32, 1, 1, 1, "sigmoid", False, True, "f16", None),
    (64, 64, 4, 1, 1, 1, "softmax", False, True, "f32", "some"),
    (65, 40, 6, 8, 3, 1, "softmax", True, True, "bf16", "some"),
    (130, 256, 8, 8, 4, 2, "sigmoid", True, True, "f32", "some"),
    (77, 512, 10, 32, 5, 2, "softmax", True, False, "f16", None),
    (257, 96, 5, 4, 1, 2, "sigmoid", False, True, "f32", "none"),
    (1000, 20, 7, 10, 2, 1, "sigmoid", False, False, "f32", "some"),   # four experts stay for seven slots
    (3001, 128, 8, 1, 1, 1, "softmax", False, True, "bf16", "some"),
]


def route_inputs(tokens, experts, dtype, bias, mask, seed):
    g = torch.Generator().manual_seed(seed)
    logits = (2 * torch.randn(tokens, experts, generator=g)).to(TYPES[dtype])
    logits[torch.rand(tokens, experts, generator=g) < 0.05] = -math.inf      # excluded experts
    if tokens > 4:
        logits[2] = -math.inf                                                 # nothing to choose
        logits[3] = 0.5                                                       # all tied
    alive = None
    if mask is not None:
        alive = torch.rand(tokens, generator=g) < (0.7 if mask == "some" else 0.0)
        logits[~alive] = math.nan
        logits[~alive, ::2] = math.inf
    b = 0.3 * torch.randn(experts, generator=g) if bias else None
    return logits.cuda(), None if b is None else b.cuda(), None if alive is None else alive.cuda()


@gpu
@pytest.mark.parametrize("tokens, experts, top_k, groups, top_groups, best, score, bias, renormalize, dtype, mask",
                         ROUTES)
def test_route(tokens, experts, top_k, groups, top_groups, best, score, bias, renormalize, dtype, mask):
    logits, b, alive = route_inputs(tokens, experts, dtype, bias, mask, tokens + experts)
    r = routed.route(logits, top_k, groups=groups, top_groups=top_groups, group_best=best, score=score, bias=b,
                     mask=alive, renormalize=renormalize, scale=1.5)
    x = logits.float().cpu().numpy()
    chosen, scores = plain_choice(x, top_k, groups, top_groups, best, score == "softmax",
                                  None if b is None else wide(b), None if alive is None else alive.cpu().numpy())
    got = r.experts.cpu().numpy()
    # A choice that differs is allowed only where 32-bit choice values are closer than their rounding.
    for t in np.unique(np.nonzero(got != chosen)[0]):
        assert b is not None or best == 2, t
        value = scores[t] + (0 if b is None else wide(b))
        ours, theirs = value[got[t][got[t] >= 0]], value[chosen[t][chosen[t] >= 0]]
        assert ours.size == theirs.size and np.max(np.abs(np.sort(ours) - np.sort(theirs))) < 2.0 ** -20, t
    weights = plain_weights(got, scores, renormalize, 1.5)
    # exp, a division, a sum of up to 32 scores and another division: 32 units of 2^-23 hold them.
    near(r.weights, weights, 32 * 2.0 ** -23 * np.abs(weights) + 1e-30, "weights")
    rows, positions, offsets = plain_order(got, experts)
    assert np.array_equal(r.rows.cpu().numpy(), rows)
    assert np.array_equal(r.positions.cpu().numpy(), positions)
    assert np.array_equal(r.offsets.cpu().numpy(), offsets)


@gpu
@pytest.mark.parametrize("tokens, experts, top_k, groups, top_groups, best, score, bias, renormalize, dtype, mask",
                         ROUTES)
def test_route_backward(tokens, experts, top_k, groups, top_groups, best, score, bias, renormalize, dtype, mask):
    logits, b, alive = route_inputs(tokens, experts, dtype, bias, mask, tokens + experts)
    r = routed.route(logits, top_k, groups=groups, top_groups=top_groups, group_best=best, score=score, bias=b,
                     mask=alive, renormalize=renormalize, scale=1.5)
    g = torch.randn(tokens, top_k, generator=torch.Generator().manual_seed(9)).cuda()
    got = routed.route_backward(logits, r, g, score=score, renormalize=renormalize, scale=1.5)
    assert got.dtype == logits.dtype
    chosen = r.experts.cpu().numpy()
    x = logits.float().cpu().numpy().astype(np.float64)
    dead = np.all(chosen < 0, axis=1)
    x[dead] = 0.0
    found = chosen >= 0
    with np.errstate(all="ignore"):
        e = np.exp(x - x.max(1, keepdims=True))
        s = e / e.sum(1, keepdims=True) if score == "softmax" else 1 / (1 + np.exp(-x))
    p = np.where(found, np.take_along_axis(s, np.maximum(chosen, 0), 1), 0.0)
    up = np.where(found, wide(g) * 1.5, 0.0)
    total = p.sum(1, keepdims=True) + 1e-20
    size = np.abs(up)
    if renormalize:
        mean = (up * p / total).sum(1, keepdims=True)
        size = np.where(found, (np.abs(up) + (np.abs(up) * p / total).sum(1, keepdims=True)) / total, 0.0)
        up = np.where(found, (up - mean) / total, 0.0)
    ds, ds_size = np.zeros_like(s), np.zeros_like(s)
    for n in range(top_k):
        t = np.nonzero(found[:, n])[0]
        ds[t, chosen[t, n]] = up[t, n]
        ds_size[t, chosen[t, n]] = size[t, n]
    if score == "softmax":
        expected = s * (ds - (up * p).sum(1, keepdims=True))
        magnitude = s * (ds_size + (size * p).sum(1, keepdims=True))
    else:
        expected = ds * s * (1 - s)
        magnitude = ds_size * s * 2
    expected[dead] = 0.0
    magnitude[dead] = 0.0
    unit, tiny = {"f32": (2.0 ** -24, 0.0), "f16": HALF["f16"][1:], "bf16": HALF["bf16"][1:]}[dtype]
    near(got, expected, 1.01 * unit * np.abs(expected) + tiny + 64 * 2.0 ** -23 * magnitude + 1e-37, "logits")


@gpu
def test_route_gradient_against_differences():
    """The gradient against central differences of the plain weights in 64 bits, for a choice that does not change."""
    logits, _, _ = route_inputs(6, 24, "f32", False, None, 3)
    logits = logits.nan_to_num(neginf=-3.0)
    for score, renormalize in (("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)):
        r = routed.route(logits, 5, score=score, renormalize=renormalize)
        g = torch.randn(6, 5, generator=torch.Generator().manual_seed(2)).cuda()
        got = wide(routed.route_backward(logits, r, g, score=score, renormalize=renormalize))
        x, chosen, up = wide(logits), r.experts.cpu().numpy(), wide(g)

        def loss(values):
            e = np.exp(values - values.max(1, keepdims=True))
            s = e / e.sum(1, keepdims=True) if score == "softmax" else 1 / (1 + np.exp(-values))
            return (up * plain_weights(chosen, s, renormalize, 1.0)).sum(1)

        step = 1e-5
        for e in range(24):
            shift = np.zeros_like(x)
            shift[:, e] = step
            slope = (loss(x + shift) - loss(x - shift)) / (2 * step)
            # Truncation step^2, cancellation 1e-16 / step, and 32-bit rounding of terms below about 10.
            assert np.max(np.abs(got[:, e] - slope)) <= 1e-9 + 1e-10 + 64 * 2.0 ** -23 * 10


@gpu
@pytest.mark.parametrize("experts", [8, 60, 128, 200, 512])
def test_route_tells_neighbouring_logits_apart(experts):
    """Logits that differ in their last bits only, some of them equal, of both signs: the order is by all bits, then
    by index."""
    g = torch.Generator().manual_seed(experts)
    steps = torch.stack([torch.randperm(2 * experts, generator=g)[:experts] // 2 for _ in range(200)])
    logits = (1 + steps.double() * 2.0 ** -23).float()
    logits[1::2] *= -1
    logits[::3, ::2] += 0.25                                # a few far from the others
    r = routed.route(logits.cuda(), 8)
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :8]
    assert torch.equal(r.experts.cpu().long(), order)


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens", [1, 100])
def test_a_single_renormalised_choice_is_exact(tokens, score):
    """One expert of weight 1: no logit moves it."""
    logits = torch.randn(tokens, 20, generator=torch.Generator().manual_seed(1)).cuda()
    logits[:, 3:] -= 40.0 if tokens == 1 else 0.0
    r = routed.route(logits, 1, score=score)
    assert (r.weights == 1).all()
    grad = routed.route_backward(logits, r, torch.randn(tokens, 1).cuda(), score=score)
    assert (grad == 0).all()


@gpu
def test_route_surfaces_numbers_that_are_not():
    logits = torch.randn(3, 16).cuda()
    logits[0, 5] = math.nan
    logits[1, 5] = math.inf
    r = routed.route(logits, 3)
    assert 5 not in r.experts[0].tolist() and r.experts[1, 0].item() == 5
    assert torch.isnan(r.weights[:2]).all() and torch.isfinite(r.weights[2]).all()


@gpu
def test_route_takes_strided_logits_preallocated_results_and_a_stream():
    store = torch.randn(300, 72).cuda()
    logits = store[:, 4:68]
    expected = routed.route(logits.contiguous(), 6)
    out = routed.empty_routing(300, 6, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r = routed.route(logits, 6, out=out)
    torch.cuda.current_stream().wait_stream(side)
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(r, out))
    assert all(torch.equal(a, b) for a, b in zip(r, expected))


# ----------------------------------------------------------------------------------------------------------------
# Products

PRODUCTS = [
    # tokens, experts, top_k, inner, outer, absent, only
    (0, 3, 2, 16, 16, 0.0, None),
    (1, 4, 1, 8, 8, 0.0, None),
    (1, 4, 3, 24, 40, 1.0, None),              # no entry has an expert
    (5, 9, 2, 64, 256, 0.3, None),
    (70, 5, 3, 72, 136, 0.2, (0, 4)),          # experts without rows between and around
    (129, 2, 2, 200, 264, 0.0, None),          # one row past a tile
    (300, 1, 1, 64, 512, 0.0, None),
    (260, 24, 4, 136, 648, 0.1, None),
    (40, 6, 2, 33, 17, 0.2, None),             # rows that no 16-byte copy can start on
    (40, 6, 2, 40, 19, 0.2, None),
    (40, 6, 2, 21, 48, 0.2, None),
    (513, 3, 2, 1032, 520, 0.05, None),
    (300, 30, 2, 72, 640, 0.1, None),          # enough tiles for the wider ones, forward and transposed
    (300, 30, 2, 640, 72, 0.1, None),
    (700, 40, 2, 72, 1032, 0.1, None),
    (700, 40, 2, 1032, 72, 0.1, None),
]


def product_inputs(tokens, inner, outer, experts, dtype, seed, rows):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, inner, generator=g).to(dtype)
    w = (torch.randn(experts, inner, outer, generator=g) / math.sqrt(inner)).to(dtype)
    return x.cuda(), w.cuda()


def plain_product(host, x, w, gather, top_k, transpose=False):
    """(values, sums of magnitudes) of the products of expert-ordered rows."""
    chosen, _, rows, _, offsets = host
    width = w.shape[1] if transpose else w.shape[2]
    y, size = np.zeros((rows.size, width)), np.zeros((rows.size, width))
    for e in range(w.shape[0]):
        part = np.arange(offsets[e], offsets[e + 1])
        left = x[rows[part] // top_k if gather else part]
        right = w[e].T if transpose else w[e]
        y[part] = left @ right
        size[part] = np.abs(left) @ np.abs(right)
    return y, size


@gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("tokens, experts, top_k, inner, outer, absent, only", PRODUCTS)
def test_routed_matmul(tokens, experts, top_k, inner, outer, absent, only, transpose, gather, dtype):
    kind, unit, tiny = HALF[dtype]
    host, r = make_routing(tokens, experts, top_k, 7, absent, only)
    rows = tokens if gather else tokens * top_k
    x, w = product_inputs(tokens, inner, outer, experts, kind, 3, rows)
    if transpose:
        x = product_inputs(tokens, outer, inner, 1, kind, 4, rows)[0]
    if absent and not gather:
        live = host[4][-1]
        x[live:] = math.nan                    # rows without an expert are nobody's business
    got = routed.routed_matmul(x, w, r, gather=gather, transpose=transpose)
    y, size = plain_product(host, wide(x), wide(w), gather, top_k, transpose)
    deep = outer if transpose else inner
    near(got, y, 1.01 * unit * np.abs(y) + tiny + deep * 2.0 ** -23 * size, "rows")


@gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("gather_x, gather_y", [(True, False), (False, True), (False, False), (True, True)])
@pytest.mark.parametrize("tokens, experts, top_k, inner, outer, absent, only", PRODUCTS)
def test_routed_weight_grad(tokens, experts, top_k, inner, outer, absent, only, gather_x, gather_y, dtype):
    kind, unit, tiny = HALF[dtype]
    host, r = make_routing(tokens, experts, top_k, 8, absent, only)
    chosen, _, rows, _, offsets = host
    x = product_inputs(tokens, inner, 1, 1, kind, 5, tokens if gather_x else tokens * top_k)[0]
    y = product_inputs(tokens, outer, 1, 1, kind, 6, tokens if gather_y else tokens * top_k)[0]
    if absent:
        for operand, gathered in ((x, gather_x), (y, gather_y)):
            if not gathered:
                operand[offsets[-1]:] = math.nan
    got = routed.routed_weight_grad(x, y, r, gather_x=gather_x, gather_y=gather_y)
    expected, size = np.zeros((experts, inner, outer)), np.zeros((experts, inner, outer))
    for e in range(experts):
        part = np.arange(offsets[e], offsets[e + 1])
        left = wide(x)[rows[part] // top_k if gather_x else part]
        right = wide(y)[rows[part] // top_k if gather_y else part]
        expected[e] = left.T @ right
        size[e] = np.abs(left).T @ np.abs(right)
    near(got, expected, 1.01 * unit * np.abs(expected) + tiny + max(1, tokens) * top_k * 2.0 ** -23 * size, "weights")


@gpu
def test_a_row_that_is_not_finite_stays_its_own():
    """An infinity or NaN in one row reaches that row's product and its own expert's gradient only."""
    host, r = make_routing(90, 4, 2, 11)
    chosen, _, rows, positions, offsets = host
    x = torch.randn(180, 64).bfloat16().cuda()
    w = torch.randn(4, 64, 128).bfloat16().cuda()
    bad = int(offsets[2])                      # the first row of expert 2: the last tile of expert 1 ends before it
    x[bad, 3] = math.nan
    x[bad + 1, 5] = math.inf
    y = routed.routed_matmul(x, w, r)
    fine = torch.isfinite(y).all(1)
    assert not fine[bad] and not fine[bad + 1] and fine[:bad].all() and fine[bad + 2:].all()
    for grad in (routed.routed_weight_grad(x, y.nan_to_num(0, 0, 0), r), routed.routed_weight_grad(x, y, r),
                 routed.routed_weight_grad(y.nan_to_num(0, 0, 0), x, r)):
        assert not torch.isfinite(grad[2]).all()
        assert torch.isfinite(grad[[0, 1, 3]]).all()


@gpu
@pytest.mark.parametrize("gather", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("inner,outer", [(128, 256), (72, 136)])
def test_weight_gradients_end_with_their_experts_rows(gather, inner, outer):
    """Row counts around the steps and slices of the sum, every second expert's rows not finite; whole numbers."""
    counts = [1, 3, 15, 2, 16, 5, 17, 1, 33, 40, 47, 48, 49, 9, 63, 64, 65, 1, 112, 7, 127, 128, 129, 30]
    offsets = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    total, expert = int(offsets[-1]), np.repeat(np.arange(len(counts)), counts)
    g = torch.Generator().manual_seed(13)
    rows = torch.randperm(total, generator=g)            # one slot: an entry is a token
    positions = torch.argsort(rows).int()
    r = routed.Routing(*(t.cuda() for t in (torch.from_numpy(expert)[positions.long()].int()[:, None],
                                            torch.ones(total, 1), rows.int(), positions[:, None],
                                            torch.from_numpy(offsets))))
    x = torch.randint(-3, 4, (total, inner), generator=g).bfloat16()
    y = torch.randint(-3, 4, (total, outer), generator=g).bfloat16()
    expected = np.zeros((len(counts), inner, outer))
    for e in range(0, len(counts), 2):
        expected[e] = wide(x[expert == e]).T @ wide(y[expert == e])
    x[expert % 2 == 1], y[expert % 2 == 1] = math.nan, math.inf

    def by_token(ordered):
        return ordered[positions.long()]
    got = routed.routed_weight_grad((by_token(x) if gather[0] else x).cuda(), (by_token(y) if gather[1] else y).cuda(), r,
                                    gather_x=gather[0], gather_y=gather[1])
    assert torch.equal(got[::2].cpu(), torch.from_numpy(expected[::2]).bfloat16())
    assert not torch.isfinite(got[1::2]).any()


@gpu
def test_products_take_strided_rows_and_repeat_their_bits():
    host, r = make_routing(200, 7, 3, 12)
    store = torch.randn(200, 160).half().cuda()
    w = torch.randn(7, 96, 64).half().cuda()
    for begin in (0, 8, 16, 3):                # 16-byte aligned rows, and rows that are not
        x = store[:, begin:begin + 96]
        y = routed.routed_matmul(x, w, r, gather=True)
        expected, size = plain_product(host, wide(x), wide(w), True, 3)
        near(y, expected, 1.01 * 2.0 ** -11 * np.abs(expected) + 2.0 ** -25 + 96 * 2.0 ** -23 * size)
        grad = routed.routed_weight_grad(x, y, r, gather_x=True)
        for _ in range(3):
            assert torch.equal(routed.routed_matmul(x, w, r, gather=True), y)
            assert torch.equal(routed.routed_weight_grad(x, y, r, gather_x=True), grad)


@gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("tokens, top_k, width", [(0, 2, 8), (1, 1, 1), (5, 3, 7), (64, 8, 264), (301, 4, 1000),
                                                  (33, 32, 513)])
def test_routed_sum(tokens, top_k, width, dtype):
    kind, unit, tiny = HALF[dtype]
    host, r = make_routing(tokens, 32, top_k, 13, absent=0.3)
    y = torch.randn(tokens * top_k, width, generator=torch.Generator().manual_seed(1)).to(kind).cuda()
    y[host[4][-1]:] = math.nan
    got = routed.routed_sum(y, r)
    values = wide(y)
    expected, size = np.zeros((tokens, width)), np.zeros((tokens, width))
    for t in range(tokens):
        for p in host[3][t]:
            if p >= 0:
                expected[t] += values[p]
                size[t] += np.abs(values[p])
    near(got, expected, 1.01 * unit * np.abs(expected) + tiny + top_k * 2.0 ** -23 * size, "sums")


# ----------------------------------------------------------------------------------------------------------------
# Gated activation and its checkpoint


def plain_codes(h, group):
    """Codes and scales by the stated rule in 32-bit steps (each step is one rounding, so the codes are exact)."""
    h = h.astype(np.float32)
    rows, width = h.shape[0], h.shape[1] // 2
    groups = -(-width // group)
    codes, scales = np.zeros((rows, 2 * width), np.int8), np.zeros((rows, 2 * groups), np.float32)
    for half in range(2):
        for j in range(groups):
            part = slice(half * width + j * group, half * width + min(width, (j + 1) * group))
            largest = np.abs(h[:, part]).max(1)
            some = largest >= np.float32(2.0 ** -100)
            with np.errstate(all="ignore"):
                unit = np.where(some, np.float32(1) / largest * np.float32(127), np.float32(0))
                scales[:, half * groups + j] = np.where(some, largest * np.float32(1 / 127), np.float32(0))
            codes[:, part] = np.clip(np.rint(h[:, part] * unit[:, None]), -127, 127)
    return codes, scales


def plain_values(codes, scales, group):
    rows, width = codes.shape[0], codes.shape[1] // 2
    groups = -(-width // group)
    column = np.arange(2 * width)
    return codes.astype(np.float64) * scales.astype(np.float64)[:, np.where(column < width, column // group,
                                                                           groups + (column - width) // group)]


GATED = [(0, 1, 8, 32), (1, 1, 1, 32), (3, 2, 7, 64), (9, 4, 64, 64), (50, 3, 136, 128), (31, 2, 1000, 32),
         (16, 8, 1416, 64), (200, 2, 513, 128)]


@gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("with_routing", [False, True])
@pytest.mark.parametrize("tokens, top_k, width, group", GATED)
def test_gated(tokens, top_k, width, group, with_routing, dtype):
    kind, unit, tiny = HALF[dtype]
    rows = tokens * top_k
    host, r = make_routing(tokens, 8, top_k, 14, absent=0.2)
    live = int(host[4][-1]) if with_routing else rows
    g = torch.Generator().manual_seed(rows + width)
    h = (2 * torch.randn(rows, 2 * width, generator=g)).to(kind)
    h[torch.rand(rows, 2 * width, generator=g) < 0.02] = 60.0
    if rows > 2:
        h[1] = 0.0
        h[2, : width // 2 + 1] = -30.0
    if with_routing:
        h[live:] = math.nan
    h = h.cuda()
    a, kept = routed.gated_save(h, routing=r if with_routing else None, group=group)
    values = wide(h)
    values[live:] = 0.0
    codes, scales = plain_codes(values, group)
    assert np.array_equal(kept.codes.cpu().numpy(), codes)
    assert np.array_equal(kept.scales.cpu().numpy(), scales)
    weight = np.zeros(rows)
    weight[:] = host[1].reshape(-1)[host[2]] if with_routing else 1.0

    def forward(v):
        gate, up = v[:, :width], v[:, width:]
        s = 1 / (1 + np.exp(-gate))
        return gate, up, s, weight[:, None] * gate * s * up

    _, _, _, expected = forward(values)
    # exp is off by up to about 2 + 1.2 |gate| units of 2^-23 (|gate| <= 60 here), the rest by a few.
    slack = 90 * 2.0 ** -23
    near(a, expected, (1.01 * unit + slack) * np.abs(expected) + tiny + 1e-36, "activation")
    loaded = plain_values(codes, scales, group)
    near(routed.checkpoint_load(kept), loaded, 2.0 ** -23 * np.abs(loaded), "values")
    near(routed.checkpoint_load(kept, kind), loaded, 1.01 * unit * np.abs(loaded) + tiny + 1e-38, "values")

    da = torch.randn(rows, width, generator=g).to(kind)
    if with_routing:
        da[live:] = math.nan
    da = da.cuda()
    dh, again, dw = routed.gated_backward(kept, da, routing=r if with_routing else None)
    gate, up, s, expected = forward(loaded)
    upstream = wide(da)
    upstream[live:] = 0.0
    silu = gate * s
    near(again, expected, (1.01 * unit + slack) * np.abs(expected) + tiny + 1e-36, "activation again")
    dg = weight[:, None] * upstream * up * (s + silu * (1 - s))
    dg_size = np.abs(weight[:, None] * upstream * up) * (s + np.abs(silu))
    du = weight[:, None] * upstream * silu
    near(dh, np.concatenate([dg, du], 1), 1.01 * unit * np.abs(np.concatenate([dg, du], 1)) + tiny + 1e-36
         + slack * np.concatenate([dg_size, np.abs(du)], 1), "input gradient")
    dots, dot_size = (upstream * silu * up).sum(1), np.abs(upstream * silu * up).sum(1)
    entry = host[2] if with_routing else np.arange(rows)
    expected_dw, dw_size = np.zeros(rows), np.zeros(rows)
    expected_dw[entry], dw_size[entry] = dots, dot_size
    near(dw.reshape(-1), expected_dw, (slack + width * 2.0 ** -23) * dw_size + 1e-36, "weight gradient")


@gpu
@pytest.mark.parametrize("with_routing", [False, True])
def test_gated_without_a_checkpoint(with_routing):
    _, r = make_routing(70, 8, 3, 14, absent=0.2)
    h = torch.randn(210, 2 * 136).bfloat16().cuda()
    a, _ = routed.gated_save(h, routing=r if with_routing else None)
    assert torch.equal(routed.gated(h, routing=r if with_routing else None), a)


@gpu
def test_gated_gradient_against_differences():
    """The gradient against central differences of the plain activation at the checkpoint's values."""
    width, group = 40, 32
    h = torch.randn(6, 2 * width, generator=torch.Generator().manual_seed(5)).half().cuda()
    da = torch.randn(6, width, generator=torch.Generator().manual_seed(6)).half().cuda()
    _, kept = routed.gated_save(h, group=group)
    dh, _, dw = routed.gated_backward(kept, da)
    x, up = wide(routed.checkpoint_load(kept)), wide(da)

    def loss(v, weight=1.0):
        return (up * weight * v[:, :width] / (1 + np.exp(-v[:, :width])) * v[:, width:]).sum(1)

    step = 1e-5
    for c in range(2 * width):
        shift = np.zeros_like(x)
        shift[:, c] = step
        slope = (loss(x + shift) - loss(x - shift)) / (2 * step)
        # Truncation and cancellation near 1e-9; the result is rounded to 11 bits.
        assert np.max(np.abs(wide(dh)[:, c] - slope) - 1.01 * 2.0 ** -11 * np.abs(slope)) <= 1e-5
    slope = (loss(x, 1 + step) - loss(x, 1 - step)) / (2 * step)
    assert np.max(np.abs(wide(dw) - slope)) <= 1e-4


@gpu
def test_checkpoint_groups_that_are_not_finite_or_tiny():
    h = torch.randn(4, 256).bfloat16()
    h[0, 5] = math.nan
    h[1, 40] = math.inf
    h[2, 64:96] = 1e-35
    h = h.cuda()
    _, kept = routed.gated_save(h, group=32)
    values = routed.checkpoint_load(kept)
    assert torch.isnan(values[0, :32]).all() and torch.isfinite(values[0, 32:]).all()
    assert torch.isnan(values[1, 32:64]).any() and torch.isfinite(values[1, 64:]).all()
    assert not torch.isfinite(values[1, 40])
    assert (values[2, 64:96] == 0).all() and torch.isfinite(values[2]).all()


# ----------------------------------------------------------------------------------------------------------------
# 4-bit products


@gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("tokens, experts, top_k, inner, outer, group, absent",
                         [(0, 2, 1, 32, 8, 32, 0.0), (1, 4, 2, 64, 1, 64, 0.0), (1, 16, 8, 512, 100, 128, 0.3),
                          (7, 3, 2, 96, 33, 32, 0.2), (40, 2, 2, 256, 24, 64, 0.0), (13, 20, 4, 1152, 257, 128, 0.1),
                          (3, 5, 2, 4256, 40, 32, 0.0), (5, 4, 2, 8320, 48, 64, 0.0)])
def test_routed_matvec(tokens, experts, top_k, inner, outer, group, absent, gather, dtype):
    kind, unit, tiny = HALF[dtype]
    host, r = make_routing(tokens, experts, top_k, 15, absent)
    g = torch.Generator().manual_seed(inner + outer)
    x = torch.randn(tokens if gather else tokens * top_k, inner, generator=g).to(kind).cuda()
    if absent and not gather:
        x[host[4][-1]:] = math.nan
    codes = torch.randint(0, 256, (experts, outer, inner // 2), generator=g, dtype=torch.uint8)
    scales = (torch.rand(experts, outer, inner // group, generator=g) / math.sqrt(inner)).to(kind)
    got = routed.routed_matvec(x, routed.Int4Weights(codes.cuda(), scales.cuda(), group), r, gather=gather)
    q = np.stack([codes.numpy() & 15, codes.numpy() >> 4], 3).reshape(experts, outer, inner).astype(np.float64) - 8
    w = q * np.repeat(wide(scales), group, axis=2)
    y, size = plain_product(host, wide(x), w.transpose(0, 2, 1), gather, top_k)
    near(got, y, 1.01 * unit * np.abs(y) + tiny + inner * 2.0 ** -23 * size, "rows")


@gpu
def test_pack_int4_halves_the_step():
    w = torch.randn(3, 128, 20, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    w[1, :64, 3] = 0.0
    packed = routed.pack_int4(w, 64)
    _, r = make_routing(128, 3, 3, 16)
    x = torch.eye(128).bfloat16().cuda()
    y = wide(routed.routed_matvec(x, packed, r, gather=True))
    rows, offsets = r.rows.cpu().numpy(), r.offsets.cpu().numpy()
    scales = wide(packed.scales)
    for e in range(3):
        for p in range(offsets[e], offsets[e + 1]):
            k = rows[p] // 3
            step = scales[e, :, k // 64]
            # Half a step, and 7 steps may end just below the largest weight: bf16 rounds the scale by 2^-9.
            assert np.max(np.abs(y[p] - wide(w)[e, k]) - step * (0.5 + 7 * 2.0 ** -8)) <= 1e-6
    assert (packed.scales[1, 3, 0] == 0) and (packed.codes[1, 3, :32] == 0x88).all()


# ----------------------------------------------------------------------------------------------------------------
# Refusals


def test_host_storage_is_refused():
    x = torch.randn(4, 8)
    with pytest.raises(ValueError, match="CUDA tensor"):
        routed.route(x, 2)
    with pytest.raises(ValueError, match="CUDA tensor"):
        routed.gated_save(x.half())


def call(name, *arguments):
    """(status, message) of a C entry point; the arguments are refused before anything is launched."""
    build.build()
    err = _native.error_buffer()
    status = getattr(_native.lib(), name)(*arguments, None, err, len(err))
    return status, err.value.decode()


A, B, C, D, E, F, G, H = (0x10000000 * (i + 1) for i in range(8))   # addresses that no check reads


@pytest.mark.parametrize("change, message", [
    ({"dtype": 12}, "F32, F16 or BF16"), ({"tokens": -1}, "nonnegative"), ({"experts": 0}, "1 to 512"),
    ({"experts": 513}, "1 to 512"), ({"top_k": 0}, "top_k"), ({"top_k": 9}, "top_k"), ({"tokens": 1 << 30}, "2^31"),
    ({"groups": 3}, "divide"), ({"top_groups": 3}, "top_groups"), ({"best": 3}, "group_best"),
    ({"score": 2}, "score"), ({"renormalize": 2}, "renormalize"), ({"scale": math.nan}, "finite"),
    ({"logits": None}, "null"), ({"logits": A + 2}, "aligned"), ({"stride": 7}, "stride"),
    ({"weights": B}, "overlap"), ({"rows": A}, "overlap"), ({"workspace": 0}, "too small"),
])
def test_route_refusals(change, message):
    a = {"dtype": 11, "tokens": 1000, "experts": 8, "top_k": 2, "groups": 2, "top_groups": 1, "best": 1, "score": 0,
         "renormalize": 1, "scale": 1.0, "logits": A, "stride": 8, "weights": C, "rows": D, "workspace": 1 << 20}
    a.update(change)
    status, text = call("t0b_route", a["dtype"], a["tokens"], a["experts"], a["top_k"], a["groups"], a["top_groups"],
                        a["best"], a["score"], a["renormalize"], a["scale"], a["logits"], a["stride"], None, None, B,
                        a["weights"], a["rows"], E, F, G, a["workspace"])
    assert status == 1 and message in text, text


@pytest.mark.parametrize("change, message", [
    ({"dtype": 11}, "F16 or BF16"), ({"transposed": 2}, "transposed"), ({"entries": 7}, "multiple of top_k"),
    ({"entries": 1 << 31}, "2^31"), ({"inner": 0}, "widths"), ({"gather": 2}, "gather"), ({"x_rows": 8}, "per token"),
    ({"x": None}, "null"), ({"x": A + 1}, "aligned"), ({"x_stride": 15}, "stride"), ({"w": None}, "null"),
    ({"output": A}, "overlap"), ({"output": D}, "overlap"),
])
def test_product_refusals(change, message):
    a = {"dtype": 10, "transposed": 0, "entries": 8, "experts": 2, "inner": 16, "outer": 32, "gather": 1, "x": A,
         "x_rows": 4, "x_stride": 16, "w": B, "rows": D, "output": C}
    a.update(change)
    status, text = call("t0b_routed_product", a["dtype"], a["transposed"], a["entries"], a["experts"], 2, a["inner"],
                        a["outer"], a["gather"], a["x"], a["x_rows"], a["x_stride"], a["w"], a["rows"], E, a["output"])
    assert status == 1 and message in text, text


@pytest.mark.parametrize("name, arguments, message", [
    ("t0b_route_backward", (11, 4, 8, 2, 0, 1, 1.0, A, 8, B, C, A), "overlap"),
    ("t0b_route_backward", (11, 4, 8, 2, 0, 1, math.inf, A, 8, B, C, D), "finite"),
    ("t0b_routed_weight_grad", (10, 8, 2, 2, 16, 32, 0, A, 4, 16, 0, B, 8, 32, D, E, C), "per entry"),
    ("t0b_routed_weight_grad", (10, 8, 2, 2, 16, 32, 1, A, 4, 16, 0, B, 8, 31, D, E, C), "stride"),
    ("t0b_routed_weight_grad", (10, 8, 2, 2, 16, 32, 1, A, 4, 16, 0, B, 8, 32, D, E, B), "overlap"),
    ("t0b_routed_sum", (11, 4, 2, 8, A, 8, B, C), "F16 or BF16"),
    ("t0b_routed_sum", (10, 4, 33, 8, A, 8, B, C), "top_k"),
    ("t0b_routed_sum", (10, 4, 2, 8, A, 8, B, A), "overlap"),
    ("t0b_gated_save", (10, 4, 0, 32, A, 16, None, None, None, 0, B, C, D), "width"),
    ("t0b_gated_save", (10, 4, 8, 48, A, 16, None, None, None, 0, B, C, D), "group"),
    ("t0b_gated_save", (10, 4, 8, 32, A, 15, None, None, None, 0, B, C, D), "stride"),
    ("t0b_gated_save", (10, 4, 8, 32, A, 16, E, None, None, 2, B, C, D), "routing"),
    ("t0b_gated_save", (10, 4, 8, 32, A, 16, None, None, None, 0, A, C, D), "overlap"),
    ("t0b_gated_save", (10, 4, 8, 32, A, 16, None, None, None, 0, B, C, None), "codes and its scales"),
    ("t0b_gated_backward", (10, 4, 8, 32, A, B, C, 8, None, None, None, 0, D, D, E), "overlap"),
    ("t0b_checkpoint_load", (12, 4, 8, 32, A, B, C), "F32, F16 or BF16"),
    ("t0b_routed_matvec4", (10, 8, 2, 2, 48, 32, 32, 1, A, 4, 48, B, C, D, E, F), "divide"),
    ("t0b_routed_matvec4", (10, 8, 2, 2, 64, 32, 32, 1, A, 4, 64, B + 8, C, D, E, F), "16-byte"),
    ("t0b_routed_matvec4", (11, 8, 2, 2, 64, 32, 32, 1, A, 4, 64, B, C, D, E, F), "F16 or BF16"),
    ("t0b_routed_matvec4", (10, 8, 2, 2, 64, 32, 32, 0, A, 4, 64, B, C, D, E, F), "one row"),
])
def test_other_refusals(name, arguments, message):
    status, text = call(name, *arguments)
    assert status == 1 and message in text, text


@gpu
def test_python_refusals():
    _, r = make_routing(6, 4, 2, 1)
    x = torch.randn(6, 32).half().cuda()
    w = torch.randn(4, 32, 16).half().cuda()
    with pytest.raises(ValueError, match="share|bfloat16"):
        routed.routed_matmul(x, w.bfloat16(), r, gather=True)
    with pytest.raises(ValueError, match="expert-ordered"):
        routed.routed_matmul(x, w, r)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        routed.routed_matmul(x.float(), w.float(), r, gather=True)
    with pytest.raises(ValueError, match="contiguous"):
        routed.routed_matmul(x, w.transpose(1, 2), r._replace(offsets=r.offsets), gather=True)
    with pytest.raises(ValueError, match="contiguous rows"):
        routed.routed_matmul(x.t().contiguous().t(), w, r, gather=True)
    shared = torch.zeros(12, 16).half().cuda()
    with pytest.raises(ValueError, match="overlap"):
        routed.routed_matmul(shared.view(6, 32), w, r, gather=True, out=shared)
    with pytest.raises(ValueError, match="score"):
        routed.route(torch.randn(4, 8).cuda(), 2, score="entropy")
    with pytest.raises(ValueError, match="top_k"):
        routed.route(torch.randn(4, 8).cuda(), 9)
    with pytest.raises(ValueError, match="mask"):
        routed.route(torch.randn(4, 8).cuda(), 2, mask=torch.ones(5, dtype=torch.bool).cuda())
    with pytest.raises(ValueError, match="entries"):
        routed.gated_save(torch.randn(5, 32).half().cuda(), routing=r)
    with pytest.raises(ValueError, match="group"):
        routed.gated_save(x, group=16)


@gpu
def test_launch_counts_show_the_kernels():
    before = _native.lib().t0b_kernel_launches()
    routed.route(torch.randn(4, 8).cuda(), 2)
    assert _native.lib().t0b_kernel_launches() == before + 1
