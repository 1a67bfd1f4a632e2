"""Cases of the routed (mixture-of-experts) operators: what each computes in plain torch, and the calls that a
user makes of ``tensor0_b200.routed``.

Four operators belong together.  ``route`` grades every token into sectors (experts) chosen at run time and orders
the rows by sector; the products are the block-sparse contraction over those sectors, forward and backward; the
gated activation between two products keeps its input for the backward pass in 8 bits; the 4-bit matrix-vector
products are the single-token form of the same layer.
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY = 2.0 ** -100   # a checkpoint group whose largest magnitude is below this is stored as zeros


def listed():
    return [
        # One decode step of a serving loop with eight sequences: latency is all there is.
        {"name": "route decode", "op": "route", "tokens": 8, "experts": 64, "top_k": 4, "groups": 1, "top_groups": 1,
         "best": 1, "score": "softmax", "bias": False, "renormalize": True, "dtype": "f32", "padded": False,
         "train": False},
        # A prompt, sigmoid scores with a bias for balance, experts in device groups scored by their two best.
        {"name": "route prompt", "op": "route", "tokens": 8191, "experts": 256, "top_k": 8, "groups": 8,
         "top_groups": 4, "best": 2, "score": "sigmoid", "bias": True, "renormalize": True, "dtype": "bf16",
         "padded": False, "train": False},
        # A training batch of padded sequences: choice, weights, row order and the logits' gradient.
        {"name": "route train", "op": "route", "tokens": 32768, "experts": 128, "top_k": 8, "groups": 1,
         "top_groups": 1, "best": 1, "score": "softmax", "bias": False, "renormalize": True, "dtype": "f32",
         "padded": True, "train": True},
        # A small batch's first product: few rows for each expert, so the weights are what is read.
        {"name": "product small", "op": "product", "kind": "up", "tokens": 64, "experts": 16, "top_k": 2,
         "inner": 512, "outer": 1024, "dtype": "bf16", "padded": False},
        # A prompt of odd length and widths that no tile divides, with padding.
        {"name": "product ragged", "op": "product", "kind": "up", "tokens": 1537, "experts": 40, "top_k": 6,
         "inner": 1000, "outer": 1416, "dtype": "f16", "padded": True},
        # A training batch's second product and the sum over each token's experts.
        {"name": "product down", "op": "product", "kind": "down", "tokens": 8192, "experts": 64, "top_k": 4,
         "inner": 1024, "outer": 2048, "dtype": "bf16", "padded": False},
        # The backward pass of a first product: the tokens' gradient and every expert's weight gradient.
        {"name": "product gradient", "op": "product", "kind": "grad", "tokens": 8192, "experts": 32, "top_k": 4,
         "inner": 2048, "outer": 2048, "dtype": "bf16", "padded": True},
        # The activation of a prompt's rows with its 8-bit checkpoint, of a width that the groups do not divide.
        {"name": "gated save", "op": "gated", "kind": "save", "tokens": 2049, "top_k": 6, "width": 1416,
         "group": 64, "dtype": "f16"},
        # A training batch's activation gradient from the checkpoint.
        {"name": "gated gradient", "op": "gated", "kind": "grad", "tokens": 16384, "top_k": 4, "width": 2048,
         "group": 128, "dtype": "bf16"},
        # One token through 4-bit experts.
        {"name": "matvec token", "op": "matvec", "tokens": 1, "experts": 64, "top_k": 8, "inner": 2048,
         "outer": 1024, "group": 128, "dtype": "bf16"},
        # A serving batch: several tokens share an expert, most experts are read.
        {"name": "matvec batch", "op": "matvec", "tokens": 16, "experts": 64, "top_k": 4, "inner": 4096,
         "outer": 2048, "group": 64, "dtype": "f16"},
    ]


def _spread(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["route", "product", "product", "gated", "matvec"])
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * _spread(rng, 16 // groups, 256 // groups)
        train = rng.random() < 0.5
        return {"op": op, "tokens": _spread(rng, 1, 32768 * 128 // max(experts, 128)), "experts": experts,
                "top_k": rng.randint(1, 8), "groups": groups, "top_groups": max(1, groups // 2),
                "best": rng.choice([1, 2]) if groups > 1 else 1, "score": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.5, "renormalize": rng.random() < 0.7,
                "dtype": rng.choice(["f32", "bf16", "f16"]), "padded": rng.random() < 0.5, "train": train}
    if op == "product":
        inner, outer = 8 * _spread(rng, 16, 256), 8 * _spread(rng, 16, 256)
        top_k = rng.randint(1, 8)
        tokens = _spread(rng, 1, 32768 // top_k)
        return {"op": op, "kind": rng.choice(["up", "down", "grad"]), "tokens": tokens,
                "experts": _spread(rng, 8, 64), "top_k": top_k, "inner": inner, "outer": outer,
                "dtype": rng.choice(["bf16", "f16"]), "padded": rng.random() < 0.5}
    if op == "gated":
        top_k = rng.randint(1, 8)
        return {"op": op, "kind": rng.choice(["save", "grad"]), "tokens": _spread(rng, 1, 65536 // top_k),
                "top_k": top_k, "width": _spread(rng, 64, 2048), "group": rng.choice([32, 64, 128]),
                "dtype": rng.choice(["bf16", "f16"])}
    group = rng.choice([32, 64, 128])
    top_k = rng.randint(1, 8)
    return {"op": op, "tokens": _spread(rng, 1, 64 // top_k), "experts": _spread(rng, 8, 64), "top_k": top_k,
            "inner": group * _spread(rng, 512 // group, 4096 // group), "outer": _spread(rng, 256, 2048),
            "group": group, "dtype": rng.choice(["bf16", "f16"])}


def work(case):
    op = case["op"]
    if op == "route":
        size = 4 if case["dtype"] == "f32" else 2
        tokens, experts, entries = case["tokens"], case["experts"], case["tokens"] * case["top_k"]
        count = tokens * experts * size + 16 * entries + 4 * (experts + 1)
        if case["train"]:
            count += tokens * experts * size + 4 * entries
        return {"bytes": count, "flops": 8 * tokens * experts}
    if op == "product":
        tokens, rows, inner, outer = case["tokens"], _live(case) * case["top_k"], case["inner"], case["outer"]
        weights = min(case["experts"], rows) * inner * outer
        if case["kind"] == "up":
            return {"bytes": 2 * (tokens * inner + weights + rows * outer), "flops": 2 * rows * inner * outer}
        if case["kind"] == "down":
            return {"bytes": 2 * (rows * inner + weights + tokens * outer), "flops": 2 * rows * inner * outer}
        return {"bytes": 2 * (2 * tokens * inner + rows * outer + weights + case["experts"] * inner * outer),
                "flops": 4 * rows * inner * outer}
    if op == "gated":
        rows, width = case["tokens"] * case["top_k"], case["width"]
        kept = 2 * width + 8 * -(-width // case["group"])
        if case["kind"] == "save":   # the input and the activation; the checkpoint; the values it stands for
            return {"bytes": rows * (4 * width + 2 * width + kept + 4 * width + 8), "flops": 20 * rows * width}
        return {"bytes": rows * (kept + 2 * width + 4 * width + 2 * width + 12), "flops": 30 * rows * width}
    rows = case["tokens"] * case["top_k"]
    read = case["experts"] * (1 - (1 - min(1, case["top_k"] / case["experts"])) ** case["tokens"])
    matrix = case["inner"] * case["outer"]
    return {"bytes": int(read * (matrix / 2 + 2 * matrix / case["group"]))
            + 2 * (case["tokens"] * case["inner"] + rows * case["outer"]), "flops": 2 * rows * matrix}


# ---------------------------------------------------------------------------------------------------------------
# Inputs


def _live(case):
    """Tokens that are no padding: the last sixteenth of a padded batch is."""
    return case["tokens"] - case["tokens"] // 16 if case.get("padded") else case["tokens"]


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _a_routing(g, tokens, live, experts, top_k):
    """A routing with uneven experts: (experts, weights, rows, positions, offsets), as ``route`` lays it out."""
    logits = _normal(g, tokens, experts) + 0.25 * _normal(g, experts)
    value, chosen = logits.topk(top_k, dim=1)
    weights = torch.softmax(value, 1)
    alive = (torch.arange(tokens, device="cuda") < live)[:, None]
    chosen = torch.where(alive, chosen, -1).to(torch.int32)
    weights = torch.where(alive, weights, 0.0)
    return (chosen, weights, *_row_order(chosen, experts))


def _row_order(chosen, experts):
    """Entries ordered by expert, absent ones last: their numbers, each entry's place, each expert's first row."""
    key = torch.where(chosen < 0, experts, chosen).reshape(-1)
    rows = torch.sort(key, stable=True).indices
    place = torch.empty_like(rows)
    place[rows] = torch.arange(rows.numel(), device=rows.device)
    positions = torch.where(chosen < 0, -1, place.view_as(chosen))
    count = (key[:, None] == torch.arange(experts, device=key.device)).sum(0)
    offsets = torch.cat([torch.zeros_like(count[:1]), count.cumsum(0)])
    return rows.to(torch.int32), positions.to(torch.int32), offsets.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op, tokens, top_k = case["op"], case["tokens"], case["top_k"]
    state = {"case": dict(case)}
    entries = tokens * top_k
    if op == "route":
        experts = case["experts"]
        live = _live(case)
        logits = 1.5 * _normal(g, tokens, experts) + 0.5 * _normal(g, experts)
        if case["padded"]:   # what a padded token's logits hold is nobody's business
            logits[live:] = float("nan")
            state["mask"] = torch.arange(tokens, device="cuda") < live
        state["logits"] = logits.to(TYPES[case["dtype"]])
        if case["bias"]:
            state["bias"] = 0.1 * _normal(g, experts)
        if case["train"]:
            state["weights_grad"] = _normal(g, tokens, top_k)
        # The buffers that a serving loop keeps from step to step.
        state["out"] = (torch.empty(tokens, top_k, dtype=torch.int32, device="cuda"),
                        torch.empty(tokens, top_k, dtype=torch.float32, device="cuda"),
                        torch.empty(entries, dtype=torch.int32, device="cuda"),
                        torch.empty(tokens, top_k, dtype=torch.int32, device="cuda"),
                        torch.empty(experts + 1, dtype=torch.int32, device="cuda"))
        return state
    if op == "gated":
        width, dtype = case["width"], TYPES[case["dtype"]]
        state["routing"] = _a_routing(g, tokens, tokens, max(16, top_k), top_k)
        h = _normal(g, entries, 2 * width) * (1 + 4 * (torch.rand(2 * width, generator=g, device="cuda") < 0.01))
        h = h.to(dtype)
        if case["kind"] == "save":
            state["h"] = h
        else:
            codes, scales = _to_8_bits(h.float(), case["group"])
            state["codes"], state["scales"] = codes.to(torch.int8), scales
            state["a_grad"] = _normal(g, entries, width).to(dtype)
        return state
    experts, inner, outer, dtype = case["experts"], case["inner"], case["outer"], TYPES[case["dtype"]]
    routing = _a_routing(g, tokens, _live(case), experts, min(top_k, experts))
    state["routing"] = routing
    if op == "matvec":
        state["x"] = _normal(g, tokens, inner).to(dtype)
        state["codes"] = torch.randint(0, 256, (experts, outer, inner // 2), generator=g, device="cuda",
                                       dtype=torch.uint8)
        state["scales"] = ((0.5 + torch.rand(experts, outer, inner // case["group"], generator=g, device="cuda"))
                           * (0.2 / math.sqrt(inner))).to(dtype)
        return state
    state["most"] = max(1, int((routing[4][1:] - routing[4][:-1]).max()))   # rows of the fullest expert
    state["w"] = (_normal(g, experts, inner, outer) / math.sqrt(inner)).to(dtype)
    if case["kind"] == "down":
        state["x"] = _normal(g, entries, inner).to(dtype)
    else:
        state["x"] = _normal(g, tokens, inner).to(dtype)
    if case["kind"] == "grad":
        state["y_grad"] = _normal(g, entries, outer).to(dtype)
    return state


# ---------------------------------------------------------------------------------------------------------------
# One pass


def run(state):
    return _own_run(state) if own else _plain_run(state)


def _own_run(state):
    from tensor0_b200 import routed
    case = state["case"]
    op = case["op"]
    if op == "route":
        r = routed.route(state["logits"], case["top_k"], groups=case["groups"], top_groups=case["top_groups"],
                         group_best=case["best"], score=case["score"], renormalize=case["renormalize"],
                         bias=state.get("bias"), mask=state.get("mask"), out=routed.Routing(*state["out"]))
        if not case["train"]:
            return tuple(r)
        return (*r, routed.route_backward(state["logits"], r, state["weights_grad"], score=case["score"],
                                          renormalize=case["renormalize"]))
    r = routed.Routing(*state["routing"])
    if op == "gated":
        if case["kind"] == "save":
            a, checkpoint = routed.gated_save(state["h"], routing=r, group=case["group"])
            return a, routed.checkpoint_load(checkpoint, state["h"].dtype)
        checkpoint = routed.Checkpoint(state["codes"], state["scales"], case["group"])
        return routed.gated_backward(checkpoint, state["a_grad"], routing=r)
    if op == "matvec":
        weights = routed.Int4Weights(state["codes"], state["scales"], case["group"])
        return routed.routed_matvec(state["x"], weights, r, gather=True)
    if case["kind"] == "up":
        return routed.routed_matmul(state["x"], state["w"], r, gather=True)
    if case["kind"] == "down":
        return routed.routed_sum(routed.routed_matmul(state["x"], state["w"], r), r)
    x_grad = routed.routed_sum(routed.routed_matmul(state["y_grad"], state["w"], r, transpose=True), r)
    return x_grad, routed.routed_weight_grad(state["x"], state["y_grad"], r, gather_x=True)


def _plain_run(state):
    case = state["case"]
    return {"route": _plain_route, "product": _plain_product, "gated": _plain_gated,
            "matvec": _plain_matvec}[case["op"]](case, state)


def _plain_route(case, state):
    x = state["logits"].float()
    tokens, experts = x.shape
    top_k, groups = case["top_k"], case["groups"]
    live = x > -math.inf
    if "mask" in state:
        live = live & state["mask"][:, None]
    if case["score"] == "softmax":
        e = torch.exp(x - x.amax(1, keepdim=True))
        # The normaliser is rounded from a 64-bit sum, so that it does not depend on the order of the terms.
        scores = e / e.double().sum(1, keepdim=True).float()
    else:
        scores = torch.reciprocal(1 + torch.exp(-x))
    if case["bias"]:
        choice = scores + state["bias"]
    else:
        choice = scores if case["best"] == 2 else x
    choice = torch.where(live, choice, -math.inf)
    if groups > 1:
        best = torch.sort(choice.view(tokens, groups, -1), dim=2, descending=True).values
        by_group = best[..., 0]
        if case["best"] == 2 and best.shape[2] > 1:
            by_group = by_group + torch.where(best[..., 1] > -math.inf, best[..., 1], 0.0)
        order = torch.sort(by_group, dim=1, descending=True, stable=True).indices
        rank = torch.argsort(order, dim=1)
        kept = (rank < case["top_groups"]).repeat_interleave(experts // groups, dim=1)
        choice = torch.where(kept, choice, -math.inf)
    ordered = torch.sort(choice, dim=1, descending=True, stable=True)
    found = ordered.values[:, :top_k] > -math.inf
    at = ordered.indices[:, :top_k]
    chosen = torch.where(found, at, -1).to(torch.int32)
    picked = torch.where(found, scores.gather(1, at), 0.0)
    total = picked.sum(1, keepdim=True) + 1e-20
    weights = picked / total if case["renormalize"] else picked
    out = (chosen, weights, *_row_order(chosen, experts))
    if not case["train"]:
        return out
    grad = torch.where(found, state["weights_grad"], 0.0)
    if case["renormalize"]:
        grad = torch.where(found, (grad - (grad * weights).sum(1, keepdim=True)) / total, 0.0)
    scores_grad = torch.zeros_like(scores).scatter_add_(1, at, grad)
    if case["score"] == "softmax":
        inner = (grad * picked).sum(1, keepdim=True)
        logits_grad = scores * (scores_grad - inner)
    else:
        logits_grad = scores_grad * scores * (1 - scores)
    if "mask" in state:
        logits_grad = torch.where(state["mask"][:, None], logits_grad, 0.0)
    return (*out, logits_grad.to(state["logits"].dtype))


def _padded(rows, routing, most):
    """[experts, most, width] of sorted rows: each expert's, with zeros after its last."""
    offsets = routing[4].long()
    place = offsets[:-1, None] + torch.arange(most, device=rows.device)
    inside = place < offsets[1:, None]
    return torch.where(inside[..., None], rows[place.clamp(max=rows.shape[0] - 1)].float(), 0.0)


def _unpadded(blocks, routing, most):
    """The sorted rows of ``_padded``'s layout; absent entries' rows are zero."""
    chosen, _, rows, _, offsets = routing
    expert = chosen.reshape(-1)[rows.long()].long()
    at = torch.arange(rows.numel(), device=rows.device) - offsets.long()[expert.clamp(min=0)]
    flat = blocks.reshape(-1, blocks.shape[2])[(expert.clamp(min=0) * most + at).clamp(0, blocks.shape[0] * most - 1)]
    return torch.where(expert[:, None] < 0, 0.0, flat)


def _summed(rows, routing):
    """Each token's sum over its experts' rows."""
    positions = routing[3].long()
    return torch.where(positions[..., None] < 0, 0.0, rows[positions.clamp(min=0)]).sum(1)


def _plain_product(case, state):
    routing, most, dtype = state["routing"], state["most"], state["x"].dtype
    w = state["w"].float()
    token = routing[2].long() // routing[0].shape[1]
    if case["kind"] == "up":
        blocks = torch.bmm(_padded(state["x"][token], routing, most), w)
        return _unpadded(blocks, routing, most).to(dtype)
    if case["kind"] == "down":
        blocks = torch.bmm(_padded(state["x"], routing, most), w)
        return _summed(_unpadded(blocks, routing, most), routing).to(dtype)
    y_grad = _padded(state["y_grad"], routing, most)
    x_rows = _unpadded(torch.bmm(y_grad, w.transpose(1, 2)), routing, most)
    x = _padded(state["x"][token], routing, most)
    return _summed(x_rows, routing).to(dtype), torch.bmm(x.transpose(1, 2), y_grad).to(dtype)


def _to_8_bits(h, group):
    """Whole numbers from -127 to 127 and each group's scale; a group is ``group`` neighbours of one half of a row."""
    rows, width = h.shape[0], h.shape[1] // 2
    most = -(-width // group)
    x = torch.nn.functional.pad(h.view(rows, 2, width), (0, most * group - width)).view(rows, 2, most, group)
    largest = x.abs().amax(3)
    some = largest >= TINY
    per_unit = torch.where(some, torch.reciprocal(largest) * 127.0, 0.0)
    scales = torch.where(some, largest * (1.0 / 127.0), 0.0)
    codes = torch.round(x * per_unit[..., None]).clamp(-127, 127)
    return codes.view(rows, 2, -1)[..., :width].reshape(rows, 2 * width), scales.view(rows, 2 * most)


def _from_8_bits(codes, scales, group):
    rows, width = codes.shape[0], codes.shape[1] // 2
    spread = scales.view(rows, 2, -1).repeat_interleave(group, dim=2)[..., :width].reshape(rows, 2 * width)
    return codes.float() * spread


def _plain_gated(case, state):
    _, weights, rows, _, _ = state["routing"]
    width, entry = case["width"], rows.long()
    weight = weights.reshape(-1)[entry][:, None]
    if case["kind"] == "save":
        h = state["h"].float()
        gate, up = h[:, :width], h[:, width:]
        a = weight * (gate / (1 + torch.exp(-gate))) * up
        values = _from_8_bits(*_to_8_bits(h, case["group"]), case["group"])
        return a.to(state["h"].dtype), values.to(state["h"].dtype)
    h = _from_8_bits(state["codes"], state["scales"], case["group"])
    gate, up = h[:, :width], h[:, width:]
    sigmoid = 1 / (1 + torch.exp(-gate))
    silu = gate * sigmoid
    a_grad = state["a_grad"].float()
    gate_grad = weight * a_grad * up * (sigmoid + silu * (1 - sigmoid))
    up_grad = weight * a_grad * silu
    weights_grad = torch.zeros_like(weights).view(-1).scatter(0, entry, (a_grad * silu * up).sum(1))
    dtype = state["a_grad"].dtype
    return (torch.cat([gate_grad, up_grad], 1).to(dtype), (weight * silu * up).to(dtype),
            weights_grad.view_as(weights))


def _plain_matvec(case, state):
    chosen, _, rows, _, _ = state["routing"]
    expert = chosen.reshape(-1)[rows.long()].long()
    codes = state["codes"][expert]
    values = torch.stack([codes & 15, codes >> 4], 3).flatten(2).float() - 8
    w = values * state["scales"][expert].float().repeat_interleave(case["group"], dim=2)
    x = state["x"].float()[rows.long() // chosen.shape[1]]
    return torch.bmm(w, x[..., None])[..., 0].to(state["x"].dtype)


# ---------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    return {"route": _exact_route, "product": _exact_product, "gated": _exact_gated,
            "matvec": _exact_matvec}[case["op"]](case, state)


def _exact_route(case, state):
    """Which experts are chosen is compared as whole numbers; the weights and gradients are taken for that choice."""
    chosen, _, _, _, _ = _plain_route({**case, "train": False}, state)
    x = state["logits"].double()
    if case["score"] == "softmax":
        log_scores = x - torch.logsumexp(x, 1, keepdim=True)
        scores = torch.exp(log_scores)
    else:
        scores = torch.sigmoid(x)
    at = chosen.long().clamp(min=0)
    found = chosen >= 0
    weights = torch.where(found, scores.gather(1, at), 0.0)
    if case["renormalize"]:
        weights = weights / (weights.sum(1, keepdim=True) + 1e-20)
    out = (None, weights, None, None, None)
    if not case["train"]:
        return out
    # The gradient as the sum over slots of d weight[slot] / d logit[j], slot by slot.
    dead = ~state["mask"] if "mask" in state else torch.zeros_like(found[:, 0])
    grad = torch.zeros_like(x)
    upstream = torch.where(found, state["weights_grad"].double(), 0.0)
    for i in range(at.shape[1]):
        own_slot = torch.nn.functional.one_hot(at[:, i], x.shape[1]).double() * found[:, i:i + 1]
        if case["score"] == "softmax":
            log_slope = own_slot - scores * found[:, i:i + 1]                        # d log s_i / d x_j
        else:
            log_slope = own_slot * (1 - scores)
        if case["renormalize"]:
            for j in range(at.shape[1]):
                other = torch.nn.functional.one_hot(at[:, j], x.shape[1]).double() * found[:, j:j + 1]
                slope = other - scores * found[:, j:j + 1] if case["score"] == "softmax" else other * (1 - scores)
                log_slope = log_slope - weights[:, j:j + 1] * slope * found[:, i:i + 1]
        grad += (upstream[:, i] * weights[:, i])[:, None] * log_slope
    grad[dead] = 0.0
    return (*out, grad)


def _exact_product(case, state):
    chosen, _, rows, positions, offsets = state["routing"]
    bounds = offsets.tolist()
    x, w = state["x"], state["w"]
    top_k = chosen.shape[1]
    token = rows.long() // top_k
    entries = rows.numel()
    if case["kind"] == "grad":
        rows_out = torch.zeros(entries, case["inner"], dtype=torch.float64, device="cuda")
        w_grad = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            part = slice(bounds[e], bounds[e + 1])
            dy = state["y_grad"][part].double()
            rows_out[part] = dy @ w[e].double().T
            w_grad[e] = x[token[part]].double().T @ dy
        x_grad = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
        x_grad.index_add_(0, token[:bounds[-1]], rows_out[:bounds[-1]])
        return x_grad, w_grad
    y = torch.zeros(entries, case["outer"], dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        part = slice(bounds[e], bounds[e + 1])
        y[part] = (x[token[part]] if case["kind"] == "up" else x[part]).double() @ w[e].double()
    if case["kind"] == "up":
        return y
    out = torch.zeros(case["tokens"], case["outer"], dtype=torch.float64, device="cuda")
    out.index_add_(0, token[:bounds[-1]], y[:bounds[-1]])
    return out


def _exact_gated(case, state):
    _, weights, rows, _, _ = state["routing"]
    width, group = case["width"], case["group"]
    entry = rows.long()
    weight = weights.reshape(-1)[entry].double()[:, None]
    if case["kind"] == "save":
        h = state["h"].double()
        gate, up = h[:, :width], h[:, width:]
        return weight * gate * torch.sigmoid(gate) * up, None
    most = -(-width // group)
    column = torch.arange(2 * width, device="cuda")
    of = torch.where(column < width, column // group, most + (column - width) // group)
    h = state["codes"].double() * state["scales"].double()[:, of]
    gate, up = h[:, :width], h[:, width:]
    s, da = torch.sigmoid(gate), state["a_grad"].double()
    h_grad = torch.cat([weight * da * up * s * (1 + gate * (1 - s)), weight * da * gate * s], 1)
    weights_grad = torch.empty(weights.numel(), dtype=torch.float64, device="cuda")
    weights_grad[entry] = (da * gate * s * up).sum(1)
    return h_grad, weight * gate * s * up, weights_grad.view(weights.shape)


def _exact_matvec(case, state):
    chosen, _, rows, _, _ = state["routing"]
    entry = rows.tolist()
    expert = chosen.reshape(-1).tolist()
    top_k, group = chosen.shape[1], case["group"]
    out = torch.empty(len(entry), case["outer"], dtype=torch.float64, device="cuda")
    for p, i in enumerate(entry):
        codes = state["codes"][expert[i]].to(torch.int64)
        w = torch.empty(case["outer"], case["inner"], dtype=torch.float64, device="cuda")
        w[:, 0::2] = (codes % 16 - 8).double()
        w[:, 1::2] = (codes // 16 - 8).double()
        w = w.view(case["outer"], -1, group) * state["scales"][expert[i]].double()[..., None]
        out[p] = w.view(case["outer"], -1) @ state["x"][i // top_k].double()
    return out
