"""Routed operators: block-sparse products whose sectors are chosen at run time.

``stride.sector_gemm`` multiplies sectors whose sizes the host knows.  Here a
router picks each token's sectors ("experts") on the device, the products run
over whatever rows each expert got, and every step has its gradient:

    r = route(logits, top_k)                              # experts, weights, row order
    h = routed_matmul(x, w_in, r, gather=True)            # [entries, 2 * width]
    a, kept = gated_save(h, routing=r)                    # weight * silu(gate) * up; h kept in 8 bits
    y = routed_sum(routed_matmul(a, w_out, r), r)         # [tokens, outer]

An entry is one (token, slot) pair, number ``token * top_k + slot``.  Rows of
the products are ordered by expert: row p holds entry ``rows[p]`` and expert
e's rows are ``offsets[e]:offsets[e + 1]``.  Entries without an expert (masked
tokens, excluded experts) come last; their rows are zeros.

As for the stride engine, storage is CUDA tensors, calls are ordered on the
current stream of the storage's device, nothing synchronizes, and there is no
CPU fallback.  ``out`` takes preallocated results; what is not given comes
from torch's allocator, as the workspace of a route of more than 64 tokens does.

The operators record nothing for autograd: an operand that requires a gradient
is refused while gradients are recorded.  A ``torch.autograd.Function`` around
them calls the backward operators in its own backward pass.
"""

from __future__ import annotations

import importlib.machinery
import importlib.util
from typing import NamedTuple

import torch

from . import _native
from . import build as _build

_HALF = {torch.float16: _native.F16, torch.bfloat16: _native.BF16}
_FLOAT = {torch.float32: _native.F32, **_HALF}


class _Binding:
    """The compiled binding (``binding/routed.cpp``), loaded at its first use.

    It checks the tensors' types, shapes, strides and devices, allocates the results and calls the C entry points.
    """

    def __getattr__(self, name: str):
        if not _build.BINDING.exists():
            raise RuntimeError(f"tensor0_b200 binding not found at {_build.BINDING}; run "
                               "tensor0_b200.build.build_binding() (there is no CPU fallback for the routed operators)")
        _native.lib()
        loader = importlib.machinery.ExtensionFileLoader("_routed", str(_build.BINDING))
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_routed", loader))
        loader.exec_module(module)
        self.__dict__.update({key: value for key, value in vars(module).items() if not key.startswith("__")})
        return self.__dict__[name]


_routed = _Binding()


class Routing(NamedTuple):
    """A router's result on the device."""

    experts: torch.Tensor     # int32 [tokens, top_k], -1 where there is none
    weights: torch.Tensor     # float32 [tokens, top_k]
    rows: torch.Tensor        # int32 [tokens * top_k]: entry of each expert-ordered row
    positions: torch.Tensor   # int32 [tokens, top_k]: row of each entry, -1 where there is none
    offsets: torch.Tensor     # int32 [experts + 1]: first row of each expert


class Checkpoint(NamedTuple):
    """A gated activation's input in 8 bits (``gated_save``)."""

    codes: torch.Tensor    # int8 [rows, 2 * width]
    scales: torch.Tensor   # float32 [rows, 2 * ceil(width / group)]
    group: int


class Int4Weights(NamedTuple):
    """Weights in 4 bits: value ``(q - 8) * scale``, two to a byte, the even one in the low half."""

    codes: torch.Tensor    # uint8 [experts, outer, inner / 2]
    scales: torch.Tensor   # [experts, outer, inner / group], of the type of the rows they multiply
    group: int


def empty_routing(tokens: int, top_k: int, experts: int, device="cuda") -> Routing:
    """Uninitialised buffers for ``route(..., out=...)``."""
    def ints(*shape):
        return torch.empty(shape, dtype=torch.int32, device=device)
    return Routing(ints(tokens, top_k), torch.empty(tokens, top_k, dtype=torch.float32, device=device),
                   ints(tokens * top_k), ints(tokens, top_k), ints(experts + 1))


def route(logits: torch.Tensor, top_k: int, *, groups: int = 1, top_groups: int | None = None, group_best: int = 1,
          score: str = "softmax", renormalize: bool = True, scale: float = 1.0, bias: torch.Tensor | None = None,
          mask: torch.Tensor | None = None, out: Routing | None = None) -> Routing:
    """Each token's ``top_k`` experts, their weights, and the order of the rows by expert.

    ``logits`` [tokens, experts]: float32, float16 or bfloat16, rows contiguous.  Scores are the softmax or sigmoid
    of a token's logits.  The choice goes by score + ``bias`` (float32 [experts], a balance term that enters the
    choice only), or by the logits where there is no bias and ``group_best`` is 1; ties go to the lowest index.
    ``groups``: the experts lie in that many equal groups, of which the ``top_groups`` with the highest best value
    (``group_best`` 1) or sum of the two best (2) stay.  ``renormalize`` divides the chosen scores by their sum.
    ``mask`` (bool [tokens]): tokens that are False take no expert, whatever their logits hold.

    A logit of -inf or NaN takes no expert, and an expert whose bias is either is not chosen.  Under softmax a NaN or
    +inf logit makes its token's weights NaN; the choice then goes by the scores without the NaN logits, and by their
    limits at +inf.
    """
    if out is None:
        if logits.dim() != 2:
            raise ValueError("logits must be [tokens, experts]")
        out = empty_routing(logits.shape[0], max(top_k, 0), logits.shape[1], logits.device)
    return _routed.route(logits, top_k, groups, top_groups, group_best, score, renormalize, scale, bias, mask, out)


def route_backward(logits: torch.Tensor, routing: Routing, weights_grad: torch.Tensor, *, score: str = "softmax",
                   renormalize: bool = True, scale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of ``routing.weights`` with respect to the logits, for the same arguments as ``route``.

    The choice of experts is piecewise constant and the bias enters it only, so neither has a gradient.  Tokens
    without an expert get zeros, whatever their logits hold.
    """
    return _routed.route_backward(logits, routing, weights_grad, score, renormalize, scale, out)


def routed_matmul(x: torch.Tensor, w: torch.Tensor, routing: Routing, *, gather: bool = False,
                  transpose: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x[r] @ w[e]`` (or ``@ w[e].T``) for every row of every expert: [entries, outer or inner].

    ``w`` [experts, inner, outer], float16 or bfloat16 as ``x``.  ``x`` holds token rows with ``gather`` (row p reads
    its entry's token), else expert-ordered rows.  Summed in 32 bits, rounded once; rows without an expert are zero.

    Operands whose rows start on 16-byte boundaries (widths and strides that 8 divides) run on the tensor cores.
    Others take the general kernel, which is some 50 times slower: pad odd widths where that matters.
    """
    return _routed.routed_matmul(x, w, routing, gather, transpose, out)


def routed_weight_grad(x: torch.Tensor, y_grad: torch.Tensor, routing: Routing, *, gather_x: bool = False,
                       gather_y: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Every expert's weight gradient ``sum over its rows of x[r]^T y_grad[q]``: [experts, inner, outer].

    Either operand holds token rows (``gather_x``, ``gather_y``) or expert-ordered ones.  An expert without rows
    gets zeros.
    """
    return _routed.routed_weight_grad(x, y_grad, routing, gather_x, gather_y, out)


def routed_sum(y: torch.Tensor, routing: Routing, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """Each token's sum over its experts' rows: [tokens, width].  Also the gradient of gathering token rows.

    Summed in 32 bits and rounded once.  The rows come rounded to 16 bits by their product: together about 1.4 times
    the error of one rounding (1.5 at times in float16), and a float16 row beyond 65504 is infinite in the sum too.
    """
    return _routed.routed_sum(y, routing, out)


def gated_save(h: torch.Tensor, *, routing: Routing | None = None, group: int = 128,
               out: tuple[torch.Tensor, Checkpoint] | None = None) -> tuple[torch.Tensor, Checkpoint]:
    """``weight * silu(gate) * up`` of rows ``h = [gate | up]``, and ``h`` in 8 bits for ``gated_backward``.

    ``group`` (32, 64 or 128) neighbours of one half share a scale, their largest magnitude / 127.  A row's weight is
    its entry's in ``routing``, or 1 without one; with one, rows without an expert are not read and give zeros.
    """
    a, kept = (None, (None, None, group)) if out is None else out
    if kept[2] != group:
        raise ValueError("out's checkpoint has another group")
    a, codes, scales = _routed.gated_save(h, routing, group, a, kept[0], kept[1])
    return a, Checkpoint(codes, scales, group)


def gated(h: torch.Tensor, *, routing: Routing | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``gated_save``'s activation alone, for a pass that has no backward one."""
    return _routed.gated_save(h, routing, None, out, None, None)


def gated_backward(checkpoint: Checkpoint, a_grad: torch.Tensor, *, routing: Routing | None = None,
                   ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of ``gated_save`` from its checkpoint: ``(h_grad, a, weights_grad)``.

    ``a`` is the activation again, from the checkpoint (the next product's weight gradient needs it).
    ``weights_grad`` is the gradient of the routing's weights [tokens, top_k], or of a weight of 1 per row [rows]
    without a routing.
    """
    return _routed.gated_backward(checkpoint, a_grad, routing)


def checkpoint_load(checkpoint: Checkpoint, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values a checkpoint stands for, as float32, float16 or bfloat16."""
    if dtype not in _FLOAT:
        raise ValueError("checkpoints load as float32, float16 or bfloat16")
    return _routed.checkpoint_load(checkpoint, _FLOAT[dtype])


@torch.no_grad()
def pack_int4(w: torch.Tensor, group: int = 128) -> Int4Weights:
    """``w`` [experts, inner, outer] in 4 bits: per group of ``group`` inner neighbours the scale max|w| / 7 (in w's
    type) and whole numbers from -7 to 7.  A NaN or infinity makes its group NaN.  Done once per model, in plain torch."""
    if w.dim() != 3 or w.dtype not in _HALF:
        raise ValueError("weights must be [experts, inner, outer] of float16 or bfloat16")
    if group not in (32, 64, 128) or w.shape[1] % group:
        raise ValueError("weight group must be 32, 64 or 128 and divide the inner width")
    experts, inner, outer = w.shape
    by_group = w.transpose(1, 2).float().reshape(experts, outer, inner // group, group)
    scales = (by_group.abs().amax(3) / 7).to(w.dtype)
    fine = torch.isfinite(scales)
    unit = torch.where(fine & (scales != 0), scales, 1).float()
    scales = torch.where(fine, scales, torch.nan)
    codes = (torch.round(by_group / unit[..., None]).nan_to_num().clamp(-7, 7) + 8).to(torch.uint8).reshape(experts, outer, inner)
    return Int4Weights((codes[..., 0::2] | (codes[..., 1::2] << 4)).contiguous(), scales.contiguous(), group)


def routed_matvec(x: torch.Tensor, weights: Int4Weights, routing: Routing, *, gather: bool = False,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """``routed_matmul`` for few rows (single tokens) with 4-bit weights: [entries, outer].

    Memory bound on the weights: a chosen expert's are read once for every eight of its rows, so many rows per expert
    are better served by ``routed_matmul`` with 16-bit weights.
    """
    codes, scales, group = weights
    return _routed.routed_matvec(x, codes, scales, group, routing, gather, out)
