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
CPU fallback.  ``out`` takes preallocated results, so that a captured or
latency-bound step allocates nothing.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _native

_HALF = {torch.float16: _native.F16, torch.bfloat16: _native.BF16}
_FLOAT = {torch.float32: _native.F32, **_HALF}
_SCORE = {"softmax": 0, "sigmoid": 1}


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


def _device(*tensors: torch.Tensor) -> int:
    """Index of the CUDA device that holds all the tensors."""
    index = tensors[0].get_device()
    for tensor in tensors:
        other = tensor.get_device()   # -1 for host storage
        if other < 0 or not tensor.is_cuda:
            raise ValueError("routed storage must be a CUDA tensor (there is no CPU fallback)")
        if other != index:
            raise ValueError("routed operands must be on one device")
    return index


def _packed(tensor: torch.Tensor, shape: tuple, dtype: torch.dtype, what: str) -> int:
    if tensor.dtype is not dtype or tensor.shape != shape or not tensor.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {list(shape)}, got {tensor.dtype} "
                         f"{list(tensor.shape)} with strides {list(tensor.stride())}")
    return tensor.data_ptr()


def _matrix(tensor: torch.Tensor, what: str) -> int:
    """Row stride of a 2-d tensor whose rows are contiguous."""
    rows, width = tensor.shape
    stride, step = tensor.stride()
    if step != 1 and width > 1:
        raise ValueError(f"{what} must be 2-d with contiguous rows")
    return stride if rows > 1 or stride > width else width


def _code(table: dict, tensor: torch.Tensor, what: str) -> int:
    code = table.get(tensor.dtype)
    if code is None:
        raise ValueError(f"{what} must be {' or '.join(str(t)[6:] for t in table)}, got {tensor.dtype}")
    return code


def _call(name: str, device: int, *arguments) -> None:
    function = getattr(_native.lib(), name)
    err = _native.error_buffer()
    # The stream's handle alone: building a Stream object costs more than the checks.
    stream = torch._C._cuda_getCurrentRawStream(device)
    if torch._C._cuda_getDevice() == device:
        status = function(*arguments, stream, err, len(err))
    else:
        with torch.cuda.device(device):
            status = function(*arguments, stream, err, len(err))
    if status != 0:
        _native.check(status, err)


def _entries(routing: Routing) -> tuple[int, int, int]:
    """(tokens, top_k, experts) of a routing whose arrays agree."""
    if routing.experts.ndim != 2:
        raise ValueError("routing experts must be [tokens, top_k]")
    tokens, top_k = routing.experts.shape
    _packed(routing.rows, (tokens * top_k,), torch.int32, "routing rows")
    experts = routing.offsets.numel() - 1
    if experts < 1:
        raise ValueError("routing offsets must be [experts + 1]")
    _packed(routing.offsets, (experts + 1,), torch.int32, "routing offsets")
    return tokens, top_k, experts


def empty_routing(tokens: int, top_k: int, experts: int, device="cuda") -> Routing:
    """Uninitialised buffers for ``route(..., out=...)``."""
    def ints(*shape):
        return torch.empty(shape, dtype=torch.int32, device=device)
    return Routing(ints(tokens, top_k), torch.empty(tokens, top_k, dtype=torch.float32, device=device),
                   ints(tokens * top_k), ints(tokens, top_k), ints(experts + 1))


def _score(score: str) -> int:
    code = _SCORE.get(score)
    if code is None:
        raise ValueError("score must be 'softmax' or 'sigmoid'")
    return code


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
    """
    if logits.ndim != 2:
        raise ValueError("logits must be [tokens, experts]")
    tokens, experts = logits.shape
    device = _device(logits, *(t for t in (bias, mask) if t is not None))
    code = _code(_FLOAT, logits, "logits")
    bias_pointer = None if bias is None else _packed(bias, (experts,), torch.float32, "bias")
    mask_pointer = None if mask is None else _packed(mask, (tokens,), torch.bool, "mask")
    if out is None:
        out = empty_routing(tokens, top_k, experts, logits.device)
    else:
        _device(logits, *out)
    entry = (tokens, top_k)
    pointers = (_packed(out.experts, entry, torch.int32, "routing experts"),
                _packed(out.weights, entry, torch.float32, "routing weights"),
                _packed(out.rows, (tokens * top_k,), torch.int32, "routing rows"),
                _packed(out.positions, entry, torch.int32, "routing positions"),
                _packed(out.offsets, (experts + 1,), torch.int32, "routing offsets"))
    size = _native.lib().t0b_route_workspace(tokens, experts)
    workspace = logits.new_empty(size, dtype=torch.uint8) if size else None
    _call("t0b_route", device, code, tokens, experts, top_k, groups, groups if top_groups is None else top_groups,
          group_best, _score(score), int(renormalize), scale, logits.data_ptr(), _matrix(logits, "logits"),
          bias_pointer, mask_pointer, *pointers, None if workspace is None else workspace.data_ptr(), size)
    return out


def route_backward(logits: torch.Tensor, routing: Routing, weights_grad: torch.Tensor, *, score: str = "softmax",
                   renormalize: bool = True, scale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of ``routing.weights`` with respect to the logits, for the same arguments as ``route``.

    The choice of experts is piecewise constant and the bias enters it only, so neither has a gradient.  Tokens
    without an expert get zeros, whatever their logits hold.
    """
    if logits.ndim != 2:
        raise ValueError("logits must be [tokens, experts]")
    tokens, experts = logits.shape
    device = _device(logits, routing.experts, weights_grad)
    code = _code(_FLOAT, logits, "logits")
    top_k = routing.experts.shape[-1]
    chosen = _packed(routing.experts, (tokens, top_k), torch.int32, "routing experts")
    grad = _packed(weights_grad, (tokens, top_k), torch.float32, "weights_grad")
    if out is None:
        out = logits.new_empty((tokens, experts))
    result = _packed(out, (tokens, experts), logits.dtype, "out")
    _call("t0b_route_backward", device, code, tokens, experts, top_k, _score(score), int(renormalize), scale,
          logits.data_ptr(), _matrix(logits, "logits"), chosen, grad, result)
    return out


def _operand(x: torch.Tensor, width: int, gather: bool, tokens: int, top_k: int, what: str) -> None:
    rows = tokens if gather else tokens * top_k
    if x.ndim != 2 or x.shape[0] != rows or x.shape[1] != width:
        raise ValueError(f"{what} must be [{rows}, {width}] ({'token' if gather else 'expert-ordered'} rows), "
                         f"got {list(x.shape)}")


def routed_matmul(x: torch.Tensor, w: torch.Tensor, routing: Routing, *, gather: bool = False,
                  transpose: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x[r] @ w[e]`` (or ``@ w[e].T``) for every row of every expert: [entries, outer or inner].

    ``w`` [experts, inner, outer], float16 or bfloat16 as ``x``.  ``x`` holds token rows with ``gather`` (row p reads
    its entry's token), else expert-ordered rows.  Summed in 32 bits, rounded once; rows without an expert are zero.
    """
    tokens, top_k, experts = _entries(routing)
    device = _device(x, w, routing.rows, routing.offsets)
    code = _code(_HALF, x, "product operands")
    if w.ndim != 3 or w.shape[0] != experts:
        raise ValueError(f"weights must be [{experts}, inner, outer]")
    _, inner, outer = w.shape
    weights = _packed(w, w.shape, x.dtype, "weights")
    _operand(x, outer if transpose else inner, gather, tokens, top_k, "x")
    width = inner if transpose else outer
    if out is None:
        out = x.new_empty((tokens * top_k, width))
    else:
        _device(x, out)
    result = _packed(out, (tokens * top_k, width), x.dtype, "out")
    _call("t0b_routed_product", device, code, int(transpose), tokens * top_k, experts, top_k, inner, outer,
          int(gather), x.data_ptr(), x.shape[0], _matrix(x, "x"), weights, routing.rows.data_ptr(),
          routing.offsets.data_ptr(), result)
    return out


def routed_weight_grad(x: torch.Tensor, y_grad: torch.Tensor, routing: Routing, *, gather_x: bool = False,
                       gather_y: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Every expert's weight gradient ``sum over its rows of x[r]^T y_grad[q]``: [experts, inner, outer].

    Either operand holds token rows (``gather_x``, ``gather_y``) or expert-ordered ones.  An expert without rows
    gets zeros.
    """
    tokens, top_k, experts = _entries(routing)
    device = _device(x, y_grad, routing.rows, routing.offsets)
    code = _code(_HALF, x, "product operands")
    if y_grad.dtype != x.dtype:
        raise ValueError("product operands must share a dtype")
    inner, outer = x.shape[-1], y_grad.shape[-1]
    _operand(x, inner, gather_x, tokens, top_k, "x")
    _operand(y_grad, outer, gather_y, tokens, top_k, "y_grad")
    if out is None:
        out = x.new_empty((experts, inner, outer))
    else:
        _device(x, out)
    result = _packed(out, (experts, inner, outer), x.dtype, "out")
    _call("t0b_routed_weight_grad", device, code, tokens * top_k, experts, top_k, inner, outer, int(gather_x),
          x.data_ptr(), x.shape[0], _matrix(x, "x"), int(gather_y), y_grad.data_ptr(), y_grad.shape[0],
          _matrix(y_grad, "y_grad"), routing.rows.data_ptr(), routing.offsets.data_ptr(), result)
    return out


def routed_sum(y: torch.Tensor, routing: Routing, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """Each token's sum over its experts' rows: [tokens, width].  Also the gradient of gathering token rows."""
    if routing.positions.ndim != 2:
        raise ValueError("routing positions must be [tokens, top_k]")
    tokens, top_k = routing.positions.shape
    device = _device(y, routing.positions)
    code = _code(_HALF, y, "sum operands")
    positions = _packed(routing.positions, (tokens, top_k), torch.int32, "routing positions")
    if y.ndim != 2 or y.shape[0] != tokens * top_k:
        raise ValueError(f"y must be [{tokens * top_k}, width]")
    width = y.shape[1]
    if out is None:
        out = y.new_empty((tokens, width))
    else:
        _device(y, out)
    result = _packed(out, (tokens, width), y.dtype, "out")
    _call("t0b_routed_sum", device, code, tokens, top_k, width, y.data_ptr(), _matrix(y, "y"), positions, result)
    return out


def _row_weights(routing: Routing | None, rows: int) -> tuple:
    """(weights, rows, offsets, experts) arguments of the gated entry points."""
    if routing is None:
        return None, None, None, 0
    tokens, top_k, experts = _entries(routing)
    if tokens * top_k != rows:
        raise ValueError(f"the routing has {tokens * top_k} entries, the activation {rows} rows")
    weights = _packed(routing.weights, (tokens, top_k), torch.float32, "routing weights")
    return weights, routing.rows.data_ptr(), routing.offsets.data_ptr(), experts


def gated_save(h: torch.Tensor, *, routing: Routing | None = None, group: int = 128,
               out: tuple[torch.Tensor, Checkpoint] | None = None) -> tuple[torch.Tensor, Checkpoint]:
    """``weight * silu(gate) * up`` of rows ``h = [gate | up]``, and ``h`` in 8 bits for ``gated_backward``.

    ``group`` (32, 64 or 128) neighbours of one half share a scale, their largest magnitude / 127.  A row's weight is
    its entry's in ``routing``, or 1 without one; with one, rows without an expert are not read and give zeros.
    """
    if h.ndim != 2 or h.shape[1] % 2 or h.shape[1] == 0:
        raise ValueError("h must be [rows, 2 * width]")
    rows, width = h.shape[0], h.shape[1] // 2
    device = _device(h, *(() if routing is None else (routing.weights, routing.rows, routing.offsets)))
    code = _code(_HALF, h, "gated activations")
    if group not in (32, 64, 128):
        raise ValueError("checkpoint group must be 32, 64 or 128")
    scales = 2 * -(-width // group)
    if out is None:
        a = h.new_empty((rows, width))
        kept = Checkpoint(h.new_empty((rows, 2 * width), dtype=torch.int8),
                          h.new_empty((rows, scales), dtype=torch.float32), group)
    else:
        a, kept = out
        if kept.group != group:
            raise ValueError("out's checkpoint has another group")
        _device(h, a, kept.codes, kept.scales)
    _call("t0b_gated_save", device, code, rows, width, group, h.data_ptr(), _matrix(h, "h"),
          *_row_weights(routing, rows), _packed(a, (rows, width), h.dtype, "out"),
          _packed(kept.codes, (rows, 2 * width), torch.int8, "checkpoint codes"),
          _packed(kept.scales, (rows, scales), torch.float32, "checkpoint scales"))
    return a, kept


def _checkpoint(checkpoint: Checkpoint) -> tuple[int, int, int, int]:
    """(rows, width, codes, scales) of a checkpoint whose arrays agree."""
    codes, scales, group = checkpoint
    if group not in (32, 64, 128):
        raise ValueError("checkpoint group must be 32, 64 or 128")
    if codes.ndim != 2 or codes.shape[1] % 2 or codes.shape[1] == 0:
        raise ValueError("checkpoint codes must be [rows, 2 * width]")
    rows, width = codes.shape[0], codes.shape[1] // 2
    return (rows, width, _packed(codes, codes.shape, torch.int8, "checkpoint codes"),
            _packed(scales, (rows, 2 * -(-width // group)), torch.float32, "checkpoint scales"))


def gated_backward(checkpoint: Checkpoint, a_grad: torch.Tensor, *, routing: Routing | None = None,
                   ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of ``gated_save`` from its checkpoint: ``(h_grad, a, weights_grad)``.

    ``a`` is the activation again, from the checkpoint (the next product's weight gradient needs it).
    ``weights_grad`` is the gradient of the routing's weights [tokens, top_k], or of a weight of 1 per row [rows]
    without a routing.
    """
    rows, width, codes, scales = _checkpoint(checkpoint)
    device = _device(a_grad, checkpoint.codes, checkpoint.scales,
                     *(() if routing is None else (routing.weights, routing.rows, routing.offsets)))
    code = _code(_HALF, a_grad, "gated activations")
    if a_grad.shape != (rows, width):
        raise ValueError(f"a_grad must be [{rows}, {width}]")
    weights = _row_weights(routing, rows)
    h_grad = a_grad.new_empty((rows, 2 * width))
    a = a_grad.new_empty((rows, width))
    weights_grad = a_grad.new_empty((rows,) if routing is None else routing.weights.shape, dtype=torch.float32)
    _call("t0b_gated_backward", device, code, rows, width, checkpoint.group, codes, scales, a_grad.data_ptr(),
          _matrix(a_grad, "a_grad"), *weights, h_grad.data_ptr(), a.data_ptr(), weights_grad.data_ptr())
    return h_grad, a, weights_grad


def checkpoint_load(checkpoint: Checkpoint, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values a checkpoint stands for, as float32, float16 or bfloat16."""
    rows, width, codes, scales = _checkpoint(checkpoint)
    device = _device(checkpoint.codes, checkpoint.scales)
    if dtype not in _FLOAT:
        raise ValueError("checkpoints load as float32, float16 or bfloat16")
    values = checkpoint.codes.new_empty((rows, 2 * width), dtype=dtype)
    _call("t0b_checkpoint_load", device, _FLOAT[dtype], rows, width, checkpoint.group, codes, scales,
          values.data_ptr())
    return values


def pack_int4(w: torch.Tensor, group: int = 128) -> Int4Weights:
    """``w`` [experts, inner, outer] in 4 bits: per group of ``group`` inner neighbours the scale max|w| / 7 (in w's
    type) and whole numbers from -7 to 7.  Done once per model, in plain torch."""
    if w.ndim != 3 or w.dtype not in _HALF:
        raise ValueError("weights must be [experts, inner, outer] of float16 or bfloat16")
    if group not in (32, 64, 128) or w.shape[1] % group:
        raise ValueError("weight group must be 32, 64 or 128 and divide the inner width")
    experts, inner, outer = w.shape
    by_group = w.transpose(1, 2).float().reshape(experts, outer, inner // group, group)
    scales = (by_group.abs().amax(3) / 7).to(w.dtype)
    unit = torch.where(scales == 0, 1, scales).float()
    codes = (torch.round(by_group / unit[..., None]).clamp(-7, 7) + 8).to(torch.uint8).reshape(experts, outer, inner)
    return Int4Weights((codes[..., 0::2] | (codes[..., 1::2] << 4)).contiguous(), scales.contiguous(), group)


def routed_matvec(x: torch.Tensor, weights: Int4Weights, routing: Routing, *, gather: bool = False,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """``routed_matmul`` for few rows (single tokens) with 4-bit weights: [entries, outer].

    Memory bound on the weights: each chosen expert's are read once however many rows it has.
    """
    tokens, top_k, experts = _entries(routing)
    codes, scales, group = weights
    device = _device(x, codes, scales, routing.rows, routing.offsets)
    code = _code(_HALF, x, "4-bit product operands")
    if group not in (32, 64, 128) or x.ndim != 2 or x.shape[1] % group:
        raise ValueError("weight group must be 32, 64 or 128 and divide the inner width")
    inner = x.shape[1]
    if codes.ndim != 3:
        raise ValueError("4-bit weight codes must be [experts, outer, inner / 2]")
    outer = codes.shape[1]
    code_pointer = _packed(codes, (experts, outer, inner // 2), torch.uint8, "4-bit weight codes")
    scale_pointer = _packed(scales, (experts, outer, inner // group), x.dtype, "4-bit weight scales")
    _operand(x, inner, gather, tokens, top_k, "x")
    if out is None:
        out = x.new_empty((tokens * top_k, outer))
    else:
        _device(x, out)
    result = _packed(out, (tokens * top_k, outer), x.dtype, "out")
    _call("t0b_routed_matvec4", device, code, tokens * top_k, experts, top_k, inner, outer, group, int(gather),
          x.data_ptr(), x.shape[0], _matrix(x, "x"), code_pointer, scale_pointer, routing.rows.data_ptr(),
          routing.offsets.data_ptr(), result)
    return out
