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

import threading
from typing import NamedTuple

import torch

from . import _native

_HALF = {torch.float16: _native.F16, torch.bfloat16: _native.BF16}
_FLOAT = {torch.float32: _native.F32, **_HALF}
_SCORE = {"softmax": 0, "sigmoid": 1}
_INT, _REAL = torch.int32, torch.float32


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
    index = tensors[0].get_device()   # -1 for host storage
    for tensor in tensors:
        if tensor.get_device() != index or not tensor.is_cuda:
            if not tensor.is_cuda or not tensors[0].is_cuda:
                raise ValueError("routed storage must be a CUDA tensor (there is no CPU fallback)")
            raise ValueError("routed operands must be on one device")
    return index


def _packed(tensor: torch.Tensor, shape: tuple, dtype: torch.dtype, what: str) -> int:
    if tensor.dtype is dtype and tensor.shape == shape and tensor.is_contiguous():
        return tensor.data_ptr()
    raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {list(shape)}, got {tensor.dtype} "
                     f"{list(tensor.shape)} with strides {list(tensor.stride())}")


def _output(like: torch.Tensor, out: torch.Tensor | None, shape: tuple) -> tuple[torch.Tensor, int]:
    """The result of an operator and its address: new, or ``out`` if that fits."""
    if out is None:
        out = like.new_empty(shape)
        return out, out.data_ptr()
    _device(like, out)
    return out, _packed(out, shape, like.dtype, "out")


def _rows(x: torch.Tensor, rows: int, width: int, what: str, gather: bool = False) -> tuple[int, int]:
    """(address, row stride) of a matrix of that shape whose rows are contiguous."""
    if x.shape != (rows, width):
        kind = "token" if gather else "expert-ordered"
        raise ValueError(f"{what} must be [{rows}, {width}] ({kind} rows), got {list(x.shape)}")
    stride, step = x.stride()
    if step != 1 and width > 1:
        raise ValueError(f"{what} must have contiguous rows")
    return x.data_ptr(), stride if rows > 1 or stride > width else width


def _code(table: dict, tensor: torch.Tensor, what: str) -> int:
    code = table.get(tensor.dtype)
    if code is None:
        raise ValueError(f"{what} must be {' or '.join(str(t)[6:] for t in table)}, got {tensor.dtype}")
    return code


class _Entry:
    """A C entry point: called with its arguments up to the stream, on the device's current stream.

    Small operators take less time than their checks, so a call costs as little as it can: the function is looked up
    once, a thread keeps its error buffer, and the stream is asked for its handle alone.
    """

    local = threading.local()

    def __init__(self, name: str):
        self.name = name
        self.function = None

    def __call__(self, device: int, *arguments) -> None:
        function = self.function
        if function is None:
            function = self.function = getattr(_native.lib(), self.name)
        try:
            err = self.local.err
        except AttributeError:
            err = self.local.err = _native.error_buffer()
        stream = torch._C._cuda_getCurrentRawStream(device)
        if torch._C._cuda_getDevice() == device:
            status = function(*arguments, stream, err, 512)
        else:
            with torch.cuda.device(device):
                status = function(*arguments, stream, err, 512)
        if status != 0:
            _native.check(status, err)


_route, _route_backward = _Entry("t0b_route"), _Entry("t0b_route_backward")
_product, _weight_grad, _sum = _Entry("t0b_routed_product"), _Entry("t0b_routed_weight_grad"), _Entry("t0b_routed_sum")
_gated_save, _gated_backward = _Entry("t0b_gated_save"), _Entry("t0b_gated_backward")
_checkpoint_load, _matvec4 = _Entry("t0b_checkpoint_load"), _Entry("t0b_routed_matvec4")


def _entries(routing: Routing) -> tuple[int, int, int, int, int]:
    """(tokens, top_k, experts, rows, offsets) of a routing whose arrays agree; the last two are addresses."""
    chosen, _, rows, _, offsets = routing
    if chosen.dim() != 2:
        raise ValueError("routing experts must be [tokens, top_k]")
    tokens, top_k = chosen.shape
    experts = offsets.numel() - 1
    if experts < 1:
        raise ValueError("routing offsets must be [experts + 1]")
    return (tokens, top_k, experts, _packed(rows, (tokens * top_k,), _INT, "routing rows"),
            _packed(offsets, (experts + 1,), _INT, "routing offsets"))


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
    if logits.dim() != 2:
        raise ValueError("logits must be [tokens, experts]")
    tokens, experts = logits.shape
    device = _device(logits, *[t for t in (bias, mask) if t is not None])
    code = _code(_FLOAT, logits, "logits")
    address, stride = _rows(logits, tokens, experts, "logits")
    bias_pointer = None if bias is None else _packed(bias, (experts,), _REAL, "bias")
    mask_pointer = None if mask is None else _packed(mask, (tokens,), torch.bool, "mask")
    if out is None:
        out = empty_routing(tokens, top_k, experts, logits.device)
    else:
        _device(logits, *out)
    chosen, weights, rows, positions, offsets = out
    entry = (tokens, top_k)
    size = _native.lib().t0b_route_workspace(tokens, experts)
    workspace = logits.new_empty(size, dtype=torch.uint8).data_ptr() if size else None
    _route(device, code, tokens, experts, top_k, groups, groups if top_groups is None else top_groups, group_best,
           _score(score), int(renormalize), scale, address, stride, bias_pointer, mask_pointer,
           _packed(chosen, entry, _INT, "routing experts"), _packed(weights, entry, _REAL, "routing weights"),
           _packed(rows, (tokens * top_k,), _INT, "routing rows"),
           _packed(positions, entry, _INT, "routing positions"),
           _packed(offsets, (experts + 1,), _INT, "routing offsets"), workspace, size)
    return out


def route_backward(logits: torch.Tensor, routing: Routing, weights_grad: torch.Tensor, *, score: str = "softmax",
                   renormalize: bool = True, scale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of ``routing.weights`` with respect to the logits, for the same arguments as ``route``.

    The choice of experts is piecewise constant and the bias enters it only, so neither has a gradient.  Tokens
    without an expert get zeros, whatever their logits hold.
    """
    if logits.dim() != 2:
        raise ValueError("logits must be [tokens, experts]")
    tokens, experts = logits.shape
    device = _device(logits, routing.experts, weights_grad)
    code = _code(_FLOAT, logits, "logits")
    address, stride = _rows(logits, tokens, experts, "logits")
    top_k = routing.experts.shape[-1]
    chosen = _packed(routing.experts, (tokens, top_k), _INT, "routing experts")
    grad = _packed(weights_grad, (tokens, top_k), _REAL, "weights_grad")
    out, result = _output(logits, out, (tokens, experts))
    _route_backward(device, code, tokens, experts, top_k, _score(score), int(renormalize), scale, address, stride,
                    chosen, grad, result)
    return out


def routed_matmul(x: torch.Tensor, w: torch.Tensor, routing: Routing, *, gather: bool = False,
                  transpose: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x[r] @ w[e]`` (or ``@ w[e].T``) for every row of every expert: [entries, outer or inner].

    ``w`` [experts, inner, outer], float16 or bfloat16 as ``x``.  ``x`` holds token rows with ``gather`` (row p reads
    its entry's token), else expert-ordered rows.  Summed in 32 bits, rounded once; rows without an expert are zero.
    """
    tokens, top_k, experts, rows, offsets = _entries(routing)
    device = _device(x, w, routing.rows, routing.offsets)
    code = _code(_HALF, x, "product operands")
    if w.dim() != 3 or w.shape[0] != experts:
        raise ValueError(f"weights must be [{experts}, inner, outer]")
    _, inner, outer = w.shape
    entries = tokens * top_k
    x_rows = tokens if gather else entries
    weights = _packed(w, w.shape, x.dtype, "weights")
    address, stride = _rows(x, x_rows, outer if transpose else inner, "x", gather)
    out, result = _output(x, out, (entries, inner if transpose else outer))
    _product(device, code, int(transpose), entries, experts, top_k, inner, outer, int(gather), address, x_rows, stride,
             weights, rows, offsets, result)
    return out


def routed_weight_grad(x: torch.Tensor, y_grad: torch.Tensor, routing: Routing, *, gather_x: bool = False,
                       gather_y: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Every expert's weight gradient ``sum over its rows of x[r]^T y_grad[q]``: [experts, inner, outer].

    Either operand holds token rows (``gather_x``, ``gather_y``) or expert-ordered ones.  An expert without rows
    gets zeros.
    """
    tokens, top_k, experts, rows, offsets = _entries(routing)
    device = _device(x, y_grad, routing.rows, routing.offsets)
    code = _code(_HALF, x, "product operands")
    if y_grad.dtype != x.dtype:
        raise ValueError("product operands must share a dtype")
    inner, outer = x.shape[-1], y_grad.shape[-1]
    entries = tokens * top_k
    x_rows, y_rows = tokens if gather_x else entries, tokens if gather_y else entries
    x_address, x_stride = _rows(x, x_rows, inner, "x", gather_x)
    y_address, y_stride = _rows(y_grad, y_rows, outer, "y_grad", gather_y)
    out, result = _output(x, out, (experts, inner, outer))
    _weight_grad(device, code, entries, experts, top_k, inner, outer, int(gather_x), x_address, x_rows, x_stride,
                 int(gather_y), y_address, y_rows, y_stride, rows, offsets, result)
    return out


def routed_sum(y: torch.Tensor, routing: Routing, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """Each token's sum over its experts' rows: [tokens, width].  Also the gradient of gathering token rows."""
    if routing.positions.dim() != 2:
        raise ValueError("routing positions must be [tokens, top_k]")
    tokens, top_k = routing.positions.shape
    device = _device(y, routing.positions)
    code = _code(_HALF, y, "sum operands")
    positions = _packed(routing.positions, (tokens, top_k), _INT, "routing positions")
    width = y.shape[-1]
    address, stride = _rows(y, tokens * top_k, width, "y")
    out, result = _output(y, out, (tokens, width))
    _sum(device, code, tokens, top_k, width, address, stride, positions, result)
    return out


def _row_weights(routing: Routing | None, rows: int) -> tuple:
    """(weights, rows, offsets, experts) arguments of the gated entry points."""
    if routing is None:
        return None, None, None, 0
    tokens, top_k, experts, entries, offsets = _entries(routing)
    if tokens * top_k != rows:
        raise ValueError(f"the routing has {tokens * top_k} entries, the activation {rows} rows")
    return _packed(routing.weights, (tokens, top_k), _REAL, "routing weights"), entries, offsets, experts


def gated_save(h: torch.Tensor, *, routing: Routing | None = None, group: int = 128,
               out: tuple[torch.Tensor, Checkpoint] | None = None) -> tuple[torch.Tensor, Checkpoint]:
    """``weight * silu(gate) * up`` of rows ``h = [gate | up]``, and ``h`` in 8 bits for ``gated_backward``.

    ``group`` (32, 64 or 128) neighbours of one half share a scale, their largest magnitude / 127.  A row's weight is
    its entry's in ``routing``, or 1 without one; with one, rows without an expert are not read and give zeros.
    """
    if h.dim() != 2 or h.shape[1] % 2 or h.shape[1] == 0:
        raise ValueError("h must be [rows, 2 * width]")
    rows, width = h.shape[0], h.shape[1] // 2
    device = _device(h, *(() if routing is None else (routing.weights, routing.rows, routing.offsets)))
    code = _code(_HALF, h, "gated activations")
    if group not in (32, 64, 128):
        raise ValueError("checkpoint group must be 32, 64 or 128")
    scales = 2 * -(-width // group)
    address, stride = _rows(h, rows, 2 * width, "h")
    if out is None:
        a = h.new_empty((rows, width))
        kept = Checkpoint(h.new_empty((rows, 2 * width), dtype=torch.int8),
                          h.new_empty((rows, scales), dtype=torch.float32), group)
    else:
        a, kept = out
        if kept.group != group:
            raise ValueError("out's checkpoint has another group")
        _device(h, a, kept.codes, kept.scales)
    _gated_save(device, code, rows, width, group, address, stride, *_row_weights(routing, rows),
                _packed(a, (rows, width), h.dtype, "out"),
                _packed(kept.codes, (rows, 2 * width), torch.int8, "checkpoint codes"),
                _packed(kept.scales, (rows, scales), _REAL, "checkpoint scales"))
    return a, kept


def gated(h: torch.Tensor, *, routing: Routing | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``gated_save``'s activation alone, for a pass that has no backward one."""
    if h.dim() != 2 or h.shape[1] % 2 or h.shape[1] == 0:
        raise ValueError("h must be [rows, 2 * width]")
    rows, width = h.shape[0], h.shape[1] // 2
    device = _device(h, *(() if routing is None else (routing.weights, routing.rows, routing.offsets)))
    code = _code(_HALF, h, "gated activations")
    address, stride = _rows(h, rows, 2 * width, "h")
    out, result = _output(h, out, (rows, width))
    _gated_save(device, code, rows, width, 128, address, stride, *_row_weights(routing, rows), result, None, None)
    return out


def _checkpoint(checkpoint: Checkpoint) -> tuple[int, int, int, int]:
    """(rows, width, codes, scales) of a checkpoint whose arrays agree."""
    codes, scales, group = checkpoint
    if group not in (32, 64, 128):
        raise ValueError("checkpoint group must be 32, 64 or 128")
    if codes.dim() != 2 or codes.shape[1] % 2 or codes.shape[1] == 0:
        raise ValueError("checkpoint codes must be [rows, 2 * width]")
    rows, width = codes.shape[0], codes.shape[1] // 2
    return (rows, width, _packed(codes, codes.shape, torch.int8, "checkpoint codes"),
            _packed(scales, (rows, 2 * -(-width // group)), _REAL, "checkpoint scales"))


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
    address, stride = _rows(a_grad, rows, width, "a_grad")
    weights = _row_weights(routing, rows)
    h_grad = a_grad.new_empty((rows, 2 * width))
    a = a_grad.new_empty((rows, width))
    weights_grad = a_grad.new_empty((rows,) if routing is None else routing.weights.shape, dtype=torch.float32)
    _gated_backward(device, code, rows, width, checkpoint.group, codes, scales, address, stride, *weights,
                    h_grad.data_ptr(), a.data_ptr(), weights_grad.data_ptr())
    return h_grad, a, weights_grad


def checkpoint_load(checkpoint: Checkpoint, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values a checkpoint stands for, as float32, float16 or bfloat16."""
    rows, width, codes, scales = _checkpoint(checkpoint)
    device = _device(checkpoint.codes, checkpoint.scales)
    if dtype not in _FLOAT:
        raise ValueError("checkpoints load as float32, float16 or bfloat16")
    values = checkpoint.codes.new_empty((rows, 2 * width), dtype=dtype)
    _checkpoint_load(device, _FLOAT[dtype], rows, width, checkpoint.group, codes, scales,
                     values.data_ptr())
    return values


def pack_int4(w: torch.Tensor, group: int = 128) -> Int4Weights:
    """``w`` [experts, inner, outer] in 4 bits: per group of ``group`` inner neighbours the scale max|w| / 7 (in w's
    type) and whole numbers from -7 to 7.  Done once per model, in plain torch."""
    if w.dim() != 3 or w.dtype not in _HALF:
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
    tokens, top_k, experts, rows, offsets = _entries(routing)
    codes, scales, group = weights
    device = _device(x, codes, scales, routing.rows, routing.offsets)
    code = _code(_HALF, x, "4-bit product operands")
    if group not in (32, 64, 128) or x.dim() != 2 or x.shape[1] % group:
        raise ValueError("weight group must be 32, 64 or 128 and divide the inner width")
    inner = x.shape[1]
    if codes.dim() != 3:
        raise ValueError("4-bit weight codes must be [experts, outer, inner / 2]")
    outer = codes.shape[1]
    code_pointer = _packed(codes, (experts, outer, inner // 2), torch.uint8, "4-bit weight codes")
    scale_pointer = _packed(scales, (experts, outer, inner // group), x.dtype, "4-bit weight scales")
    entries = tokens * top_k
    x_rows = tokens if gather else entries
    address, stride = _rows(x, x_rows, inner, "x", gather)
    out, result = _output(x, out, (entries, outer))
    _matvec4(device, code, entries, experts, top_k, inner, outer, group, int(gather), address, x_rows, stride,
             code_pointer, scale_pointer, rows, offsets, result)
    return out
