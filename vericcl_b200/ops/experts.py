"""Mixture-of-experts operators on both sides of an AllToAll of tokens.

* :func:`route` — the router's choice: the ``k`` largest logits of each token and their softmax weights.
* :func:`sort_by_expert` — a stable sort of the (token, choice) assignments by expert, packed or with an equal
  number of rows per expert (the equal parts an AllToAll exchanges).
* :func:`dispatch` — every token copied to its rows; :func:`combine` — its rows weighted and summed back.
* :func:`expert_matmul_int4` — the experts' matrix-vector products with 4-bit weights and group scales
  (:func:`quantize_int4` lays weights out).

All run on the current stream of their tensors' GPU, allocate nothing but their results, read nothing back to
the host and can be captured into a CUDA graph.  ``route``, ``dispatch`` and ``combine`` take part in autograd;
``route_backward``, ``dispatch_backward`` and ``combine_backward`` are the same gradients as plain calls, which is
the form to capture: autograd refuses under capture, because the accumulation into a leaf that an eager graph
still holds would run on a stream outside the capture.  Forward-mode gradients are refused.

Matrices are ``[rows, hidden]`` with contiguous rows at any row stride (a column slice of a wider matrix, a row
broadcast by ``expand``); ``out`` may be such a view too, must not overlap an input (columns of one matrix beside each
other do not) and is written whole, which autograd sees as an in-place change of it.
:class:`~vericcl_b200.models.ExpertExchange` puts these around an engine's AllToAll.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from vericcl_b200.errors import RuntimeFailure
from vericcl_b200.ops import native

MAX_EXPERTS = 1024
MAX_CHOICES = 32
MAX_COLUMNS = 1 << 22
INT4_GROUPS = (32, 64, 128)
_DTYPES = frozenset({torch.float32, torch.bfloat16, torch.float16})
_INT_MAX = 2 ** 31 - 1
_GIVE_UP = False             # True: 4-bit products wait for no weights, as if they arrived too late

_module = None


def _mod():
    global _module
    if _module is None:
        _module = native.cuda()
    return _module


def _call(name, check, *args):
    """The native call ``name(*args)``, which refuses bad arguments before it launches anything; ``check()`` then says
    what was wrong.  Tensors off the GPU never reach it."""
    if args[0].is_cuda:
        try:
            return getattr(_module or _mod(), name)(*args)
        except torch.OutOfMemoryError:
            raise
        except (RuntimeError, TypeError) as error:
            check()
            raise RuntimeFailure("%s: %s" % (name, str(error).splitlines()[0])) from error
    check()
    raise RuntimeFailure("the expert operators need CUDA tensors")


class ExpertOrder:
    """Where each assignment's row is: the result of :func:`sort_by_expert`.

    ``slot`` [tokens, k]: row of each assignment, -1 where it has none; ``source`` [rows]: assignment
    (``token * k + choice``) of each row, -1 where a row has none; ``counts`` [experts]: rows in use;
    ``starts`` [experts]: first row.  All int32 on the GPU.
    """

    __slots__ = ("slot", "source", "counts", "starts")

    def __init__(self, slot, source, counts, starts):
        self.slot, self.source, self.counts, self.starts = slot, source, counts, starts

    @property
    def rows(self) -> int:
        return self.source.numel()


# -- checks -----------------------------------------------------------------------------------------------

def _no_tangent(t, name):
    if forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeFailure("%s carries a forward-mode gradient: these operators have reverse-mode gradients only" % name)


def _matrix(t, name):
    if t.dim() != 2 or t.dtype not in _DTYPES:
        raise RuntimeFailure("%s must be a [rows, columns] matrix of float32, bfloat16 or float16" % name)
    if t.size(1) > MAX_COLUMNS:
        raise RuntimeFailure("%s has more than %d columns" % (name, MAX_COLUMNS))
    if t.size(1) > 1 and t.stride(1) != 1:
        raise RuntimeFailure("%s must have contiguous rows (stride 1 in the last dimension)" % name)
    _no_tangent(t, name)


def _table(t, shape, dtype, name):
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise RuntimeFailure("%s must be a contiguous %s tensor of shape %s" % (name, dtype, list(shape)))
    _no_tangent(t, name)


def _order(order):
    slot, source = order.slot, order.source
    if slot.dtype != torch.int32 or slot.dim() != 2 or not slot.is_contiguous() or \
            source.dtype != torch.int32 or source.dim() != 1 or not source.is_contiguous():
        raise RuntimeFailure("an order holds contiguous int32 slot [tokens, k] and source [rows]")
    if not 1 <= slot.size(1) <= MAX_CHOICES or max(slot.numel(), source.numel()) > _INT_MAX:
        raise RuntimeFailure("an order has 1 to %d choices, and fewer than 2^31 assignments and rows" % MAX_CHOICES)
    return slot, source


def _on_gpu(first, *others):
    if not first.is_cuda:
        raise RuntimeFailure("the expert operators need CUDA tensors")
    for t in others:
        if t is not None and t.device != first.device:
            raise RuntimeFailure("the tensors are on different devices")


def _result(out, rows, like, name, columns=None):
    """Refuse an ``out`` that is not the result's shape and dtype, whose rows overlap each other, or that autograd
    follows."""
    if out is None:
        return
    columns = like.size(1) if columns is None else columns
    if tuple(out.shape) != (rows, columns) or out.dtype != like.dtype:
        raise RuntimeFailure("%s must be [%d, %d] of %s" % (name, rows, columns, like.dtype))
    if (columns > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < columns):
        raise RuntimeFailure("%s must have contiguous rows that do not overlap" % name)
    if out.requires_grad and torch.is_grad_enabled():
        raise RuntimeFailure("%s requires a gradient, which a call that writes into it would lose" % name)


def _extent(t):
    """``(address, bytes of a row, bytes between rows, rows)``; a contiguous tensor of other dimensions is one row."""
    size = t.element_size()
    if not t.numel():
        return t.data_ptr(), 0, 0, 0
    if t.dim() != 2:
        return t.data_ptr(), t.numel() * size, 0, 1
    return t.data_ptr(), t.size(1) * size, t.stride(0) * size, t.size(0)


def _meet(a, b) -> bool:
    """Whether two extents may share a byte.  Column ranges of one matrix lie in one span of memory without meeting:
    with one pitch, what counts is the distance of the first columns within it.  Different pitches are compared by
    their spans."""
    (a_lo, a_width, a_pitch, a_rows), (b_lo, b_width, b_pitch, b_rows) = a, b
    if not a_rows or not b_rows:
        return False
    if a_lo + (a_rows - 1) * a_pitch + a_width <= b_lo or b_lo + (b_rows - 1) * b_pitch + b_width <= a_lo:
        return False
    pitch = a_pitch if a_rows > 1 else b_pitch
    if (b_rows > 1 and b_pitch != pitch) or a_rows == b_rows == 1 or pitch < max(a_width, b_width):
        return True
    between = (b_lo - a_lo) % pitch
    return between < a_width or between + b_width > pitch


def _apart(out, name, *inputs):
    if out is not None and any(_meet(_extent(out), _extent(t)) for t in inputs if t is not None):
        raise RuntimeFailure("%s overlaps an input" % name)


def _learns() -> bool:
    """Whether an input that requires a gradient is recorded by autograd."""
    if not torch.is_grad_enabled():
        return False
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeFailure("autograd under graph capture: capture the plain calls (detached inputs and the "
                             "*_backward functions) instead")
    return True


def _no_out(out):
    if out is not None:
        raise RuntimeFailure("out= cannot be used with inputs that require gradients")


def _rows_of(grad):
    """A gradient from autograd as a matrix of contiguous rows (it may be expanded or transposed)."""
    return grad if grad.size(1) <= 1 or grad.stride(1) == 1 else grad.contiguous()


# -- router -----------------------------------------------------------------------------------------------

def _check_route(logits, k):
    _matrix(logits, "logits")
    if not 1 <= logits.size(1) <= MAX_EXPERTS:
        raise RuntimeFailure("logits must cover 1 to %d experts" % MAX_EXPERTS)
    if not 1 <= k <= min(MAX_CHOICES, logits.size(1)):
        raise RuntimeFailure("k must be 1 to min(%d, experts)" % MAX_CHOICES)
    if logits.size(0) * logits.size(1) > 2 ** 40 or logits.size(0) * k > _INT_MAX:
        raise RuntimeFailure("more than 2^31 - 1 assignments")
    _on_gpu(logits)


def route(logits: torch.Tensor, k: int, *, renormalize: bool = True):
    """``(ids, weights)``, int32 and float32 [tokens, k]: each token's ``k`` largest logits, the largest first
    (ties to the lower expert), and their weights: the softmax over the chosen logits, or with
    ``renormalize=False`` their share of the softmax over all.

    A logit of -inf takes its expert out: a token with fewer than ``k`` experts left gets id -1 and weight 0 for
    the rest.  A NaN logit is never chosen and makes the weights of its token NaN, and so does +inf, which is.
    """
    if logits.requires_grad and _learns():
        return _Route.apply(logits, k, renormalize)
    return _call("route", lambda: _check_route(logits, k), logits, k, renormalize)


def route_backward(logits, ids, weights, grad_weights, *, renormalize: bool = True) -> torch.Tensor:
    """Gradient of ``route``'s weights with respect to ``logits`` [tokens, experts], in the logits' dtype."""
    def check():
        shape = (logits.size(0) if logits.dim() else 0, ids.size(-1) if ids.dim() else 0)
        _table(ids, shape, torch.int32, "ids")
        _table(weights, shape, torch.float32, "weights")
        _table(grad_weights, shape, torch.float32, "grad_weights")
        _check_route(logits, shape[1])
        _on_gpu(logits, ids, weights, grad_weights)
    return _call("route_backward", check, logits, ids, weights, grad_weights, renormalize)


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, renormalize):
        ids, weights = _call("route", lambda: _check_route(logits, k), logits, k, renormalize)
        ctx.renormalize = renormalize
        ctx.save_for_backward(logits, ids, weights)
        ctx.mark_non_differentiable(ids)
        return ids, weights

    @staticmethod
    @once_differentiable
    def backward(ctx, _, grad):
        return route_backward(*ctx.saved_tensors, grad.contiguous(), renormalize=ctx.renormalize), None, None


# -- sort, dispatch, combine ------------------------------------------------------------------------------

def sort_by_expert(ids: torch.Tensor, experts: int, *, capacity: int | None = None) -> ExpertOrder:
    """Rows for the assignments ``ids`` [tokens, k] (int32 or int64), grouped by expert and, within an expert, in
    the order of the assignments.

    Without ``capacity`` every assignment has a row: ``tokens * k`` rows, expert after expert without gaps.  With
    it expert ``e`` owns the rows ``e * capacity ... (e + 1) * capacity - 1`` and assignments beyond them have
    none.  An id outside ``[0, experts)`` (-1 for a padded token) has no row.
    """
    def check():
        if ids.dim() != 2 or ids.dtype not in (torch.int32, torch.int64) or not ids.is_contiguous():
            raise RuntimeFailure("ids must be a contiguous int32 or int64 tensor [tokens, k]")
        if not 1 <= experts <= MAX_EXPERTS:
            raise RuntimeFailure("1 to %d experts" % MAX_EXPERTS)
        if capacity is not None and capacity < 1:
            raise RuntimeFailure("a capacity is at least one row per expert")
        if ids.size(1) < 1 or ids.size(1) > MAX_CHOICES:
            raise RuntimeFailure("1 to %d choices per token" % MAX_CHOICES)
        if ids.numel() > _INT_MAX or experts * (capacity or 0) > _INT_MAX:
            raise RuntimeFailure("more than 2^31 - 1 assignments or rows")
    # a capacity of 0 would mean none to the native call
    return ExpertOrder(*_call("sort_by_expert", check, ids, experts, 0 if capacity is None else capacity or -1))


def _check_dispatch(x, order, out, name):
    slot, source = _order(order)
    _matrix(x, name)
    if x.size(0) != slot.size(0):
        raise RuntimeFailure("%s has %d tokens, the order %d" % (name, x.size(0), slot.size(0)))
    _result(out, source.numel(), x, "out")
    _apart(out, "out", x, slot, source)
    _on_gpu(x, slot, source, out)


def _check_combine(rows, weights, order, out, name):
    slot, source = _order(order)
    _matrix(rows, name)
    if rows.size(0) != source.numel():
        raise RuntimeFailure("%s has %d rows, the order %d" % (name, rows.size(0), source.numel()))
    if weights is not None:
        _table(weights, slot.shape, torch.float32, "weights")
    _result(out, slot.size(0), rows, "out")
    _apart(out, "out", rows, slot, source, weights)
    _on_gpu(rows, slot, source, weights, out)


def dispatch(x: torch.Tensor, order: ExpertOrder, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """``rows[r] = x[token of row r]`` [rows, hidden]; a row without an assignment is zero."""
    if x.requires_grad and _learns():
        _no_out(out)
        return _Dispatch.apply(x, order)
    return _call("dispatch", lambda: _check_dispatch(x, order, out, "x"), x, order.slot, order.source, out)


def dispatch_backward(grad_rows: torch.Tensor, order: ExpertOrder, *, out: torch.Tensor | None = None):
    """Gradient of :func:`dispatch` with respect to ``x``: the sum of each token's rows, in fp32, rounded once."""
    return _call("combine", lambda: _check_combine(grad_rows, None, order, out, "grad_rows"), grad_rows, None,
                 order.slot, order.source, out)


def combine(rows: torch.Tensor, weights: torch.Tensor, order: ExpertOrder, *, out: torch.Tensor | None = None):
    """``out[t] = sum over j of weights[t, j] * rows[slot[t, j]]`` [tokens, hidden], summed in fp32 in the order of
    the choices and rounded once.  An assignment without a row adds nothing, whatever its weight; ``weights`` is
    float32 [tokens, k]."""
    if (rows.requires_grad or weights.requires_grad) and _learns():
        _no_out(out)
        return _Combine.apply(rows, weights, order)
    return _call("combine", lambda: _check_combine(rows, weights, order, out, "rows"), rows, weights, order.slot,
                 order.source, out)


def combine_backward(grad_out, rows, weights, order: ExpertOrder, *, out: torch.Tensor | None = None):
    """``(grad_rows, grad_weights)`` of :func:`combine`: ``w * grad_out[t]`` at each assignment's row (zero in rows
    without one; written to ``out`` where given) and the fp32 products ``<grad_out[t], rows[slot]>``, zero where an
    assignment has no row."""
    def check():
        _order(order)
        _matrix(grad_out, "grad_out")
        _matrix(rows, "rows")
        if tuple(rows.shape) != (order.source.numel(), grad_out.size(1)) or rows.dtype != grad_out.dtype:
            raise RuntimeFailure("rows must be [%d, %d] of %s" % (order.source.numel(), grad_out.size(1), grad_out.dtype))
        _table(weights, order.slot.shape, torch.float32, "weights")
        _apart(out, "out", rows, weights)
        _check_dispatch(grad_out, order, out, "grad_out")
        _on_gpu(grad_out, rows, weights)
    return _call("combine_backward", check, grad_out, rows, weights, order.slot, order.source, out)


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order):
        rows = dispatch(x.detach(), order)
        ctx.save_for_backward(order.slot, order.source)
        return rows

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return dispatch_backward(_rows_of(grad), ExpertOrder(*ctx.saved_tensors, None, None)), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, order):
        out = combine(rows.detach(), weights.detach(), order)
        ctx.save_for_backward(rows, weights, order.slot, order.source)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        rows, weights, slot, source = ctx.saved_tensors
        return *combine_backward(_rows_of(grad), rows, weights, ExpertOrder(slot, source, None, None)), None


# -- 4-bit products ---------------------------------------------------------------------------------------

def quantize_int4(weight: torch.Tensor, group: int = 128, *, scale_dtype: torch.dtype | None = None):
    """``(packed, scales)`` of a weight [..., n, inner]: uint8 [..., n, inner / 2] and [..., n, inner / group].

    Value ``k`` of a row is ``(q - 8) * scale``: two 4-bit ``q`` a byte, the even ``k`` in the low half.  The scale of
    a group, its largest magnitude / 7, is rounded to ``scale_dtype`` (the weight's by default) before the values
    are, so its rounding moves the grid and adds no error of its own but to a largest magnitude that it leaves
    beyond 7 steps, which is clamped.  A scale that would round to 0 is the smallest positive value instead (1 in a
    group of zeros); one beyond the range of ``scale_dtype`` is refused.  Weights must be finite.  Done once when they
    are loaded.
    """
    if weight.dim() < 2 or weight.dtype not in _DTYPES:
        raise RuntimeFailure("a weight is [..., n, inner] of float32, bfloat16 or float16")
    if group not in INT4_GROUPS or weight.size(-1) % group or not weight.size(-1):
        raise RuntimeFailure("groups of 32, 64 or 128 that divide the inner size")
    dtype = weight.dtype if scale_dtype is None else scale_dtype
    if dtype not in _DTYPES:
        raise RuntimeFailure("scales are float32, bfloat16 or float16")
    w = weight.detach().float().unflatten(-1, (-1, group))
    if not bool(torch.isfinite(w).all()):
        raise RuntimeFailure("a weight to quantize holds infinities or NaN")
    largest = w.abs().amax(-1)
    scales = (largest / 7.0).to(dtype)
    if not bool(torch.isfinite(scales).all()):
        raise RuntimeFailure("a group's largest magnitude / 7 is beyond the range of %s scales" % dtype)
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps     # the smallest subnormal
    scales = torch.where(scales == 0, torch.full_like(scales, least).masked_fill_(largest == 0, 1.0), scales)
    q = (torch.round(w / scales.float()[..., None]).clamp_(-8, 7) + 8).to(torch.uint8).flatten(-2)
    return (q[..., 0::2] | (q[..., 1::2] << 4)).contiguous(), scales.contiguous()


def _check_product(rows, starts, counts, packed, scales, out):
    _matrix(rows, "rows")
    if rows.dtype == torch.float32:
        raise RuntimeFailure("rows must be bfloat16 or float16")
    if packed.dim() != 3 or packed.dtype != torch.uint8 or not packed.is_contiguous() or not packed.size(0) \
            or packed.size(2) * 2 != rows.size(1):
        raise RuntimeFailure("packed must be a contiguous uint8 tensor [experts, n, inner / 2]")
    if scales.dim() != 3 or scales.shape[:2] != packed.shape[:2] or not scales.is_contiguous() or \
            scales.dtype not in (torch.float32, rows.dtype):
        raise RuntimeFailure("scales must be a contiguous tensor [experts, n, inner / group] of the rows' dtype or float32")
    if not scales.size(2) or rows.size(1) % scales.size(2) or rows.size(1) // scales.size(2) not in INT4_GROUPS:
        raise RuntimeFailure("groups of 32, 64 or 128 that divide the inner size")
    _no_tangent(scales, "scales")
    segments = starts.numel()
    if not 1 <= segments <= MAX_EXPERTS or segments % packed.size(0):
        raise RuntimeFailure("1 to %d segments, a multiple of the experts" % MAX_EXPERTS)
    _table(starts, (segments,), torch.int32, "starts")
    _table(counts, (segments,), torch.int32, "counts")
    if rows.size(0) > _INT_MAX or packed.size(0) * packed.size(1) > _INT_MAX or rows.size(1) > _INT_MAX:
        raise RuntimeFailure("more than 2^31 - 1 rows, weight rows or inner values")
    if packed.data_ptr() % 16:
        raise RuntimeFailure("packed must start on a 16-byte boundary")
    if rows.requires_grad and torch.is_grad_enabled():
        raise RuntimeFailure("4-bit products have no gradient: detach the rows")
    _result(out, rows.size(0), rows, "out", packed.size(1))
    _apart(out, "out", rows, starts, counts, packed, scales)
    _on_gpu(rows, starts, counts, packed, scales, out)


def expert_matmul_int4(rows: torch.Tensor, starts: torch.Tensor, counts: torch.Tensor, packed: torch.Tensor,
                       scales: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[r] = W[e] @ rows[r]`` [rows, n] for the rows ``starts[s] ... starts[s] + counts[s] - 1`` of every
    segment ``s``, whose expert is ``e = s % experts``; a row no segment covers is zero.

    ``rows`` [rows, inner] is bfloat16 or float16; ``starts`` and ``counts`` int32 [segments] (an order's, or one
    segment per source rank and expert after an AllToAll), a multiple of the experts, at most 1024, in any order but
    without overlap (segments that share rows leave every row of the result undefined); ``packed`` uint8
    [experts, n, inner / 2] and ``scales`` [experts, n, inner / group] of the rows' dtype or float32, as
    :func:`quantize_int4` gives them, in groups of 32, 64 or 128.  Products and sums are fp32, rounded once.  No
    gradients: 4-bit weights are for serving.  The kernel's waits are bounded: outputs whose weights did not arrive
    within a second of the GPU's timer are NaN, and :func:`check_status` says so.
    """
    return _call("int4_product", lambda: _check_product(rows, starts, counts, packed, scales, out), rows, starts, counts,
                 packed, scales, out, _GIVE_UP)


def check_status() -> None:
    """Raise when a 4-bit product on the current GPU gave up waiting for its weights since the last check.  It waits
    for all streams of that GPU, so it is refused while the current stream is being captured; other GPUs have their
    own status."""
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeFailure("check_status waits for the GPU and cannot be called under graph capture")
    if _mod().int4_late_copies():
        raise RuntimeFailure("a 4-bit product's copy of weights did not arrive in time; its outputs are NaN")
