"""Expert-parallel token exchange: tokens sorted to the experts of every rank, an AllToAll, and the way back.

``ExpertExchange`` puts the operators of :mod:`vericcl_b200.ops.experts` on both sides of
:meth:`CollectiveEngine.all_to_all`.  Experts are dealt to the ranks in order (rank ``r`` owns ``experts / world``
of them from ``r * experts / world`` on) and every source rank has ``capacity`` rows at every expert, the equal parts
an AllToAll exchanges.  The rows that ``dispatch`` and ``combine_backward`` send and what every exchange receives lie
in the communicator's heap and need no copy; rows that a caller brings (the experts' results, the gradient of the
dispatched rows) are first copied to a heap buffer of the engine, unless they lie in the heap themselves
(``comm.empty``).  One rank exchanges nothing and uses its rows in place.
"""
from __future__ import annotations

import torch

from vericcl_b200.errors import RuntimeFailure
from vericcl_b200.ops import experts as ops


class ExpertExchange:
    """The rows of one mixture layer.

    >>> exchange = ExpertExchange(engine, experts=64, hidden=4096, capacity=512)
    >>> ids, weights = ops.route(logits, 8)
    >>> rows = exchange.dispatch(x, ids)                  # [world * local * capacity, hidden], this rank's experts
    >>> y = exchange.matmul_int4(rows, *quantized)        # or any per-expert computation of the same rows
    >>> out = exchange.combine(y, weights)                # [tokens, hidden]

    Rows are ordered by (source rank, local expert, place); ``starts`` and ``counts`` say which of them hold tokens,
    the others are zero.  Rows that a call returns are the exchange's own buffers: they hold until the same call of
    this object runs again, so a layer whose backward pass is still to come keeps its own exchange (autograd refuses a
    graph whose saved rows were overwritten).  Calls run on the current stream, in the same order on every rank.

    Autograd stops here: no call records anything, results require no gradient whatever the inputs do, and
    :meth:`combine_backward` and :meth:`dispatch_backward` are the gradients, to be handed on by the caller
    (``weights.backward(grad_weights)``, ``x.backward(grad_x)``, or inside a ``torch.autograd.Function``).
    """

    def __init__(self, engine, *, experts: int, hidden: int, capacity: int, dtype: torch.dtype = torch.bfloat16):
        comm = engine.comm
        if experts < 1 or experts > ops.MAX_EXPERTS or experts % comm.world:
            raise RuntimeFailure("experts must be 1 to %d, a multiple of the world size" % ops.MAX_EXPERTS)
        if hidden < 1 or hidden > ops.MAX_COLUMNS or capacity < 1 or experts * capacity > 2 ** 31 - 1:
            raise RuntimeFailure("hidden and capacity must be positive, and the rows fewer than 2^31")
        if dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise RuntimeFailure("rows are float32, bfloat16 or float16")
        self.local = experts // comm.world
        if comm.world > 1 and self.local * capacity * hidden * dtype.itemsize % 16:
            raise RuntimeFailure("a rank's part of the rows must be a multiple of 16 bytes")
        self.engine, self.comm = engine, comm
        self.experts, self.hidden, self.capacity, self.dtype = experts, hidden, capacity, dtype
        self.rows = experts * capacity
        self.order = None
        self._returned = None        # rows of the last combine, until another dispatch
        self._grad_of = None         # the order of a combine gradient whose dispatch gradient is to come
        self._heap: dict = {}
        segments = torch.arange(experts, dtype=torch.int32, device=torch.device("cuda", comm.device))
        self.starts = segments * capacity
        self.counts = torch.zeros_like(segments)

    def _buffer(self, name: str) -> torch.Tensor:
        """A heap matrix of all rows, allocated on first use (every rank makes the same calls in the same order)."""
        buf = self._heap.get(name)
        if buf is None:
            buf = self._heap[name] = self.comm.empty(self.rows * self.hidden, self.dtype)
        return buf.view(self.rows, self.hidden)

    def _check_rows(self, rows, name):
        if tuple(rows.shape) != (self.rows, self.hidden) or rows.dtype != self.dtype:
            raise RuntimeFailure("%s must be [%d, %d] of %s" % (name, self.rows, self.hidden, self.dtype))

    def _check_tokens(self, x, name):
        if x.dim() != 2 or x.size(1) != self.hidden or x.dtype != self.dtype:
            raise RuntimeFailure("%s must be [tokens, %d] of %s" % (name, self.hidden, self.dtype))

    def _dispatched(self):
        if self.order is None:
            raise RuntimeFailure("dispatch comes first")
        return self.order

    def _exchange(self, rows: torch.Tensor, name: str) -> torch.Tensor:
        if self.comm.world == 1:
            return rows
        out = self._buffer(name)
        self.engine.all_to_all(rows, out)
        torch.autograd.graph.increment_version(out)               # a graph that has saved these rows sees the write
        return out

    def _exchange_counts(self, counts: torch.Tensor) -> torch.Tensor:
        """Counts per (source rank, local expert); they travel as float32, exact up to a capacity of 2^24."""
        world = self.comm.world
        if world == 1:
            return counts
        pad = (self.local + 3) // 4 * 4                       # 16 bytes a rank
        bufs = self._heap.get("counts")
        if bufs is None:
            bufs = self._heap["counts"] = (self.comm.empty(world * pad), self.comm.empty(world * pad))
        mine, theirs = bufs
        mine.view(world, pad)[:, :self.local].copy_(counts.view(world, self.local))
        self.engine.all_to_all(mine, theirs)
        return theirs.view(world, pad)[:, :self.local].to(torch.int32).reshape(-1)

    def dispatch(self, x: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
        """Rows of this rank's experts from every rank's tokens ``x`` [tokens, hidden] and choices ``ids`` [tokens, k].

        Ranks may hold different numbers of tokens; a choice beyond an expert's ``capacity`` rows is dropped
        (``order.slot`` is -1 there).  The gradients of an earlier ``combine`` and dispatch end here."""
        self._check_tokens(x, "x")
        if self.comm.world > 1 and self.capacity > 1 << 24:
            raise RuntimeFailure("a capacity above 2^24 cannot be exchanged")
        order = ops.sort_by_expert(ids, self.experts, capacity=self.capacity)
        rows = ops.dispatch(x.detach(), order, out=self._buffer("sent"))
        self.order, self._returned = order, None
        self.counts = self._exchange_counts(self.order.counts)
        return self._exchange(rows, "received")

    def matmul_int4(self, rows: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, *, out=None) -> torch.Tensor:
        """The local experts' 4-bit products of dispatched rows (:func:`vericcl_b200.ops.experts.expert_matmul_int4`)."""
        self._dispatched()
        if packed.dim() != 3 or packed.size(0) != self.local:
            raise RuntimeFailure("packed must hold the %d experts of this rank" % self.local)
        return ops.expert_matmul_int4(rows, self.starts, self.counts, packed, scales, out=out)

    def combine(self, rows: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        """``out`` [tokens, hidden]: the experts' rows back at their tokens, weighted with ``weights`` and summed."""
        order = self._dispatched()
        self._check_rows(rows, "rows")
        self._returned = None
        back = self._exchange(rows.detach(), "returned")
        out = ops.combine(back, weights.detach(), order)
        self._returned = back
        return out

    def combine_backward(self, grad_out: torch.Tensor, weights: torch.Tensor):
        """``(grad_rows, grad_weights)`` of the last :meth:`combine`: the gradient of this rank's expert rows and of
        its tokens' weights.  On one rank the rows given to ``combine`` must still hold."""
        order = self._dispatched()
        self._check_tokens(grad_out, "grad_out")
        if self._returned is None:
            raise RuntimeFailure("combine comes before its gradient, without another dispatch between them")
        grad, grad_weights = ops.combine_backward(grad_out, self._returned, weights.detach(), order,
                                                  out=self._buffer("grad_sent"))
        self._grad_of = order
        return self._exchange(grad, "grad_received"), grad_weights

    def dispatch_backward(self, grad_rows: torch.Tensor) -> torch.Tensor:
        """Gradient of the last :meth:`dispatch`'s ``x`` [tokens, hidden] from the gradient of its rows; refused when
        that dispatch came after the :meth:`combine_backward` whose rows' gradient is on its way."""
        order = self._dispatched()
        self._check_rows(grad_rows, "grad_rows")
        if self._grad_of is not None and self._grad_of is not order:
            raise RuntimeFailure("another dispatch came between the gradients of combine and dispatch")
        grad = ops.dispatch_backward(self._exchange(grad_rows, "grad_returned"), order)
        self._grad_of = None
        return grad

    def close(self) -> None:
        """Give the exchange's heap buffers back (none may be in flight); the engine keeps its copy buffers."""
        for buf in self._heap.values():
            for t in buf if isinstance(buf, tuple) else (buf,):
                self.comm.free(t)
        self._heap.clear()
        self.order = self._returned = self._grad_of = None
