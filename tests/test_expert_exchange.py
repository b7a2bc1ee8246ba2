"""Expert-parallel token exchange: one rank through the engine, two ranks as threads that exchange host-side."""
import threading
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")

from vericcl_b200.errors import RuntimeFailure                    # noqa: E402
from vericcl_b200.models import ExpertExchange                    # noqa: E402
from vericcl_b200.ops import experts as ex                        # noqa: E402


def test_refusals():
    engine = SimpleNamespace(comm=SimpleNamespace(world=2))
    good = dict(experts=4, hidden=8, capacity=2, dtype=torch.bfloat16)
    for change in (dict(experts=3), dict(experts=0), dict(experts=2048), dict(hidden=0), dict(capacity=0),
                   dict(capacity=1 << 30), dict(dtype=torch.float64), dict(hidden=3, capacity=1)):
        with pytest.raises(RuntimeFailure):
            ExpertExchange(engine, **{**good, **change})


def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def tokens_for(rank, tokens, experts, k, hidden, dtype):
    g = torch.Generator(device="cuda").manual_seed(100 + rank)
    x = torch.randn(tokens, hidden, device="cuda", generator=g).to(dtype)
    logits = torch.randn(tokens, experts, device="cuda", generator=g)
    grad = torch.randn(tokens, hidden, device="cuda", generator=g).to(dtype)
    return x, logits, grad


def layer(exchange, x, logits, grad, k, scale):
    """A mixture whose expert e multiplies its rows with scale[e]; forward and backward."""
    ids, w = ex.route(logits, k)
    rows = exchange.dispatch(x, ids)
    per_row = scale.repeat_interleave(exchange.capacity).repeat(exchange.comm.world)[:, None].to(x.dtype)
    out = exchange.combine(rows * per_row, w)
    grad_rows, grad_w = exchange.combine_backward(grad, w)
    grad_x = exchange.dispatch_backward(grad_rows * per_row)
    return [t.clone() for t in (out, grad_x, grad_w, ids, exchange.counts, exchange.order.slot)]


def plain_layer(x, logits, grad, k, scale, capacity):
    """The same on one rank's tokens without any exchange, in 64 bits; powers of two as scales keep rows exact."""
    ids, w = ex.route(logits, k)
    order = ex.sort_by_expert(ids, scale.numel(), capacity=capacity)
    kept = (order.slot >= 0).double()
    factor = scale.double()[ids.long()] * kept
    out = (x.double()[:, None] * (factor * w.double())[..., None]).sum(1)
    grad_x = (grad.double()[:, None] * (factor * w.double())[..., None]).sum(1)
    grad_w = (grad.double()[:, None] * x.double()[:, None] * factor[..., None]).sum(2)
    return out, grad_x, grad_w


def compare(got, want, x, grad, scale, dtype):
    half = torch.finfo(dtype).eps / 2
    k, hidden, top = got[3].size(1), x.size(1), scale.abs().max().item()
    fp32 = (2 * k + 2) * 2.0 ** -24
    # out: one rounding of sums of at most k products of magnitude |x| top (weights sum to at most 1)
    assert bool(((got[0].double() - want[0]).abs() <= half * want[0].abs() + fp32 * x.abs().max().double() * top).all())
    # grad_x: w * grad is rounded once per row before the k rows are added, then once more
    bound = (half * 2.01 + fp32) * grad.abs().max().double() * top
    assert bool(((got[1].double() - want[1]).abs() <= bound).all())
    size = (grad.double().abs() * x.double().abs()).sum(1, keepdim=True) * top
    assert bool(((got[2].double() - want[2]).abs() <= (hidden + 1) * 2.0 ** -24 * size).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_rank(dtype):
    gpu()
    from vericcl_b200.models import CollectiveEngine
    from vericcl_b200.parallel import Communicator
    comm = Communicator(heap_bytes=64 << 20)
    try:
        exchange = ExpertExchange(CollectiveEngine(comm), experts=6, hidden=72, capacity=9, dtype=dtype)
        with pytest.raises(RuntimeFailure, match="first"):
            exchange.combine(torch.zeros(54, 72, dtype=dtype, device="cuda"), torch.zeros(1, 1, device="cuda"))
        scale = torch.tensor([1.0, 2, 0.5, -1, 4, -0.25], device="cuda")
        for tokens in (25, 1, 0):
            x, logits, grad = tokens_for(0, tokens, 6, 2, 72, dtype)
            if tokens:
                compare(layer(exchange, x, logits, grad, 2, scale), plain_layer(x, logits, grad, 2, scale, 9), x, grad,
                        scale, dtype)
            else:
                rows = exchange.dispatch(x, torch.zeros(0, 2, dtype=torch.int32, device="cuda"))
                assert bool((rows == 0).all()) and int(exchange.counts.sum()) == 0
        with pytest.raises(RuntimeFailure):
            exchange.dispatch(x[:, :8], torch.zeros(0, 2, dtype=torch.int32, device="cuda"))
        used = comm.heap.used()
        exchange.close()
        assert comm.heap.used() < used
    finally:
        comm.close()


class Threads:
    """Two ranks' AllToAll as copies between two barriers: nothing on the GPU waits."""

    def __init__(self, world):
        self.world, self.gate, self.parts = world, threading.Barrier(world, timeout=60), {}

    def engine(self, rank):
        comm = SimpleNamespace(world=self.world, rank=rank, device=0, free=lambda t: None,
                               empty=lambda n, dtype=torch.float32: torch.empty(n, dtype=dtype, device="cuda"))

        def all_to_all(inp, out):
            torch.cuda.synchronize()
            self.parts[rank] = inp.reshape(self.world, -1)
            self.gate.wait()
            for r in range(self.world):
                out.view(self.world, -1)[r].copy_(self.parts[r][rank])
            torch.cuda.synchronize()
            self.gate.wait()
        return SimpleNamespace(comm=comm, all_to_all=all_to_all)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_two_ranks(dtype):
    gpu()
    world, experts, k, hidden, capacity = 2, 6, 2, 64, 5
    scale = torch.tensor([1.0, 2, 0.5, -1, 4, -0.25], device="cuda")
    links, results, errors = Threads(world), {}, []

    def rank_main(rank):
        try:
            exchange = ExpertExchange(links.engine(rank), experts=experts, hidden=hidden, capacity=capacity, dtype=dtype)
            x, logits, grad = tokens_for(rank, 17 + rank, experts, k, hidden, dtype)
            local = scale[rank * 3:rank * 3 + 3]
            results[rank] = layer(exchange, x, logits, grad, k, local)
        except Exception as error:                               # noqa: BLE001  (reported by the test)
            errors.append(error)
            links.gate.abort()

    threads = [threading.Thread(target=rank_main, args=(r,)) for r in range(world)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for rank in range(world):
        x, logits, grad = tokens_for(rank, 17 + rank, experts, k, hidden, dtype)
        compare(results[rank], plain_layer(x, logits, grad, k, scale, capacity), x, grad, scale, dtype)
        # the counts a rank holds are those of its experts, by source rank
        want = []
        for source in range(world):
            slot = results[source][5]
            ids = results[source][3]
            want += [int(((ids == e) & (slot >= 0)).sum()) for e in range(rank * 3, rank * 3 + 3)]
        assert results[rank][4].tolist() == want


@pytest.mark.gpu
def test_int4_products_of_exchanged_rows():
    gpu()
    world, experts, hidden, capacity = 2, 4, 64, 3
    links, results, errors = Threads(world), {}, []
    g = torch.Generator(device="cuda").manual_seed(7)
    packed, scales = ex.quantize_int4(torch.randn(experts, hidden, hidden, device="cuda", generator=g).bfloat16(), 32)

    def rank_main(rank):
        try:
            exchange = ExpertExchange(links.engine(rank), experts=experts, hidden=hidden, capacity=capacity)
            x, logits, _ = tokens_for(rank, 4, experts, 1, hidden, torch.bfloat16)
            ids, w = ex.route(logits, 1)
            mine = slice(rank * 2, rank * 2 + 2)
            rows = exchange.dispatch(x, ids)
            out = exchange.combine(exchange.matmul_int4(rows, packed[mine].contiguous(), scales[mine].contiguous()), w)
            with pytest.raises(RuntimeFailure):
                exchange.matmul_int4(rows, packed, scales)
            results[rank] = (out.clone(), ids.clone(), exchange.order.slot.clone(), x)
        except Exception as error:                               # noqa: BLE001  (reported by the test)
            errors.append(error)
            links.gate.abort()

    threads = [threading.Thread(target=rank_main, args=(r,)) for r in range(world)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    q = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).double() - 8
    dense = (q.unflatten(-1, (-1, 32)) * scales.double()[..., None]).flatten(-2)
    for out, ids, slot, x in results.values():
        for t in range(4):
            want = dense[ids[t, 0]] @ x[t].double() if slot[t, 0] >= 0 else torch.zeros(hidden, dtype=torch.float64,
                                                                                       device="cuda")
            # one weight (1.0), one rounding of the product; fp32 sums of 64 terms
            size = dense[ids[t, 0]].abs() @ x[t].double().abs()
            assert bool(((out[t].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -15 * size).all())


def alone(**kwargs):
    """An exchange of one rank without a communicator's heap."""
    comm = SimpleNamespace(world=1, rank=0, device=0, free=lambda t: None,
                           empty=lambda n, dtype=torch.float32: torch.empty(n, dtype=dtype, device="cuda"))
    return ExpertExchange(SimpleNamespace(comm=comm), **kwargs)


@pytest.mark.gpu
def test_gradients_of_another_dispatch_are_refused():
    gpu()
    exchange = alone(experts=4, hidden=16, capacity=8, dtype=torch.float32)
    x, logits, grad = tokens_for(0, 6, 4, 2, 16, torch.float32)
    ids, w = ex.route(logits, 2)
    other = (ids + 1) % 4

    def forward(choices):
        rows = exchange.dispatch(x, choices)
        return exchange.combine(rows * 2, w)

    forward(ids)
    want_rows, want_w = (t.clone() for t in exchange.combine_backward(grad, w))
    want_x = exchange.dispatch_backward(want_rows * 2)
    # a dispatch between combine and its gradient
    exchange.dispatch(x, other)
    with pytest.raises(RuntimeFailure, match="combine"):
        exchange.combine_backward(grad, w)
    # between the gradient of combine and that of dispatch
    forward(ids)
    grad_rows = exchange.combine_backward(grad, w)[0].clone()
    exchange.dispatch(x, other)
    with pytest.raises(RuntimeFailure, match="dispatch"):
        exchange.dispatch_backward(grad_rows * 2)
    # the next step has its own
    forward(other)
    exchange.combine_backward(grad, w)
    forward(ids)
    got_rows, got_w = exchange.combine_backward(grad, w)
    assert torch.equal(got_rows, want_rows) and torch.equal(got_w, want_w)
    assert torch.equal(exchange.dispatch_backward(got_rows * 2), want_x)
    # without a combine, the gradient of dispatch is that of the last one
    exchange.dispatch(x, other)
    direct = exchange.dispatch_backward(torch.ones(32, 16, device="cuda"))
    assert torch.equal(direct, (exchange.order.slot >= 0).sum(1, keepdim=True).float().expand(6, 16))


@pytest.mark.gpu
def test_a_refused_call_leaves_the_exchange_as_it_was():
    gpu()
    exchange = alone(experts=4, hidden=16, capacity=8, dtype=torch.float32)
    x, logits, grad = tokens_for(0, 6, 4, 2, 16, torch.float32)
    ids, w = ex.route(logits, 2)
    rows = exchange.dispatch(x, ids)
    out = exchange.combine(rows * 2, w)
    want = exchange.combine_backward(grad, w)[1]
    with pytest.raises(RuntimeFailure):
        exchange.dispatch(x, ids[:5])                             # choices of fewer tokens
    assert torch.equal(exchange.combine_backward(grad, w)[1], want)
    assert torch.equal(exchange.combine(rows * 2, w), out)
    with pytest.raises(RuntimeFailure):
        exchange.combine(rows * 3, w[:5])
    with pytest.raises(RuntimeFailure, match="combine"):          # that combine did not finish, and its rows are gone
        exchange.combine_backward(grad, w)


@pytest.mark.gpu
@pytest.mark.parametrize("world", [1, 2])
def test_autograd_sees_that_rows_were_overwritten(world):
    """Rows that a learnable expert's graph has saved: its backward pass works until the next dispatch overwrites them."""
    gpu()
    links, errors = Threads(world), []

    def rank_main(rank):
        try:
            engine = links.engine(rank)
            copy = engine.all_to_all
            engine.all_to_all = lambda inp, out: copy(inp, out.data)          # as a kernel writes: unseen by autograd
            exchange = ExpertExchange(engine, experts=4, hidden=16, capacity=8, dtype=torch.float32)
            x, logits, grad = tokens_for(rank, 6, 4, 2, 16, torch.float32)
            ids, w = ex.route(logits, 2)
            expert = torch.ones(16, device="cuda", requires_grad=True)
            rows = exchange.dispatch(x, ids)
            y = rows * expert
            exchange.combine(y, w)
            grad_rows, _ = exchange.combine_backward(grad, w)
            exchange.dispatch_backward(grad_rows)
            parts = grad_rows.double() * rows.double()
            y.backward(grad_rows)
            # products and sums of the rows: as many roundings as there are rows, and one for the product
            bound = (rows.size(0) + 1) * 2.0 ** -24 * parts.abs().sum(0)
            assert bool(((expert.grad.double() - parts.sum(0)).abs() <= bound).all())
            y = exchange.dispatch(x, ids) * expert
            z = exchange.combine(y, w) * expert                   # rows that came back to the tokens
            exchange.dispatch(x, ids)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward(grad_rows)
            z.backward(grad)
        except BaseException as error:                           # noqa: BLE001  (reported by the test; pytest's own too)
            errors.append(error)
            links.gate.abort()

    threads = [threading.Thread(target=rank_main, args=(r,)) for r in range(world)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.gpu
def test_explicit_gradients_are_handed_on_by_the_caller():
    """Inputs that require gradients: the exchange records nothing, and its gradients reach the leaves through backward
    calls of the caller, as autograd's own through the operators do."""
    gpu()
    exchange = alone(experts=4, hidden=16, capacity=8, dtype=torch.float32)
    base, logits, grad = tokens_for(0, 6, 4, 2, 16, torch.float32)
    x, l = (t.requires_grad_() for t in (base, logits))
    tokens = x * 3                                                # an activation, no leaf
    ids, w = ex.route(l, 2)
    rows = exchange.dispatch(tokens, ids)
    out = exchange.combine(rows * 2, w)
    assert w.requires_grad and not rows.requires_grad and not out.requires_grad
    grad_rows, grad_w = exchange.combine_backward(grad, w)
    tokens.backward(exchange.dispatch_backward(grad_rows * 2))
    w.backward(grad_w)
    x2, l2 = (t.detach().clone().requires_grad_() for t in (x, l))
    ids2, w2 = ex.route(l2, 2)
    order = ex.sort_by_expert(ids2, 4, capacity=8)
    want = ex.combine(ex.dispatch(x2 * 3, order) * 2, w2, order)
    want.backward(grad)
    assert torch.equal(out, want) and torch.equal(x.grad, x2.grad) and torch.equal(l.grad, l2.grad)


@pytest.mark.gpu
def test_products_of_another_number_of_experts_and_foreign_rows_are_refused():
    gpu()
    exchange = alone(experts=4, hidden=64, capacity=3)
    x, logits, _ = tokens_for(0, 4, 4, 1, 64, torch.bfloat16)
    ids, w = ex.route(logits, 1)
    packed, scales = ex.quantize_int4(torch.ones(5, 64, 64, device="cuda").bfloat16(), 32)
    with pytest.raises(RuntimeFailure, match="first"):
        exchange.matmul_int4(x, packed[:4], scales[:4])
    rows = exchange.dispatch(x, ids)
    for count in (3, 5):
        with pytest.raises(RuntimeFailure, match="experts"):
            exchange.matmul_int4(rows, packed[:count], scales[:count])
    assert exchange.matmul_int4(rows, packed[:4], scales[:4]).shape == (12, 64)
    for wrong in (rows[:11], rows[:, :63], rows.float()):
        with pytest.raises(RuntimeFailure, match="rows"):
            exchange.combine(wrong, w)
