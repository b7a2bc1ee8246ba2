"""Mixture-of-experts operators: refusals and weight layout (CPU), numerics against 64-bit references (GPU)."""
import math

import pytest

torch = pytest.importorskip("torch")

from vericcl_b200.errors import RuntimeFailure                    # noqa: E402
from vericcl_b200.ops import experts as ex                        # noqa: E402

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def close(got, want, magnitude, dtype, terms):
    """|got - want| <= one rounding of the result + the fp32 sum's error: ``terms`` roundings of at most 2^-24 of
    the sum of the terms' magnitudes (each of the products and partial sums is no larger), + the smallest
    subnormal step of ``dtype``."""
    err = (got.double() - want).abs()
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bound = half_step(dtype) * want.abs() + (1 + half_step(dtype)) * terms * 2.0 ** -24 * magnitude + tiny
    assert bool((err <= bound).all()), (err - bound).max().item()


# -- refusals (no GPU needed: every check runs before the device is touched) ---------------------------------

def _cpu_order(tokens=3, k=2, rows=6):
    return ex.ExpertOrder(torch.zeros(tokens, k, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32),
                          torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))


REFUSED = [
    lambda: ex.route(torch.zeros(3), 1),
    lambda: ex.route(torch.zeros(3, 4, dtype=torch.float64), 1),
    lambda: ex.route(torch.zeros(3, 4), 0),
    lambda: ex.route(torch.zeros(3, 4), 5),
    lambda: ex.route(torch.zeros(3, 2000), 2),
    lambda: ex.route(torch.zeros(3, 64), 33),
    lambda: ex.route(torch.zeros(4, 3).t(), 1),
    lambda: ex.route_backward(torch.zeros(3, 4), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2),
                              torch.zeros(3, 2)),
    lambda: ex.route_backward(torch.zeros(3, 4), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2),
                              torch.zeros(2, 2)),
    lambda: ex.sort_by_expert(torch.zeros(3, 2), 4),
    lambda: ex.sort_by_expert(torch.zeros(6, dtype=torch.int32), 4),
    lambda: ex.sort_by_expert(torch.zeros(2, 3, dtype=torch.int32).t(), 4),
    lambda: ex.sort_by_expert(torch.zeros(3, 2, dtype=torch.int32), 0),
    lambda: ex.sort_by_expert(torch.zeros(3, 2, dtype=torch.int32), 1025),
    lambda: ex.sort_by_expert(torch.zeros(3, 2, dtype=torch.int32), 4, capacity=0),
    lambda: ex.sort_by_expert(torch.zeros(3, 2, dtype=torch.int32), 1024, capacity=1 << 21),
    lambda: ex.sort_by_expert(torch.zeros(3, 0, dtype=torch.int32), 4),
    lambda: ex.sort_by_expert(torch.zeros(3, 33, dtype=torch.int32), 4),
    lambda: ex.dispatch(torch.zeros(4, 8), _cpu_order()),
    lambda: ex.dispatch(torch.zeros(3, 8, dtype=torch.int32), _cpu_order()),
    lambda: ex.dispatch(torch.zeros(8, 3).t(), _cpu_order()),
    lambda: ex.dispatch(torch.zeros(3, 8), _cpu_order(), out=torch.zeros(5, 8)),
    lambda: ex.dispatch(torch.zeros(3, 8), _cpu_order(), out=torch.zeros(6, 8, dtype=torch.float16)),
    lambda: ex.dispatch(torch.zeros(3, 8), _cpu_order(), out=torch.zeros(1, 8).expand(6, 8)),
    lambda: ex.dispatch(torch.zeros(3, 8), _cpu_order(k=33, rows=99)),
    lambda: ex.dispatch(torch.zeros(3, 8), _cpu_order(k=0)),
    lambda: ex.dispatch_backward(torch.zeros(5, 8), _cpu_order()),
    lambda: ex.combine(torch.zeros(5, 8), torch.zeros(3, 2), _cpu_order()),
    lambda: ex.combine(torch.zeros(6, 8), torch.zeros(3, 2, dtype=torch.bfloat16), _cpu_order()),
    lambda: ex.combine(torch.zeros(6, 8), torch.zeros(2, 3), _cpu_order()),
    lambda: ex.combine_backward(torch.zeros(3, 8), torch.zeros(6, 9), torch.zeros(3, 2), _cpu_order()),
    lambda: ex.combine_backward(torch.zeros(3, 8), torch.zeros(6, 8, dtype=torch.float16), torch.zeros(3, 2),
                                _cpu_order()),
    lambda: ex.quantize_int4(torch.zeros(8)),
    lambda: ex.quantize_int4(torch.zeros(8, 100), 32),
    lambda: ex.quantize_int4(torch.zeros(8, 96), 48),
    lambda: ex.quantize_int4(torch.full((8, 32), float("nan")), 32),
    lambda: ex.quantize_int4(torch.zeros(8, 128), 128, scale_dtype=torch.float64),
]


@pytest.mark.parametrize("call", REFUSED)
def test_refusals(call):
    with pytest.raises(RuntimeFailure):
        call()


@pytest.mark.gpu
def test_the_same_calls_are_refused_on_the_gpu():
    cuda()
    for call in REFUSED:
        with torch.device("cuda"), pytest.raises(RuntimeFailure):
            call()
    for change in PRODUCT_REFUSED:
        with pytest.raises(RuntimeFailure):
            # a view that starts off the 16-byte grid stays one
            ex.expert_matmul_int4(**{k: on_gpu(v) for k, v in _product_args(**change).items()})
    with pytest.raises(RuntimeFailure, match="different devices"):
        ex.dispatch(torch.zeros(3, 8, device="cuda"), _cpu_order())


def on_gpu(t):
    return t.detach().cuda().as_strided(t.shape, t.stride()).requires_grad_(t.requires_grad) if t.is_contiguous() and \
        t.storage_offset() == 0 else torch.empty(t.untyped_storage().nbytes() // t.element_size(), dtype=t.dtype,
                                                 device="cuda").as_strided(t.shape, t.stride(), t.storage_offset())


def _product_args(**change):
    args = dict(rows=torch.zeros(5, 128, dtype=torch.bfloat16), starts=torch.zeros(2, dtype=torch.int32),
                counts=torch.zeros(2, dtype=torch.int32), packed=torch.zeros(2, 7, 64, dtype=torch.uint8),
                scales=torch.zeros(2, 7, 1, dtype=torch.bfloat16))
    args.update(change)
    return args


PRODUCT_REFUSED = [
    dict(rows=torch.zeros(5, 128)), dict(rows=torch.zeros(5, 126, dtype=torch.bfloat16)),
    dict(rows=torch.zeros(128, 5, dtype=torch.bfloat16).t()),
    dict(starts=torch.zeros(3, dtype=torch.int32)), dict(starts=torch.zeros(2, dtype=torch.int64)),
    dict(counts=torch.zeros(4, dtype=torch.int32)),
    dict(starts=torch.zeros(3, dtype=torch.int32), counts=torch.zeros(3, dtype=torch.int32)),
    dict(starts=torch.zeros(0, dtype=torch.int32), counts=torch.zeros(0, dtype=torch.int32)),
    dict(starts=torch.zeros(1026, dtype=torch.int32), counts=torch.zeros(1026, dtype=torch.int32)),
    dict(packed=torch.zeros(2, 7, 64, dtype=torch.int8)), dict(packed=torch.zeros(2, 7, 63, dtype=torch.uint8)),
    dict(packed=torch.zeros(7, 2, 64, dtype=torch.uint8).transpose(0, 1)),
    dict(packed=torch.zeros(2 * 7 * 64 + 1, dtype=torch.uint8)[1:].view(2, 7, 64)),
    dict(scales=torch.zeros(2, 7, 1, dtype=torch.float16)), dict(scales=torch.zeros(2, 7, 3, dtype=torch.bfloat16)),
    dict(scales=torch.zeros(2, 7, 8, dtype=torch.bfloat16)), dict(scales=torch.zeros(2, 7, 0, dtype=torch.bfloat16)),
    dict(scales=torch.zeros(2, 8, 1, dtype=torch.bfloat16)),
    dict(rows=torch.zeros(5, 128, dtype=torch.bfloat16, requires_grad=True)),
    dict(out=torch.zeros(5, 8, dtype=torch.bfloat16)), dict(out=torch.zeros(5, 7, dtype=torch.float16)),
]


@pytest.mark.parametrize("change", PRODUCT_REFUSED)
def test_product_refusals(change):
    with pytest.raises(RuntimeFailure):
        ex.expert_matmul_int4(**_product_args(**change))


def test_cpu_tensors_are_refused():
    for call in (lambda: ex.route(torch.zeros(3, 4), 2),
                 lambda: ex.sort_by_expert(torch.zeros(3, 2, dtype=torch.int32), 4),
                 lambda: ex.dispatch(torch.zeros(3, 8), _cpu_order()),
                 lambda: ex.combine(torch.zeros(6, 8), torch.zeros(3, 2), _cpu_order()),
                 lambda: ex.expert_matmul_int4(**_product_args())):
        with pytest.raises(RuntimeFailure, match="CUDA"):
            call()


def dequantized(packed, scales, group):
    q = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).double() - 8
    return (q.unflatten(-1, (-1, group)) * scales.double()[..., None]).flatten(-2)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_int4_is_within_half_a_step(group, dtype):
    g = torch.Generator().manual_seed(group)
    w = torch.randn(3, 5, 256, generator=g).to(dtype)
    w[0, 0] = 0
    packed, scales = ex.quantize_int4(w, group)
    assert packed.shape == (3, 5, 128) and packed.dtype == torch.uint8
    assert scales.shape == (3, 5, 256 // group) and scales.dtype == dtype
    back = dequantized(packed, scales, group)
    step = scales.double().repeat_interleave(group, -1)
    # half a step, plus what the largest magnitudes lose when the rounded scale is below magnitude / 7, plus the
    # fp32 quotient's rounding (a quotient of up to 7 is off by 2^-24 relative)
    bound = step * (0.5 + 7 * (half_step(dtype) + 2.0 ** -22))
    assert bool(((back - w.double()).abs() <= bound).all())
    assert bool((back[0, 0] == 0).all())


# -- numerics -----------------------------------------------------------------------------------------------

def cuda(seed=0):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def reference_route(logits, k, renormalize):
    x = logits.double().cpu()
    ids = torch.full((x.size(0), k), -1, dtype=torch.int32)
    w = torch.zeros(x.size(0), k, dtype=torch.float64)
    for t in range(x.size(0)):
        row = x[t]
        order = sorted((e for e in range(len(row)) if row[e] > -math.inf), key=lambda e: (-row[e].item(), e))[:k]
        if not order:
            continue
        ids[t, :len(order)] = torch.tensor(order, dtype=torch.int32)
        chosen = row[order]
        total = chosen if renormalize else row[row > -math.inf]
        w[t, :len(order)] = torch.exp(chosen - row.max()) / torch.exp(total - row.max()).sum()
    return ids.cuda(), w.cuda()


# exp is within 2 units in the last place for arguments of any size (2^-22 relative), its argument's difference is
# rounded once (2^-24 of at most 2 max|l|), the sum adds log2(32) + 32 roundings and the quotient one
def route_bound(logits):
    fine = logits.double().masked_fill(~torch.isfinite(logits.double()), 0)
    return 2.0 ** -24 * (2 * 2 * fine.abs().max().item() + 2 * 4 + 40)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (1, 128, 8), (9, 5, 5), (17, 33, 2), (64, 257, 32), (7, 1024, 9)])
def test_route_matches_reference(dtype, renormalize, tokens, experts, k):
    g = cuda(tokens + experts)
    logits = normal(g, tokens, experts, dtype=dtype, scale=3.0)
    ids, w = ex.route(logits, k, renormalize=renormalize)
    want_ids, want = reference_route(logits, k, renormalize)
    assert torch.equal(ids, want_ids)
    assert bool(((w.double() - want).abs() <= route_bound(logits) * want + 1e-38).all())
    grad = normal(g, tokens, k)
    got = ex.route_backward(logits, ids, w, grad, renormalize=renormalize)
    inner = (want * grad.double()).sum(1, keepdim=True)
    if renormalize:
        expect = torch.zeros(tokens, experts, dtype=torch.float64, device="cuda")
        expect.scatter_(1, ids.long(), want * (grad.double() - inner))
    else:
        share = torch.softmax(logits.double(), 1)
        expect = share * (torch.zeros_like(share).scatter_(1, ids.long(), grad.double()) - inner)
    # each factor carries the weights' relative error, on magnitudes of at most w (|g| + sum w |g|)
    size = grad.abs().max().item() * 2
    bound = half_step(dtype) * expect.abs() + (4 * route_bound(logits) + 40 * 2.0 ** -24) * size * \
        torch.softmax(logits.double(), 1).clamp(min=0 if not renormalize else 1) + \
        torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert bool(((got.double() - expect).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_masks_ties_and_nan(renormalize):
    cuda()
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    logits = torch.tensor([[1.0, 1, 1, 1], [-inf, 2, -inf, -inf], [-inf] * 4, [low] * 4, [0.0, -0.0, -1, low],
                           [nan, 1, 2, 0], [5, low, -inf, low]], device="cuda")
    ids, w = ex.route(logits, 3, renormalize=renormalize)
    assert ids.tolist() == [[0, 1, 2], [1, -1, -1], [-1, -1, -1], [0, 1, 2], [0, 1, 2], [2, 1, 3], [0, 1, 3]]
    third, quarter = 1 / 3, 1 / 4
    each = third if renormalize else quarter
    assert torch.allclose(w[0], torch.full((3,), each, device="cuda"))
    assert w[1].tolist() == [1, 0, 0] and w[2].tolist() == [0, 0, 0]
    assert torch.allclose(w[3], torch.full((3,), each, device="cuda"))
    assert bool(w[5].isnan().all()) and w[6].tolist() == [1, 0, 0]
    grad = ex.route_backward(logits, ids, w, torch.ones_like(w), renormalize=renormalize)
    assert bool((grad[[1, 2]] == 0).all()) and bool(grad[[0, 3, 4, 6]].isfinite().all())


def reference_order(ids, experts, capacity):
    flat = ids.reshape(-1).tolist()
    buckets = [[a for a, e in enumerate(flat) if e == want] for want in range(experts)]
    rows = experts * capacity if capacity else len(flat)
    slot, source, starts, counts = [-1] * len(flat), [-1] * rows, [], []
    at = 0
    for e, bucket in enumerate(buckets):
        start = e * capacity if capacity else at
        kept = bucket[:capacity] if capacity else bucket
        for i, a in enumerate(kept):
            slot[a], source[start + i] = start + i, a
        starts.append(start)
        counts.append(len(kept))
        at += len(bucket)
    make = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
    return make(slot).view(ids.shape), make(source), make(counts), make(starts)


def random_ids(g, tokens, k, experts, dtype=torch.int32):
    ids = torch.randint(-1, experts + 1, (tokens, k), device="cuda", generator=g).to(dtype)   # -1 and experts: none
    return ids


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,k,experts,capacity", [
    (0, 2, 4, None), (0, 2, 4, 3), (1, 1, 1, None), (1, 8, 64, None), (1, 8, 64, 2), (33, 3, 7, None), (33, 3, 7, 5),
    (1000, 2, 1024, None), (4099, 6, 60, 300), (5000, 8, 3, None), (40000, 4, 256, None), (40000, 4, 256, 700)])
def test_sort_is_stable_and_complete(dtype, tokens, k, experts, capacity):
    g = cuda(tokens)
    ids = random_ids(g, tokens, k, experts, dtype)
    order = ex.sort_by_expert(ids, experts, capacity=capacity)
    want = reference_order(ids.cpu(), experts, capacity)
    for got, expect in zip((order.slot, order.source, order.counts, order.starts), want):
        assert torch.equal(got, expect)
    again = ex.sort_by_expert(ids, experts, capacity=capacity)
    assert torch.equal(again.slot, order.slot)


@pytest.mark.gpu
def test_sort_all_on_one_expert_and_none_at_all():
    cuda()
    ids = torch.full((3000, 4), 5, dtype=torch.int32, device="cuda")
    order = ex.sort_by_expert(ids, 9)
    assert order.counts.tolist() == [0] * 5 + [12000] + [0] * 3
    assert torch.equal(order.slot.view(-1), torch.arange(12000, dtype=torch.int32, device="cuda"))
    order = ex.sort_by_expert(ids, 9, capacity=7)
    assert order.counts.tolist() == [0] * 5 + [7] + [0] * 3 and int((order.slot >= 0).sum()) == 7
    order = ex.sort_by_expert(torch.full_like(ids, -1), 9)
    assert bool((order.slot == -1).all()) and bool((order.source == -1).all()) and int(order.counts.sum()) == 0


CASES = [(1, 1, 1, None, 1), (1, 8, 64, None, 4096), (5, 2, 4, None, 7), (33, 3, 7, 5, 1030), (64, 8, 16, 40, 96),
         (257, 4, 8, None, 2048), (1000, 6, 60, 90, 515)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,k,experts,capacity,hidden", CASES)
def test_dispatch_and_combine_match_reference(dtype, tokens, k, experts, capacity, hidden):
    g = cuda(hidden)
    order = ex.sort_by_expert(random_ids(g, tokens, k, experts), experts, capacity=capacity)
    slot, kept = order.slot.long(), order.slot >= 0
    x = normal(g, tokens, hidden, dtype=dtype)
    rows = ex.dispatch(x, order)
    expect = torch.zeros(order.rows, hidden, dtype=dtype, device="cuda")
    expect[slot[kept]] = x.repeat_interleave(k, 0).view(tokens, k, hidden)[kept]
    assert torch.equal(rows, expect)

    def gathered(r):
        return torch.where(kept[..., None], r.double()[slot.clamp(min=0)], 0.0)

    # rows nobody owns must not be read: NaN there may not reach a result
    values = normal(g, order.rows, hidden, dtype=dtype)
    values[order.source < 0] = math.nan
    weights = normal(g, tokens, k)
    parts = gathered(values)
    close(ex.dispatch_backward(values, order), parts.sum(1), parts.abs().sum(1), dtype, k)
    parts = parts * weights.double()[..., None]
    close(ex.combine(values, weights, order), parts.sum(1), parts.abs().sum(1), dtype, 2 * k)

    grad = normal(g, tokens, hidden, dtype=dtype)
    grad_rows, grad_weights = ex.combine_backward(grad, values, weights, order)
    expect = torch.zeros(order.rows, hidden, dtype=torch.float64, device="cuda")
    expect[slot[kept]] = (grad.double()[:, None] * weights.double()[..., None])[kept]
    close(grad_rows, expect, expect.abs(), dtype, 1)
    parts = gathered(values) * grad.double()[:, None]
    close(grad_weights, parts.sum(2), parts.abs().sum(2), torch.float32, hidden)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hidden,offset,pitch", [(64, 8, 96), (64, 1, 67), (66, 2, 72), (128, 3, 1024)])
def test_strided_and_broadcast_rows(dtype, hidden, offset, pitch):
    g = cuda(pitch)
    order = ex.sort_by_expert(random_ids(g, 50, 3, 6), 6)
    wide = normal(g, 150, pitch + offset, dtype=dtype)
    view = wide[:50, offset:offset + hidden]
    store = torch.full((order.rows, pitch + offset), 7.0, device="cuda").to(dtype)
    rows = ex.dispatch(view, order, out=store[:, offset:offset + hidden])
    assert torch.equal(rows, ex.dispatch(view.contiguous(), order))
    assert bool((store[:, :offset] == 7).all()) and bool((store[:, offset + hidden:] == 7).all())
    values, weights = wide[:, offset:offset + hidden], normal(g, 50, 3)
    assert torch.equal(ex.combine(values, weights, order), ex.combine(values.contiguous(), weights, order))
    grads = ex.combine_backward(view, values, weights, order, out=store[:, offset:offset + hidden])
    plain = ex.combine_backward(view.contiguous(), values.contiguous(), weights, order)
    assert torch.equal(grads[0], plain[0])
    # the order of a product's fp32 additions follows the widest vector the addresses allow, so its sums may differ
    # by the roundings of hidden additions: both are held to the 64-bit value
    parts = torch.where((order.slot >= 0)[..., None], values.double()[order.slot.clamp(min=0).long()], 0.0) * \
        view.double()[:, None]
    close(grads[1], parts.sum(2), parts.abs().sum(2), torch.float32, hidden)
    close(plain[1], parts.sum(2), parts.abs().sum(2), torch.float32, hidden)
    assert bool((store[:, :offset] == 7).all()) and bool((store[:, offset + hidden:] == 7).all())
    one = wide[:1, offset:offset + hidden].expand(50, hidden)
    assert torch.equal(ex.dispatch(one, order), ex.dispatch(one.contiguous(), order))


@pytest.mark.gpu
def test_no_tokens_and_no_columns():
    cuda()
    order = ex.sort_by_expert(torch.zeros(0, 2, dtype=torch.int32, device="cuda"), 4, capacity=3)
    rows = ex.dispatch(torch.zeros(0, 8, device="cuda"), order)
    assert rows.shape == (12, 8) and bool((rows == 0).all())
    assert ex.combine(rows, torch.zeros(0, 2, device="cuda"), order).shape == (0, 8)
    grad_rows, grad_weights = ex.combine_backward(torch.zeros(0, 8, device="cuda"), rows,
                                                  torch.zeros(0, 2, device="cuda"), order)
    assert bool((grad_rows == 0).all()) and grad_weights.shape == (0, 2)
    order = ex.sort_by_expert(torch.zeros(3, 2, dtype=torch.int32, device="cuda"), 4)
    empty = torch.zeros(3, 0, device="cuda")
    assert ex.dispatch(empty, order).shape == (6, 0)
    got = ex.combine_backward(empty, torch.zeros(6, 0, device="cuda"), torch.ones(3, 2, device="cuda"), order)
    assert bool((got[1] == 0).all())
    ids, w = ex.route(torch.zeros(0, 4, device="cuda"), 2)
    assert ids.shape == (0, 2) and w.shape == (0, 2)


@pytest.mark.gpu
def test_a_user_made_order_is_kept_inside_its_rows():
    """Slots beyond the rows are treated like assignments without a row."""
    cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    order = ex.ExpertOrder(torch.tensor([[0, 99], [-7, 1]], **i32), torch.tensor([0, 3], **i32),
                           torch.tensor([2], **i32), torch.tensor([0], **i32))
    x = torch.tensor([[1.0, 2], [3, 4]], device="cuda")
    assert ex.dispatch(x, order).tolist() == [[1, 2], [3, 4]]
    w = torch.full((2, 2), 2.0, device="cuda")
    assert ex.combine(x, w, order).tolist() == [[2, 4], [6, 8]]
    grad_rows, grad_weights = ex.combine_backward(x, x, w, order)
    assert grad_rows.tolist() == [[2, 4], [6, 8]] and grad_weights.tolist() == [[5, 0], [0, 25]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("renormalize", [True, False])
def test_autograd_agrees_with_the_plain_calls(dtype, renormalize):
    g = cuda(3)
    logits = normal(g, 40, 12, dtype=dtype).requires_grad_()
    x = normal(g, 40, 72, dtype=dtype).requires_grad_()
    ids, w = ex.route(logits, 3, renormalize=renormalize)
    order = ex.sort_by_expert(ids, 12, capacity=8)
    rows = ex.dispatch(x, order)
    y = ex.combine(rows * 2, w, order)
    grad = normal(g, 40, 72, dtype=dtype)
    y.backward(grad)
    grad_rows, grad_w = ex.combine_backward(grad, rows.detach() * 2, w.detach(), order)
    assert torch.equal(x.grad, ex.dispatch_backward(grad_rows * 2, order))
    assert torch.equal(logits.grad, ex.route_backward(logits.detach(), ids, w.detach(), grad_w, renormalize=renormalize))


@pytest.mark.gpu
def test_gradients_against_differences():
    """Central differences in fp32: the functions are smooth, a step of 2^-6 leaves a relative error of about 2^-12
    from the third derivative and 2^-24 * 2^6 * |loss| from the rounding of the loss."""
    g = cuda(5)
    logits, x = normal(g, 6, 5), normal(g, 6, 9)
    ids, _ = ex.route(logits, 2)
    order = ex.sort_by_expert(ids, 5)
    up, mix = normal(g, 6, 9).double(), normal(g, 12, 9)

    def loss(l, t):
        # the choice is held: the gradient is that of the weights
        p = torch.softmax(l.double(), 1).gather(1, ids.long()).float()
        got = ex.combine(ex.dispatch(t, order) * mix, p, order)
        return (got.double() * up).sum().item()

    lg, xg = logits.clone().requires_grad_(), x.clone().requires_grad_()
    got_ids, w = ex.route(lg, 2, renormalize=False)
    assert torch.equal(got_ids, ids)
    ex.combine(ex.dispatch(xg, order) * mix, w, order).backward(up.float())
    h, size = 2.0 ** -6, (up.abs().sum() * 8).item()
    for value, grad, which in ((logits, lg.grad, 0), (x, xg.grad, 1)):
        for i in range(0, value.numel(), 4):
            step = torch.zeros_like(value)
            step.view(-1)[i] = h
            pair = [(logits + s * step, x) if which == 0 else (logits, x + s * step) for s in (1, -1)]
            difference = (loss(*pair[0]) - loss(*pair[1])) / (2 * h)
            assert abs(difference - grad.view(-1)[i].item()) <= size * (2.0 ** -12 + 2.0 ** -24 * 2 ** 6)


PRODUCTS = [(1, 1, 1, 1, 32, 32), (1, 64, 8, 64, 128, 64), (3, 4, 7, 33, 160, 32), (8, 64, 8, 256, 512, 128),
            (17, 3, 17, 100, 384, 128), (37, 16, 13, 131, 2080, 32), (40, 2, 2, 16, 4096, 64), (100, 5, 4, 515, 896, 128),
            (300, 2, 2, 130, 192, 64)]


def product_case(g, rows, experts, active, n, inner, group, dtype, scale_dtype):
    counts = torch.zeros(experts, dtype=torch.int64)
    pick = torch.randint(0, min(active, experts), (rows,), generator=torch.Generator().manual_seed(rows))
    chosen = torch.randperm(experts, generator=torch.Generator().manual_seed(n))[:min(active, experts)]
    counts.scatter_add_(0, chosen[pick], torch.ones(rows, dtype=torch.int64))
    starts = counts.cumsum(0) - counts
    x = normal(g, rows, inner, dtype=dtype)
    packed = torch.randint(0, 256, (experts, n, inner // 2), dtype=torch.uint8, device="cuda", generator=g)
    scales = (0.01 + 0.02 * torch.rand(experts, n, inner // group, device="cuda", generator=g)).to(scale_dtype)
    return x, starts.int().cuda(), counts.int().cuda(), packed, scales


def product_reference(x, starts, counts, packed, scales, group):
    """(values, sums of magnitudes) in 64 bits."""
    out = torch.zeros(x.size(0), packed.size(1), dtype=torch.float64, device="cuda")
    size = torch.zeros_like(out)
    for s, (at, c) in enumerate(zip(starts.tolist(), counts.tolist())):
        w = dequantized(packed[s % packed.size(0)], scales[s % packed.size(0)], group)
        out[at:at + c] = x[at:at + c].double() @ w.T
        size[at:at + c] = x[at:at + c].double().abs() @ w.abs().T
    return out, size


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wide_scales", [False, True])
@pytest.mark.parametrize("rows,experts,active,n,inner,group", PRODUCTS)
def test_int4_product_matches_reference(dtype, wide_scales, rows, experts, active, n, inner, group):
    g = cuda(inner + n)
    args = product_case(g, rows, experts, active, n, inner, group, dtype, torch.float32 if wide_scales else dtype)
    want, size = product_reference(*args, group)
    got = ex.expert_matmul_int4(*args)
    # products and partial sums: at most inner additions, each of them and each group's scaling off by 2^-23 (the
    # matrix unit may cut instead of rounding)
    close(got, want, size, dtype, 2 * (inner + 3 * inner // group))
    ex.check_status()
    # that bound is the worst case; the fp32 errors have random signs, so over all outputs they stay near the error
    # of one rounding of values as large as the partial sums (32 of which is 2^-19), far under the result's rounding
    assert (got.double() - want).norm() <= (half_step(dtype) + 2.0 ** -16) * want.norm()
    assert torch.equal(got, ex.expert_matmul_int4(*args))


@pytest.mark.gpu
def test_int4_product_segments_gaps_and_views():
    """Segments of two source ranks, rows between them that no segment covers, strided rows and outputs."""
    g = cuda(11)
    i32 = dict(dtype=torch.int32, device="cuda")
    starts, counts = torch.tensor([0, 4, 8, 12], **i32), torch.tensor([3, 0, 4, 2], **i32)
    _, _, _, packed, scales = product_case(g, 4, 2, 2, 50, 128, 64, torch.bfloat16, torch.bfloat16)
    wide = normal(g, 17, 200, dtype=torch.bfloat16)
    x = wide[:, 3:131]
    store = torch.full((17, 60), 7.0, device="cuda", dtype=torch.bfloat16)
    got = ex.expert_matmul_int4(x, starts, counts, packed, scales, out=store[:, 5:55])
    want, size = product_reference(x, starts, counts, packed, scales, 64)
    close(got, want, size, torch.bfloat16, 2 * (128 + 6))
    for r in (3, 4, 5, 6, 7, 14, 15, 16):
        assert bool((got[r] == 0).all())
    assert bool((store[:, :5] == 7).all()) and bool((store[:, 55:] == 7).all())
    none = ex.expert_matmul_int4(x, starts, torch.zeros_like(counts), packed, scales)
    assert bool((none == 0).all())
    assert ex.expert_matmul_int4(x[:0], starts, counts, packed, scales).shape == (0, 50)


@pytest.mark.gpu
def test_int4_product_keeps_segments_inside_the_rows():
    g = cuda(12)
    i32 = dict(dtype=torch.int32, device="cuda")
    _, _, _, packed, scales = product_case(g, 4, 2, 2, 20, 64, 32, torch.float16, torch.float16)
    x = normal(g, 6, 64, dtype=torch.float16)
    got = ex.expert_matmul_int4(x, torch.tensor([-3, 4], **i32), torch.tensor([5, 1000], **i32), packed, scales)
    want, size = product_reference(x, torch.tensor([0, 4]), torch.tensor([2, 2]), packed, scales, 32)
    close(got, want, size, torch.float16, 2 * (64 + 6))


@pytest.mark.gpu
def test_int4_product_infinities_and_nan_follow_the_formula():
    cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.full((1, 3, 64), 8, dtype=torch.uint8, device="cuda")
    q[0, 0, 5], q[0, 1, 5] = 11, 2                       # +3, -6 and (row 2) 0 times infinity
    packed = q[..., 0::2] | (q[..., 1::2] << 4)
    scales = torch.ones(1, 3, 2, device="cuda", dtype=torch.bfloat16)
    x = torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16)
    x[0, 5] = math.inf
    got = ex.expert_matmul_int4(x, torch.zeros(1, **i32), torch.full((1,), 2, **i32), packed, scales)
    assert got[0, 0] == math.inf and got[0, 1] == -math.inf and bool(got[0, 2].isnan())
    assert bool((got[1] == 0).all())


@pytest.mark.gpu
def test_the_set_together_eager_and_replayed_on_a_side_stream():
    """Router, sort, dispatch, two 4-bit products and combine, as a serving step calls them; the captured step on
    new inputs equals the eager one bit for bit."""
    g = cuda(21)
    tokens, experts, k, hidden, inner = 13, 8, 2, 256, 384
    up = ex.quantize_int4(normal(g, experts, inner, hidden, dtype=torch.bfloat16, scale=0.05), 64)
    down = ex.quantize_int4(normal(g, experts, hidden, inner, dtype=torch.bfloat16, scale=0.05), 128)
    gate = normal(g, hidden, experts, dtype=torch.bfloat16, scale=0.1)

    def step(x):
        ids, w = ex.route(x @ gate, k)
        order = ex.sort_by_expert(ids, experts)
        h = ex.expert_matmul_int4(ex.dispatch(x, order), order.starts, order.counts, *up)
        y = ex.expert_matmul_int4(h.relu(), order.starts, order.counts, *down)
        return ex.combine(y, w, order), ids, w, h, y

    x = normal(g, tokens, hidden, dtype=torch.bfloat16)
    out, ids, w, h, y = step(x)
    wu, wd = dequantized(*up, 64), dequantized(*down, 128)
    for t in range(tokens):
        total = torch.zeros(hidden, dtype=torch.float64, device="cuda")
        for j in range(k):
            e = ids[t, j]
            mid = (wu[e] @ x[t].double()).to(torch.bfloat16).double().relu()
            total += w[t, j].double() * (wd[e] @ mid).to(torch.bfloat16).double()
        # the kernel and this loop round the middle and the expert's result to bf16 on sums that differ in fp32, so
        # to neighbours at most (2 half steps each); the last rounding is one half step, fp32 errors less than one
        mids = torch.stack([(wu[e].abs() @ x[t].double().abs()) for e in ids[t]])
        size = sum(w[t, j].double() * (wd[ids[t, j]].abs() @ mids[j]) for j in range(k))
        assert bool(((out[t].double() - total).abs() <= 6 * half_step(torch.bfloat16) * size).all())

    stream = torch.cuda.Stream()
    held = x.clone()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(held)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured = step(held)[0]
        for seed in (1, 2):
            fresh = normal(cuda(seed), tokens, hidden, dtype=torch.bfloat16)
            stream.wait_stream(torch.cuda.current_stream())
            held.copy_(fresh)
            graph.replay()
            assert torch.equal(captured, step(fresh)[0])
    torch.cuda.current_stream().wait_stream(stream)


@pytest.mark.gpu
def test_autograd_is_refused_under_capture_and_plain_gradients_replay():
    g = cuda(31)
    x = normal(g, 16, 64).requires_grad_()
    ids = torch.randint(0, 4, (16, 2), device="cuda", generator=g, dtype=torch.int32)
    w = torch.rand(16, 2, device="cuda", generator=g)
    order = ex.sort_by_expert(ids, 4)
    eager = ex.dispatch(x, order)                      # an eager graph of the same leaf stays alive
    grad = normal(g, 16, 64)
    plain = x.detach()

    def training_step():
        rows = ex.dispatch(plain, order)
        out = ex.combine(rows, w, order)
        grad_rows, grad_w = ex.combine_backward(grad, rows, w, order)
        return out, ex.dispatch_backward(grad_rows, order), grad_w

    want = training_step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeFailure, match="capture"):
            ex.dispatch(x, order)
        got = training_step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    eager.sum().backward()
    assert bool((x.grad == 2).all())


@pytest.mark.gpu
def test_out_over_an_input_is_refused():
    cuda()
    order = ex.sort_by_expert(torch.zeros(4, 1, dtype=torch.int32, device="cuda"), 1)
    x = torch.zeros(6, 8, device="cuda")
    with pytest.raises(RuntimeFailure, match="overlaps"):
        ex.dispatch(x[:4], order, out=x[2:6])
    with pytest.raises(RuntimeFailure, match="overlaps"):
        ex.combine(x[:4], torch.zeros(4, 1, device="cuda"), order, out=x[:4])


@pytest.mark.gpu
@pytest.mark.parametrize("kernel", ["expert_route", "expert_sort", "expert_dispatch", "expert_combine",
                                    "expert_combine_backward", "expert_matmul_int4"])
def test_kernel_bench_runs_the_expert_kernels(kernel, capsys):
    cuda()
    import json
    from vericcl_b200.ops import kernel_bench
    assert kernel_bench.main(["--kernel", kernel, "--tokens", "33", "--experts", "8", "--choices", "2", "--hidden", "256",
                              "--outputs", "48", "--group", "64", "--iters", "2"]) == 0
    line = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert line["us"] > 0 and kernel in line["kernel"]


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements of rows (and 2^32 bytes of weights): the last rows are where a 32-bit offset would wrap."""
    g = cuda(41)
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    tokens, k, hidden = 270_000, 2, 4096
    ids = torch.randint(0, 16, (tokens, k), device="cuda", generator=g, dtype=torch.int32)
    order = ex.sort_by_expert(ids, 16)
    x = torch.zeros(tokens, hidden, device="cuda", dtype=torch.bfloat16)
    x[:, :8] = torch.randn(tokens, 8, device="cuda", generator=g).bfloat16()
    rows = ex.dispatch(x, order)
    source = order.source.long()
    assert torch.equal(rows[:, :8], x[source // k, :8])
    w = torch.full((tokens, k), 0.5, device="cuda")
    assert torch.equal(ex.combine(rows, w, order), x)                 # two halves of the same value: exact
    grad_rows, grad_w = ex.combine_backward(x, rows, w, order)
    assert torch.equal(grad_rows[:, :8], (x * 0.5)[source // k, :8])
    parts = x[:, :8].double().square()
    close(grad_w, parts.sum(1, keepdim=True).expand(tokens, k), parts.sum(1, keepdim=True).expand(tokens, k),
          torch.float32, 8)
    assert torch.equal(ex.dispatch_backward(rows, order), (x.float() * 2).bfloat16())
    del rows, grad_rows
    experts, n, inner = 40, 16384, 16384                              # 5.4 GB of weights
    packed = torch.full((experts, n, inner // 2), 0x88, dtype=torch.uint8, device="cuda")
    packed[-1] = torch.randint(0, 256, (n, inner // 2), dtype=torch.uint8, device="cuda", generator=g)
    scales = torch.ones(experts, n, inner // 128, device="cuda", dtype=torch.bfloat16)
    counts = torch.zeros(experts, dtype=torch.int32, device="cuda")
    counts[0], counts[-1] = 1, 2
    starts = (counts.cumsum(0) - counts).int()
    y = normal(g, 3, inner, dtype=torch.bfloat16)
    got = ex.expert_matmul_int4(y, starts, counts, packed, scales)
    assert bool((got[0] == 0).all())
    q = torch.stack([packed[-1] & 15, packed[-1] >> 4], -1).flatten(-2).double() - 8
    want, size = y[1:].double() @ q.T, y[1:].double().abs() @ q.abs().T
    close(got[1:], want, size, torch.bfloat16, 2 * (inner + 3 * inner // 128))
    assert (got[1:].double() - want).norm() <= (half_step(torch.bfloat16) + 2.0 ** -16) * want.norm()


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls keep nothing between them: the same operators on two streams, many times, give the eager results."""
    g = cuda(51)
    work = []
    for tokens, experts in ((700, 30), (41, 5)):
        x, w = normal(g, tokens, 512, dtype=torch.bfloat16), torch.rand(tokens, 4, device="cuda", generator=g)
        ids = torch.randint(0, experts, (tokens, 4), device="cuda", generator=g, dtype=torch.int32)
        packed = torch.randint(0, 256, (experts, 256, 256), dtype=torch.uint8, device="cuda", generator=g)
        scales = torch.rand(experts, 256, 8, device="cuda", generator=g).bfloat16()
        work.append((x, w, ids, packed, scales, experts))

    def step(x, w, ids, packed, scales, experts):
        order = ex.sort_by_expert(ids, experts)
        rows = ex.dispatch(x, order)
        return ex.expert_matmul_int4(rows, order.starts, order.counts, packed, scales), ex.combine(rows, w, order)

    want = [step(*w) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(step(*work[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for a in got[i]:
            assert torch.equal(a[0], want[i][0]) and torch.equal(a[1], want[i][1])


@pytest.mark.gpu
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_infinity_is_chosen_and_spoils_the_weights(renormalize):
    cuda()
    ids, w = ex.route(torch.tensor([[1.0, math.inf, 2]], device="cuda"), 2, renormalize=renormalize)
    assert ids.tolist() == [[1, 2]] and bool(w.isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("experts,k", [(128, 8), (300, 16), (1000, 32)])
def test_route_many_equal_logits(experts, k):
    """Few distinct values: more candidates than a warp has lanes, ties everywhere."""
    g = cuda(experts)
    logits = torch.randint(0, 3, (50, experts), device="cuda", generator=g).to(torch.bfloat16)
    logits[:10] = 1.0
    logits[10:20, k // 2:] = -math.inf
    ids, _ = ex.route(logits, k)
    assert torch.equal(ids, reference_route(logits, k, True)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("group,scale_dtype", [(32, torch.float32), (64, torch.float16), (128, torch.float16)])
def test_int4_product_segments_in_any_order_and_of_all_lengths(group, scale_dtype):
    """Segments of 0, 1, 8, 9, 32, 33, 41 and 65 rows, later ones first: every number of columns, items that are
    sorted by their length, and more than one stage of x and scales."""
    g = cuda(group)
    lengths = [65, 0, 9, 33, 1, 41, 32, 8]
    starts, at = [0] * 8, 0
    for s in reversed(range(8)):
        starts[s] = at
        at += lengths[s]
    inner = 5 * 512 + group                                           # the last tile holds one group
    i32 = dict(dtype=torch.int32, device="cuda")
    starts, counts = torch.tensor(starts, **i32), torch.tensor(lengths, **i32)
    x = normal(g, at, inner, dtype=torch.float16)
    packed = torch.randint(0, 256, (4, 145, inner // 2), dtype=torch.uint8, device="cuda", generator=g)
    scales = (0.01 + 0.02 * torch.rand(4, 145, inner // group, device="cuda", generator=g)).to(scale_dtype)
    got = ex.expert_matmul_int4(x, starts, counts, packed, scales)
    want, size = product_reference(x, starts, counts, packed, scales, group)
    close(got, want, size, torch.float16, 2 * (inner + 3 * inner // group))
    assert (got.double() - want).norm() <= (half_step(torch.float16) + 2.0 ** -16) * want.norm()


@pytest.mark.gpu
def test_gradients_of_broadcast_tokens_and_of_expanded_gradients():
    """One row of x for every token (its gradient is the sum over them), and a gradient that is one number expanded."""
    g = cuda(61)
    base, w = normal(g, 1, 40).requires_grad_(), torch.rand(7, 2, device="cuda", generator=g).requires_grad_()
    order = ex.sort_by_expert(random_ids(g, 7, 2, 3), 3)
    rows = ex.dispatch(base.expand(7, 40), order)
    out = ex.combine(rows, w, order)
    out.sum().backward()
    kept = (order.slot >= 0).double()
    share = (w.detach().double() * kept).sum()
    # every row adds its weight once: sums of 14 positive terms, each addition off by 2^-24 of at most the sum
    assert bool(((base.grad.double() - share).abs() <= 32 * 2.0 ** -24 * share).all())
    total = base.detach().double().sum()
    size = base.detach().double().abs().sum()
    assert bool(((w.grad.double() - kept * total).abs() <= 41 * 2.0 ** -24 * size).all())


@pytest.mark.parametrize("weight_dtype,scale_dtype,magnitude", [
    (torch.float32, torch.float16, 1e6), (torch.bfloat16, torch.float16, 1e6), (torch.float32, torch.float16, 7 * 65520.0)])
def test_quantize_int4_refuses_scales_beyond_their_type(weight_dtype, scale_dtype, magnitude):
    """65520 is the lowest magnitude that rounds to fp16's infinity."""
    w = torch.ones(2, 128, dtype=weight_dtype)
    w[1, 70] = magnitude
    with pytest.raises(RuntimeFailure, match="range"):
        ex.quantize_int4(w, 64, scale_dtype=scale_dtype)
    packed, scales = ex.quantize_int4(w, 64, scale_dtype=torch.float32)          # a wider type holds it
    assert bool(scales.isfinite().all())
    w[1, 70] = 7 * 65000.0                                                       # near the largest fp16 value, 65504
    assert 64000 < ex.quantize_int4(w, 64, scale_dtype=scale_dtype)[1][1, 1] <= 65504


@pytest.mark.parametrize("dtype,scale_dtype", [(torch.float16, torch.float16), (torch.float32, torch.float16),
                                               (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                               (torch.float32, torch.bfloat16)])
def test_quantize_int4_keeps_groups_whose_scale_underflows(dtype, scale_dtype):
    """Magnitudes of at most 3.5 smallest scales: their seventh rounds to 0, and the smallest positive scale holds
    them to half a step.  A group of zeros stays zeros."""
    least = torch.finfo(scale_dtype).smallest_normal * torch.finfo(scale_dtype).eps
    w = torch.zeros(3, 64, dtype=torch.float64)
    w[0, :32] = torch.linspace(-3.0, 3.0, 32, dtype=torch.float64) * least
    w[1, 3] = least
    w = w.to(dtype)
    packed, scales = ex.quantize_int4(w, 32, scale_dtype=scale_dtype)
    assert bool((scales > 0).all()) and scales[0, 0] == least and scales[1, 0] == least
    back = dequantized(packed, scales, 32)
    assert bool(((back - w.double()).abs() <= least * 0.5).all())
    assert bool((back[2] == 0).all()) and back[1, 3] == least


def calls_with_out(g, device="cuda"):
    """Each call that takes ``out``, as (call of out, the shape of out), on small inputs of bfloat16."""
    i32 = dict(dtype=torch.int32, device=device)
    order = ex.ExpertOrder(torch.tensor([[0, 2], [1, 3], [4, 5]], **i32), torch.tensor([0, 2, 1, 3, 4, 5], **i32),
                           torch.tensor([6], **i32), torch.tensor([0], **i32))
    x, rows = (torch.randn(n, 32, generator=g, device=device).bfloat16() for n in (3, 6))
    w = torch.rand(3, 2, generator=g, device=device)
    packed = torch.zeros(1, 5, 16, dtype=torch.uint8, device=device)
    scales = torch.ones(1, 5, 1, dtype=torch.bfloat16, device=device)
    return [(lambda out: ex.dispatch(x, order, out=out), (6, 32)),
            (lambda out: ex.dispatch_backward(rows, order, out=out), (3, 32)),
            (lambda out: ex.combine(rows, w, order, out=out), (3, 32)),
            (lambda out: ex.combine_backward(x, rows, w, order, out=out), (6, 32)),
            (lambda out: ex.expert_matmul_int4(rows, order.starts, order.counts, packed, scales, out=out), (6, 5))]


def test_an_out_that_requires_a_gradient_is_refused():
    for call, shape in calls_with_out(torch.Generator().manual_seed(1), "cpu"):
        with pytest.raises(RuntimeFailure, match="gradient"):
            call(torch.zeros(shape, dtype=torch.bfloat16, requires_grad=True))


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(5))
def test_autograd_sees_writes_into_out(which):
    """A buffer that a graph has saved and that a call overwrites stops that graph's backward pass, as torch's own
    ``out=`` does; a slice of it too."""
    g = cuda(71)
    call, shape = calls_with_out(g)[which]
    wide = torch.zeros(shape[0], shape[1] + 8, dtype=torch.bfloat16, device="cuda")
    leaf = torch.ones_like(wide, requires_grad=True)
    loss = (leaf * wide).sum()
    call(wide[:, 8:])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    held = torch.zeros(shape, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeFailure, match="gradient"):
        call(held)
    with torch.no_grad():
        call(held)
    with torch.inference_mode():
        kept = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
        call(kept)
    call(kept)                                                    # it has no versions, and no graph can have saved it
    assert torch.equal(kept, held)


@pytest.mark.gpu
def test_check_status_waits_for_products_on_any_stream():
    g = cuda(81)
    args = product_case(g, 3, 2, 2, 40, 128, 64, torch.bfloat16, torch.bfloat16)
    a = torch.zeros(8192, 8192, dtype=torch.bfloat16, device="cuda")
    a @ a
    ex.expert_matmul_int4(*args)
    ex.check_status()                                             # whatever is set up once is
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(100):                                      # tens of milliseconds before the product starts
            a = a @ a
        ex.expert_matmul_int4(*args)
    ex.check_status()
    assert stream.query()


@pytest.mark.gpu
def test_check_status_is_refused_under_capture():
    cuda()
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(8, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = x + 1
        with pytest.raises(RuntimeFailure, match="capture"):
            ex.check_status()
    graph.replay()
    ex.check_status()
    assert bool((y == 1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,experts,active,n,inner,group", [(3, 4, 2, 33, 32, 32), (8, 8, 8, 256, 4096, 128),
                                                               (40, 2, 2, 130, 1600, 64)])
def test_int4_product_whose_waits_run_out(monkeypatch, rows, experts, active, n, inner, group):
    """Every wait given up at once (the copies themselves arrive): covered rows are NaN, the others zero, the
    status is raised once, and the next product is right.  Sizes of one tile, of a cluster and of several tiles."""
    g = cuda(91)
    x, starts, counts, packed, scales = product_case(g, rows, experts, active, n, inner, group, torch.bfloat16,
                                                     torch.bfloat16)
    x = torch.cat([x, x[:2]])                                     # two rows that no segment covers
    ex.check_status()
    with monkeypatch.context() as patch:
        patch.setattr(ex, "_GIVE_UP", True)
        late = ex.expert_matmul_int4(x, starts, counts, packed, scales)
    with pytest.raises(RuntimeFailure, match="in time"):
        ex.check_status()
    ex.check_status()
    assert bool(late[:rows].isnan().all()) and bool((late[rows:] == 0).all())
    got = ex.expert_matmul_int4(x, starts, counts, packed, scales)
    want, size = product_reference(x, starts, counts, packed, scales, group)
    close(got, want, size, torch.bfloat16, 2 * (inner + 3 * inner // group))
    ex.check_status()


def float_calls(g, device):
    """(call of its float tensors, those tensors) of every operator, on small inputs."""
    i32 = dict(dtype=torch.int32, device=device)
    order = ex.ExpertOrder(torch.tensor([[0, 2], [1, 3]], **i32), torch.tensor([0, 2, 1, 3], **i32),
                           torch.tensor([4], **i32), torch.tensor([0], **i32))
    draw = lambda *shape: torch.randn(shape, generator=g, device=device)     # noqa: E731
    ids = torch.tensor([[0, 2], [1, 0]], **i32)
    packed = torch.zeros(1, 5, 16, dtype=torch.uint8, device=device)
    return [(lambda l: ex.route(l, 2), [draw(2, 3)]),
            (lambda l, w, u: ex.route_backward(l, ids, w, u), [draw(2, 3), draw(2, 2), draw(2, 2)]),
            (lambda x: ex.dispatch(x, order), [draw(2, 8)]),
            (lambda r: ex.dispatch_backward(r, order), [draw(4, 8)]),
            (lambda r, w: ex.combine(r, w, order), [draw(4, 8), draw(2, 2)]),
            (lambda u, r, w: ex.combine_backward(u, r, w, order), [draw(2, 8), draw(4, 8), draw(2, 2)]),
            (lambda r, s: ex.expert_matmul_int4(r.bfloat16(), order.starts, order.counts, packed, s),
             [draw(4, 32), draw(1, 5, 1)])]


def tangents_are_refused(device):
    import torch.autograd.forward_ad as fwd
    for call, inputs in float_calls(torch.Generator(device=device).manual_seed(3), device):
        for which in range(len(inputs)):
            with fwd.dual_level():
                given = list(inputs)
                given[which] = fwd.make_dual(given[which], torch.ones_like(given[which]))
                with pytest.raises(RuntimeFailure, match="forward-mode"):
                    call(*given)
        if device == "cuda":
            call(*inputs)


def test_forward_mode_tangents_are_refused():
    tangents_are_refused("cpu")


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused_on_the_gpu():
    cuda()
    tangents_are_refused("cuda")


def overlapping_calls(device):
    """Calls whose out lies over an input that is not the matrix the rows come from."""
    i32 = dict(dtype=torch.int32, device=device)
    pool = torch.zeros(4096, device=device)                       # every tensor is a part of it
    order = ex.ExpertOrder(pool[:8].view(torch.int32).view(4, 2), pool[8:16].view(torch.int32), torch.tensor([8], **i32),
                           torch.tensor([0], **i32))
    w, x, rows = pool[16:24].view(4, 2), pool[64:96].view(4, 8), pool[128:192].view(8, 8)
    elsewhere = pool[1024:1056].view(4, 8)
    half = pool.view(torch.bfloat16)                              # element 2 i is at pool[i]
    r16 = half[4096:4096 + 8 * 32].view(8, 32)
    packed = pool[512:512 + 20].view(torch.uint8).view(1, 5, 16)
    scales, starts, counts = half[1200:1205].view(1, 5, 1), pool[700:701].view(torch.int32), pool[704:705].view(torch.int32)

    def product(at):
        return lambda: ex.expert_matmul_int4(r16, starts, counts, packed, scales, out=half[at:at + 40].view(8, 5))
    return [lambda: ex.dispatch(x, order, out=pool[4:68].view(8, 8)),               # slot
            lambda: ex.dispatch(elsewhere, order, out=pool[15:79].view(8, 8)),      # source
            lambda: ex.dispatch_backward(rows, order, out=pool[15:47].view(4, 8)),
            lambda: ex.combine(rows, w, order, out=pool[7:39].view(4, 8)),
            lambda: ex.combine(rows, w, order, out=pool[23:55].view(4, 8)),         # weights
            lambda: ex.combine_backward(elsewhere, rows, w, order, out=pool[23:87].view(8, 8)),
            lambda: ex.combine_backward(elsewhere, rows, w, order, out=pool[100:164].view(8, 8)),
            product(2 * 512 - 39), product(2 * 512 + 39), product(1204), product(1200 - 39), product(1400), product(1409)]


def test_an_out_over_any_input_is_refused():
    for i, call in enumerate(overlapping_calls("cpu")):
        with pytest.raises(RuntimeFailure, match="overlaps"):
            call()


@pytest.mark.gpu
def test_an_out_over_any_input_is_refused_on_the_gpu():
    cuda()
    for call in overlapping_calls("cuda"):
        with pytest.raises(RuntimeFailure, match="overlaps"):
            call()


def beside(device):
    """One matrix whose column ranges are the tokens, the rows and the results."""
    i32 = dict(dtype=torch.int32, device=device)
    order = ex.ExpertOrder(torch.tensor([[0, 2], [1, 3]], **i32), torch.tensor([0, 2, 1, 3], **i32),
                           torch.tensor([4], **i32), torch.tensor([0], **i32))
    wide = torch.arange(4 * 24, dtype=torch.float32, device=device).view(4, 24)
    return wide, order, torch.tensor([[1.0, 2], [0.5, 1]], device=device)


def test_columns_that_meet_are_refused():
    wide, order, w = beside("cpu")
    for call in (lambda: ex.dispatch(wide[:2, :8], order, out=wide[:, 7:15]),
                 lambda: ex.dispatch(wide[:2, 8:16], order, out=wide[:, 1:9]),
                 lambda: ex.dispatch(wide[:2, :8], order, out=wide[:, :8]),
                 lambda: ex.dispatch(wide.view(8, 12)[:2, :6], order, out=wide[:, 6:12]),     # other strides
                 lambda: ex.dispatch_backward(wide[:1, :8].expand(4, 8), order, out=wide[:2, 4:12]),
                 lambda: ex.combine(wide[:, 8:16], w, order, out=wide[:2, 15:23]),
                 # the last column of a row and the first of the next
                 lambda: ex.combine(wide[:, :8], w, order, out=wide.view(-1)[17:17 + 48].view(2, 24)[:, :8])):
        with pytest.raises(RuntimeFailure, match="overlaps"):
            call()


def test_columns_beside_each_other_are_not_an_overlap():
    wide, order, w = beside("cpu")
    for call in (lambda: ex.dispatch(wide[:2, :8], order, out=wide[:, 8:16]),
                 lambda: ex.dispatch(wide[1:3, 16:], order, out=wide[:, 8:16]),
                 lambda: ex.combine(wide[:, 8:16], w, order, out=wide[:2, 16:24]),
                 lambda: ex.combine(wide[:, :8], w, order, out=wide.view(-1)[16:16 + 48].view(2, 24)[:, :8]),
                 lambda: ex.combine_backward(wide[:2, 16:], wide[:, :8], w, order, out=wide[:, 8:16])):
        with pytest.raises(RuntimeFailure, match="CUDA"):         # nothing else is wrong with them
            call()


@pytest.mark.gpu
def test_columns_of_one_matrix_as_inputs_and_out():
    cuda()
    wide, order, w = beside("cuda")
    start = wide.clone()
    rows = ex.dispatch(wide[:2, :8], order, out=wide[:, 8:16])
    assert torch.equal(rows, start[[0, 1, 0, 1], :8])
    assert torch.equal(wide[:, :8], start[:, :8]) and torch.equal(wide[:, 16:], start[:, 16:])
    ex.combine(wide[:, 8:16], w, order, out=wide[1:3, 16:])
    assert torch.equal(wide[1:3, 16:], start[:2, :8] * torch.tensor([[3.0], [1.5]], device="cuda"))
    grad, got_w = ex.combine_backward(wide[1:3, 16:], wide[:, 8:16], w, order, out=wide[:, :8])
    up = wide[1:3, 16:]
    assert torch.equal(grad, up.repeat(2, 1) * torch.tensor([[1.0], [0.5], [2], [1]], device="cuda"))
    assert torch.allclose(got_w, (up * wide[:2, 8:16]).sum(1, keepdim=True).expand(2, 2))
    with pytest.raises(RuntimeFailure, match="overlaps"):
        ex.dispatch(wide[:2, :8], order, out=wide[:, 7:15])


@pytest.mark.gpu
def test_int4_product_of_the_longest_segment():
    """One segment of 2^31 - 1 rows (one row repeated): its length rounded up to whole items passes 31 bits."""
    g = cuda(101)
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    rows, i32 = 2 ** 31 - 1, dict(dtype=torch.int32, device="cuda")
    x = normal(g, 1, 32, dtype=torch.bfloat16)
    packed = torch.randint(0, 256, (1, 1, 16), dtype=torch.uint8, device="cuda", generator=g)
    scales = torch.ones(1, 1, 1, dtype=torch.bfloat16, device="cuda")
    one = ex.expert_matmul_int4(x, torch.zeros(1, **i32), torch.ones(1, **i32), packed, scales)
    assert one[0, 0] != 0 and one[0, 0].isfinite()
    out = torch.zeros(rows, 1, dtype=torch.bfloat16, device="cuda")
    ex.expert_matmul_int4(x.expand(rows, 32), torch.zeros(1, **i32), torch.full((1,), rows, **i32), packed, scales, out=out)
    assert all(bool((part == one[0, 0]).all()) for part in out.split(1 << 28))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("experts,k", [(96, 6), (128, 8), (300, 16), (1000, 32)])
def test_route_masks_nan_and_infinity_among_many_experts(dtype, renormalize, experts, k):
    """The paths of more than 64 experts: few finite logits, none, the type's lowest value, NaN and +inf."""
    g = cuda(experts + k)
    logits = normal(g, 60, experts, dtype=dtype, scale=3.0)
    scattered = torch.rand(60, experts, device="cuda", generator=g)
    for t, finite in enumerate([0, 1, k - 1, k, k + 1, 33, 64]):  # so many experts are left, anywhere
        logits[t].masked_fill_(scattered[t].argsort().argsort() >= finite, -math.inf)
    logits[10:20].masked_fill_(scattered[10:20] < 0.5, -math.inf)
    low = torch.finfo(dtype).min
    logits[20] = low
    logits[21:25].masked_fill_(scattered[21:25] < 0.9, low)
    logits[25, 1:] = low
    finite_rows = list(range(30))
    logits[30:35, 7] = math.nan
    logits[35] = math.nan
    logits[36] = -math.inf
    logits[36, 70] = math.nan
    logits[40:45, 90] = math.inf
    logits[45:48] = math.inf
    logits[48, 3], logits[48, 88] = math.inf, math.nan
    spoiled = list(range(30, 36)) + list(range(40, 49))
    finite_rows += [t for t in range(30, 60) if t not in spoiled]  # 36, a token without a choice, has weights of 0
    ids, w = ex.route(logits, k, renormalize=renormalize)
    want_ids, want = reference_route(logits, k, renormalize)
    assert torch.equal(ids, want_ids)
    fine = torch.tensor(finite_rows, device="cuda")
    bound = route_bound(logits[50:])                              # differences to a masked logit do not reach a weight
    # exp of a difference beyond the type's finite range is 0 on both sides, or below 2^-126 where a subnormal is cut
    assert bool(((w[fine].double() - want[fine]).abs() <= bound * want[fine] + 2.0 ** -125).all())
    assert bool(w[spoiled][ids[spoiled] >= 0].isnan().all()) and bool((w[ids < 0] == 0).all())
    up = normal(g, 60, k)
    got = ex.route_backward(logits, ids, w, up, renormalize=renormalize)
    up64 = torch.where(ids >= 0, up.double(), 0.0)
    inner = (want * up64).sum(1, keepdim=True)
    expect = torch.zeros(60, experts + 1, dtype=torch.float64, device="cuda")
    spot = torch.where(ids >= 0, ids.long(), experts)             # a column for what is not chosen
    if renormalize:
        expect.scatter_(1, spot, want * (up64 - inner))
        expect, share = expect[:, :experts], 1.0
    else:
        share = torch.softmax(logits.double(), 1).nan_to_num()
        expect = share * (expect.scatter_(1, spot, up64)[:, :experts] - inner)
    size = up.abs().max().item() * 2
    limit = half_step(dtype) * expect.abs() + (4 * bound + 40 * 2.0 ** -24) * size * share + \
        torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps + 2.0 ** -124
    rows = [t for t in finite_rows if t != 36]
    assert bool(((got.double() - expect).abs() <= limit)[rows].all())
    for t in spoiled:                                             # the chosen experts' gradients are spoiled, or all
        assert bool(got[t][ids[t][ids[t] >= 0].long()].isnan().all())
        if renormalize:
            others = torch.ones(experts, dtype=torch.bool, device="cuda")
            others[ids[t][ids[t] >= 0].long()] = False
            assert bool((got[t][others] == 0).all())
        elif bool((ids[t] >= 0).any()):
            assert bool(got[t].isnan().all())


def torch_order(ids, experts, capacity):
    """``reference_order`` for many assignments."""
    flat = ids.reshape(-1).long().cpu()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    total = torch.bincount(key, minlength=experts + 1)
    by_expert = torch.sort(key, stable=True).indices
    place = torch.empty_like(key)
    place[by_expert] = torch.arange(len(key)) - (total.cumsum(0) - total)[key[by_expert]]
    starts = torch.arange(experts) * capacity if capacity else (total.cumsum(0) - total)[:experts]
    kept = (key < experts) & (place < (capacity or len(key)))
    slot = torch.where(kept, starts[key.clamp(max=experts - 1)] + place, -1)
    source = torch.full((experts * capacity if capacity else len(key),), -1)
    source[slot[kept]] = torch.arange(len(key))[kept]
    counts = total[:experts].clamp(max=capacity or len(key))
    return [t.int().cuda() for t in (slot.view(ids.shape), source, counts, starts)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,k,experts,capacity", [(65536, 8, 1024, None), (65536, 8, 1024, 500), (16397, 8, 1023, 3),
                                                       (300000, 1, 1, 299999), (40000, 4, 2, 90000)])
def test_sort_across_the_largest_cluster(dtype, tokens, k, experts, capacity):
    """16 CTAs with the most experts, whose counts take the most shared memory; few experts with long empty parts."""
    g = cuda(tokens)
    ids = random_ids(g, tokens, k, experts, dtype)
    order = ex.sort_by_expert(ids, experts, capacity=capacity)
    for got, expect in zip((order.slot, order.source, order.counts, order.starts), torch_order(ids, experts, capacity)):
        assert torch.equal(got, expect)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hidden", [(torch.float32, 1030), (torch.float32, 1028), (torch.float32, 1027),
                                          (torch.bfloat16, 2052), (torch.float16, 2051), (torch.bfloat16, 1544)])
def test_rows_beyond_half_the_l2_with_empty_ones(dtype, hidden):
    """More than 64 MB of rows, a third of them without a token, in vectors of 16, 8, 4 and 2 bytes."""
    test_dispatch_and_combine_match_reference(dtype, 6000, 3, 40, 600, hidden)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_int4_product_of_the_smallest_and_largest_rows(dtype, group):
    """Rows whose products are subnormal in fp32 for bf16 rows (fp16's smallest are not), and rows near the type's largest
    value with scales that bring the sum back."""
    g = cuda(group)
    fine = torch.finfo(dtype)
    i32 = dict(dtype=torch.int32, device="cuda")
    inner, n = 4 * group, 21
    packed = torch.randint(0, 256, (1, n, inner // 2), dtype=torch.uint8, device="cuda", generator=g)
    signs = torch.randint(0, 2, (3, inner), device="cuda", generator=g) * 2.0 - 1
    for magnitude, scale in ((fine.smallest_normal, 1.0), (fine.smallest_normal * fine.eps, 1.0),
                             (fine.smallest_normal, 2.0 ** 14), (fine.max / 2 ** 12, 2.0 ** -14)):
        x = (signs * magnitude).to(dtype)
        scales = torch.full((1, n, inner // group), scale, dtype=dtype, device="cuda")
        args = x, torch.zeros(1, **i32), torch.full((1,), 3, **i32), packed, scales
        want, size = product_reference(*args, group)
        close(ex.expert_matmul_int4(*args), want, size, dtype, 2 * (inner + 3 * inner // group))


@pytest.mark.gpu
def test_int4_product_with_overlapping_segments_stays_inside_its_result():
    """Segments that cover rows twice leave the result undefined, and everything around it as it was."""
    g = cuda(111)
    i32 = dict(dtype=torch.int32, device="cuda")
    _, _, _, packed, scales = product_case(g, 4, 2, 2, 50, 128, 64, torch.bfloat16, torch.bfloat16)
    x = normal(g, 40, 128, dtype=torch.bfloat16)
    store = torch.full((42, 60), 7.0, device="cuda", dtype=torch.bfloat16)
    for starts, counts in (([0, 0, 0, 0], [40, 40, 40, 40]), ([0, 3, 20, 39], [20, 9, 20, 7])):
        ex.expert_matmul_int4(x, torch.tensor(starts, **i32), torch.tensor(counts, **i32), packed, scales,
                              out=store[1:41, 5:55])
        assert bool((store[[0, 41]] == 7).all()) and bool((store[:, :5] == 7).all()) and bool((store[:, 55:] == 7).all())
    ex.check_status()
