"""Measured cases of the mixture-of-experts operators (``vericcl_b200.ops.experts``).

Four operators around an AllToAll of tokens: the router's choice (top-k softmax, with its gradient), tokens
sorted by expert and copied to their rows (with the gradient), the experts' rows weighted and summed back per
token (with both gradients), and the experts' matrix-vector products with 4-bit weights and group scales.  With
``own`` false ``run`` computes them from elementary torch operations in 32 bits, with ``own`` true it makes the
framework's calls.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one decoded token: latency only
        dict(name="route one token", kind="route", tokens=1, experts=128, k=8, dtype="bf16", renorm=True, train=False),
        # a training micro-batch of a fine-grained mixture, with the router's gradient
        dict(name="route training", kind="route", tokens=16384, experts=256, k=8, dtype="fp32", renorm=False, train=True),
        # a few decoded tokens on their way to the experts
        dict(name="dispatch decode", kind="dispatch", tokens=4, experts=64, k=8, hidden=4096, capacity=0, pad=0,
             dtype="bf16", train=False),
        # the largest: a training micro-batch, every assignment kept, forward and backward
        dict(name="dispatch training", kind="dispatch", tokens=16384, experts=128, k=8, hidden=4096, capacity=0, pad=0,
             dtype="bf16", train=True),
        # odd sizes in the equal parts of an AllToAll: experts with a capacity, padded tokens, rows that stay empty
        dict(name="dispatch odd capacity", kind="dispatch", tokens=4099, experts=60, k=6, hidden=1030, capacity=512,
             pad=131, dtype="fp32", train=True),
        # one decoded token's experts summed
        dict(name="combine one token", kind="combine", tokens=1, experts=64, k=8, hidden=4096, capacity=0, pad=0,
             dtype="bf16", train=False),
        # training, forward and both gradients
        dict(name="combine training", kind="combine", tokens=8192, experts=64, k=8, hidden=2048, capacity=0, pad=0,
             dtype="bf16", train=True),
        # odd sizes with a capacity that drops some rows
        dict(name="combine odd capacity", kind="combine", tokens=4097, experts=48, k=3, hidden=1544, capacity=256,
             pad=65, dtype="fp16", train=True),
        # one decoded token: each of its 8 experts reads a whole matrix for one row
        dict(name="product one token", kind="product", rows=8, active=8, experts=64, n=4096, inner=4096, group=128,
             dtype="bf16"),
        # a small ragged batch: odd output size, the smallest groups
        dict(name="product ragged", kind="product", rows=37, active=13, experts=16, n=2051, inner=2080, group=32,
             dtype="fp16"),
        # a decode batch that touches every expert
        dict(name="product decode batch", kind="product", rows=256, active=32, experts=32, n=2048, inner=4096,
             group=128, dtype="bf16"),
        # a short prompt: many rows an expert
        dict(name="product prompt", kind="product", rows=1024, active=8, experts=8, n=1024, inner=2048, group=64,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["route", "dispatch", "combine", "product"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "route":
        experts = _log(rng, 4, 512)
        return dict(kind=kind, tokens=_log(rng, 1, 16384), experts=experts, k=rng.randint(1, min(8, experts)),
                    dtype=dtype, renorm=rng.random() < 0.5, train=rng.random() < 0.5)
    if kind == "product":
        group = rng.choice([32, 64, 128])
        inner = group * _log(rng, 4, 4096 // group)
        n = _log(rng, 64, 4096)
        experts = _log(rng, 1, 64)
        rows = min(_log(rng, 1, 1024), max(1, (1 << 31) // (n * inner)))
        return dict(kind=kind, rows=rows, active=rng.randint(1, min(rows, experts)), experts=experts, n=n, inner=inner,
                    group=group, dtype=rng.choice(["bf16", "fp16"]))
    experts = _log(rng, 4, 256)
    k = rng.randint(1, min(8, experts))
    hidden = _log(rng, 64, 4096)
    if rng.random() < 0.7:
        hidden = max(64, hidden // 64 * 64)
    tokens = _log(rng, 1, 16384)
    pad = rng.choice([0, tokens // 9])
    capacity = max(1, round(tokens * k / experts * rng.uniform(0.7, 1.5))) if rng.random() < 0.4 else 0
    if tokens * k * hidden * BYTES[dtype] > (1 << 30):
        tokens = (1 << 30) // (k * hidden * BYTES[dtype])
        pad, capacity = min(pad, tokens // 9), 0
    return dict(kind=kind, tokens=tokens, experts=experts, k=k, hidden=hidden, capacity=capacity, pad=pad, dtype=dtype,
                train=rng.random() < 0.6)


# -- inputs -----------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def _choices(g, case):
    """Distinct experts per token, some experts more popular than others; the padded last tokens have none (-1)."""
    t, e, k = case["tokens"], case["experts"], case["k"]
    popular = 0.5 * torch.randn(e, device="cuda", generator=g)
    noise = -torch.log(-torch.log(torch.rand(t, e, device="cuda", generator=g).clamp_(1e-9, 1 - 1e-7)))
    ids = (popular + noise).topk(k, dim=1).indices.to(torch.int32)
    if case["pad"]:
        ids[t - case["pad"]:] = -1
    return ids


def _rows(case):
    return case["experts"] * case["capacity"] if case["capacity"] else case["tokens"] * case["k"]


def prepare(case, seed):
    g, dtype, kind = _generator(seed), DTYPES[case["dtype"]], case["kind"]
    state = dict(case)
    if kind == "route":
        state["logits"] = _normal(g, (case["tokens"], case["experts"]), dtype, 2.0)
        state["grad"] = _normal(g, (case["tokens"], case["k"]), torch.float32)
    elif kind == "dispatch":
        state["ids"] = _choices(g, case)
        state["x"] = _normal(g, (case["tokens"], case["hidden"]), dtype)
        if case["train"]:
            state["grad"] = _normal(g, (_rows(case), case["hidden"]), dtype)
    elif kind == "combine":
        # a user has the order from the dispatch before it
        slot, source, counts, starts = _order(_choices(g, case), case["experts"], case["capacity"])
        state.update(slot=slot, source=source, counts=counts, starts=starts)
        state["rows"] = _normal(g, (_rows(case), case["hidden"]), dtype)
        state["weights"] = torch.rand(case["tokens"], case["k"], device="cuda", generator=g)
        if case["train"]:
            state["grad"] = _normal(g, (case["tokens"], case["hidden"]), dtype)
    else:
        e, n, inner, groups = case["experts"], case["n"], case["inner"], case["inner"] // case["group"]
        chosen = torch.randperm(e, device="cuda", generator=g)[:case["active"]]
        extra = torch.randint(0, case["active"], (case["rows"] - case["active"],), device="cuda", generator=g)
        counts = torch.zeros(e, dtype=torch.int32, device="cuda")
        counts[chosen] = 1
        counts.scatter_add_(0, chosen[extra], torch.ones_like(extra, dtype=torch.int32))
        state["counts"] = counts
        state["starts"] = (counts.cumsum(0) - counts).to(torch.int32)
        state["rows_in"] = _normal(g, (case["rows"], inner), dtype)
        # two 4-bit values a byte, the even inner index in the low half; value = (q - 8) * scale
        state["packed"] = torch.randint(0, 256, (e, n, inner // 2), dtype=torch.uint8, device="cuda", generator=g)
        state["scales"] = (0.004 + 0.016 * torch.rand(e, n, groups, device="cuda", generator=g)).to(dtype)
    return state


# -- the plain forms --------------------------------------------------------------------------------------

def _order(ids, experts, capacity):
    """(slot, source, counts, starts): rows by expert, in each expert by the assignment's number."""
    flat = ids.reshape(-1).long()
    a = flat.numel()
    known = (flat >= 0) & (flat < experts)
    key = torch.where(known, flat, experts)
    number = torch.arange(a, device=flat.device)
    sorted_key, perm = torch.sort(key, stable=True)
    total = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device).scatter_add_(0, key, torch.ones_like(key))
    first = total.cumsum(0) - total
    place = number - first[sorted_key]
    kept = sorted_key < experts
    if capacity:
        kept = kept & (place < capacity)
        starts = torch.arange(experts, device=flat.device) * capacity
        counts, rows = total[:experts].clamp(max=capacity), experts * capacity
    else:
        starts, counts, rows = first[:experts], total[:experts], a
    row = torch.where(kept, starts[sorted_key.clamp(max=experts - 1)] + place, -1)
    slot = torch.empty_like(flat).scatter_(0, perm, row)
    # a row more than there are takes what is not kept
    source = torch.full((rows + 1,), -1, dtype=torch.int64, device=flat.device)
    source.scatter_(0, torch.where(kept, row, rows), perm)
    source = source[:rows]
    return slot.view(ids.shape).int(), source.int(), counts.int(), starts.int()


def _gather(rows, slot):
    """rows[slot] in 32 bits, zero where the slot is -1."""
    got = rows.float()[slot.clamp(min=0).long()]
    return torch.where((slot >= 0)[..., None], got, 0.0)


def _plain_route(s):
    logits = s["logits"].float()
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :s["k"]]
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    if s["renorm"]:
        chosen = logits.gather(1, ids)
        w = torch.exp(chosen - chosen.amax(1, keepdim=True))
        w = w / w.sum(1, keepdim=True)
    else:
        w = p.gather(1, ids)
    out = {"ids": ids.int(), "weights": w}
    if s["train"]:
        inner = (s["grad"] * w).sum(1, keepdim=True)
        if s["renorm"]:
            grad = torch.zeros_like(logits).scatter_(1, ids, w * (s["grad"] - inner))
        else:
            grad = p * (torch.zeros_like(logits).scatter_(1, ids, s["grad"]) - inner)
        out["grad_logits"] = grad.to(s["logits"].dtype)
    return out


def _plain_dispatch(s):
    slot, source, counts, starts = _order(s["ids"], s["experts"], s["capacity"])
    x = s["x"]
    token = torch.where(source >= 0, source // s["k"], -1)
    out = {"slot": slot, "source": source, "counts": counts, "starts": starts,
           "rows": _gather(x, token).to(x.dtype)}
    if s["train"]:
        out["grad_x"] = _gather(s["grad"], slot).sum(1).to(x.dtype)
    return out


def _plain_combine(s):
    rows, w, slot, source = s["rows"], s["weights"], s["slot"], s["source"]
    got = _gather(rows, slot)
    out = {"out": (got * w[..., None]).sum(1).to(rows.dtype)}
    if s["train"]:
        grad = s["grad"].float()
        out["grad_weights"] = (got * grad[:, None]).sum(2)
        number = source.clamp(min=0).long()
        scaled = grad[number // s["k"]] * w.reshape(-1)[number][:, None]
        out["grad_rows"] = torch.where((source >= 0)[:, None], scaled, 0.0).to(rows.dtype)
    return out


def _dequantized(packed, scales, group):
    q = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2).float() - 8.0
    return (q.unflatten(-1, (-1, group)) * scales.float()[..., None]).flatten(-2)


def _plain_product(s):
    x, number = s["rows_in"], torch.arange(s["rows"], device="cuda")[:, None]
    expert = ((number >= s["starts"]) & (number < s["starts"] + s["counts"])).int().argmax(1)
    if s["rows"] < s["experts"]:       # fewer rows than matrices: only the rows' own matrices are opened
        w = _dequantized(s["packed"][expert], s["scales"][expert], s["group"])
    else:
        w = _dequantized(s["packed"], s["scales"], s["group"])[expert]
    return {"out": torch.bmm(w, x.float()[..., None])[..., 0].to(x.dtype)}


PLAIN = {"route": _plain_route, "dispatch": _plain_dispatch, "combine": _plain_combine, "product": _plain_product}


# -- the framework's calls --------------------------------------------------------------------------------

def _own_route(s):
    from vericcl_b200.ops import experts
    ids, w = experts.route(s["logits"], s["k"], renormalize=s["renorm"])
    out = {"ids": ids, "weights": w}
    if s["train"]:
        out["grad_logits"] = experts.route_backward(s["logits"], ids, w, s["grad"], renormalize=s["renorm"])
    return out


def _own_dispatch(s):
    from vericcl_b200.ops import experts
    order = experts.sort_by_expert(s["ids"], s["experts"], capacity=s["capacity"] or None)
    out = {"slot": order.slot, "source": order.source, "counts": order.counts, "starts": order.starts,
           "rows": experts.dispatch(s["x"], order)}
    if s["train"]:
        out["grad_x"] = experts.dispatch_backward(s["grad"], order)
    return out


def _own_combine(s):
    from vericcl_b200.ops import experts
    order = experts.ExpertOrder(s["slot"], s["source"], s["counts"], s["starts"])
    out = {"out": experts.combine(s["rows"], s["weights"], order)}
    if s["train"]:
        out["grad_rows"], out["grad_weights"] = experts.combine_backward(s["grad"], s["rows"], s["weights"], order)
    return out


def _own_product(s):
    from vericcl_b200.ops import experts
    return {"out": experts.expert_matmul_int4(s["rows_in"], s["starts"], s["counts"], s["packed"], s["scales"])}


OWN = {"route": _own_route, "dispatch": _own_dispatch, "combine": _own_combine, "product": _own_product}


def run(state):
    return (OWN if own else PLAIN)[state["kind"]](state)


# -- floors and 64-bit values -----------------------------------------------------------------------------

def work(case):
    b = BYTES[case["dtype"]]
    if case["kind"] == "product":
        n, inner, groups = case["n"], case["inner"], case["inner"] // case["group"]
        return {"bytes": case["active"] * n * (inner // 2 + groups * b) + case["rows"] * (inner + n) * b
                + 8 * case["experts"], "flops": 2.0 * case["rows"] * n * inner}
    t, k = case["tokens"], case["k"]
    if case["kind"] == "route":
        e = case["experts"]
        grad = t * (e * b + 4 * k) if case["train"] else 0
        return {"bytes": t * e * b + 8 * t * k + grad, "flops": t * e * (10.0 if case["train"] else 4.0)}
    h, rows = case["hidden"], _rows(case)
    kept = min((t - case["pad"]) * k, rows)
    if case["kind"] == "dispatch":
        grad = (kept + t) * h * b if case["train"] else 0
        return {"bytes": 8 * t * k + 4 * rows + 8 * case["experts"] + (t + rows) * h * b + grad,
                "flops": float(2 * t * k + (kept * h if case["train"] else 0))}
    grad = (t + rows) * h * b + 4 * t * k + 4 * rows if case["train"] else 0
    return {"bytes": 8 * t * k + (kept + t) * h * b + grad, "flops": kept * h * (5.0 if case["train"] else 2.0)}


def exact(case, seed):
    s = prepare(case, seed)
    k = s.get("k")
    if s["kind"] == "route":
        x = s["logits"].double()
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
        taken = torch.zeros_like(x).scatter_(1, ids, 1.0)
        share = torch.softmax(x.masked_fill(taken == 0, -math.inf) if s["renorm"] else x, dim=1)
        out = {"ids": None, "weights": share.gather(1, ids)}
        if s["train"]:
            up = torch.zeros_like(x).scatter_(1, ids, s["grad"].double())
            out["grad_logits"] = share * up - share * (share * up).sum(1, keepdim=True)
        return out
    if s["kind"] == "product":
        outs = torch.zeros(s["rows"], s["n"], dtype=torch.float64, device="cuda")
        starts, counts = s["starts"].tolist(), s["counts"].tolist()
        for e in range(s["experts"]):
            if counts[e]:
                w = torch.empty(s["n"], s["inner"], dtype=torch.float64, device="cuda")
                w[:, 0::2], w[:, 1::2] = (s["packed"][e] % 16).double() - 8, (s["packed"][e] // 16).double() - 8
                w *= s["scales"][e].double().repeat_interleave(s["group"], dim=1)
                at = slice(starts[e], starts[e] + counts[e])
                outs[at] = s["rows_in"][at].double() @ w.T
        return {"out": outs}
    t, h = s["tokens"], s["hidden"]
    if s["kind"] == "dispatch":
        ids = s["ids"].reshape(-1).cpu().numpy()
        starts, taken, slot = [], [0] * s["experts"], [-1] * len(ids)
        known = [0] * s["experts"]
        for i in ids.tolist():
            if i >= 0:
                known[i] += 1
        for e in range(s["experts"]):
            starts.append(e * s["capacity"] if s["capacity"] else sum(known[:e]))
        for a, i in enumerate(ids.tolist()):
            if i >= 0 and (not s["capacity"] or taken[i] < s["capacity"]):
                slot[a] = starts[i] + taken[i]
                taken[i] += 1
        slot = torch.tensor(slot, device="cuda")
        out = {"slot": None, "source": None, "counts": None, "starts": None,
               "rows": torch.zeros(_rows(case), h, dtype=torch.float64, device="cuda")}
        kept = (slot >= 0).nonzero()[:, 0]
        out["rows"][slot[kept]] = s["x"].double()[kept // k]
        if s["train"]:
            out["grad_x"] = torch.zeros(t, h, dtype=torch.float64, device="cuda")
            out["grad_x"].index_add_(0, kept // k, s["grad"][slot[kept]].double())
        return out
    flat, w = s["slot"].reshape(-1).long(), s["weights"].double().reshape(-1)
    kept = (flat >= 0).nonzero()[:, 0]
    rows = s["rows"][flat[kept]].double()
    out = {"out": torch.zeros(t, h, dtype=torch.float64, device="cuda")}
    out["out"].index_add_(0, kept // k, rows * w[kept][:, None])
    if s["train"]:
        grad = s["grad"].double()[kept // k]
        out["grad_rows"] = torch.zeros(_rows(case), h, dtype=torch.float64, device="cuda")
        out["grad_rows"][flat[kept]] = grad * w[kept][:, None]
        out["grad_weights"] = torch.zeros(t * k, dtype=torch.float64, device="cuda")
        out["grad_weights"][kept] = (grad * rows).sum(1)
        out["grad_weights"] = out["grad_weights"].view(t, k)
    return out
