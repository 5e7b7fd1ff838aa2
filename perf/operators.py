"""What is measured of the routed operators: rows that are each multiplied by the matrix they are routed to.

Four operators, each with its plain torch form, its 64-bit definition and the call a user makes:

    route     a router's choice of experts per row, the weights, and the rows listed by expert     (+ gradient)
    product   every routed row times its expert's matrix                                           (+ both gradients)
    combine   the weighted sum of the rows an input row was routed to                              (+ both gradients)
    adapters  a shared projection plus the low-rank pair of the adapter each row asks for          (+ gradients)

A case is a dict of plain values; `op` names the operator and `grad` its backward pass.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------------ cases

def _route(name, rows, experts, top, dtype, score="softmax", bias=False, groups=1, top_groups=1, group_top=1, renorm=True, scale=1.0,
           masked=False, grad=False):
    return dict(name=name, op="route", rows=rows, experts=experts, top=top, dtype=dtype, score=score, bias=bias, groups=groups,
                top_groups=top_groups, group_top=group_top, renorm=renorm, scale=scale, masked=masked, grad=grad)


def _product(name, rows, experts, top, k, n, dtype, padded=False, grad=False):
    return dict(name=name, op="product", rows=rows, experts=experts, top=top, k=k, n=n, dtype=dtype, padded=padded, grad=grad)


def _combine(name, rows, top, dim, dtype, padded=False, grad=False):
    return dict(name=name, op="combine", rows=rows, top=top, dim=dim, dtype=dtype, padded=padded, grad=grad)


def _adapters(name, rows, adapters, rank, k, n, dtype, single, grad=False):
    return dict(name=name, op="adapters", rows=rows, adapters=adapters, rank=rank, k=k, n=n, dtype=dtype, single=single, grad=grad)


def listed():
    return [
        # one generated token asks 64 experts for 8: nothing but latency
        _route("route_token", 1, 64, 8, "bf16"),
        # a long prompt under the grouped choice with a balancing bias: 8 groups, 4 of them kept
        _route("route_prompt", 16384, 256, 8, "f32", "sigmoid", True, 8, 4, 2, True, 2.5),
        # a training batch of odd length, 60 experts of which a few are masked out, weights not renormalised
        _route("route_grad", 4099, 60, 4, "f16", renorm=False, masked=True, grad=True),
        # a small batch of generated tokens: the experts' matrices are read once each and bound it
        _product("product_tokens", 8, 64, 4, 2048, 1024, "bf16"),
        # a long prompt: every expert has about a thousand rows, the arithmetic bounds it
        _product("product_prompt", 8192, 32, 4, 2048, 2048, "bf16"),
        # odd numbers of rows and experts, widths that end inside every tile, padded rows
        _product("product_odd", 1003, 17, 2, 1000, 712, "f16", padded=True),
        # the backward pass of a training step: the rows' gradient and the matrices'
        _product("product_grad", 4096, 16, 2, 1024, 2048, "bf16", padded=True, grad=True),
        # the sum over a long prompt's four experts per token: moves bytes only
        _combine("combine_prompt", 16384, 4, 2048, "bf16"),
        # its gradient on an odd batch: rows' and weights' gradients in one pass
        _combine("combine_grad", 5001, 2, 1000, "f16", padded=True, grad=True),
        # one generated token for each of 64 requests, 24 adapters in use among them
        _adapters("adapters_tokens", 64, 24, 16, 4096, 4096, "bf16", True),
        # prompts of several requests beside one another, some without an adapter
        _adapters("adapters_prompt", 4096, 8, 64, 4096, 4096, "bf16", False),
        # training several adapters in one odd batch
        _adapters("adapters_grad", 2500, 5, 8, 2048, 1024, "f16", False, grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    op = rng.choice(["route", "product", "product", "combine", "adapters", "adapters"])
    grad = rng.random() < 0.35
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        per = _log(rng, 8 if groups == 1 else 4, 512 // groups)
        experts = groups * per
        top_groups = rng.randint(1, groups)
        top = rng.randint(1, min(16, top_groups * per))
        return _route(None, _log(rng, 1, 16384), experts, top, rng.choice(["f32", "f16", "bf16"]), rng.choice(["softmax", "sigmoid"]),
                      rng.random() < 0.5, groups, top_groups, rng.choice([1, 2]), rng.random() < 0.6, rng.choice([1.0, 2.5]),
                      rng.random() < 0.3, grad)
    if op == "product":
        experts = _log(rng, 2, 128)
        return _product(None, _log(rng, 1, 8192), experts, min(rng.choice([1, 2, 4, 8]), experts), 8 * _log(rng, 8, 512),
                        8 * _log(rng, 8, 512), rng.choice(["f16", "bf16"]), rng.random() < 0.3, grad)
    if op == "combine":
        return _combine(None, _log(rng, 1, 16384), rng.choice([1, 2, 4, 8]), _log(rng, 16, 4096), rng.choice(["f32", "f16", "bf16"]),
                        rng.random() < 0.3, grad)
    single = rng.random() < 0.5
    return _adapters(None, _log(rng, 1, 256 if single else 4096), _log(rng, 1, 64), 8 * rng.randint(1, 8), 8 * _log(rng, 16, 512),
                     8 * _log(rng, 16, 512), rng.choice(["f16", "bf16"]), single, grad)


def draw(rng):
    largest = {key: max(work(case)[key] for case in listed()) for key in ("bytes", "flops")}
    while True:  # a case that would cost more than the largest listed one is drawn again
        case = _draw_once(rng)
        cost = work(case)
        if all(cost[key] <= largest[key] for key in largest):
            return case


# ------------------------------------------------------------------------------------------------ inputs

def _groups_of(ids, n_groups):
    """Rows listed by group: where each group starts, the row behind every slot, the slot of every (row, choice)."""
    flat = ids.reshape(-1).to(torch.int64)
    key = torch.where(flat < 0, torch.full_like(flat, n_groups), flat)
    order = torch.sort(key, stable=True).indices
    counts = torch.bincount(key, minlength=n_groups + 1)
    ptr = torch.zeros(n_groups + 1, dtype=torch.int64, device=ids.device)
    ptr[1:] = torch.cumsum(counts[:n_groups], 0)
    place = torch.arange(flat.numel(), device=ids.device)
    used = place < ptr[-1]
    per_row = ids.numel() // ids.shape[0]
    row = torch.where(used, order // per_row, torch.full_like(order, -1))
    slot = torch.empty_like(order)
    slot[order] = torch.where(used, place, torch.full_like(place, -1))
    return ptr.to(torch.int32), row.to(torch.int32), slot.to(torch.int32).reshape(ids.shape)


def _choices(case, gen):
    """Experts of every row, some far more popular than others; a padded batch ends in rows that ask for none."""
    rows, experts, top = case["rows"], case["experts"], case["top"]
    popularity = -0.4 * torch.log(torch.arange(1, experts + 1, device="cuda", dtype=torch.float32))
    popularity = popularity[torch.randperm(experts, generator=gen, device="cuda")]
    noise = -torch.log(-torch.log(torch.rand(rows, experts, generator=gen, device="cuda").clamp(1e-9, 1 - 1e-7)))
    ids = torch.topk(popularity + noise, top, dim=1).indices.to(torch.int32)
    if case["padded"]:
        ids[rows - rows // 16:] = -1
    return ids


def _normal(gen, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "route":
        rows, experts = case["rows"], case["experts"]
        logits = torch.randn(rows, experts, generator=gen, device="cuda") * 1.5
        if case["masked"]:  # experts that are switched off, and rows of padding that may choose none
            logits[:, torch.rand(experts, generator=gen, device="cuda") < 0.1] = -math.inf
            logits[rows - rows // 32:] = -math.inf
        state["logits"] = logits.to(dtype)
        state["bias"] = torch.randn(experts, generator=gen, device="cuda") * 0.05 if case["bias"] else None
        if case["grad"]:
            state["ids"] = _route_plain(case, state["logits"], state["bias"])[0]
            state["d_weights"] = torch.randn(rows, case["top"], generator=gen, device="cuda")
    elif case["op"] == "product":
        ids = _choices(case, gen)
        state["ptr"], state["row"], state["slot"] = _groups_of(ids, case["experts"])
        slots = ids.numel()
        state["x"] = _normal(gen, dtype, case["rows"], case["k"])
        state["w"] = torch.empty(case["experts"], case["n"], case["k"], dtype=dtype, device="cuda")
        for e in range(case["experts"]):
            state["w"][e] = _normal(gen, dtype, case["n"], case["k"], scale=case["k"] ** -0.5)
        if case["grad"]:
            state["dy"] = _normal(gen, dtype, slots, case["n"], scale=0.1)
            state["out_x"] = torch.zeros(slots, case["k"], dtype=dtype, device="cuda")
            state["out_w"] = torch.zeros_like(state["w"])
        else:
            state["out"] = torch.zeros(slots, case["n"], dtype=dtype, device="cuda")
    elif case["op"] == "combine":
        ids = _choices(dict(case, experts=max(16, case["top"])), gen)
        _, _, state["slot"] = _groups_of(ids, max(16, case["top"]))
        slots = ids.numel()
        state["rows"] = _normal(gen, dtype, slots, case["dim"])
        weights = torch.rand(case["rows"], case["top"], generator=gen, device="cuda") + 0.05
        state["weights"] = weights / weights.sum(1, keepdim=True)
        if case["grad"]:
            state["dy"] = _normal(gen, dtype, case["rows"], case["dim"], scale=0.1)
            state["out_rows"] = torch.zeros_like(state["rows"])
    else:
        rows, n_adapters = case["rows"], case["adapters"]
        if case["single"]:
            ids = torch.randint(-1, n_adapters, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        else:  # requests beside one another, of about equal length, each with an adapter of its own or none
            requests = min(rows, 2 * n_adapters)
            cut = torch.sort(torch.rand(requests, generator=gen, device="cuda")).values
            cut[0] = 0
            asks = torch.randint(-1, n_adapters, (requests,), generator=gen, device="cuda", dtype=torch.int32)
            at = torch.arange(rows, device="cuda", dtype=torch.float32) / rows
            ids = asks[torch.searchsorted(cut, at, right=True) - 1]
        state["ids"] = ids.contiguous()
        state["ptr"], state["row"], state["slot"] = _groups_of(ids, n_adapters)
        state["x"] = _normal(gen, dtype, rows, case["k"])
        state["w"] = _normal(gen, dtype, case["n"], case["k"], scale=case["k"] ** -0.5)
        state["a"] = _normal(gen, dtype, n_adapters, case["rank"], case["k"], scale=case["k"] ** -0.5)
        state["b"] = _normal(gen, dtype, n_adapters, case["n"], case["rank"], scale=case["rank"] ** -0.5)
        state["scale"] = torch.rand(n_adapters, generator=gen, device="cuda") + 0.5
        if case["grad"]:
            state["dy"] = _normal(gen, dtype, rows, case["n"], scale=0.1)
    return state


# ------------------------------------------------------------------------------------------------ plain forms

def _pick(key, count):
    """Columns of the `count` largest keys of each row in falling order, the lowest column first among equals; -1 where
    nothing above -inf is left."""
    key = key.clone()
    column = torch.arange(key.shape[1], device=key.device)
    out = []
    for _ in range(count):
        best = key.max(1, keepdim=True).values
        at = torch.where(key == best, column, key.shape[1]).min(1).values
        out.append(torch.where(best[:, 0] > -math.inf, at, -1))
        key[torch.arange(key.shape[0], device=key.device), at] = -math.inf
    return torch.stack(out, 1)


def _scores(case, logits):
    if case["score"] == "sigmoid":
        return 1 / (1 + torch.exp(-logits))
    top = logits.max(1, keepdim=True).values
    e = torch.exp(logits - torch.where(top > -math.inf, top, 0))
    total = e.sum(1, keepdim=True)
    return e / torch.where(total > 0, total, 1)


def _route_plain(case, logits, bias):
    wide = logits.double()  # the choice between close candidates needs more than 32 bits
    score = _scores(case, wide)
    key = wide if bias is None else torch.where(wide > -math.inf, score + bias.double(), -math.inf)
    if case["groups"] > 1:
        rows, groups = key.shape[0], case["groups"]
        member = key.reshape(rows, groups, -1)
        if case["group_top"] == 2:
            value = torch.where(key > -math.inf, score if bias is None else key, -math.inf).reshape(rows, groups, -1)
            first = value.max(2, keepdim=True).values
            column = torch.arange(value.shape[2], device=key.device)
            at = torch.where(value == first, column, value.shape[2]).min(2, keepdim=True).values
            second = torch.where(column == at, -math.inf, value).max(2).values
            group_key = first[:, :, 0] + torch.where(second > -math.inf, second, 0)
        else:
            group_key = member.max(2).values
        kept = _pick(group_key, case["top_groups"])
        keep = (kept[:, :, None] == torch.arange(groups, device=key.device)).any(1)
        key = torch.where(keep[:, :, None], member, -math.inf).reshape(rows, -1)
    ids = _pick(key, case["top"])
    chosen = ids >= 0
    weights = torch.where(chosen, _scores(case, logits.float()).gather(1, ids.clamp(min=0)), 0)
    if case["renorm"]:
        total = weights.sum(1, keepdim=True)
        weights = weights / torch.where(total > 0, total, 1)
    return ids.to(torch.int32), (weights * case["scale"]).float()


def _route_grad_plain(case, logits, ids, d_weights):
    score = _scores(case, logits.float())
    chosen = ids >= 0
    at = ids.clamp(min=0).long()
    d = torch.where(chosen, d_weights, 0) * case["scale"]
    s = torch.where(chosen, score.gather(1, at), 0)
    if case["renorm"]:
        total = s.sum(1, keepdim=True)
        total = torch.where(total > 0, total, 1)
        d = (d - (d * s).sum(1, keepdim=True) / total) / total
    d_score = torch.zeros_like(score).scatter_add(1, at, torch.where(chosen, d, 0))
    if case["score"] == "sigmoid":
        out = d_score * score * (1 - score)
    else:
        out = score * (d_score - (d_score * score).sum(1, keepdim=True))
    return out.to(logits.dtype)


def _product_plain(state):
    x, w, row = state["x"], state["w"], state["row"]
    bounds = state["ptr"].tolist()
    out = torch.zeros(row.numel(), w.shape[1], dtype=torch.float32, device=x.device)
    for e in range(w.shape[0]):
        lo, hi = bounds[e], bounds[e + 1]
        if hi > lo:
            out[lo:hi] = x[row[lo:hi].long()].float() @ w[e].float().t()
    return out.to(x.dtype)


def _product_grad_plain(state):
    x, w, row, dy = state["x"], state["w"], state["row"], state["dy"]
    bounds = state["ptr"].tolist()
    dx = torch.zeros(row.numel(), w.shape[2], dtype=torch.float32, device=x.device)
    dw = torch.zeros_like(w)
    for e in range(w.shape[0]):
        lo, hi = bounds[e], bounds[e + 1]
        if hi > lo:
            d = dy[lo:hi].float()
            dx[lo:hi] = d @ w[e].float()
            dw[e] = (d.t() @ x[row[lo:hi].long()].float()).to(w.dtype)
    return dx.to(x.dtype), dw


def _combine_plain(rows, slot, weights):
    out = torch.zeros(slot.shape[0], rows.shape[1], dtype=torch.float32, device=rows.device)
    for j in range(slot.shape[1]):
        at = slot[:, j]
        term = rows[at.clamp(min=0).long()].float() * weights[:, j:j + 1]
        out += torch.where((at >= 0)[:, None], term, 0)
    return out.to(rows.dtype)


def _combine_grad_plain(dy, rows, slot, weights):
    d_rows, d_weights = torch.zeros_like(rows), torch.zeros_like(weights)
    wide = dy.float()
    for j in range(slot.shape[1]):
        used = torch.nonzero(slot[:, j] >= 0)[:, 0]
        at = slot[used, j].long()
        d_rows[at] = (wide[used] * weights[used, j:j + 1]).to(rows.dtype)
        d_weights[used, j] = (wide[used] * rows[at].float()).sum(1)
    return d_rows, d_weights


def _adapters_plain(state):
    x, ids = state["x"].float(), state["ids"]
    y = x @ state["w"].float().t()
    for i in range(state["a"].shape[0]):
        at = torch.nonzero(ids == i)[:, 0]
        y[at] += state["scale"][i] * ((x[at] @ state["a"][i].float().t()) @ state["b"][i].float().t())
    return y.to(state["x"].dtype)


def _adapters_grad_plain(state):
    x, dy, ids = state["x"].float(), state["dy"].float(), state["ids"]
    dx = dy @ state["w"].float()
    da, db = torch.zeros_like(state["a"]), torch.zeros_like(state["b"])
    for i in range(state["a"].shape[0]):
        at = torch.nonzero(ids == i)[:, 0]
        a, b = state["a"][i].float(), state["b"][i].float()
        v = state["scale"][i] * (dy[at] @ b)
        u = state["scale"][i] * (x[at] @ a.t())
        dx[at] += v @ a
        da[i] = (v.t() @ x[at]).to(da.dtype)
        db[i] = (dy[at].t() @ u).to(db.dtype)
    return dx.to(state["x"].dtype), da, db


# ------------------------------------------------------------------------------------------------ one pass

def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


def run(state):
    case = state["case"]
    op, grad = case["op"], case["grad"]
    if own:
        mps = _package()
        if op == "route":
            if grad:
                return mps.route_backward(state["logits"], state["ids"], state["d_weights"], score=case["score"], renormalise=case["renorm"],
                                          scale=case["scale"])
            ids, weights, groups = mps.route(state["logits"], case["top"], score=case["score"], bias=state["bias"], n_groups=case["groups"],
                                             top_groups=case["top_groups"], group_top=case["group_top"], renormalise=case["renorm"],
                                             scale=case["scale"])
            return ids, weights, groups.ptr, groups.row, groups.slot
        if op == "product":
            groups = mps.Groups(state["ptr"], state["row"], state["slot"])
            if grad:
                return (mps.routed_product(state["dy"], state["w"], groups, gather=False, transpose=True, out=state["out_x"]),
                        mps.routed_wgrad(state["x"], state["dy"], groups, out=state["out_w"]))
            return mps.routed_product(state["x"], state["w"], groups, out=state["out"])
        if op == "combine":
            if grad:
                return mps.routed_combine_backward(state["dy"], state["rows"], state["slot"], state["weights"], out=state["out_rows"])
            return mps.routed_combine(state["rows"], state["slot"], state["weights"])
        groups = mps.Groups(state["ptr"], state["row"], state["slot"])
        if grad:
            return mps.adapters_backward(state["dy"], state["x"], state["w"], state["a"], state["b"], state["ids"], groups, state["scale"])
        return mps.adapters(state["x"], state["w"], state["a"], state["b"], state["ids"], groups, state["scale"])
    if op == "route":
        if grad:
            return _route_grad_plain(case, state["logits"], state["ids"], state["d_weights"])
        ids, weights = _route_plain(case, state["logits"], state["bias"])
        return (ids, weights) + _groups_of(ids, case["experts"])
    if op == "product":
        return _product_grad_plain(state) if grad else _product_plain(state)
    if op == "combine":
        if grad:
            return _combine_grad_plain(state["dy"], state["rows"], state["slot"], state["weights"])
        return _combine_plain(state["rows"], state["slot"], state["weights"])
    return _adapters_grad_plain(state) if grad else _adapters_plain(state)


# ------------------------------------------------------------------------------------------------ work

def _touched(groups, slots):
    """Groups that `slots` rows meet when they choose evenly."""
    return groups * (1 - (1 - 1 / groups) ** slots)


def work(case):
    s, rows = SIZE[case["dtype"]], case["rows"]
    if case["op"] == "route":
        experts, top = case["experts"], case["top"]
        if case["grad"]:
            return {"bytes": 2 * rows * experts * s + rows * top * 8, "flops": 10 * rows * experts}
        return {"bytes": rows * experts * s + 16 * rows * top + 4 * (experts + 1) + (4 * experts if case["bias"] else 0),
                "flops": 10 * rows * experts}
    if case["op"] == "product":
        slots, k, n = rows * case["top"], case["k"], case["n"]
        if case["padded"]:
            slots -= case["top"] * (rows // 16)
        weights = _touched(case["experts"], slots) * k * n * s
        if case["grad"]:  # dy, x and the matrices read, the rows' gradients written, and every matrix's
            return {"bytes": slots * n * s + rows * k * s + weights + slots * k * s + case["experts"] * k * n * s + 4 * slots,
                    "flops": 4 * slots * k * n}
        return {"bytes": min(rows, slots) * k * s + weights + slots * n * s + 4 * slots, "flops": 2 * slots * k * n}
    if case["op"] == "combine":
        slots, dim = rows * case["top"], case["dim"]
        if case["grad"]:
            return {"bytes": rows * dim * s + 2 * slots * dim * s + 12 * slots, "flops": 3 * slots * dim}
        return {"bytes": slots * dim * s + rows * dim * s + 8 * slots, "flops": 2 * slots * dim}
    k, n, r = case["k"], case["n"], case["rank"]
    pairs = _touched(case["adapters"], rows) * r * (k + n) * s
    if case["grad"]:
        return {"bytes": rows * n * s + rows * k * s + n * k * s + pairs + rows * k * s + case["adapters"] * r * (k + n) * s + 4 * rows,
                "flops": 2 * rows * k * n + 2 * rows * r * (3 * k + 2 * n)}
    return {"bytes": rows * k * s + n * k * s + pairs + rows * n * s + 4 * rows, "flops": 2 * rows * k * n + 2 * rows * r * (k + n)}


# ------------------------------------------------------------------------------------------------ 64 bits

def _ranked(key, count):
    """The `count` best columns per row by a stable sort of the negated keys, host arrays."""
    order = np.argsort(-key, axis=1, kind="stable")[:, :count]
    best = np.take_along_axis(key, order, 1)
    return np.where(best > -np.inf, order, -1)


def _score64(case, logits):
    with np.errstate(over="ignore", invalid="ignore"):
        if case["score"] == "sigmoid":
            return np.where(logits >= 0, 1 / (1 + np.exp(-np.abs(logits))), np.exp(-np.abs(logits)) / (1 + np.exp(-np.abs(logits))))
        peak = logits.max(1, keepdims=True)
        part = np.exp(logits - np.where(np.isfinite(peak), peak, 0))
        total = part.sum(1, keepdims=True)
        return np.divide(part, total, out=np.zeros_like(part), where=total > 0)


def _exact_route(case, state):
    logits = state["logits"].double().cpu().numpy()
    score = _score64(case, logits)
    rows, experts = logits.shape
    if case["grad"]:
        ids, d_w = state["ids"].cpu().numpy(), state["d_weights"].double().cpu().numpy()
        grad = np.zeros((rows, experts))
        line = np.arange(rows)[:, None]
        mask = ids >= 0
        at = np.where(mask, ids, 0)
        s = np.where(mask, score[line, at], 0)
        if case["renorm"]:
            share = np.divide(s, s.sum(1, keepdims=True), out=np.zeros_like(s), where=s.sum(1, keepdims=True) > 0)
            pull = case["scale"] * share * (d_w - (d_w * share).sum(1, keepdims=True))  # gradient by the logarithm of each score
            slope = 1 - score[line, at] if case["score"] == "sigmoid" else np.ones_like(s)
            np.add.at(grad, (np.broadcast_to(line, ids.shape)[mask], at[mask]), (pull * slope)[mask])
        else:
            pull = case["scale"] * d_w * s
            if case["score"] == "sigmoid":
                pull = pull * (1 - score[line, at])
            else:
                grad -= score * pull.sum(1, keepdims=True)
            np.add.at(grad, (np.broadcast_to(line, ids.shape)[mask], at[mask]), pull[mask])
        return torch.from_numpy(grad)
    open_ = logits > -np.inf
    key = logits if state["bias"] is None else np.where(open_, score + state["bias"].double().cpu().numpy(), -np.inf)
    if case["groups"] > 1:
        cells = key.reshape(rows, case["groups"], -1)
        if case["group_top"] == 2:
            value = np.where(open_, score, -np.inf).reshape(cells.shape) if state["bias"] is None else cells
            two = -np.sort(-value, axis=2)[:, :, :2]
            rank = two[:, :, 0] + (np.where(two[:, :, 1] > -np.inf, two[:, :, 1], 0) if two.shape[2] > 1 else 0)
        else:
            rank = cells.max(2)
        kept = _ranked(rank, case["top_groups"])
        allowed = np.zeros((rows, case["groups"] + 1), bool)
        np.put_along_axis(allowed, kept, True, 1)  # -1 marks the spare last column
        key = np.where(allowed[:, :case["groups"], None], cells, -np.inf).reshape(rows, experts)
    ids = _ranked(key, case["top"])
    weights = np.where(ids >= 0, np.take_along_axis(score, np.maximum(ids, 0), 1), 0)
    if case["renorm"]:
        total = weights.sum(1, keepdims=True)
        weights = np.divide(weights, total, out=np.zeros_like(weights), where=total > 0)
    flat = ids.reshape(-1)
    listed_ = np.concatenate([np.nonzero(flat == e)[0] for e in range(experts)])
    ptr = np.concatenate([[0], np.cumsum([(flat == e).sum() for e in range(experts)])])
    row, slot = np.full(flat.size, -1), np.full(flat.size, -1)
    row[:listed_.size] = listed_ // case["top"]
    slot[listed_] = np.arange(listed_.size)
    as_int = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32)
    return as_int(ids), torch.from_numpy(weights * case["scale"]), as_int(ptr), as_int(row), as_int(slot.reshape(ids.shape))


def exact(case, seed):
    state = prepare(case, seed)
    op, grad = case["op"], case["grad"]
    if op == "route":
        return _exact_route(case, state)
    if op == "product":
        ptr = state["ptr"].cpu().numpy()
        slots = state["row"].numel()
        gathered = state["x"].double()[state["row"].clamp(min=0).long()]
        if not grad:
            out = torch.zeros(slots, case["n"], dtype=torch.float64, device="cuda")
            for e in np.nonzero(np.diff(ptr))[0]:
                torch.matmul(gathered[ptr[e]:ptr[e + 1]], state["w"][int(e)].double().mT, out=out[ptr[e]:ptr[e + 1]])
            return out
        dx = torch.zeros(slots, case["k"], dtype=torch.float64, device="cuda")
        dw = torch.zeros(case["experts"], case["n"], case["k"], dtype=torch.float64, device="cuda")
        dy = state["dy"].double()
        for e in np.nonzero(np.diff(ptr))[0]:
            part = slice(int(ptr[e]), int(ptr[e + 1]))
            dx[part] = torch.einsum("sn,nk->sk", dy[part], state["w"][int(e)].double())
            dw[int(e)] = torch.einsum("sn,sk->nk", dy[part], gathered[part])
        return dx, dw
    if op == "combine":
        rows, weights = state["rows"].double(), state["weights"].double()
        live = state["slot"] >= 0
        if not grad:
            out = torch.zeros(case["rows"], case["dim"], dtype=torch.float64, device="cuda")
            line, choice = torch.nonzero(live, as_tuple=True)
            return out.index_add_(0, line, rows[state["slot"][live].long()] * weights[line, choice][:, None])
        dy = state["dy"].double()
        line, choice = torch.nonzero(live, as_tuple=True)
        at = state["slot"][live].long()
        d_rows = torch.zeros_like(rows)
        d_rows[at] = dy[line] * weights[line, choice][:, None]
        d_weights = torch.zeros_like(weights)
        d_weights[line, choice] = torch.einsum("pd,pd->p", dy[line], rows[at])
        return d_rows, d_weights
    x, w = state["x"].double(), state["w"].double()
    a, b, scale = state["a"].double(), state["b"].double(), state["scale"].double()
    live = [(i, torch.nonzero(state["ids"] == i).flatten()) for i in range(case["adapters"])]
    if not grad:
        y = torch.einsum("tk,nk->tn", x, w)
        for i, at in live:
            if at.numel():
                y.index_add_(0, at, x[at] @ (scale[i] * (b[i] @ a[i])).mT)  # the pair multiplied out
        return y
    dy = state["dy"].double()
    dx = torch.einsum("tn,nk->tk", dy, w)
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    for i, at in live:
        if at.numel():
            outer = scale[i] * torch.einsum("tn,tk->nk", dy[at], x[at])  # gradient by the pair's product b a
            dx.index_add_(0, at, dy[at] @ (scale[i] * (b[i] @ a[i])))
            da[i] = b[i].mT @ outer
            db[i] = outer @ a[i].mT
    return dx, da, db
