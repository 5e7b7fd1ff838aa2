"""Plain 64-bit forms of the routed operators on the CPU (numpy), and the tolerances their kernels are held to.

Every result r of a kernel is compared with its 64-bit value R by |r - R| <= half(type) |R| + sums * magnitude + floor: one
rounding to the stored type, and a fp32 sum of n terms whose every addition may lose one unit in the last place (2^-23 of at
most the sum of the magnitudes)."""
import math

import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
FLOOR = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half a step among the subnormals
# relative error of a low-rank intermediate kept as a pair of stored-type values: half a step of the rest after half a step
PAIR = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -16}


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def close(got, want, dtype, terms, magnitude, extra=0.0):
    got, want, magnitude = np.asarray(got, np.float64), np.asarray(want, np.float64), np.asarray(magnitude, np.float64)
    bound = HALF[dtype] * np.abs(want) + (terms + 2) * 2.0 ** -23 * (1 + HALF[dtype]) * magnitude + FLOOR[dtype] + extra
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.size} outside, first at {tuple(np.argwhere(bad)[0])}: got {got[bad][0]}, want {want[bad][0]}, "
                           f"bound {np.broadcast_to(bound, got.shape)[bad][0]}")


# ---------------------------------------------------------------------------------------------- routing

def _rank(key, count):
    """The `count` best of (index, key) above -inf, falling, the lowest index first among equals."""
    order = sorted((i for i in range(len(key)) if key[i] > -math.inf), key=lambda i: (-key[i], i))
    return order[:count]


def row_scores(l, score):
    live = [v for v in l if v > -math.inf]
    if score == "sigmoid":
        return [1 / (1 + math.exp(-v)) if v >= 0 else math.exp(v) / (1 + math.exp(v)) if v > -700 else 0.0 for v in l]
    peak = max(live, default=0.0)
    e = [math.exp(v - peak) if v > -math.inf else 0.0 for v in l]
    total = sum(e)
    return [v / total if total else 0.0 for v in e]


def route(logits, top_k, score="softmax", bias=None, n_groups=1, top_groups=1, group_top=1, renormalise=True, scale=1.0):
    rows, experts = logits.shape
    ids, weights = np.full((rows, top_k), -1), np.zeros((rows, top_k))
    for t in range(rows):
        nan = np.isnan(logits[t]).any()
        l = [-math.inf if math.isnan(v) else float(v) for v in logits[t]]
        s = row_scores(l, score)
        key = l if bias is None else [s[e] + float(bias[e]) if l[e] > -math.inf and not math.isnan(bias[e]) else -math.inf for e in range(experts)]
        if n_groups > 1:
            per = experts // n_groups
            rank = []
            for g in range(n_groups):
                if group_top == 2:
                    cell = sorted((s[e] if bias is None else key[e] for e in range(g * per, g * per + per) if key[e] > -math.inf), reverse=True)[:2]
                    rank.append(sum(cell) if cell else -math.inf)
                else:
                    rank.append(max(key[g * per:g * per + per]))
            kept = set(_rank(rank, top_groups))
            key = [key[e] if e // per in kept else -math.inf for e in range(experts)]
        chosen = _rank(key, top_k)
        ids[t, :len(chosen)] = chosen
        if renormalise and chosen:  # ratios of the scores, by their logarithms so that they hold where the scores underflow
            log = [l[e] if score == "softmax" else (-math.log1p(math.exp(-l[e])) if l[e] > -30 else l[e]) for e in chosen]
            part = [math.exp(v - max(log)) for v in log]
            w = [v / sum(part) for v in part]
        else:
            w = [s[e] for e in chosen]
        weights[t, :len(chosen)] = np.array(w) * scale
        if nan:
            weights[t] = np.nan
    return ids, weights


def route_grad(logits, ids, d_weights, score="softmax", renormalise=True, scale=1.0):
    out = np.zeros(logits.shape)
    for t in range(logits.shape[0]):
        s = np.array(row_scores(list(logits[t]), score))
        d = np.zeros_like(s)
        live = [j for j in range(ids.shape[1]) if ids[t, j] >= 0]
        total = sum(s[ids[t, j]] for j in live)
        for j in live:
            g = d_weights[t, j] * scale
            if renormalise:
                g = (g - sum(d_weights[t, i] * scale * s[ids[t, i]] for i in live) / total) / total if total else 0.0
            d[ids[t, j]] += g
        out[t] = d * s * (1 - s) if score == "sigmoid" else s * (d - (d * s).sum())
    return out


def group_rows(ids, n_groups):
    flat = np.asarray(ids).reshape(-1)
    per = flat.size // max(len(ids), 1) if flat.size else 1
    ptr, row, slot, at = [0], np.full(flat.size, -1), np.full(flat.size, -1), 0
    for g in range(n_groups):
        for i in np.nonzero(flat == g)[0]:
            row[at], slot[i] = i // per, at
            at += 1
        ptr.append(at)
    return np.array(ptr), row, slot.reshape(np.shape(ids))


# ---------------------------------------------------------------------------------------------- products

def product(x, w, ptr, row, out):
    """(y, magnitude); rows of `out` (and magnitude 0) outside the groups."""
    y, mag = np.array(out, np.float64), np.zeros(out.shape)
    for g in range(len(ptr) - 1):
        part = slice(ptr[g], ptr[g + 1])
        xs = x[row[part]]
        y[part], mag[part] = xs @ w[g].T, np.abs(xs) @ np.abs(w[g]).T
    return y, mag


def wgrad(x, dy, ptr, row):
    n_groups = len(ptr) - 1
    dw, mag = np.zeros((n_groups, dy.shape[1], x.shape[1])), np.zeros((n_groups, dy.shape[1], x.shape[1]))
    for g in range(n_groups):
        xs, d = x[row[ptr[g]:ptr[g + 1]]], dy[ptr[g]:ptr[g + 1]]
        dw[g], mag[g] = d.T @ xs, np.abs(d).T @ np.abs(xs)
    return dw, mag


def combine(rows, slot, weights):
    y, mag = np.zeros((slot.shape[0], rows.shape[1])), np.zeros((slot.shape[0], rows.shape[1]))
    for t, j in np.argwhere(slot >= 0):
        y[t] += weights[t, j] * rows[slot[t, j]]
        mag[t] += np.abs(weights[t, j] * rows[slot[t, j]])
    return y, mag


def combine_grad(dy, rows, slot, weights, out):
    d_rows, d_w, mag = np.array(out, np.float64), np.zeros(slot.shape), np.zeros(slot.shape)
    for t, j in np.argwhere(slot >= 0):
        d_rows[slot[t, j]] = weights[t, j] * dy[t]
        d_w[t, j], mag[t, j] = dy[t] @ rows[slot[t, j]], np.abs(dy[t]) @ np.abs(rows[slot[t, j]])
    return d_rows, d_w, mag


def adapters(x, w, a, b, ids, scale):
    """(y, magnitude of the sums, magnitude that an intermediate's relative error meets, sum of |b| that its floor meets)."""
    y, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    pair, ones = np.zeros_like(y), np.zeros_like(y)
    for i in range(len(a)):
        at = np.nonzero(ids == i)[0]
        u, um = scale[i] * (x[at] @ a[i].T), abs(scale[i]) * (np.abs(x[at]) @ np.abs(a[i]).T)
        y[at] += u @ b[i].T
        mag[at] += um @ np.abs(b[i]).T
        pair[at] = np.abs(u) @ np.abs(b[i]).T
        ones[at] = np.abs(b[i]).sum(1)
    return y, mag, pair, ones


def adapters_grad(dy, x, w, a, b, ids, scale):
    """dx, da, db, each with its three magnitudes as in adapters."""
    dx = adapters(dy, w.T, b.transpose(0, 2, 1), a.transpose(0, 2, 1), ids, scale)
    da, db = [np.zeros_like(a) for _ in range(4)], [np.zeros_like(b) for _ in range(4)]
    for i in range(len(a)):
        at = np.nonzero(ids == i)[0]
        u, um = scale[i] * (x[at] @ a[i].T), abs(scale[i]) * (np.abs(x[at]) @ np.abs(a[i]).T)
        v, vm = scale[i] * (dy[at] @ b[i]), abs(scale[i]) * (np.abs(dy[at]) @ np.abs(b[i]))
        da[0][i], da[1][i], da[2][i], da[3][i] = v.T @ x[at], vm.T @ np.abs(x[at]), np.abs(v).T @ np.abs(x[at]), np.abs(x[at]).sum(0)[None, :]
        db[0][i], db[1][i], db[2][i], db[3][i] = dy[at].T @ u, np.abs(dy[at]).T @ um, np.abs(dy[at]).T @ np.abs(u), np.abs(dy[at]).sum(0)[:, None]
    return dx, tuple(da), tuple(db)
