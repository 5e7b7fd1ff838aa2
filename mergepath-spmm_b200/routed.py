"""Rows that are each multiplied by the matrix they are routed to: experts, weights per node type, low-rank adapters.

The routing is kept as the rows listed by group (`Groups`): `ptr` is the row_ptr over groups, `row` the col_idx (the input row
in every slot), `slot` the slot of every (row, choice).  Thin wrappers of the mps_route* / mps_routed_* / mps_adapters* entry
points of include/mps.h over torch CUDA tensors (float32, float16 or bfloat16); no reference counterpart.  Results are not part
of an autograd graph, whatever the inputs ask for: gradients are functions of their own, which a user's autograd function calls.
`stream` is where a call runs and what it returns belongs to.  Nothing synchronises; `routed_check()`
waits and reports what the device met out of range.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import NamedTuple

from . import capi

try:
    import torch
except Exception:  # pragma: no cover
    torch = None

__all__ = ["Groups", "route", "route_backward", "group_rows", "routed_product", "routed_wgrad", "routed_combine", "routed_combine_backward",
           "adapters", "adapters_backward", "routed_check"]

_DTYPES = {} if torch is None else {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}


class Groups(NamedTuple):
    """Rows listed by group: int32 CUDA tensors ptr (groups + 1), row (slots, -1 behind the last one in use) and slot (the
    shape of the ids, -1 for none)."""
    ptr: "torch.Tensor"
    row: "torch.Tensor"
    slot: "torch.Tensor"


def _dtype(t) -> int:
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise ValueError(f"expected float32, float16 or bfloat16, got {t.dtype}")
    return d


def _is(t, dtype, shape, index) -> bool:
    """A contiguous tensor of that dtype and shape on CUDA device `index`, or None (not given)."""
    return t is None or (t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous())


def _explain(device, *named):
    """Raises for the first (name, tensor, dtype, shape) that is not what `_is` asks for."""
    for name, t, dtype, shape in named:
        if _is(t, dtype, shape, device.index):
            continue
        if not t.is_cuda:
            raise ValueError(f"{name}: expected a CUDA tensor (there is no CPU path)")
        if t.device != device:
            raise ValueError(f"{name}: on {t.device}, expected {device}")
        if not t.is_contiguous():
            raise ValueError(f"{name}: expected a contiguous tensor")
        if t.dtype != dtype:
            raise ValueError(f"{name}: expected {dtype}, got {t.dtype}")
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")


def _ptr(t):
    return None if t is None else t.data_ptr()


# the current stream's handle without a Stream object around it (5 us of a 14 us call), where this torch has it
_raw_stream = getattr(getattr(torch, "_C", None), "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(device, stream, name, *args):
    """The entry point on `device` and `stream` (default: torch's current stream of that device)."""
    fn = getattr(capi.lib(), name)
    if stream is not None and stream.device != device:
        raise ValueError(f"stream: on {stream.device}, expected {device}")
    handle = _raw_stream(device.index) if stream is None else stream.cuda_stream
    if device.index == torch.cuda.current_device():
        rc = fn(*args, handle)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, handle)
    if rc:
        capi.check(rc)


def _new(stream, like, shape, dtype=None):
    """Memory of the stream that is going to write it: work of another one may still be under way on what that one has freed.
    By `new_empty` on the device of `like`: `torch.empty` with a dtype and a device takes a microsecond longer."""
    if stream is None:
        return like.new_empty(shape) if dtype is None else like.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _like(stream, t):
    if stream is None:
        return torch.empty_like(t)
    with torch.cuda.stream(stream):
        return torch.empty_like(t)


def _shape(name, t, dims=2):
    shape = t.shape
    if len(shape) != dims:
        raise ValueError(f"{name}: expected {dims} dimensions, got {len(shape)}")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor (there is no CPU path)")
    return shape


def _spec(n_experts, top_k, score, n_groups, top_groups, group_top, renormalise, scale):
    if score not in capi.SCORES:
        raise ValueError(f"score: expected one of {sorted(capi.SCORES)}, got {score!r}")
    return capi.RouteSpec(n_experts, top_k, capi.SCORES[score], n_groups, top_groups, group_top, int(renormalise), scale)


def route(logits, top_k: int, *, score: str = "softmax", bias=None, n_groups: int = 1, top_groups: int = 1, group_top: int = 1,
          renormalise: bool = True, scale: float = 1.0, group: bool = True, stream=None):
    """(ids, weights, groups): the top_k experts of every row of `logits` (rows, experts) by score + bias among the best
    `top_groups` of `n_groups` expert groups, their weights (fp32), and the rows listed by expert (None with group=False).  Gradient: route_backward."""
    rows, experts = _shape("logits", logits)
    dev = logits.device
    at = dev.index
    if not (_is(logits, logits.dtype, (rows, experts), at) and _is(bias, torch.float32, (experts,), at)):
        _explain(dev, ("logits", logits, logits.dtype, (rows, experts)), ("bias", bias, torch.float32, (experts,)))
    spec = _spec(experts, top_k, score, n_groups, top_groups, group_top, renormalise, scale)
    # one allocation and few views: five of each take longer than the kernels of a small batch
    k = max(top_k, 0)  # what is wrong with it the entry point says
    n = rows * k
    if group:
        by_row, row, ptr = _new(stream, logits, 4 * n + experts + 1, torch.int32).split_with_sizes((3 * n, n, experts + 1))
        ids, weights, slot = by_row.view(3, rows, k).unbind(0)
        groups = Groups(ptr, row, slot)
    else:
        (ids, weights), ptr, row, slot, groups = _new(stream, logits, (2, rows, k), torch.int32).unbind(0), None, None, None, None
    weights = weights.view(torch.float32)
    _call(dev, stream, "mps_route", rows, C.byref(spec), _dtype(logits), _ptr(logits), _ptr(bias), _ptr(ids), _ptr(weights), _ptr(ptr), _ptr(row), _ptr(slot))
    return ids, weights, groups


def route_backward(logits, ids, d_weights, *, score: str = "softmax", renormalise: bool = True, scale: float = 1.0, stream=None):
    """Gradient by the logits of route's weights for the choice `ids` and the weights' gradient (fp32)."""
    rows, experts = _shape("logits", logits)
    dev = logits.device
    top_k = _shape("ids", ids)[1]
    at = dev.index
    if not (_is(logits, logits.dtype, (rows, experts), at) and _is(ids, torch.int32, (rows, top_k), at)
            and _is(d_weights, torch.float32, (rows, top_k), at)):
        _explain(dev, ("logits", logits, logits.dtype, (rows, experts)), ("ids", ids, torch.int32, (rows, top_k)),
               ("d_weights", d_weights, torch.float32, (rows, top_k)))
    spec = _spec(experts, top_k, score, 1, 1, 1, renormalise, scale)
    out = _like(stream, logits)
    _call(dev, stream, "mps_route_backward", rows, C.byref(spec), _dtype(logits), _ptr(logits), _ptr(ids), _ptr(d_weights), _ptr(out))
    return out


def group_rows(ids, n_groups: int, *, stream=None) -> Groups:
    """Rows listed by group from int32 `ids` of shape (rows,) or (rows, choices); a negative id is no group."""
    dev = ids.device
    if ids.dim() not in (1, 2):
        raise ValueError(f"ids: expected 1 or 2 dimensions, got {ids.dim()}")
    at = dev.index
    if not (_is(ids, torch.int32, ids.shape, at)):
        _explain(dev, ("ids", ids, torch.int32, ids.shape))
    rows, per_row = ids.shape[0], 1 if ids.dim() == 1 else ids.shape[1]
    groups = Groups(_new(stream, ids, max(n_groups, 0) + 1), _new(stream, ids, ids.numel()), _like(stream, ids))
    _call(dev, stream, "mps_group_rows", rows, per_row, n_groups, _ptr(ids), _ptr(groups.ptr), _ptr(groups.row), _ptr(groups.slot))
    return groups


def routed_product(x, w, groups: Groups, *, gather: bool = True, transpose: bool = False, out=None, stream=None):
    """y[s] = x[groups.row[s]] @ w[g].T for the slots s of every group g (x[s] itself with gather=False); transpose=True
    multiplies by w[g] instead.  w (groups, n, k).  Rows of `out` behind the last slot in use are left as they were.  Gradients: this
    with transpose the other way (of the slots) and routed_wgrad."""
    n_groups, n, k = _shape("w", w, 3)
    inner, outer = (n, k) if transpose else (k, n)
    dev, rows, slots = x.device, _shape("x", x)[0], groups.row.numel()
    if out is None:
        out = _new(stream, x, (slots, outer))
    at = dev.index
    if not (_is(x, x.dtype, (rows, inner), at) and _is(w, x.dtype, (n_groups, n, k), at) and _is(groups.ptr, torch.int32, (n_groups + 1,), at)
            and _is(groups.row, torch.int32, (slots,), at) and _is(out, x.dtype, (slots, outer), at)):
        _explain(dev, ("x", x, x.dtype, (rows, inner)), ("w", w, x.dtype, (n_groups, n, k)), ("groups.ptr", groups.ptr, torch.int32, (n_groups + 1,)),
               ("groups.row", groups.row, torch.int32, (slots,)), ("out", out, x.dtype, (slots, outer)))
    _call(dev, stream, "mps_routed_product", slots, rows, n_groups, k, n, _dtype(x), int(transpose), _ptr(groups.ptr),
          _ptr(groups.row) if gather else None, _ptr(x), _ptr(w), _ptr(out))
    return out


def routed_wgrad(x, dy, groups: Groups, *, gather: bool = True, out=None, stream=None):
    """dw[g] = sum over the slots s of g of outer(dy[s], x[groups.row[s]]) (x[s] with gather=False): (groups, n, k), zero for
    a group without slots."""
    dev, slots, n_groups = x.device, groups.row.numel(), groups.ptr.numel() - 1
    (rows, k), n = _shape("x", x), _shape("dy", dy)[1]
    if out is None:
        out = _new(stream, x, (n_groups, n, k))
    at = dev.index
    if not (_is(x, x.dtype, (rows, k), at) and _is(dy, x.dtype, (slots, n), at) and _is(groups.ptr, torch.int32, (n_groups + 1,), at)
            and _is(groups.row, torch.int32, (slots,), at) and _is(out, x.dtype, (n_groups, n, k), at)):
        _explain(dev, ("x", x, x.dtype, (rows, k)), ("dy", dy, x.dtype, (slots, n)), ("groups.ptr", groups.ptr, torch.int32, (n_groups + 1,)),
               ("groups.row", groups.row, torch.int32, (slots,)), ("out", out, x.dtype, (n_groups, n, k)))
    _call(dev, stream, "mps_routed_wgrad", slots, rows, n_groups, k, n, _dtype(x), _ptr(groups.ptr), _ptr(groups.row) if gather else None,
          _ptr(x), _ptr(dy), _ptr(out))
    return out


def routed_combine(rows, slot, weights=None, *, out=None, stream=None):
    """y[t] = sum over j of weights[t, j] * rows[slot[t, j]]; no term for a negative slot, weights None: 1 each.  Gradients:
    routed_combine_backward."""
    dev, (n_slots, dim), (n, per_row) = rows.device, _shape("rows", rows), _shape("slot", slot)
    if out is None:
        out = _new(stream, rows, (n, dim))
    at = dev.index
    if not (_is(rows, rows.dtype, (n_slots, dim), at) and _is(slot, torch.int32, (n, per_row), at) and _is(weights, torch.float32, (n, per_row), at)
            and _is(out, rows.dtype, (n, dim), at)):
        _explain(dev, ("rows", rows, rows.dtype, (n_slots, dim)), ("slot", slot, torch.int32, (n, per_row)), ("weights", weights, torch.float32, (n, per_row)),
               ("out", out, rows.dtype, (n, dim)))
    _call(dev, stream, "mps_routed_combine", n, per_row, n_slots, dim, _dtype(rows), _ptr(slot), _ptr(weights), _ptr(rows), _ptr(out))
    return out


def routed_combine_backward(dy, rows, slot, weights=None, *, out=None, stream=None):
    """(d_rows, d_weights) of routed_combine; `out` receives d_rows, whose rows that no slot names are left as they were."""
    dev, (n_slots, dim), (n, per_row) = rows.device, _shape("rows", rows), _shape("slot", slot)
    if out is None:
        out = _like(stream, rows)
    at = dev.index
    if not (_is(dy, rows.dtype, (n, dim), at) and _is(rows, rows.dtype, (n_slots, dim), at) and _is(slot, torch.int32, (n, per_row), at)
            and _is(weights, torch.float32, (n, per_row), at) and _is(out, rows.dtype, (n_slots, dim), at)):
        _explain(dev, ("dy", dy, rows.dtype, (n, dim)), ("rows", rows, rows.dtype, (n_slots, dim)), ("slot", slot, torch.int32, (n, per_row)),
               ("weights", weights, torch.float32, (n, per_row)), ("out", out, rows.dtype, (n_slots, dim)))
    d_weights = _new(stream, rows, (n, per_row), torch.float32)
    _call(dev, stream, "mps_routed_combine_backward", n, per_row, n_slots, dim, _dtype(rows), _ptr(slot), _ptr(weights), _ptr(dy), _ptr(rows), _ptr(out),
          _ptr(d_weights))
    return out, d_weights


def _adapter_sizes(x, w, a, b, ids, groups, scale):
    rows, (n, k), (n_adapters, rank) = _shape("x", x)[0], _shape("w", w), _shape("a", a, 3)[:2]
    at = x.device.index
    if not (_is(x, x.dtype, (rows, k), at) and _is(w, x.dtype, (n, k), at) and _is(a, x.dtype, (n_adapters, rank, k), at)
            and _is(b, x.dtype, (n_adapters, n, rank), at) and _is(ids, torch.int32, (rows,), at)
            and _is(groups.ptr, torch.int32, (n_adapters + 1,), at) and _is(groups.row, torch.int32, (rows,), at)
            and _is(scale, torch.float32, (n_adapters,), at)):
        _explain(x.device, ("x", x, x.dtype, (rows, k)), ("w", w, x.dtype, (n, k)), ("a", a, x.dtype, (n_adapters, rank, k)),
               ("b", b, x.dtype, (n_adapters, n, rank)), ("ids", ids, torch.int32, (rows,)), ("groups.ptr", groups.ptr, torch.int32, (n_adapters + 1,)),
               ("groups.row", groups.row, torch.int32, (rows,)), ("scale", scale, torch.float32, (n_adapters,)))
    return rows, k, n, n_adapters, rank


@functools.lru_cache(maxsize=64)
def _workspace_bytes(*sizes) -> int:
    need = capi.lib().mps_adapters_workspace(*sizes)
    if need < 0:
        capi.check(int(need))
    return need


def adapters(x, w, a, b, ids, groups: Groups, scale=None, *, out=None, stream=None):
    """y[t] = x[t] @ w.T + scale[i] * (x[t] @ a[i].T) @ b[i].T with i = ids[t] (a negative id: the projection alone).
    w (n, k), a (adapters, rank, k), b (adapters, n, rank), groups = group_rows(ids, adapters), scale fp32 or None (1).
    Gradients: adapters_backward."""
    sizes = rows, k, n, _, _ = _adapter_sizes(x, w, a, b, ids, groups, scale)
    if out is None:
        out = _new(stream, x, (rows, n))
    at = x.device.index
    if not (_is(out, x.dtype, (rows, n), at)):
        _explain(x.device, ("out", out, x.dtype, (rows, n)))
    dtype = _dtype(x)
    ws = _new(stream, x, _workspace_bytes(*sizes, dtype, 0), torch.uint8)
    _call(x.device, stream, "mps_adapters", *sizes, dtype, _ptr(ids), _ptr(groups.ptr), _ptr(groups.row), _ptr(scale), _ptr(x), _ptr(w), _ptr(a), _ptr(b),
          _ptr(out), _ptr(ws), ws.numel())
    return out


def adapters_backward(dy, x, w, a, b, ids, groups: Groups, scale=None, *, stream=None):
    """(dx, da, db) of adapters; the shared projection and the scales are constants."""
    sizes = rows, k, n, _, _ = _adapter_sizes(x, w, a, b, ids, groups, scale)
    at = x.device.index
    if not (_is(dy, x.dtype, (rows, n), at)):
        _explain(x.device, ("dy", dy, x.dtype, (rows, n)))
    dx, da, db = _like(stream, x), _like(stream, a), _like(stream, b)
    dtype = _dtype(x)
    ws = _new(stream, x, _workspace_bytes(*sizes, dtype, 1), torch.uint8)
    _call(x.device, stream, "mps_adapters_backward", *sizes, dtype, _ptr(ids), _ptr(groups.ptr), _ptr(groups.row), _ptr(scale), _ptr(dy), _ptr(x), _ptr(w),
          _ptr(a), _ptr(b), _ptr(dx), _ptr(da), _ptr(db), _ptr(ws), ws.numel())
    return dx, da, db


def routed_check(device=None, stream=None) -> None:
    """Waits for the stream and raises if a routed operator on the device (default: the stream's, or the current one) met an index
    out of range or gave up a wait since the last check."""
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device()) if stream is None else stream.device
    device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
    if device.index is None:
        device = torch.device(device.type, torch.cuda.current_device())
    _call(device, stream, "mps_routed_check")
