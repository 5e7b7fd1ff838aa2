"""Routed operators, what is decided on the host: every refused argument comes back as a code with a message, before any
device call (these run without a GPU), and the wrappers refuse tensors that the entry points could not see are wrong."""
import ctypes as C

import numpy as np
import pytest
import torch

P = 1 << 20  # an address that is never followed: every call below is refused first


def spec(mps, **kw):
    d = dict(n_experts=64, top_k=8, score=0, n_groups=1, top_groups=1, group_top=1, renormalise=1, scale=1.0)
    d.update(kw)
    return C.byref(mps.capi.RouteSpec(*d.values()))


def code(mps, rc, want, word):
    assert rc == want, (rc, mps.capi.lib().mps_last_error())
    assert word in mps.capi.lib().mps_last_error().decode()


@pytest.mark.parametrize("change,want,word", [
    (dict(n_experts=0), "ARG", "experts"), (dict(top_k=0), "ARG", "top"), (dict(top_k=65), "ARG", "top 65"), (dict(score=2), "ARG", "score"),
    (dict(n_groups=0), "ARG", "groups"), (dict(n_groups=7), "ARG", "groups"), (dict(n_groups=8, top_groups=0), "ARG", "top_groups"),
    (dict(n_groups=8, top_groups=9), "ARG", "top_groups"), (dict(group_top=3), "ARG", "group_top"), (dict(n_groups=64, top_groups=7), "ARG", "top 8"),
    (dict(scale=float("nan")), "ARG", "scale"), (dict(n_experts=1025), "UNSUPPORTED", "1024"), (dict(top_k=33), "UNSUPPORTED", "32"),
    (dict(n_groups=64, top_groups=64), "UNSUPPORTED", "32"),
])
def test_route_specs_refused(mps, change, want, word):
    L = mps.capi.lib()
    want = getattr(mps.capi, "ERR_" + want)
    code(mps, L.mps_route(4, spec(mps, **change), 0, P, None, P, P, None, None, None, None), want, word)
    code(mps, L.mps_route_backward(4, spec(mps, **change), 0, P, P, P, P, None), want, word)


def test_route_arguments_refused(mps):
    L, c = mps.capi.lib(), mps.capi
    ok = spec(mps)
    code(mps, L.mps_route(4, None, 0, P, None, P, P, None, None, None, None), c.ERR_ARG, "spec")
    code(mps, L.mps_route(-1, ok, 0, P, None, P, P, None, None, None, None), c.ERR_ARG, "n_rows")
    code(mps, L.mps_route(4, ok, 3, P, None, P, P, None, None, None, None), c.ERR_ARG, "dtype")
    code(mps, L.mps_route(4, ok, 0, None, None, P, P, None, None, None, None), c.ERR_ARG, "NULL")
    code(mps, L.mps_route(4, ok, 0, P, None, P, P, P, None, None, None), c.ERR_ARG, "together")
    code(mps, L.mps_route(4, ok, 0, P, None, P, P, None, P, P, None), c.ERR_ARG, "together")
    code(mps, L.mps_route(4, ok, 0, P + 2, None, P, P, None, None, None, None), c.ERR_ALIGN, "aligned")
    code(mps, L.mps_route(4, ok, 1, P + 1, None, P, P, None, None, None, None), c.ERR_ALIGN, "aligned")
    code(mps, L.mps_route(2**28, ok, 1, P, None, P, P, None, None, None, None), c.ERR_UNSUPPORTED, "31 bits")
    code(mps, L.mps_route_backward(4, ok, 0, P, P, None, P, None), c.ERR_ARG, "NULL")
    code(mps, L.mps_route_backward(4, ok, 0, P, P, P + 2, P, None), c.ERR_ALIGN, "aligned")
    assert L.mps_route(0, ok, 0, None, None, None, None, None, None, None, None) == c.OK
    assert L.mps_route_backward(0, ok, 0, None, None, None, None, None) == c.OK


def test_group_rows_arguments_refused(mps):
    L, c = mps.capi.lib(), mps.capi
    code(mps, L.mps_group_rows(-1, 1, 4, P, P, P, P, None), c.ERR_ARG, "rows")
    code(mps, L.mps_group_rows(4, 0, 4, P, P, P, P, None), c.ERR_ARG, "per row")
    code(mps, L.mps_group_rows(4, 1, 0, P, P, P, P, None), c.ERR_ARG, "groups")
    code(mps, L.mps_group_rows(4, 1, 1025, P, P, P, P, None), c.ERR_UNSUPPORTED, "1024")
    code(mps, L.mps_group_rows(2**30, 2, 4, P, P, P, P, None), c.ERR_UNSUPPORTED, "31 bits")
    code(mps, L.mps_group_rows(4, 1, 4, None, P, P, P, None), c.ERR_ARG, "NULL")
    code(mps, L.mps_group_rows(4, 1, 4, P, P, P, P + 2, None), c.ERR_ALIGN, "aligned")


def test_product_arguments_refused(mps):
    L, c = mps.capi.lib(), mps.capi
    for name in ("mps_routed_product", "mps_routed_wgrad"):
        fn = getattr(L, name)
        t = (0,) if name == "mps_routed_product" else ()
        code(mps, fn(-1, 4, 2, 8, 8, 1, *t, P, P, P, P, P, None), c.ERR_ARG, "slots")
        code(mps, fn(4, 4, 0, 8, 8, 1, *t, P, P, P, P, P, None), c.ERR_ARG, "groups")
        code(mps, fn(4, 4, 2, 0, 8, 1, *t, P, P, P, P, P, None), c.ERR_ARG, "k = 0")
        code(mps, fn(4, 4, 2, 8, 8, 7, *t, P, P, P, P, P, None), c.ERR_ARG, "dtype")
        code(mps, fn(4, 4, 1025, 8, 8, 1, *t, P, P, P, P, P, None), c.ERR_UNSUPPORTED, "1024")
        code(mps, fn(4, 4, 2, 8, 2**22, 1, *t, P, P, P, P, P, None), c.ERR_UNSUPPORTED, "up to")
        code(mps, fn(4, 4, 2, 8, 8, 1, *t, P, P, None, P, P, None), c.ERR_ARG, "NULL")
        code(mps, fn(4, 3, 2, 8, 8, 1, *t, P, None, P, P, P, None), c.ERR_ARG, "in order")
        code(mps, fn(4, 4, 2, 8, 8, 1, *t, P, P, P + 1, P, P, None), c.ERR_ALIGN, "aligned")
    assert L.mps_routed_product(0, 0, 2, 8, 8, 1, 0, None, None, None, None, None, None) == c.OK


def test_combine_arguments_refused(mps):
    L, c = mps.capi.lib(), mps.capi
    code(mps, L.mps_routed_combine(4, 0, 8, 16, 1, P, P, P, P, None), c.ERR_ARG, "terms")
    code(mps, L.mps_routed_combine(4, 2, 8, 0, 1, P, P, P, P, None), c.ERR_ARG, "dim")
    code(mps, L.mps_routed_combine(4, 2, 8, 16, 9, P, P, P, P, None), c.ERR_ARG, "dtype")
    code(mps, L.mps_routed_combine(2**30, 2, 8, 16, 1, P, P, P, P, None), c.ERR_UNSUPPORTED, "31 bits")
    code(mps, L.mps_routed_combine(4, 2, 8, 16, 1, P, P, None, P, None), c.ERR_ARG, "NULL")
    code(mps, L.mps_routed_combine(4, 2, 8, 16, 0, P, P, P, P + 2, None), c.ERR_ALIGN, "aligned")
    code(mps, L.mps_routed_combine_backward(4, 2, 8, 16, 1, P, P, P, None, P, P, None), c.ERR_ARG, "NULL")
    code(mps, L.mps_routed_combine_backward(4, 2, 8, 16, 1, P, P, P, P, P, P + 2, None), c.ERR_ALIGN, "aligned")
    assert L.mps_routed_combine(0, 2, 0, 16, 1, None, None, None, None, None) == c.OK


def test_adapters_arguments_refused(mps):
    L, c = mps.capi.lib(), mps.capi
    need = L.mps_adapters_workspace(16, 64, 32, 4, 8, 2, 1)
    assert need > 0 and L.mps_adapters_workspace(0, 64, 32, 4, 8, 2, 0) >= 0
    code(mps, L.mps_adapters_workspace(16, 64, 32, 0, 8, 2, 0), c.ERR_ARG, "adapters")

    def fwd(rows=16, k=64, n=32, na=4, r=8, dtype=2, ids=P, ptr=P, row=P, scale=P, x=P, ws=P, size=need):
        return L.mps_adapters(rows, k, n, na, r, dtype, ids, ptr, row, scale, x, P, P, P, P, ws, size, None)

    def bwd(rows=16, k=64, n=32, na=4, r=8, dtype=2, ids=P, ptr=P, row=P, scale=P, x=P, ws=P, size=need):
        return L.mps_adapters_backward(rows, k, n, na, r, dtype, ids, ptr, row, scale, P, x, P, P, P, P, P, P, ws, size, None)

    for fn in (fwd, bwd):
        code(mps, fn(rows=-1), c.ERR_ARG, "rows")
        code(mps, fn(k=0), c.ERR_ARG, "k = 0")
        code(mps, fn(r=0), c.ERR_ARG, "rank 0")
        code(mps, fn(dtype=5), c.ERR_ARG, "dtype")
        code(mps, fn(na=1025), c.ERR_UNSUPPORTED, "1024")
        code(mps, fn(r=5000), c.ERR_UNSUPPORTED, "rank")
        code(mps, fn(ids=None), c.ERR_ARG, "NULL")
        code(mps, fn(ptr=None), c.ERR_ARG, "NULL")
        code(mps, fn(x=None), c.ERR_ARG, "NULL")
        code(mps, fn(x=P + 1), c.ERR_ALIGN, "aligned")
        code(mps, fn(ids=P + 2), c.ERR_ALIGN, "aligned")
        code(mps, fn(ws=None), c.ERR_ARG, "workspace")
        code(mps, fn(size=16), c.ERR_ARG, "workspace")
        code(mps, fn(ws=P + 16), c.ERR_ALIGN, "256")


def test_other_operators_still_refuse_the_third_type(mps):
    h = C.c_void_p()
    assert mps.capi.lib().mps_plan_create(100, 100, 16, mps.BF16, 8, 1, C.byref(h)) == mps.capi.ERR_ARG
    assert mps.capi.lib().mps_csr_transpose_device(4, 4, 0, mps.BF16, P, None, None, P, None, None, None) == mps.capi.ERR_ARG


def test_wrappers_refuse_host_tensors_and_wrong_shapes(mps):
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        mps.route(x, 2)
    with pytest.raises(ValueError, match="CUDA"):
        mps.group_rows(torch.zeros(4, dtype=torch.int32), 2)
    with pytest.raises(ValueError, match="dimensions"):
        mps.route(torch.zeros(4), 2)
    with pytest.raises(ValueError, match="dimensions"):
        mps.group_rows(torch.zeros(2, 2, 2, dtype=torch.int32), 2)
    g = mps.Groups(*(torch.zeros(3, dtype=torch.int32) for _ in range(3)))
    for call in (lambda: mps.routed_product(x, torch.zeros(2, 8, 8), g), lambda: mps.routed_wgrad(x, x, g),
                 lambda: mps.routed_combine(x, torch.zeros(4, 2, dtype=torch.int32)),
                 lambda: mps.routed_combine_backward(x, x, torch.zeros(4, 2, dtype=torch.int32)),
                 lambda: mps.adapters(x, torch.zeros(8, 8), torch.zeros(2, 2, 8), torch.zeros(2, 8, 2), torch.zeros(4, dtype=torch.int32), g)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_oracle_forms_agree_with_differences():
    """The 64-bit gradients the kernels are compared with are those of the 64-bit forward forms."""
    import routed_oracle as o
    rng = np.random.default_rng(0)
    l = rng.normal(size=(3, 7))
    for score in ("softmax", "sigmoid"):
        for renorm in (False, True):
            ids, w = o.route(l, 3, score, renormalise=renorm, scale=1.7)
            g = rng.normal(size=w.shape)
            d = o.route_grad(l, ids, g, score, renorm, 1.7)
            step = rng.normal(size=l.shape) * 1e-6
            up, down = (o.route(l + s * step, 3, score, renormalise=renorm, scale=1.7) for s in (1, -1))
            assert (up[0] == ids).all() and (down[0] == ids).all()
            assert abs(((up[1] - down[1]) * g).sum() / 2 - (d * step).sum()) < 1e-12
    x, w, a, b = rng.normal(size=(5, 6)), rng.normal(size=(4, 6)), rng.normal(size=(2, 3, 6)), rng.normal(size=(2, 4, 3))
    ids, scale, dy = np.array([0, 1, -1, 1, 1]), np.array([0.5, 2.0]), rng.normal(size=(5, 4))
    grads = o.adapters_grad(dy, x, w, a, b, ids, scale)
    for at, (p, d) in enumerate(zip((x, a, b), grads)):
        step = rng.normal(size=p.shape) * 1e-6
        args = [[x, a, b], [x, a, b]]
        args[0][at], args[1][at] = p + step, p - step
        up, down = (o.adapters(q[0], w, q[1], q[2], ids, scale)[0] for q in args)
        assert abs(((up - down) * dy).sum() / 2 - (d[0] * step).sum()) < 1e-10
