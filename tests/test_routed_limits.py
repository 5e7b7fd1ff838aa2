"""Routed operators: calls that are refused on the host because the kernels' own arithmetic or their order of reads and writes does
not cover them (no GPU needed: every call below is refused before any device call)."""
import ctypes as C

import pytest

P = 1 << 33  # addresses that are never followed
MOST = 2**31 - 1


def code(mps, rc, want, word):
    assert rc == want, (rc, mps.capi.lib().mps_last_error())
    assert word in mps.capi.lib().mps_last_error().decode()


@pytest.mark.parametrize("dtype,k", [(0, 8), (2, 8), (2, 5)])
@pytest.mark.parametrize("slots,rows", [(MOST, 4), (MOST - 100, 4), (4, MOST)])
def test_slot_numbers_whose_tiles_pass_31_bits(mps, dtype, k, slots, rows):
    """A tile's end behind the last slot is still counted in 32 bits."""
    L, c = mps.capi.lib(), mps.capi
    code(mps, L.mps_routed_product(slots, rows, 2, k, 8, dtype, 0, P, P, P, P << 1, P << 2, None), c.ERR_UNSUPPORTED, "slots")
    code(mps, L.mps_routed_wgrad(slots, rows, 2, k, 8, dtype, P, P, P, P << 1, P << 2, None), c.ERR_UNSUPPORTED, "slots")


def test_rows_too_wide_to_combine(mps):
    L, c = mps.capi.lib(), mps.capi
    for dim in (2**24 + 1, MOST):
        code(mps, L.mps_routed_combine(4, 2, 8, dim, 1, P, P, P << 1, P << 3, None), c.ERR_UNSUPPORTED, "dim")
        code(mps, L.mps_routed_combine_backward(4, 2, 8, dim, 1, P, P, P << 1, P << 2, P << 3, P, None), c.ERR_UNSUPPORTED, "dim")


def test_workspace_of_sizes_the_adapters_refuse(mps):
    L, c = mps.capi.lib(), mps.capi
    code(mps, L.mps_adapters_workspace(16, 64, 32, 1025, 8, 2, 0), c.ERR_UNSUPPORTED, "1024")
    code(mps, L.mps_adapters_workspace(16, 64, 32, 4, 5000, 2, 1), c.ERR_UNSUPPORTED, "rank")
    code(mps, L.mps_adapters_workspace(2**30, 64, 32, 4, 8, 2, 1), c.ERR_UNSUPPORTED, "rows")
    for backward in (0, 1):  # what a call needs grows with the call, and a call without rows needs nothing
        sizes = [L.mps_adapters_workspace(rows, 256, 512, 8, 16, 2, backward) for rows in (0, 1, 64, 4096)]
        assert sizes[0] == 0 and sizes[1] > 0 and sizes[1] < sizes[2] < sizes[3]


def test_results_over_what_is_read(mps):
    """A result that lies over an operand would be read after it was written."""
    L, c = mps.capi.lib(), mps.capi
    x, w, y = P, P << 1, P << 2
    size = 2

    def product(x, w, y, transpose=0):
        return L.mps_routed_product(8, 4, 2, 16, 32, 2, transpose, P, P, x, w, y, None)

    for rc in (product(x, w, x), product(x, w, x + (4 * 16 - 1) * size // 2 * 2), product(x, w, w), product(x, w, w - 16), product(x, w, x, 1)):
        code(mps, rc, c.ERR_ARG, "overlap")
    for rc in (L.mps_routed_wgrad(8, 4, 2, 16, 32, 2, P, P, x, w, x, None), L.mps_routed_wgrad(8, 4, 2, 16, 32, 2, P, P, x, w, w + 2, None)):
        code(mps, rc, c.ERR_ARG, "overlap")
    code(mps, L.mps_routed_combine(4, 2, 8, 16, 2, P, P, x, x, None), c.ERR_ARG, "overlap")
    code(mps, L.mps_routed_combine(4, 2, 8, 16, 2, P, P, x, x - 2, None), c.ERR_ARG, "overlap")
    code(mps, L.mps_routed_combine_backward(4, 2, 8, 16, 2, P, P, x, w, x, P, None), c.ERR_ARG, "overlap")
    code(mps, L.mps_routed_combine_backward(4, 2, 8, 16, 2, P, P, x, w, w + 2, P, None), c.ERR_ARG, "overlap")  # in place, but shifted

    need = L.mps_adapters_workspace(16, 64, 64, 4, 8, 2, 1)
    at = {name: P * (i + 1) for i, name in enumerate(("dy", "x", "w", "a", "b", "y", "dx", "da", "db", "ws"))}

    def forward(**change):
        t = {**at, **change}
        return L.mps_adapters(16, 64, 64, 4, 8, 2, P, P, P, None, t["x"], t["w"], t["a"], t["b"], t["y"], t["ws"], need, None)

    def backward(**change):
        t = {**at, **change}
        return L.mps_adapters_backward(16, 64, 64, 4, 8, 2, P, P, P, None, t["dy"], t["x"], t["w"], t["a"], t["b"], t["dx"], t["da"], t["db"], t["ws"], need, None)

    for operand in ("x", "w", "a", "b"):
        code(mps, forward(y=at[operand]), c.ERR_ARG, "overlap")
        for result in ("dx", "da", "db"):
            code(mps, backward(**{result: at[operand]}), c.ERR_ARG, "overlap")
    code(mps, backward(dx=at["dy"]), c.ERR_ARG, "overlap")
    code(mps, forward(ws=at["x"]), c.ERR_ARG, "overlap")
    code(mps, backward(ws=at["dx"]), c.ERR_ARG, "overlap")
    code(mps, backward(da=at["db"]), c.ERR_ARG, "overlap")
