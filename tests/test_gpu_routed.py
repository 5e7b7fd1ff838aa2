"""Routed operators on the GPU against their plain 64-bit forms (routed_oracle.py): choices, row lists, products, combination
and adapters, each with its gradient, at the sizes and masks where they can go wrong; and a run of them together."""
import math

import numpy as np
import pytest
import torch

import routed_oracle as o
from routed_oracle import close, f64

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SENTINEL = 7.0


def rand(gen, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def gen_of(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def lists(ids, n_groups):
    """Groups on the device from the oracle's lists, so that the products are tested apart from group_rows."""
    import __graft_entry__ as entry
    parts = o.group_rows(np.asarray(ids), n_groups)
    return entry.load_package().Groups(*(torch.from_numpy(np.ascontiguousarray(p, dtype=np.int32)).cuda() for p in parts)), parts


# ---------------------------------------------------------------------------------------------- route

def check_route(mps, logits, top, **kw):
    """Choice equal, weights within fp32 rounding: the exponent's argument is rounded once (2^-24 of its size), exponentials,
    sums over at most 37 levels and quotient add at most 48 half units."""
    kwargs = dict(kw)
    bias = kwargs.pop("bias", None)
    ids, weights, groups = mps.route(logits, top, bias=bias, **kwargs)
    mps.routed_check()
    want_ids, want_w = o.route(f64(logits), top, bias=None if bias is None else f64(bias), **kwargs)
    got = ids.cpu().numpy()
    assert (got == want_ids).all(), np.argwhere(got != want_ids)[:5]
    l = f64(logits)
    live = np.where(np.isfinite(l), l, np.nan)
    span = np.nan_to_num(np.nanmax(live, 1, initial=-1e300, where=~np.isnan(live)) - np.nanmin(live, 1, initial=1e300, where=~np.isnan(live)),
                         nan=0.0, posinf=0.0, neginf=0.0).clip(0, 1e4)[:, None]
    got_w = f64(weights)
    assert (np.isnan(got_w) == np.isnan(want_w)).all()
    bad = ~(np.abs(got_w - want_w) <= (span + 48) * 2.0 ** -23 * np.abs(want_w) + 2.0 ** -126) & ~np.isnan(want_w)
    assert not bad.any(), (got_w[bad][:4], want_w[bad][:4])
    for a, b in zip(groups, o.group_rows(got, logits.shape[1])):
        assert (a.cpu().numpy() == b).all()
    return ids, weights


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,experts,top,kw", [
    (1, 1, 1, {}), (1, 64, 8, {}), (1, 256, 8, dict(score="sigmoid", with_bias=True, n_groups=8, top_groups=4, group_top=2, scale=2.5)),
    (3, 33, 5, dict(renormalise=False)), (67, 60, 4, dict(score="sigmoid", renormalise=False)), (129, 7, 7, dict(with_bias=True)),
    (40, 1024, 32, {}), (17, 1000, 9, dict(score="sigmoid", with_bias=True, n_groups=5, top_groups=3, group_top=2)),
    (33, 96, 6, dict(n_groups=32, top_groups=7, group_top=1)), (50, 130, 16, dict(n_groups=13, top_groups=2, group_top=2, renormalise=False)),
    (300, 24, 3, dict(score="sigmoid", n_groups=4, top_groups=1, group_top=1, with_bias=True)), (9, 31, 1, dict(n_groups=31, top_groups=1, group_top=2)),
])
def test_route(mps, cuda, dtype, rows, experts, top, kw):
    gen = gen_of(rows * 1000 + experts)
    kw = dict(kw)
    bias = torch.randn(experts, generator=gen, device="cuda") * 0.05 if kw.pop("with_bias", False) else None
    logits = rand(gen, dtype, rows, experts, scale=1.5)
    check_route(mps, logits, top, bias=bias, **kw)
    logits[:, torch.rand(experts, generator=gen, device="cuda") < 0.4] = -math.inf  # masked experts, and rows with none left
    logits[::3] = -math.inf
    logits[1::7, : max(1, experts // 2)] = torch.finfo(dtype).min
    check_route(mps, logits, top, bias=bias, **kw)


def test_route_without_rows(mps, cuda):
    ids, weights, groups = mps.route(torch.empty(0, 40, device="cuda"), 3)
    assert ids.shape == weights.shape == groups.slot.shape == (0, 3) and groups.row.shape == (0,) and groups.ptr.tolist() == [0] * 41
    assert mps.route_backward(torch.empty(0, 40, device="cuda"), ids, weights).shape == (0, 40)
    ids, weights, groups = mps.route(torch.randn(5, 40, device="cuda"), 3, group=False)
    assert groups is None and ids.shape == (5, 3)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("n_groups", [1, 4])
def test_route_equal_logits_go_to_the_lowest_index(mps, cuda, score, biased, n_groups):
    gen = gen_of(5)
    for rows in (70, 2060):  # a warp per row; eight lanes per row
        logits = torch.randint(-2, 3, (rows, 64), generator=gen, device="cuda").float()
        logits[0] = 0.0
        logits[1, ::2] = -0.0
        bias = torch.randint(0, 2, (64,), generator=gen, device="cuda").float() * 0.25 if biased else None
        check_route(mps, logits, 9, score=score, bias=bias, n_groups=n_groups, top_groups=min(2, n_groups), group_top=2)
        check_route(mps, logits.bfloat16(), 9, score=score, bias=bias, n_groups=n_groups, top_groups=min(2, n_groups), group_top=1)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_top", [1, 2])
def test_route_close_keys_are_told_apart(mps, cuda, score, group_top):
    """Score + bias of many experts within 1e-8 of one another: the order of the exact sums, which fp32 does not resolve."""
    rng = np.random.default_rng(3)
    logits = rng.normal(size=(64, 32)).astype(np.float32)
    s = np.array([o.row_scores(list(r.astype(np.float64)), score) for r in logits])
    for t in range(64):  # a bias per case: the bias that levels row t, so one call per row
        bias = torch.from_numpy((0.75 - s[t] + rng.normal(size=32) * 1e-8).astype(np.float32)).cuda()
        ids, _, _ = mps.route(torch.from_numpy(logits[t:t + 1]).cuda(), 6, score=score, bias=bias, n_groups=4, top_groups=2, group_top=group_top)
        want, _ = o.route(logits[t:t + 1].astype(np.float64), 6, score, f64(bias), 4, 2, group_top)
        assert (ids.cpu().numpy() == want).all(), t
        ids, _, _ = mps.route(torch.from_numpy(logits[t:t + 1]).cuda().repeat(2048, 1), 6, score=score, bias=bias, n_groups=4, top_groups=2,
                              group_top=group_top)
        assert (ids.cpu().numpy() == want).all(), t
    close_logits = torch.from_numpy((3 + rng.random((2100, 64)) * 1e-5).astype(np.float32)).cuda()  # a few units in the last place apart
    check_route(mps, close_logits, 10, score=score)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_not_a_number_and_infinite(mps, cuda, dtype, score):
    for rows in (12, 2055):
        not_a_number(mps, rand(gen_of(1), dtype, rows, 40), score)


def not_a_number(mps, logits, score):
    logits[2, 5] = math.nan
    logits[3] = math.nan
    logits[5, :38] = -math.inf
    bias = torch.zeros(40, device="cuda")
    bias[7], bias[9] = -math.inf, math.nan
    check_route(mps, logits, 4, score=score)
    check_route(mps, logits, 4, score=score, bias=bias)
    logits[7, 11] = math.inf  # a score of one for a sigmoid; not a number for a softmax, and said so
    ids, weights, _ = mps.route(logits, 4, score=score)
    assert ids[7, 0] == 11 and bool(torch.isnan(weights[7]).all()) == (score == "softmax")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_shares_hold_where_scores_underflow(mps, cuda, score):
    logits = torch.full((4, 16), -400.0, device="cuda") + torch.arange(16, device="cuda") * 0.25
    logits[:, 15] = 0.0 if score == "softmax" else -500.0
    bias = torch.zeros(16, device="cuda")
    bias[2:6] = 2.0  # the bias chooses experts whose scores are all zero in fp32
    check_route(mps, logits, 4, score=score, bias=bias)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [False, True])
@pytest.mark.parametrize("rows,experts,top", [(1, 1, 1), (5, 33, 3), (200, 60, 4), (9, 1024, 32)])
def test_route_backward(mps, cuda, dtype, score, renormalise, rows, experts, top):
    gen = gen_of(experts)
    logits = rand(gen, dtype, rows, experts, scale=1.5)
    logits[:, 1::5] = -math.inf
    ids = mps.route(logits, top, score=score, renormalise=renormalise)[0]
    if rows > 2:
        ids[1, 0] = -1
        ids[2] = -1
        if top > 1 and not renormalise:
            ids[3, 1] = ids[3, 0]  # the same expert twice
    g = torch.randn(rows, top, generator=gen, device="cuda")
    d = mps.route_backward(logits, ids, g, score=score, renormalise=renormalise, scale=1.5)
    mps.routed_check()
    want = o.route_grad(f64(logits), ids.cpu().numpy(), f64(g), score, renormalise, 1.5)
    # score times a difference of at most 2 max|g| sums, both to fp32 rounding as in check_route (span <= 20 here)
    mag = 1.5 * 3 * np.abs(f64(g)).max(1, keepdims=True) * np.ones_like(want)
    close(f64(d), want, dtype, 68, mag)


# ---------------------------------------------------------------------------------------------- group_rows

@pytest.mark.parametrize("rows,per,n_groups", [(0, 1, 3), (1, 1, 1), (7, 3, 5), (64, 32, 1024), (2049, 1, 60), (5001, 8, 256), (30011, 1, 2), (100000, 1, 1024)])
def test_group_rows(mps, cuda, rows, per, n_groups):
    rng = np.random.default_rng(rows + per)
    ids = rng.integers(-1, n_groups, (rows, per)).astype(np.int32)
    if rows > 10:
        ids[ids == n_groups // 2] = n_groups - 1  # an empty group, and one that is larger
    g = mps.group_rows(torch.from_numpy(ids).cuda(), n_groups)
    mps.routed_check()
    for got, want in zip(g, o.group_rows(ids, n_groups)):
        assert (got.cpu().numpy() == want).all()


def test_group_rows_nothing_chosen_and_one_dimension(mps, cuda):
    g = mps.group_rows(torch.full((100,), -1, dtype=torch.int32, device="cuda"), 4)
    assert not g.ptr.any() and (g.row == -1).all() and (g.slot == -1).all() and g.slot.shape == (100,)


def test_indices_out_of_range_are_skipped_and_reported(mps, cuda):
    def reported():
        with pytest.raises(mps.MpsError) as e:
            mps.routed_check()
        assert e.value.code == mps.capi.ERR_ARG
        mps.routed_check()  # cleared

    ids = torch.tensor([0, 4, 1, 2**31 - 1, 3], dtype=torch.int32, device="cuda")
    g = mps.group_rows(ids, 4)
    assert g.ptr.tolist() == [0, 1, 2, 2, 3] and g.row.tolist() == [0, 2, 4, -1, -1]
    reported()
    for dtype, k in ((BF16, 64), (BF16, 5), (F32, 8)):
        x, w = rand(gen_of(0), dtype, 5, k), rand(gen_of(1), dtype, 2, 16, k)
        row = torch.tensor([0, 9, -5, 1, 2**31 - 1], dtype=torch.int32, device="cuda")
        out = torch.full((5, 16), SENTINEL, dtype=dtype, device="cuda")
        mps.routed_product(x, w, mps.Groups(torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda"), row, None), out=out)
        reported()
        want = f64(x)[[0]] @ f64(w)[0].T
        close(f64(out)[[0]], want, dtype, k, np.abs(f64(x)[[0]]) @ np.abs(f64(w)[0].T))
        mps.routed_wgrad(x, rand(gen_of(2), dtype, 5, 16), mps.Groups(torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda"), row, None))
        reported()
        row = torch.arange(5, dtype=torch.int32, device="cuda")
        for ptr in ([-4, 3, 9], [3, 1, 5], [2**31 - 1, -2**31, 4]):  # offsets outside, or falling
            mps.routed_product(x, w, mps.Groups(torch.tensor(ptr, dtype=torch.int32, device="cuda"), row, None), out=out)
            reported()
        mps.routed_combine(x, torch.tensor([[0, 5], [2**31 - 1, 1]], dtype=torch.int32, device="cuda"))
        reported()
        mps.routed_combine_backward(x[:2].contiguous(), x, torch.tensor([[0, 5], [2**31 - 1, 1]], dtype=torch.int32, device="cuda"))
        reported()
    logits = rand(gen_of(3), F32, 2, 8)
    mps.route_backward(logits, torch.tensor([[0, 8], [2**30, 1]], dtype=torch.int32, device="cuda"), torch.ones(2, 2, device="cuda"))
    reported()
    for rank, k in ((8, 64), (3, 10)):
        x, w, a, b = rand(gen_of(0), BF16, 4, k), rand(gen_of(1), BF16, 16, k), rand(gen_of(2), BF16, 2, rank, k), rand(gen_of(3), BF16, 2, 16, rank)
        good = torch.tensor([0, 1, -1, 1], dtype=torch.int32, device="cuda")
        bad = torch.tensor([0, 7, -1, 2**31 - 1], dtype=torch.int32, device="cuda")
        y = mps.adapters(x, w, a, b, bad, mps.group_rows(good, 2))
        reported()
        want = o.adapters(f64(x), f64(w), f64(a), f64(b), np.array([0, -1, -1, -1]), np.ones(2))
        close(f64(y), want[0], BF16, k + rank, want[1], o.PAIR[BF16] * want[2])


# ---------------------------------------------------------------------------------------------- products

def counts_ids(counts, per_row, rng, padded=0):
    """Shuffled ids with the given number of rows per group, `padded` unused pairs among them."""
    flat = np.concatenate([np.full(c, g) for g, c in enumerate(counts)] + [np.full(padded, -1)]).astype(np.int32)
    flat = flat[: len(flat) // per_row * per_row]
    rng.shuffle(flat)
    return flat.reshape(-1, per_row)


PRODUCTS = [
    # k, n, rows per group, choices per row, padded
    (64, 128, [1], 1, 0), (8, 8, [3, 0, 2], 1, 0), (64, 64, [0, 0, 5], 1, 3), (72, 136, [17, 1, 0, 33], 1, 2), (200, 328, [130, 64, 65, 1], 2, 6),
    (512, 256, [1, 1, 1, 1, 0, 1, 1, 2], 2, 0), (128, 1000, [300, 7], 1, 0), (1000, 72, [257, 255, 0, 16], 4, 8), (24, 2056, [40, 9], 1, 0),
    (1544, 384, [2, 9, 31, 0, 8, 8], 1, 0), (256, 512, [600, 128, 256, 40], 2, 8),
    (64, 100, [300, 7, 40], 1, 0), (128, 3, [5, 1], 2, 0), (320, 136, [0] * 500 + [3] + [0] * 522 + [1], 1, 0), (64, 512, [2000, 700], 1, 4),
    (7, 5, [9, 0, 70], 1, 1), (33, 130, [65, 3], 2, 0), (1, 1, [2, 2], 1, 0), (4100, 12, [5, 70], 1, 0),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("k,n,counts,per_row,padded", PRODUCTS)
def test_product_and_gradients(mps, cuda, dtype, k, n, counts, per_row, padded):
    rng, gen = np.random.default_rng(k + n), gen_of(k * 7 + n)
    ids = counts_ids(counts, per_row, rng, padded)
    groups, (ptr, row, slot) = lists(ids, len(counts))
    slots, rows = row.size, len(ids)
    x, w, dy = rand(gen, dtype, rows, k), rand(gen, dtype, len(counts), n, k, scale=k ** -0.5), rand(gen, dtype, slots, n, scale=0.1)
    dy[ptr[-1]:] = math.nan  # rows behind the last slot are not read
    held = np.full((slots, n), SENTINEL)
    out = torch.full((slots, n), SENTINEL, dtype=dtype, device="cuda")
    assert mps.routed_product(x, w, groups, out=out) is out
    want, mag = o.product(f64(x), f64(w), ptr, row, held)
    close(f64(out), want, dtype, k, mag)

    ordered = x[groups.row.clamp(min=0).long()].contiguous()  # the same rows in slot order
    again = torch.full_like(out, SENTINEL)
    mps.routed_product(ordered, w, groups, gather=False, out=again)
    assert torch.equal(again, out)

    dx = torch.full((slots, k), SENTINEL, dtype=dtype, device="cuda")
    mps.routed_product(dy, w, groups, gather=False, transpose=True, out=dx)
    want, mag = o.product(f64(dy), f64(w).transpose(0, 2, 1), ptr, np.arange(slots), np.full((slots, k), SENTINEL))
    close(f64(dx), want, dtype, n, mag)

    dw = mps.routed_wgrad(x, dy, groups)
    want, mag = o.wgrad(f64(x), f64(dy), ptr, row)
    close(f64(dw), want, dtype, max(counts), mag)
    assert torch.equal(mps.routed_wgrad(ordered, dy, groups, gather=False), dw)
    mps.routed_check()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("k,n,counts", [(128, 512, [0] * 1000 + [700] + [0] * 20 + [40, 0, 0]), (256, 72, [5] + [0] * 1022 + [70]), (64, 320, [0] * 40 + [9] + [0] * 60)])
def test_product_of_few_groups_of_many(mps, cuda, dtype, k, n, counts):
    """Groups without slots, in every place and for narrow and wide tiles: passed over by the products, zeros in the gradient."""
    test_product_and_gradients(mps, cuda, dtype, k, n, counts, 1, 0)


@pytest.mark.parametrize("dtype,k,n", [(BF16, 256, 192), (F16, 72, 40), (F32, 30, 20)])
def test_product_rows_do_not_meet(mps, cuda, dtype, k, n):
    """A row of NaN or infinity reaches its own slots and its own group's matrix gradient only."""
    gen = gen_of(4)
    ids = np.array([[0], [1], [1], [0], [2], [1]] * 20, dtype=np.int32)
    groups, (ptr, row, slot) = lists(ids, 3)
    x, w, dy = rand(gen, dtype, 120, k), rand(gen, dtype, 3, n, k), rand(gen, dtype, 120, n)
    y, dw = mps.routed_product(x, w, groups), mps.routed_wgrad(x, dy, groups)
    x2 = x.clone()
    x2[1], x2[7] = math.nan, math.inf
    y2, dw2 = mps.routed_product(x2, w, groups), mps.routed_wgrad(x2, dy, groups)
    touched = [int(slot[1, 0]), int(slot[7, 0])]
    keep = [s for s in range(120) if s not in touched]
    assert torch.equal(y[keep], y2[keep]) and not torch.isfinite(y2[touched]).any()
    assert torch.equal(dw[[0, 2]], dw2[[0, 2]])


@pytest.mark.parametrize("dtype,k", [(BF16, 64), (F32, 20)])
def test_product_without_slots(mps, cuda, dtype, k):
    x, w = torch.empty(0, k, dtype=dtype, device="cuda"), torch.ones(3, 16, k, dtype=dtype, device="cuda")
    g = mps.group_rows(torch.empty(0, 2, dtype=torch.int32, device="cuda"), 3)
    assert mps.routed_product(x, w, g).shape == (0, 16)
    assert not mps.routed_wgrad(x, torch.empty(0, 16, dtype=dtype, device="cuda"), g).any()
    x = torch.ones(4, k, dtype=dtype, device="cuda")
    g = mps.group_rows(torch.full((4, 1), -1, dtype=torch.int32, device="cuda"), 3)
    out = torch.full((4, 16), SENTINEL, dtype=dtype, device="cuda")
    assert (mps.routed_product(x, w, g, out=out) == SENTINEL).all()
    assert not mps.routed_wgrad(x, torch.ones(4, 16, dtype=dtype, device="cuda"), g).any()
    mps.routed_check()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_product_at_addresses_off_16_bytes(mps, cuda, dtype):
    """Operands at addresses that no tensor map takes, and results at addresses that no 16-byte store takes."""
    def shifted(t):
        u = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        return u.copy_(t)

    gen, rng = gen_of(9), np.random.default_rng(9)
    groups, (ptr, row, slot) = lists(counts_ids([40, 0, 300], 1, rng), 3)
    x, w, dy = rand(gen, dtype, 340, 128), rand(gen, dtype, 3, 64, 128, scale=0.1), rand(gen, dtype, 340, 64)
    y, dw = mps.routed_product(x, w, groups), mps.routed_wgrad(x, dy, groups)
    out = shifted(torch.zeros_like(y))
    assert torch.equal(mps.routed_product(x, w, groups, out=out), y)
    assert torch.equal(mps.routed_wgrad(x, dy, groups, out=shifted(torch.zeros_like(dw))), dw)
    want, mag = o.product(f64(x), f64(w), ptr, row, np.zeros(y.shape))
    for a, b in ((shifted(x), w), (x, shifted(w))):
        close(f64(mps.routed_product(a, b, groups)), want, dtype, 128, mag)
    want, mag = o.wgrad(f64(x), f64(dy), ptr, row)
    for a, b in ((shifted(x), dy), (x, shifted(dy))):
        close(f64(mps.routed_wgrad(a, b, groups)), want, dtype, 300, mag)
    a, b, scale = rand(gen, dtype, 3, 8, 128), rand(gen, dtype, 3, 64, 8), torch.ones(3, device="cuda")
    ids = torch.from_numpy(rng.integers(-1, 3, 340).astype(np.int32)).cuda()
    ag = mps.group_rows(ids, 3)
    wide = mps.adapters(x, w[0], a, b, ids, ag, scale)
    assert torch.equal(mps.adapters(x, w[0], a, b, ids, ag, scale, out=shifted(torch.zeros_like(wide))), wide)
    ref = o.adapters(f64(x), f64(w[0]), f64(a), f64(b), ids.cpu().numpy(), np.ones(3))
    close(f64(mps.adapters(x, w[0], a, shifted(b), ids, ag, scale)), ref[0], dtype, 128 + 8 + 2, ref[1], o.PAIR[dtype] * ref[2] + o.FLOOR[dtype] * ref[3])
    mps.routed_check()


def test_product_offsets_beyond_31_bits(mps, cuda):
    """x, w and y of more than 2^31 elements each: the last rows and the last group are still found."""
    k, n, slots = 512, 512, (1 << 22) + 600
    x = torch.zeros(slots, k, dtype=BF16, device="cuda")
    x[-300:] = rand(gen_of(0), BF16, 300, k)
    w = torch.zeros(2, n, k, dtype=BF16, device="cuda")
    w[1] = rand(gen_of(1), BF16, n, k, scale=k ** -0.5)
    ptr = torch.tensor([0, slots - 300, slots], dtype=torch.int32, device="cuda")
    row = torch.arange(slots, dtype=torch.int32, device="cuda")
    g = mps.Groups(ptr, row, None)
    y = mps.routed_product(x, w, g)
    a, b = f64(x[-300:]), f64(w[1])
    close(f64(y[-300:]), a @ b.T, BF16, k, np.abs(a) @ np.abs(b).T)
    assert not y[:-300].any()
    dw = mps.routed_wgrad(x, y, g)
    d = f64(y[-300:])
    close(f64(dw[1]), d.T @ a, BF16, 300, np.abs(d).T @ np.abs(a))
    s = (torch.arange(300, dtype=torch.int32, device="cuda") + (slots - 300)).reshape(150, 2)
    out = mps.routed_combine(y, s)
    close(f64(out), d.reshape(150, 2, n).sum(1), BF16, 2, np.abs(d).reshape(150, 2, n).sum(1))
    mps.routed_check()


# ---------------------------------------------------------------------------------------------- combine

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,per,dim", [(1, 1, 1), (1, 8, 2048), (40, 8, 549), (3, 2, 4099), (21, 2, 7), (70, 2, 40), (33, 3, 37), (5, 5, 1000), (300, 1, 8), (9, 33, 264)])
def test_combine_and_gradients(mps, cuda, dtype, rows, per, dim):
    rng, gen = np.random.default_rng(rows + dim), gen_of(dim)
    slots = rows * per + 3
    slot = rng.permutation(slots)[: rows * per].reshape(rows, per).astype(np.int32)
    slot[rng.random((rows, per)) < 0.2] = -1
    if rows > 3:
        slot[2] = -1  # a row with nothing to sum
    d_slot = torch.from_numpy(slot).cuda()
    r, dy = rand(gen, dtype, slots, dim), rand(gen, dtype, rows, dim)
    unnamed = np.setdiff1d(np.arange(slots), slot)
    r[unnamed] = math.nan
    w = torch.randn(rows, per, generator=gen, device="cuda")
    for weights in (w, None):
        wide = f64(w) if weights is not None else np.ones((rows, per))
        y = mps.routed_combine(r, d_slot, weights)
        want, mag = o.combine(f64(r), slot, wide)
        close(f64(y), want, dtype, per, mag)
        out = torch.full_like(r, SENTINEL)
        d_rows, d_w = mps.routed_combine_backward(dy, r, d_slot, weights, out=out)
        want_r, want_w, mag = o.combine_grad(f64(dy), f64(r), slot, wide, np.full(r.shape, SENTINEL))
        close(f64(d_rows), want_r, dtype, 1, np.abs(want_r))
        close(f64(d_w), want_w, F32, dim, mag)
    # without the weights' gradient, and from addresses that are no multiple of 16 bytes
    if dim > 1:
        wide_r = torch.empty(slots * dim + 1, dtype=dtype, device="cuda")[1:].view(slots, dim)
        wide_r.copy_(r)
        assert torch.equal(mps.routed_combine(wide_r, d_slot, w), mps.routed_combine(r, d_slot, w))
    out2 = torch.full_like(r, SENTINEL)
    lib = mps.capi.lib()
    mps.capi.check(lib.mps_routed_combine_backward(rows, per, slots, dim, mps.routed._dtype(r), d_slot.data_ptr(), None, dy.data_ptr(), None, out2.data_ptr(),
                                                   None, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out2, out)
    mps.routed_check()


# ---------------------------------------------------------------------------------------------- adapters

ADAPTERS = [
    # rows, adapters, rank, k, n, order
    (1, 1, 8, 64, 64, "one"), (1, 5, 16, 256, 512, "none"), (64, 24, 16, 512, 256, "mixed"), (5, 70, 8, 128, 1000, "mixed"),
    (300, 3, 64, 200, 136, "runs"), (700, 6, 40, 512, 264, "runs"), (130, 2, 128, 72, 72, "mixed"), (257, 200, 24, 136, 640, "mixed"),
    (90, 4, 8, 1000, 8, "runs"), (40, 3, 200, 64, 128, "mixed"), (9, 3, 8, 64, 50, "mixed"), (1500, 3, 8, 64, 100, "mixed"), (40, 1024, 8, 64, 64, "mixed"),
    (2600, 4, 16, 256, 512, "runs"), (2600, 4, 72, 128, 264, "mixed"), (3000, 1, 8, 64, 1024, "mixed"), (33, 4, 3, 20, 30, "mixed"), (20, 2, 1, 7, 9, "mixed"), (50, 3, 12, 64, 64, "runs"),
]


def adapter_ids(rows, n, order, rng):
    if order == "one":
        return np.zeros(rows, np.int32)
    if order == "none":
        return np.full(rows, -1, np.int32)
    ids = rng.integers(-1, n, rows).astype(np.int32)
    return np.sort(ids)[::-1].copy() if order == "runs" else ids


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,n_adapters,rank,k,n,order", ADAPTERS)
def test_adapters_and_gradients(mps, cuda, dtype, rows, n_adapters, rank, k, n, order):
    rng, gen = np.random.default_rng(rows + k), gen_of(rank + n)
    ids = adapter_ids(rows, n_adapters, order, rng)
    d_ids = torch.from_numpy(ids).cuda()
    groups = mps.group_rows(d_ids, n_adapters)
    x, w, dy = rand(gen, dtype, rows, k), rand(gen, dtype, n, k, scale=k ** -0.5), rand(gen, dtype, rows, n, scale=0.1)
    a, b = rand(gen, dtype, n_adapters, rank, k, scale=k ** -0.5), rand(gen, dtype, n_adapters, n, rank, scale=rank ** -0.5)
    scale = torch.rand(n_adapters, generator=gen, device="cuda") + 0.5
    y = mps.adapters(x, w, a, b, d_ids, groups, scale)
    want = o.adapters(f64(x), f64(w), f64(a), f64(b), ids, f64(scale))
    close(f64(y), want[0], dtype, k + rank + 2, want[1], o.PAIR[dtype] * want[2] + o.FLOOR[dtype] * want[3])
    got = mps.adapters_backward(dy, x, w, a, b, d_ids, groups, scale)
    terms = (n + rank + 2, n + rows + 2, k + rows + 2)
    for g, want, t in zip(got, o.adapters_grad(f64(dy), f64(x), f64(w), f64(a), f64(b), ids, f64(scale)), terms):
        close(f64(g), want[0], dtype, t, want[1], o.PAIR[dtype] * want[2] + o.FLOOR[dtype] * want[3])
    ones = torch.ones(n_adapters, device="cuda")
    assert torch.equal(mps.adapters(x, w, a, b, d_ids, groups), mps.adapters(x, w, a, b, d_ids, groups, ones))
    mps.routed_check()


@pytest.mark.parametrize("rows", [9, 1500])
def test_few_adapters_of_many(mps, cuda, rows):
    gen = gen_of(rows)
    ids = np.array([3, 700, 1023, -1, 700], np.int32)[np.random.default_rng(rows).integers(0, 5, rows)]
    n_adapters, rank, k, n = 1024, 16, 128, 192
    d_ids = torch.from_numpy(ids).cuda()
    groups = mps.group_rows(d_ids, n_adapters)
    x, w, dy = rand(gen, BF16, rows, k), rand(gen, BF16, n, k, scale=k ** -0.5), rand(gen, BF16, rows, n, scale=0.1)
    a, b = rand(gen, BF16, n_adapters, rank, k, scale=k ** -0.5), rand(gen, BF16, n_adapters, n, rank, scale=rank ** -0.5)
    scale = torch.rand(n_adapters, generator=gen, device="cuda") + 0.5
    want = o.adapters(f64(x), f64(w), f64(a), f64(b), ids, f64(scale))
    close(f64(mps.adapters(x, w, a, b, d_ids, groups, scale)), want[0], BF16, k + rank + 2, want[1], o.PAIR[BF16] * want[2] + o.FLOOR[BF16] * want[3])
    got = mps.adapters_backward(dy, x, w, a, b, d_ids, groups, scale)
    terms = (n + rank + 2, n + rows + 2, k + rows + 2)
    for g, want, t in zip(got, o.adapters_grad(f64(dy), f64(x), f64(w), f64(a), f64(b), ids, f64(scale)), terms):
        close(f64(g), want[0], BF16, t, want[1], o.PAIR[BF16] * want[2] + o.FLOOR[BF16] * want[3])
    mps.routed_check()


@pytest.mark.parametrize("repeat", [30, 700])  # rows of any adapter in one tile; tiles of one adapter each
def test_adapters_rows_do_not_meet(mps, cuda, repeat):
    """NaN in a row, in an adapter nobody asks for, or in one other rows ask for, stays with the rows concerned."""
    gen = gen_of(8)
    ids = np.array([0, 1, -1, 2, 1, 0] * repeat, dtype=np.int32)
    d_ids = torch.from_numpy(ids).cuda()
    groups = mps.group_rows(d_ids, 4)
    x, w = rand(gen, BF16, len(ids), 128), rand(gen, BF16, 256, 128)
    a, b = rand(gen, BF16, 4, 16, 128), rand(gen, BF16, 4, 256, 16)
    a[3], b[3] = math.nan, math.inf
    y = mps.adapters(x, w, a, b, d_ids, groups)
    assert torch.isfinite(y).all()
    b2 = b.clone()
    b2[1] = math.nan
    y2 = mps.adapters(x, w, a, b2, d_ids, groups)
    other = torch.from_numpy(ids != 1).cuda()
    assert torch.equal(y[other], y2[other]) and torch.isnan(y2[~other]).all()
    x2 = x.clone()
    x2[3] = math.inf
    y3 = mps.adapters(x2, w, a, b, d_ids, groups)
    keep = torch.arange(len(ids)) != 3
    assert torch.equal(y[keep], y3[keep]) and not torch.isfinite(y3[3]).any()
    dy = rand(gen, BF16, len(ids), 256)
    dx, da, db = mps.adapters_backward(dy, x, w, a, b, d_ids, groups)
    assert torch.isfinite(dx).all() and torch.isfinite(da).all() and torch.isfinite(db).all()
    dx2, da2, db2 = mps.adapters_backward(dy, x2, w, a, b, d_ids, groups)  # row 3 asks for adapter 2
    assert torch.equal(dx, dx2) and torch.equal(da[[0, 1, 3]], da2[[0, 1, 3]]) and torch.equal(db[[0, 1, 3]], db2[[0, 1, 3]])
    assert not torch.isfinite(da2[2]).all()


def test_adapters_without_rows(mps, cuda):
    ids = torch.empty(0, dtype=torch.int32, device="cuda")
    g = mps.group_rows(ids, 2)
    x, w, a, b = (torch.ones(*s, dtype=BF16, device="cuda") for s in ((0, 64), (32, 64), (2, 8, 64), (2, 32, 8)))
    assert mps.adapters(x, w, a, b, ids, g).shape == (0, 32)
    dx, da, db = mps.adapters_backward(torch.empty(0, 32, dtype=BF16, device="cuda"), x, w, a, b, ids, g)
    assert dx.shape == (0, 64) and not da.any() and not db.any()


# ---------------------------------------------------------------------------------------------- together

def layer(mps, x, router, w1, w2, top):
    """A mixture of experts as a user runs it: route, first products, relu^2, second products, combine."""
    logits = (x.float() @ router).contiguous()
    ids, weights, groups = mps.route(logits, top, score="sigmoid", renormalise=True, scale=1.5)
    h = mps.routed_product(x, w1, groups)
    act = h.relu().square()
    rows = mps.routed_product(act, w2, groups, gather=False)
    return mps.routed_combine(rows, groups.slot, weights), (logits, ids, weights, groups, h, act, rows)


def layer_backward(mps, dy, x, router, w1, w2, saved):
    logits, ids, weights, groups, h, act, rows = saved
    d_rows, d_weights = mps.routed_combine_backward(dy, rows, groups.slot, weights)
    d_act = mps.routed_product(d_rows, w2, groups, gather=False, transpose=True)
    dw2 = mps.routed_wgrad(act, d_rows, groups, gather=False)
    d_h = d_act * 2 * h.relu()
    dw1 = mps.routed_wgrad(x, d_h, groups)
    d_slots = mps.routed_product(d_h, w1, groups, gather=False, transpose=True)
    d_logits = mps.route_backward(logits, ids, d_weights, score="sigmoid", renormalise=True, scale=1.5)
    return mps.routed_combine(d_slots, groups.slot) + (d_logits @ router.t()).to(x.dtype), x.float().t() @ d_logits, dw1, dw2


def plain_layer(x, router, w1, w2, ids):
    s = torch.sigmoid(x @ router).gather(1, ids)
    weights = 1.5 * s / s.sum(1, keepdim=True)
    y = torch.zeros_like(x)
    for j in range(ids.shape[1]):
        h = torch.einsum("tk,tnk->tn", x, w1[ids[:, j]]).relu().square()
        y = y + weights[:, j:j + 1] * torch.einsum("tn,tkn->tk", h, w2[ids[:, j]])
    return y


@pytest.mark.parametrize("dtype,tol", [(F32, 2e-5), (BF16, 4e-2)])
def test_layer_and_its_gradient(mps, cuda, dtype, tol):
    """The run of operators against 64-bit autograd of the plain layer, and against differences of it.  Relative to the largest
    value: five products, each rounding its stored inputs to the type (bf16: 2^-8 each, the square twice), fp32 2^-24 per term."""
    gen = gen_of(11)
    x, router = rand(gen, dtype, 37, 48), rand(gen, F32, 48, 6, scale=0.3)
    w1, w2 = rand(gen, dtype, 6, 40, 48, scale=48 ** -0.5), rand(gen, dtype, 6, 48, 40, scale=40 ** -0.5)
    dy = rand(gen, dtype, 37, 48)
    y, saved = layer(mps, x, router, w1, w2, 2)
    grads = layer_backward(mps, dy, x, router, w1, w2, saved)
    mps.routed_check()
    ids = saved[1].long()
    leaves = [t.double().requires_grad_() for t in (x, router, w1, w2)]
    want = plain_layer(*leaves, ids)
    want.backward(dy.double())
    for got, ref in zip((y, *grads), (want, *(t.grad for t in leaves))):
        assert (got.double() - ref).abs().max() <= tol * ref.abs().max()
    step = [torch.randn(t.shape, generator=gen, device="cuda", dtype=torch.float64) * 1e-5 for t in leaves]
    with torch.no_grad():
        up, down = (plain_layer(*(t + s * d for t, d in zip(leaves, step)), ids) for s in (1, -1))
        along = sum((g.double() * d).sum() for g, d in zip(grads, step))
        size = sum((g.double() * d).pow(2).sum() for g, d in zip(grads, step)).sqrt()
    assert abs((((up - down) * dy.double()).sum() / 2 - along).item()) <= 4 * tol * size.item()


def everything(mps, t):
    """One of each operator, forward and backward; returns all results."""
    ids, weights, g = mps.route(t["logits"], 4, score="sigmoid", bias=t["bias"], n_groups=4, top_groups=2, group_top=2)
    y = mps.routed_product(t["x"], t["w1"], g)
    dw = mps.routed_wgrad(t["x"], y, g)
    dx = mps.routed_product(y, t["w1"], g, gather=False, transpose=True)
    z = mps.routed_combine(y, g.slot, weights)
    d_rows, d_w = mps.routed_combine_backward(z, y, g.slot, weights)
    d_l = mps.route_backward(t["logits"], ids, d_w, score="sigmoid")
    ag = mps.group_rows(t["ids"], 6)
    out = mps.adapters(t["x"], t["w"], t["a"], t["b"], t["ids"], ag, t["scale"])
    return [ids, weights, *g, y, dw, dx, z, d_rows, d_w, d_l, *ag, out, *mps.adapters_backward(out, t["x"], t["w"], t["a"], t["b"], t["ids"], ag, t["scale"])]


def everything_inputs(seed, rows=77):
    gen = gen_of(seed)
    return dict(logits=rand(gen, F32, rows, 32), bias=rand(gen, F32, 32, scale=0.1), x=rand(gen, BF16, rows, 256), w1=rand(gen, BF16, 32, 192, 256, scale=0.06),
                w=rand(gen, BF16, 128, 256, scale=0.06), a=rand(gen, BF16, 6, 16, 256, scale=0.06), b=rand(gen, BF16, 6, 128, 16, scale=0.2),
                scale=torch.rand(6, generator=gen, device="cuda"), ids=torch.randint(-1, 6, (rows,), generator=gen, device="cuda", dtype=torch.int32))


def test_results_do_not_depend_on_the_run(mps, cuda):
    t = everything_inputs(0)
    first = everything(mps, t)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, everything(mps, t)))


def test_two_streams_at_once(mps, cuda):
    inputs = [everything_inputs(1), everything_inputs(2, 400)]
    want = [everything(mps, t) for t in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        got = []
        for s, t in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append(everything(mps, t))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_stream_argument(mps, cuda):
    t = everything_inputs(3)
    want = everything(mps, t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    ag = mps.group_rows(t["ids"], 6, stream=s)
    out = mps.adapters(t["x"], t["w"], t["a"], t["b"], t["ids"], ag, t["scale"], stream=s)
    mps.routed_check(stream=s)
    assert torch.equal(out, want[-4])


@pytest.mark.parametrize("name", ["route", "route_backward", "group_rows", "product", "wgrad", "combine", "combine_backward", "adapters", "adapters_backward"])
def test_results_on_another_stream_are_memory_of_that_stream(mps, cuda, name):
    """The current stream is still going to write what it has freed; a call on another stream must not be given that."""
    gen = gen_of(11)
    x, dy, w = rand(gen, torch.bfloat16, 300, 64), rand(gen, torch.bfloat16, 600, 96), rand(gen, torch.bfloat16, 6, 96, 64)
    logits, weights = rand(gen, torch.float32, 300, 6), rand(gen, torch.float32, 300, 2)
    ids, _, groups = mps.route(logits, 2)
    one = ids[:, 0].contiguous()
    ag, a, b = mps.group_rows(one, 6), rand(gen, torch.bfloat16, 6, 8, 64), rand(gen, torch.bfloat16, 6, 96, 8)

    def call(s):
        if name == "route":
            ids_, weights_, groups_ = mps.route(logits, 2, stream=s)
            return (ids_, weights_, *groups_)
        if name == "route_backward":
            return (mps.route_backward(logits, ids, weights, stream=s),)
        if name == "group_rows":
            return tuple(mps.group_rows(ids, 6, stream=s))
        if name == "product":
            return (mps.routed_product(x, w, groups, stream=s),)
        if name == "wgrad":
            return (mps.routed_wgrad(x, dy, groups, stream=s),)
        if name == "combine":
            return (mps.routed_combine(dy, groups.slot, weights, stream=s),)
        if name == "combine_backward":
            return mps.routed_combine_backward(dy[:300], dy, groups.slot, weights, stream=s)
        if name == "adapters":
            return (mps.adapters(x, w[0], a, b, one, ag, stream=s),)
        return mps.adapters_backward(dy[:300], x, w[0], a, b, one, ag, stream=s)

    want = call(None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda._sleep(100_000_000)  # about 50 ms
    size = 4 * 600 + 7 if name == "route" else 0  # route's results share one allocation
    freed = [torch.empty(max(t.numel() * t.element_size(), 4 * size), dtype=torch.uint8, device="cuda") for t in want for _ in range(4)]
    for t in freed:
        t.fill_(3)
    del freed, t
    got = call(side)
    torch.cuda.synchronize()
    assert all(torch.equal(g, w_) for g, w_ in zip(got, want))


def test_stream_of_another_device_is_refused(mps, cuda):
    class Elsewhere:
        device, cuda_stream = torch.device("cuda", 99), 0

    slot = torch.zeros(4, 1, dtype=torch.int32, device="cuda")
    rows = torch.ones(4, 8, device="cuda")
    with pytest.raises(ValueError, match="stream: on cuda:99, expected cuda:0"):
        mps.routed_combine(rows, slot, out=torch.empty_like(rows), stream=Elsewhere())


def test_captured_and_replayed_on_new_inputs(mps, cuda):
    """Two graphs over the same inputs, replayed at once on two streams, after the inputs were changed in place."""
    t, other = everything_inputs(4), everything_inputs(5)
    everything(mps, t)
    torch.cuda.synchronize()
    graphs, results = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g in graphs:
        with torch.cuda.graph(g):
            results.append(everything(mps, t))
    for k in t:
        t[k].copy_(other[k])
    want = everything(mps, other)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    mps.routed_check()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, want))


def test_wrappers_refuse_what_is_not_contiguous_or_of_another_type(mps, cuda):
    t = everything_inputs(6)
    g = mps.group_rows(t["ids"], 32)
    for call in (lambda: mps.route(t["logits"].t(), 2), lambda: mps.route(t["logits"].double(), 2), lambda: mps.routed_product(t["x"][:, ::2], t["w1"], g),
                 lambda: mps.routed_product(t["x"], t["w1"].half(), g), lambda: mps.routed_product(t["x"], t["w1"][:8], g),
                 lambda: mps.routed_product(t["x"], t["w1"], g, out=torch.empty(3, 192, dtype=BF16, device="cuda")),
                 lambda: mps.routed_wgrad(t["x"], t["x"][:5], g), lambda: mps.group_rows(t["ids"].long(), 6),
                 lambda: mps.adapters(t["x"], t["w"], t["a"], t["b"], t["ids"], g, t["scale"]),
                 lambda: mps.routed_combine(t["x"], t["ids"].view(-1, 1).long()), lambda: mps.route(t["logits"], 2, score="tanh")):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(mps.MpsError) as e:
        mps.route(t["logits"], 33)
    assert e.value.code == mps.capi.ERR_ARG
