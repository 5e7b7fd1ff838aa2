"""Adapters whose low-rank intermediate is far from one: scale * x A^T and scale * dy B from 1e-10 to beyond fp16's largest value,
and infinite ones.  Results are held to the relative error of the intermediate alone, with no floor for it."""
import math

import numpy as np
import pytest
import torch

import routed_oracle as o
from routed_oracle import close, f64
from test_gpu_routed import rand, gen_of

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
# Relative error of the intermediate where the matrix gradients read it: half a step of the rest after half a step (as PAIR), and in
# fp16 2^-40 of the adapter's largest, which the tests below cover by magnitudes that differ by less than 2^18.
ROWS = [(60, "few rows: one pass over the shared matrix"), (1500, "tiles of one adapter each")]


def case(dtype, rows, n_adapters, rank, k, n, x_size, dy_size, b_size, a_size=1.0, seed=0):
    gen, rng = gen_of(seed + rows + rank), np.random.default_rng(seed + rows)
    ids = rng.integers(-1, n_adapters, rows).astype(np.int32)
    t = dict(x=rand(gen, dtype, rows, k, scale=x_size), w=rand(gen, dtype, n, k, scale=k ** -0.5), a=rand(gen, dtype, n_adapters, rank, k, scale=a_size * k ** -0.5),
             b=rand(gen, dtype, n_adapters, n, rank, scale=b_size * rank ** -0.5), dy=rand(gen, dtype, rows, n, scale=dy_size),
             scale=torch.rand(n_adapters, generator=gen, device="cuda") + 0.5)
    return ids, torch.from_numpy(ids).cuda(), t


def check(mps, dtype, ids, d_ids, t, n_adapters, forward=True, backward=True):
    rows, k = t["x"].shape
    n, rank = t["b"].shape[1:]
    groups = mps.group_rows(d_ids, n_adapters)
    wide = {name: f64(v) for name, v in t.items()}
    if forward:
        want = o.adapters(wide["x"], wide["w"], wide["a"], wide["b"], ids, wide["scale"])
        close(f64(mps.adapters(t["x"], t["w"], t["a"], t["b"], d_ids, groups, t["scale"])), want[0], dtype, k + rank + 2, want[1], o.PAIR[dtype] * want[2])
    if backward:
        got = mps.adapters_backward(t["dy"], t["x"], t["w"], t["a"], t["b"], d_ids, groups, t["scale"])
        wants = o.adapters_grad(wide["dy"], wide["x"], wide["w"], wide["a"], wide["b"], ids, wide["scale"])
        for g, want, terms in zip(got, wants, (n + rank + 2, n + rows + 2, k + rows + 2)):
            close(f64(g), want[0], dtype, terms, want[1], o.PAIR[dtype] * want[2])
    mps.routed_check()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,why", ROWS)
@pytest.mark.parametrize("rank", [8, 40, 136])
@pytest.mark.parametrize("dy_size,b_size", [(1e-3, 1e-3), (1.0, 1e-3), (1.0, 1e-5), (1e-3, 1e-5), (1e-2, 1e-5), (1.0, 1e-7)])
def test_small_intermediates(mps, cuda, dtype, rows, why, rank, dy_size, b_size):
    """The start of training: the second matrix is near zero, so dy B is."""
    ids, d_ids, t = case(dtype, rows, 4, rank, 256, 384, 1.0, dy_size, b_size)
    check(mps, dtype, ids, d_ids, t, 4)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,why", ROWS)
@pytest.mark.parametrize("size", [1e-3, 1e-5, 1e-7])
def test_small_rows(mps, cuda, dtype, rows, why, size):
    """x, dy and x A^T small; the results are small too, but for dA and dB times large rows."""
    ids, d_ids, t = case(dtype, rows, 3, 16, 256, 384, size, 1.0, 1.0, a_size=4.0)
    check(mps, dtype, ids, d_ids, t, 3)
    ids, d_ids, t = case(dtype, rows, 3, 16, 256, 384, 8.0, size, 8.0, a_size=8.0, seed=1)
    check(mps, dtype, ids, d_ids, t, 3)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,why", ROWS)
@pytest.mark.parametrize("rank", [8, 72])
def test_intermediates_beyond_half_precision(mps, cuda, dtype, rows, why, rank):
    """scale * x A^T about 1e6, the second matrix about 1e-6: their product is ordinary.  The gradient of the second matrix is
    dy^T times that, with dy about 1e-4; scale * dy B about 1e6 likewise against a first matrix about 1e-6."""
    ids, d_ids, t = case(dtype, rows, 4, rank, 256, 384, 1000.0, 1e-6, 1e-6, a_size=1000.0)
    check(mps, dtype, ids, d_ids, t, 4)
    ids, d_ids, t = case(dtype, rows, 4, rank, 256, 384, 1e-5, 1000.0, 1000.0, a_size=1e-5, seed=1)
    check(mps, dtype, ids, d_ids, t, 4)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,why", ROWS)
def test_adapters_of_different_magnitudes(mps, cuda, dtype, rows, why):
    """Adapters far apart in size beside one another: each keeps its own digits."""
    ids, d_ids, t = case(dtype, rows, 6, 24, 256, 384, 1.0, 1.0, 1.0)
    for i in range(6):
        t["a"][i] *= 10.0 ** (2 - i)
        t["b"][i] *= 10.0 ** (i - 5)
    check(mps, dtype, ids, d_ids, t, 6)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,why", ROWS)
def test_rows_of_different_magnitudes(mps, cuda, dtype, rows, why):
    """Rows of one adapter from 1e-5 to 1: y and dx of a small row keep its digits beside a large one."""
    ids, d_ids, t = case(dtype, rows, 3, 16, 256, 384, 1.0, 1.0, 1.0)
    size = torch.tensor([1e-5, 1e-3, 1.0, 1e-4], device="cuda").repeat((rows + 3) // 4)[:rows, None]
    t["x"], t["dy"] = (t["x"].float() * size).to(dtype), (t["dy"].float() * size).to(dtype)
    check(mps, dtype, ids, d_ids, t, 3)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,why", ROWS)
def test_infinite_intermediates(mps, cuda, dtype, rows, why):
    """An infinite scale * x A^T is infinite, not a NaN, wherever the second matrix is not zero, and so are its gradients; the other
    rows, adapters and ranks are what they were."""
    n_adapters, rank, k, n = 3, 16, 256, 384
    ids, d_ids, t = case(dtype, rows, n_adapters, rank, k, n, 1.0, 1.0, 1.0)
    t["x"].abs_()
    t["b"].abs_()
    t["a"].abs_()
    t["dy"].abs_()
    at = int(np.argwhere(ids == 1)[0, 0])
    groups = mps.group_rows(d_ids, n_adapters)
    y = mps.adapters(t["x"], t["w"], t["a"], t["b"], d_ids, groups, t["scale"])
    dx, da, db = mps.adapters_backward(t["dy"], t["x"], t["w"], t["a"], t["b"], d_ids, groups, t["scale"])
    assert all(torch.isfinite(v).all() for v in (y, dx, da, db))
    a = t["a"].clone()
    a[1, 5] = math.inf  # x A^T is infinite at one rank of adapter 1
    y2 = mps.adapters(t["x"], t["w"], a, t["b"], d_ids, groups, t["scale"])
    mine = d_ids == 1
    assert torch.isinf(y2[mine]).all() and torch.equal(y2[~mine], y[~mine])
    b = t["b"].clone()
    b[1, :, 5] = math.inf  # dy B likewise
    dx2, da2, db2 = mps.adapters_backward(t["dy"], t["x"], t["w"], t["a"], b, d_ids, groups, t["scale"])
    assert torch.isinf(dx2[mine]).all() and torch.equal(dx2[~mine], dx[~mine]) and torch.equal(db2, db)
    other = [r for r in range(rank) if r != 5]
    assert torch.isinf(da2[1, 5]).all() and torch.equal(da2[1, other], da[1, other]) and torch.equal(da2[[0, 2]], da[[0, 2]])
    x = t["x"].clone()
    x[at, 0] = math.inf  # one row: all ranks
    y3 = mps.adapters(x, t["w"].abs(), t["a"], t["b"], d_ids, groups, t["scale"])
    assert torch.isinf(y3[at]).all()
    _, da3, db3 = mps.adapters_backward(t["dy"], x, t["w"], t["a"], t["b"], d_ids, groups, t["scale"])
    assert torch.isinf(db3[1]).all() and torch.equal(db3[[0, 2]], db[[0, 2]])
    assert torch.isinf(da3[1, :, 0]).all() and torch.equal(da3[1, :, 1:], da[1, :, 1:]) and torch.equal(da3[[0, 2]], da[[0, 2]])
    mps.routed_check()


def test_rows_listed_in_another_order(mps, cuda):
    """The rows of a group may stand in any order in the caller's list."""
    for rows in (60, 1500):
        ids, d_ids, t = case(BF16, rows, 4, 16, 256, 384, 1.0, 1.0, 1.0)
        groups = mps.group_rows(d_ids, 4)
        row, ptr = groups.row.cpu().numpy().copy(), groups.ptr.tolist()
        rng = np.random.default_rng(0)
        for g in range(4):
            rng.shuffle(row[ptr[g]:ptr[g + 1]])
        shuffled = mps.Groups(groups.ptr, torch.from_numpy(row).cuda(), None)
        wide = {name: f64(v) for name, v in t.items()}
        want = o.adapters(wide["x"], wide["w"], wide["a"], wide["b"], ids, wide["scale"])
        close(f64(mps.adapters(t["x"], t["w"], t["a"], t["b"], d_ids, shuffled, t["scale"])), want[0], BF16, 256 + 18, want[1], o.PAIR[BF16] * want[2])
        got = mps.adapters_backward(t["dy"], t["x"], t["w"], t["a"], t["b"], d_ids, shuffled, t["scale"])
        wants = o.adapters_grad(wide["dy"], wide["x"], wide["w"], wide["a"], wide["b"], ids, wide["scale"])
        for g, want, terms in zip(got, wants, (384 + 18, 384 + rows + 2, 256 + rows + 2)):
            close(f64(g), want[0], BF16, terms, want[1], o.PAIR[BF16] * want[2])
        mps.routed_check()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("b_size", [1.0, 1e-5])
@pytest.mark.parametrize("rows,n_adapters,rank,k,n", [(3000, 4, 40, 512, 1024), (2600, 4, 16, 256, 512), (700, 2, 24, 768, 1160), (300, 2, 72, 2048, 520), (1, 1, 8, 64, 64)])
def test_every_tile(mps, cuda, dtype, b_size, rows, n_adapters, rank, k, n):
    """Tiles of 32 to 256 rows, sums cut over a cluster or not."""
    ids, d_ids, t = case(dtype, rows, n_adapters, rank, k, n, 1.0, 0.1, b_size)
    check(mps, dtype, ids, d_ids, t, n_adapters)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [60, 3000])
def test_infinite_matrices(mps, cuda, dtype, rows):
    """An infinite entry of a low-rank matrix gives what fp32 gives: the infinity of its rank's intermediate's sign."""
    ids, d_ids, t = case(dtype, rows, 3, 16, 512, 1024, 1.0, 1.0, 1.0)
    groups = mps.group_rows(d_ids, 3)
    mine = np.argwhere(ids == 2).ravel()
    y = mps.adapters(t["x"], t["w"], t["a"], t["b"], d_ids, groups, t["scale"])
    t["b"][2, 7, 3] = math.inf
    y2 = f64(mps.adapters(t["x"], t["w"], t["a"], t["b"], d_ids, groups, t["scale"]))
    u = f64(t["x"])[mine] @ f64(t["a"])[2, 3]
    assert (y2[mine, 7] == np.sign(u) * math.inf).all()
    y2[mine, 7] = 0
    same = f64(y)
    same[mine, 7] = 0
    assert (y2 == same).all()
    t["a"][2, 3, 9] = math.inf
    t["b"][2, 7, 3] = 1.0
    dx, _, _ = mps.adapters_backward(t["dy"], t["x"], t["w"], t["a"], t["b"], d_ids, groups, t["scale"])
    v = f64(t["dy"])[mine] @ f64(t["b"])[2, :, 3]
    assert (f64(dx)[mine, 9] == np.sign(v) * math.inf).all()
    assert torch.isfinite(dx).sum() == dx.numel() - len(mine)


def both(mps, t, d_ids, groups):
    return [mps.adapters(t["x"], t["w"], t["a"], t["b"], d_ids, groups, t["scale"]),
            *mps.adapters_backward(t["dy"], t["x"], t["w"], t["a"], t["b"], d_ids, groups, t["scale"])]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 60, 1500, 3000])
def test_captured_and_on_two_streams(mps, cuda, dtype, rows):
    """Two graphs replayed at once on two streams, on inputs that changed since; and eager calls side by side."""
    cases = [case(dtype, rows, 5, 40, 512, 1024, 1.0, 1.0, size, seed=i) for i, size in enumerate((1.0, 1e-4))]
    lists = [mps.group_rows(d_ids, 5) for _, d_ids, _ in cases]
    want = [both(mps, t, d_ids, g) for (_, d_ids, t), g in zip(cases, lists)]
    torch.cuda.synchronize()
    held = [{k: v.clone() for k, v in cases[0][2].items()} for _ in range(2)]
    ids = [cases[0][1].clone() for _ in range(2)]
    groups = [mps.Groups(*(p.clone() for p in lists[0])) for _ in range(2)]
    graphs, results = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            results.append(both(mps, held[i], ids[i], groups[i]))
    for k, v in cases[1][2].items():
        held[1][k].copy_(v)
    ids[1].copy_(cases[1][1])
    for p, q in zip(groups[1], lists[1]):
        p.copy_(q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        eager = []
        for s, g, (_, d_ids, t), l in zip(streams, graphs, cases, lists):
            with torch.cuda.stream(s):
                g.replay()
                eager.append(both(mps, t, d_ids, l))
                g.replay()
        torch.cuda.synchronize()
        for got in (results, eager):
            assert all(torch.equal(a, b) for r, w in zip(got, want) for a, b in zip(r, w))
    mps.routed_check()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [60, 1500])
def test_wrong_lists_are_reported_and_harmless(mps, cuda, dtype, rows):
    """Rows and offsets out of range in the caller's list: reported, nothing outside the arrays touched, and the adapters whose lists are
    right keep their gradients."""
    ids, d_ids, t = case(dtype, rows, 4, 16, 256, 384, 1.0, 1.0, 1.0)
    groups = mps.group_rows(d_ids, 4)
    want = both(mps, t, d_ids, groups)
    ptr = groups.ptr.tolist()
    row = groups.row.clone()
    row[ptr[1]], row[ptr[1] + 1] = -7, rows + 5
    got = both(mps, t, d_ids, mps.Groups(groups.ptr, row, None))
    with pytest.raises(mps.MpsError) as e:
        mps.routed_check()
    assert e.value.code == mps.capi.ERR_ARG
    for a, b in ((got[2], want[2]), (got[3], want[3])):
        assert torch.equal(a[[0, 2, 3]], b[[0, 2, 3]]) and torch.isfinite(a).all()
    for bad in ([0, ptr[1], 2**31 - 1, -5, ptr[4]], [5, 1, 3, 2, rows], [-2**31] * 5, [rows] * 5):
        both(mps, t, d_ids, mps.Groups(torch.tensor(bad, dtype=torch.int32, device="cuda"), groups.row, None))
        torch.cuda.synchronize()
        try:
            mps.routed_check()
        except mps.MpsError as x:
            assert x.code == mps.capi.ERR_ARG
    assert all(torch.equal(a, b) for a, b in zip(both(mps, t, d_ids, groups), want))
    mps.routed_check()


@pytest.mark.parametrize("rows,why", ROWS)
@pytest.mark.parametrize("x_size,b_size", [(1e-17, 1e22), (1e-18, 1e23), (1e17, 1e-20)])
def test_bf16_intermediates_at_the_ends_of_its_range(mps, cuda, rows, why, x_size, b_size):
    """Sums of eight products, so that what the intermediate itself loses shows: about 1e-34, 1e-35 and 1e34 (by matrices of the same
    size as x); the gradients likewise.  A value's second part is what bf16 rounds it to: half a step of 2^-16 of the value, or, below
    2^-118, where that part is subnormal, half a step of 2^-133 of it, which meets |b| (or |a|).  At 1e-35 some values are."""
    ids, d_ids, t = case(BF16, rows, 3, 8, 8, 64, x_size, 1.0, b_size, a_size=x_size)
    wide = {name: f64(v) for name, v in t.items()}
    want = o.adapters(wide["x"], wide["w"], wide["a"], wide["b"], ids, wide["scale"])
    close(f64(mps.adapters(t["x"], t["w"], t["a"], t["b"], d_ids, mps.group_rows(d_ids, 3), t["scale"])), want[0], BF16, 8 + 8 + 2, want[1],
          o.PAIR[BF16] * want[2] + 2.0 ** -134 * want[3])
    gen = gen_of(rows)  # dx = dy W + (scale dy B) A with dy and B small (large), A large (small)
    t = dict(x=rand(gen, BF16, rows, 64), w=rand(gen, BF16, 8, 64, scale=x_size), a=rand(gen, BF16, 3, 8, 64, scale=b_size), b=rand(gen, BF16, 3, 8, 8, scale=x_size),
             dy=rand(gen, BF16, rows, 8, scale=x_size), scale=torch.ones(3, device="cuda"))
    groups = mps.group_rows(d_ids, 3)
    wide = {name: f64(v) for name, v in t.items()}
    dx, _, _ = mps.adapters_backward(t["dy"], t["x"], t["w"], t["a"], t["b"], d_ids, groups, t["scale"])
    want = o.adapters_grad(wide["dy"], wide["x"], wide["w"], wide["a"], wide["b"], ids, wide["scale"])[0]
    close(f64(dx), want[0], BF16, 8 + 8 + 2, want[1], o.PAIR[BF16] * want[2] + 2.0 ** -134 * want[3])
    mps.routed_check()
