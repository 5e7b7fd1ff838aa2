"""The router's choice where it is hard to tell (equal keys at the last place, keys in one bucket of the packed form, group ranks
whose two keys cancel or leave fp32's range), and every form of the kernel for many rows, against the 64-bit definition."""
import math

import numpy as np
import pytest
import torch

import routed_oracle as o

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
FEW, MANY = 40, 2061  # a warp per row; eight lanes per row (from 2048 rows on)


def ids_of(mps, logits, top, **kw):
    ids = mps.route(logits, top, group=False, **kw)[0]
    mps.routed_check()
    return ids.cpu().numpy()


def same_choice(mps, logits, top, **kw):
    """As the definition has it, and the same whether the rows come at once or a few at a time."""
    want, _ = o.route(logits.detach().cpu().double().numpy(), top, kw.get("score", "softmax"), None if kw.get("bias") is None else kw["bias"].cpu().double().numpy(),
                      kw.get("n_groups", 1), kw.get("top_groups", 1), kw.get("group_top", 1))
    got = ids_of(mps, logits, top, **kw)
    bad = np.argwhere((got != want).any(1)).ravel()
    assert not bad.size, (bad.size, bad[:4], got[bad[:4]], want[bad[:4]])


@pytest.mark.parametrize("rows", [FEW, MANY])
@pytest.mark.parametrize("experts", [24, 64, 200])
@pytest.mark.parametrize("places", [(0, 1, 2), (0, 9, 18), (5, 3, 20), (2, 0, 1)])
def test_equal_logits_before_a_larger_one(mps, cuda, rows, experts, places):
    """Two equal logits, and one a unit in the last place above them, asked for the best one and the best two."""
    logits = torch.rand(rows, experts, generator=torch.Generator(device="cuda").manual_seed(experts), device="cuda") - 3
    first, second, third = places
    logits[:, first] = logits[:, second] = 1.0
    logits[:, third] = float(np.nextafter(np.float32(1.0), np.float32(2.0)))
    for top in (1, 2):
        same_choice(mps, logits, top)
        same_choice(mps, -logits, top)  # negative keys
        same_choice(mps, logits, top, n_groups=8, top_groups=8, score="sigmoid")


@pytest.mark.parametrize("rows", [FEW, MANY])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("equals", [2, 3, 7])
def test_equal_keys_at_the_last_place(mps, cuda, rows, dtype, score, equals):
    """Keys that fp32 cannot tell apart: several experts of equal logit and bias, and later ones whose score is larger or smaller
    by less than fp32 resolves."""
    logits = torch.full((rows, 64), -40.0, dtype=dtype, device="cuda")
    base = 20.0 if score == "sigmoid" else 0.0  # a sigmoid of 20 and more is 1 in fp32
    logits[:, 4:4 + equals] = base
    logits[::2, 30] = base + 0.125
    logits[1::2, 30] = base - 0.125
    logits[::3, 50] = base + 0.25
    if score == "softmax":
        logits[:, 63] = 60.0  # the others' scores are below 1e-22: nothing beside the bias
    bias = torch.zeros(64, device="cuda")
    bias[4:51] = 1.0
    for top in (1, 2, 3, equals, equals + 1, equals + 2):
        same_choice(mps, logits, top, score=score, bias=bias)
        same_choice(mps, logits, top, score=score, bias=bias, n_groups=4, top_groups=4)


@pytest.mark.parametrize("rows", [FEW * 8, 4096])
@pytest.mark.parametrize("top", [1, 2])
def test_keys_beside_a_bucket_edge(mps, cuda, rows, top):
    """Keys around a number whose last five bits are zeros: the best is just above it, one just below, and one further down with a
    lower index.  Their distance is a few units of fp32's last place, which is what the scores' errors are."""
    rng = np.random.default_rng(rows + top)
    experts = 32
    bias = (1.0 - rng.random(experts) * 0.5).astype(np.float32)
    logits = np.full((rows, experts), -9.0)
    edge = 1 + 2.0 ** -18 * rng.integers(20000, 40000, rows)  # multiples of 32 units of [1, 2)

    def put(e, key):
        logits[:, e] = np.log((key - bias[e]) / (1 - (key - bias[e])))

    unit = 2.0 ** -23
    put(0, edge - (20 + 10 * rng.random(rows)) * unit)
    put(1, edge + rng.normal(size=rows) * 2 * unit)
    put(2, edge + rng.normal(size=rows) * 2 * unit)
    if top == 2:
        put(3, edge + 0.01)
    order = np.concatenate([rng.permutation(4), np.arange(4, experts)])
    for at in (np.arange(experts), order):
        same_choice(mps, torch.from_numpy(np.ascontiguousarray(logits[:, at], dtype=np.float32)).cuda(), top, score="sigmoid", bias=torch.from_numpy(bias[at]).cuda())


@pytest.mark.parametrize("rows", [FEW * 10, MANY])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("size", [1000.0, 3e5])
def test_group_ranks_whose_keys_cancel(mps, cuda, rows, score, size):
    """Groups of two experts with biases of +size and -size: the ranks are sums of the two scores, far finer than either key."""
    rng = np.random.default_rng(int(size))
    logits = rng.normal(size=(rows, 16)).astype(np.float32)
    if score == "sigmoid":  # neighbouring groups' sums of scores within the rounding of a key of one another
        s = 1 / (1 + np.exp(-logits.astype(np.float64)))
        want = np.clip(s[:, 0] + s[:, 1] - s[:, 2] + rng.normal(size=rows) * size * 2.0 ** -24, 1e-3, 1 - 1e-3)
        logits[:, 3] = np.log(want / (1 - want))
    bias = np.tile([size, -size], 8).astype(np.float32)
    same_choice(mps, torch.from_numpy(logits).cuda(), 2, score=score, bias=torch.from_numpy(bias).cuda(), n_groups=8, top_groups=1, group_top=2)
    same_choice(mps, torch.from_numpy(logits).cuda(), 3, score=score, bias=torch.from_numpy(bias).cuda(), n_groups=8, top_groups=4, group_top=2)


@pytest.mark.parametrize("rows", [FEW, MANY])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("value", [torch.finfo(F32).min, torch.finfo(F32).max])
def test_group_ranks_beyond_the_type(mps, cuda, rows, score, value):
    """Experts masked (or forced) by a bias of the type's lowest (largest) value: the sum of two such keys has left fp32, the group
    has not left the choice."""
    logits = torch.randn(rows, 32, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    for masked in (slice(0, 16), slice(8, 32), slice(0, 32), slice(8, 30)):
        bias = torch.zeros(32, device="cuda")
        bias[masked] = value
        for n_groups, top_groups in ((4, 2), (4, 3), (8, 5), (2, 1)):
            same_choice(mps, logits, 6, score=score, bias=bias, n_groups=n_groups, top_groups=top_groups, group_top=2)


MANY_FORMS = [
    # experts, groups, top_groups, group_top, top: every width of the eight-lane form, its groups, and choices in each of its lanes' places
    (8, 1, 1, 1, 8), (64, 2, 1, 2, 17), (72, 1, 1, 1, 9), (72, 4, 2, 2, 24), (128, 1, 1, 1, 1), (128, 2, 1, 1, 16), (128, 4, 3, 2, 32), (128, 8, 4, 2, 8),
    (136, 8, 2, 1, 12), (200, 2, 2, 2, 32), (200, 1, 1, 1, 16), (256, 1, 1, 1, 8), (256, 2, 1, 2, 1), (256, 4, 2, 1, 16), (256, 8, 4, 2, 8), (256, 8, 3, 2, 32),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("experts,n_groups,top_groups,group_top,top", MANY_FORMS)
def test_many_rows(mps, cuda, dtype, experts, n_groups, top_groups, group_top, top):
    from test_gpu_routed import check_route
    gen = torch.Generator(device="cuda").manual_seed(experts + top)
    rows = MANY
    logits = (torch.randn(rows, experts, generator=gen, device="cuda") * 1.5).to(dtype)
    bias = torch.randn(experts, generator=gen, device="cuda") * 0.05
    groups = dict(n_groups=n_groups, top_groups=top_groups, group_top=group_top)
    check_route(mps, logits, top, score="sigmoid", bias=bias, scale=2.5, **groups)
    check_route(mps, logits, top, renormalise=False, **groups)
    logits[:, torch.rand(experts, generator=gen, device="cuda") < 0.4] = -math.inf  # masked experts, and rows with none left
    logits[::3] = -math.inf
    logits[1::7, : max(1, experts // 2)] = torch.finfo(dtype).min
    flat = torch.empty(rows * experts + 1, dtype=dtype, device="cuda")  # the same rows off 16 bytes
    shifted = flat[1:].view(rows, experts)
    shifted.copy_(logits)
    for score, b, renormalise in (("softmax", bias, True), ("sigmoid", None, False)):
        ids, weights = check_route(mps, logits, top, score=score, bias=b, renormalise=renormalise, **groups)
        again, same, _ = mps.route(shifted, top, score=score, bias=b, renormalise=renormalise, **groups)
        assert torch.equal(ids, again) and torch.equal(weights, same)
        few = torch.cat([mps.route(part, top, score=score, bias=b, renormalise=renormalise, group=False, **groups)[0] for part in logits.split(1000)])
        assert torch.equal(ids, few)


@pytest.mark.parametrize("experts,n_groups,top", [(128, 1, 9), (128, 8, 9), (256, 1, 20), (256, 4, 20)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_many_rows_of_equal_and_close_keys(mps, cuda, experts, n_groups, top, score, biased):
    gen = torch.Generator(device="cuda").manual_seed(7)
    equal = torch.randint(-2, 3, (MANY, experts), generator=gen, device="cuda").float()
    close = 3 + torch.rand(MANY, experts, generator=gen, device="cuda") * 1e-5  # a few units in the last place apart
    bias = torch.randint(0, 2, (experts,), generator=gen, device="cuda").float() * 0.25 if biased else None
    for logits in (equal, equal.bfloat16(), close):
        for group_top in (1, 2):
            same_choice(mps, logits, top, score=score, bias=bias, n_groups=n_groups, top_groups=max(1, n_groups // 2), group_top=group_top)
