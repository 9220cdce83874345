"""Routing to experts and the weighted sum (csrc/expert_routing.hip) against their definitions in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF, FLOAT = torch.float16, torch.float32


@pytest.fixture(scope="module")
def g():
    import gpu_util
    gpu_util.capi.init(0)
    return gpu_util


def normal(seed, shape, dtype, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale).to(dtype).cuda()


def reference(logits, k, bias, score, groups, top_groups, group_best, normalize, scale):
    x = logits.double().cpu()
    x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=torch.finfo(FLOAT).max)
    T, E = x.shape
    if score == "softmax":
        most = x.max(1, keepdim=True).values
        e = torch.exp(x - torch.where(most == -math.inf, 0.0, most))
        p = torch.where(e > 0, e / e.sum(1, keepdim=True), 0.0)
    else:
        p = torch.sigmoid(x)
    key = p if bias is None else p + bias.double().cpu()
    # (without bias and groups the logits say the same and tell apart what has one score in 64 bits)
    if bias is None and groups == 1:
        key = x
    if groups > 1:
        each = key.reshape(T, groups, -1)
        best = each.sort(dim=2, descending=True).values[:, :, :group_best].sum(2).sort(dim=1, descending=True, stable=True).indices[:, :top_groups]
        taken = torch.zeros(T, groups, dtype=torch.bool).scatter_(1, best, True).repeat_interleave(E // groups, 1)
    else:
        taken = torch.ones_like(key, dtype=torch.bool)
    experts = torch.empty(T, k, dtype=torch.int64)
    for t in range(T):
        at = taken[t].nonzero()[:, 0]
        experts[t] = at[key[t][at].sort(descending=True, stable=True).indices[:k]]
    w = p.gather(1, experts)
    if normalize:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    flat = experts.reshape(-1)
    offsets = torch.zeros(E + 1, dtype=torch.int64)
    offsets[1:] = torch.bincount(flat, minlength=E).cumsum(0)
    return experts, w * scale, torch.sort(flat, stable=True).indices, offsets


def check(g, logits, k, bias=None, score="softmax", groups=1, top_groups=None, group_best=1, normalize=True, scale=1.0):
    got = g.ops.ExpertRouting(logits, k, bias=bias, score=score, groups=groups, top_groups=top_groups, group_best=group_best, normalize=normalize, scale=scale)
    want = reference(logits, k, bias, score, groups, groups if top_groups is None else top_groups, group_best, normalize, scale)
    for i, name in ((0, "experts"), (2, "order"), (3, "offsets")):
        assert got[i].dtype == torch.int32 and torch.equal(got[i].cpu().long(), want[i]), name
    # float32: exponentials of arguments whose rounding is 2^-24 of up to 16, a sum of E and a division
    E = logits.shape[1]
    assert ((got[1].double().cpu() - want[1]).abs() <= abs(scale) * (16 + E) * 2.0 ** -24).all()
    return got


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 8), (3, 60, 5), (32, 64, 2), (33, 65, 7), (100, 300, 64), (257, 1000, 10), (1100, 128, 8), (2051, 20, 3), (5000, 513, 4)])
@pytest.mark.parametrize("dtype", [HALF, FLOAT])
def test_sizes(g, T, E, k, dtype):
    """Both launches and every width; half of the cases with a bias (in 64 bits then), float16 logits with many equal ones."""
    logits = normal(1, (T, E), dtype, 1.5)
    bias = normal(2, (E,), FLOAT, 0.1) if (T + E) % 2 else None
    check(g, logits, k, bias=bias, score="sigmoid" if T % 3 else "softmax", normalize=bool(k % 2), scale=2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,groups,top_groups,group_best", [(5, 16, 4, 4, 2, 2), (40, 256, 8, 8, 4, 2), (70, 96, 3, 3, 1, 1), (9, 64, 2, 64, 2, 1), (130, 160, 6, 8, 8, 2), (6, 1024, 20, 4, 1, 2)])
def test_groups(g, score, T, E, k, groups, top_groups, group_best):
    logits = normal(3, (T, E), FLOAT, 1.5)
    for bias in (None, normal(4, (E,), FLOAT, 0.2)):
        check(g, logits, k, bias=bias, score=score, groups=groups, top_groups=top_groups, group_best=group_best)


def test_equal_scores_take_the_lower_index(g):
    logits = torch.zeros(50, 64, device="cuda")
    logits[10:, 32:] = 1.0
    logits[20:30] = -0.0
    for bias in (None, torch.zeros(64, device="cuda")):
        for groups in (1, 8):
            check(g, logits, 6, bias=bias, groups=groups, top_groups=groups if groups == 1 else 2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("with_bias", [False, True])
def test_masked_rows(g, score, dtype, with_bias):
    """Rows with nothing but -inf, fewer experts than are asked for, the type's lowest and largest values, infinities and NaN."""
    logits = normal(5, (40, 24), dtype)
    logits[0] = -math.inf
    logits[1, 3:] = -math.inf
    logits[2, 5] = math.inf
    logits[3, ::2] = math.nan
    logits[4] = math.nan
    logits[5] = torch.finfo(dtype).min
    logits[6, 1:] = torch.finfo(dtype).min
    logits[7] = torch.finfo(dtype).max
    bias = normal(6, (24,), FLOAT, 0.1) if with_bias else None
    for normalize in (True, False):
        got = check(g, logits, 5, bias=bias, score=score, normalize=normalize)
        assert torch.isfinite(got[1]).all() and float(got[1][0].abs().max()) == 0.0


def test_a_bias_that_is_not_finite(g):
    bias = torch.zeros(16, device="cuda")
    bias[3], bias[4] = -math.inf, math.inf
    check(g, normal(7, (9, 16), FLOAT), 15, bias=bias)
    check(g, normal(7, (9, 16), FLOAT), 3, bias=bias, groups=4, top_groups=2, group_best=2)


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("E", [20, 70, 600])
@pytest.mark.parametrize("score,low,choice", [("sigmoid", (-86.0, -104.0), None), ("sigmoid", (-100.0, -690.0), None), ("sigmoid", (-86.0, -104.0), "zeros"),
                                              ("sigmoid", (-100.0, -690.0), "groups"), ("softmax", (-70.0, -110.0), "moved"), ("softmax", (-100.0, -690.0), "moved")])
def test_weights_of_very_low_scores(g, score, low, choice, E, normalize):
    """Scores that 64 bits hold and 32 do not: their shares, and what is left of them after a scale that brings them back.

    The score, the sum of four of them and their quotient are off by less than 700 * 2^-52 (an exponent of up to 700, rounded to 64 bits) and a few roundings of 2^-53; the
    result is rounded to float32 once, by 2^-24 of itself."""
    T, k = 21, 4
    first, last = low
    logits = (first + (last - first) * torch.rand(T, E, generator=torch.Generator().manual_seed(31))).cuda()
    bias, groups = None, 1
    if choice == "moved":  # the experts that have the scores are switched off, the next best ones are chosen
        logits[:, 2] = 0.5
        logits[:, 5] = 0.0
        bias = torch.zeros(E, device="cuda")
        bias[2] = bias[5] = -math.inf
    elif choice == "zeros":
        bias = torch.zeros(E, device="cuda")
    elif choice == "groups":
        groups = 5
    scale = 1.5 if normalize else 2.0 ** 100
    got = g.ops.ExpertRouting(logits, k, bias=bias, score=score, groups=groups, top_groups=groups, normalize=normalize, scale=scale)
    want = reference(logits, k, bias, score, groups, groups, 1, normalize, scale)
    for i in (0, 2, 3):
        assert torch.equal(got[i].cpu().long(), want[i])
    y = got[1].double().cpu()
    assert bool((want[1].sum(1) > 0).all()) and ((y - want[1]).abs() <= (2.0 ** -24 + 2.0 ** -40) * want[1] + 2.0 ** -150).all()
    if normalize:
        assert ((y.sum(1) - scale).abs() <= 4 * 2.0 ** -24 * scale).all()


def test_scores_that_are_equal_in_64_bits(g):
    """Sigmoids of 40, 50 and 60 are all 1, softmaxes of -900 and -800 beside 1 both 0: without bias and groups their logits tell them apart, else their index does."""
    zeros = torch.zeros(4, device="cuda")
    x = torch.tensor([[40.0, 60.0, 50.0, 1.0]], device="cuda")
    assert g.ops.ExpertRouting(x, 3, score="sigmoid")[0].cpu().tolist() == [[1, 2, 0]]
    assert g.ops.ExpertRouting(x, 3, score="sigmoid", bias=zeros)[0].cpu().tolist() == [[0, 1, 2]]
    assert g.ops.ExpertRouting(x, 3, score="sigmoid", groups=2, top_groups=2)[0].cpu().tolist() == [[0, 1, 2]]
    x = torch.tensor([[0.0, -900.0, -800.0, 1.0]], device="cuda")
    assert g.ops.ExpertRouting(x, 3)[0].cpu().tolist() == [[3, 0, 2]]
    assert g.ops.ExpertRouting(x, 3, bias=zeros)[0].cpu().tolist() == [[3, 0, 1]]


def test_strides_and_no_rows(g):
    space = normal(8, (80, 150), HALF)
    check(g, space[::2, 3:67], 4)
    check(g, space[:, ::3], 4)
    check(g, space.T, 4, bias=normal(9, (80,), FLOAT))
    empty = g.ops.ExpertRouting(space[:0], 4)
    assert empty[0].shape == (0, 4) and empty[2].shape == (0,) and empty[3].cpu().tolist() == [0] * 151


def test_numbers_that_are_refused(g):
    """Of more than 32 bits, or more experts or alternatives than there are: before results of such sizes are allocated."""
    logits = normal(18, (4096, 64), FLOAT)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.max_memory_allocated()
    for names in ({"groups": 2 ** 32 + 1}, {"groups": 2, "top_groups": 2 ** 32 + 1}, {"group_best": 2 ** 32 + 1}):
        with pytest.raises(ValueError):
            g.ops.ExpertRouting(logits, 2, **names)
    for k in (0, 65, 10 ** 6):
        with pytest.raises(ValueError):
            g.ops.ExpertRouting(logits, k)
    for top in (65, 10 ** 6):
        with pytest.raises(g.capi.ChxHipError):
            g.ops.TokenLogProbs(logits, None, top=top)
    with pytest.raises(ValueError):
        g.ops.TokenLogProbs(logits, None, top=-1)
    assert torch.cuda.max_memory_allocated() == before


@pytest.mark.parametrize("T", [20, 900])
def test_recorded_twice(g, T):
    """Two recorded calls side by side, replayed with eager calls in between."""
    logits = normal(10, (T, 96), FLOAT), normal(11, (T, 96), FLOAT)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = [g.ops.ExpertRouting(x, 6) for x in logits]
    for i in range(3):
        for j, x in enumerate(logits):
            x.copy_(normal(20 + 2 * i + j, x.shape, FLOAT))
        graph.replay()
        torch.cuda.synchronize()
        for x, got in zip(logits, recorded):
            for a, b in zip(got, g.ops.ExpertRouting(x, 6)):
                assert torch.equal(a, b)


def test_almost_2_to_the_31_rows(g):
    """The most rows there can be: the last chunk's end, and a wavefront's step behind it, are above 2^31.  (4 GB of logits, 26 GB of results.)"""
    T = 2 ** 31 - 9
    logits = torch.zeros(T, 1, dtype=HALF, device="cuda")
    experts, weights, order, offsets = g.ops.ExpertRouting(logits, 1)
    assert offsets.tolist() == [0, T]
    step = 1 << 28
    for first in range(0, T, step):
        last = min(first + step, T)
        assert not bool(experts[first:last].any()) and bool((weights[first:last] == 1).all())
        assert torch.equal(order[first:last], torch.arange(first, last, dtype=torch.int32, device="cuda"))
    del logits, experts, weights, order
    torch.cuda.empty_cache()


# ---- the weighted sum -----------------------------------------------------------------------------------

def check_sum(g, x, weights, r=None, out=None):
    y = g.ops.ExpertCombine(x, weights, r=r, out=out)
    T, k = weights.shape
    terms = x.double().reshape(T, k, -1) * weights.double()[:, :, None]
    terms = torch.where((weights == 0)[:, :, None], torch.zeros_like(terms), terms)
    want, size = terms.sum(1), terms.abs().sum(1)
    return y, want, size


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("T,k,n", [(1, 1, 1), (3, 2, 64), (17, 8, 200), (5, 6, 333), (300, 5, 1024), (2, 9, 8)])
def test_sums(g, dtype, T, k, n):
    x, weights, r = normal(12, (T * k, n), dtype), normal(13, (T, k), FLOAT), normal(14, (T, n), dtype)
    weights[0, 0] = 0.0
    x[0] = math.nan                                  # its weight is 0: it adds nothing
    half = 2.0 ** -11 if dtype == HALF else 2.0 ** -24
    for given in (None, r):
        y, want, size = check_sum(g, x, weights, given)
        if given is not None:
            want, size = want + given.double(), size + given.double().abs()
        assert y.dtype == dtype and ((y.double() - want).abs() <= half * want.abs() + (k + 2) * 2.0 ** -24 * size + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
def test_sums_of_any_strides(g, dtype):
    T, k, n = 12, 3, 64
    weights, r = normal(15, (T, k), FLOAT), normal(16, (T, n), dtype)
    plain = normal(17, (T * k, n), dtype)
    want = g.ops.ExpertCombine(plain, weights, r=r)
    for first, gap, col in [(0, 8, 1), (1, 2, 1), (0, 0, 2)]:
        space = torch.full((T * k, first + n * col + gap), math.nan, dtype=dtype, device="cuda")
        x = space[:, first: first + n * col: col]
        x.copy_(plain)
        out = torch.full((T + 1, 2 * n + 1), 7.0, dtype=dtype, device="cuda")
        y = out[:T, 1: 1 + n * col: col]
        assert g.ops.ExpertCombine(x, weights, r=r, out=y) is y and torch.equal(y, want)
        y.fill_(7.0)
        assert bool((out == 7.0).all())
    assert g.ops.ExpertCombine(plain, weights, r=r, out=r) is r and torch.equal(r, want)


def test_more_sums_than_one_launch_has(g):
    """More than 2^31 results, an element to a lane: what lies behind the first launch's part."""
    T, n = (1 << 19) + 3, 4099
    x = torch.randint(-4, 5, (64, n), dtype=torch.int8, device="cuda").half().repeat(T // 64 + 1, 1)[:T]
    weights = 2.0 * torch.ones(T, 1, device="cuda")
    y = g.ops.ExpertCombine(x, weights)
    for first in range(0, T, 1 << 16):
        assert torch.equal(y[first: first + (1 << 16)], 2 * x[first: first + (1 << 16)])
    del x, y
    torch.cuda.empty_cache()
