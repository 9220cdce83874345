"""Products with an epilogue from a plan (csrc/linear_plan.hip), against the formula in 64 bits, element by element.

The bound of an element: its rounding (half a step: 2^-11 of a float16 value, 2^-24 of a float32 one, and half the smallest float16 step), and
what float32 sums may lose: a rounding of 2^-24 for each of the K additions and a few for scale, bias, activation and residual, of at most the sum
of the magnitudes A.  The activations stretch an error by less than 1.2, and are themselves off by less than 4e-6 of their argument (float16
results: the short exponentials and the fitted polynomial) or 2^-20 (float32 ones)."""
import math

import pytest
import torch

import linear_sizes

pytestmark = pytest.mark.gpu

HALF, FLOAT = torch.float16, torch.float32
ACTS = {"": lambda v: v, "relu": lambda v: v.clamp(min=0), "silu": lambda v: v * torch.sigmoid(v), "gelu": lambda v: v * torch.special.erfc(-v / math.sqrt(2)) / 2,
        "gelu_tanh": lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))}


@pytest.fixture(scope="module")
def g():
    import gpu_util
    gpu_util.capi.init(0)
    return gpu_util


def normal(seed, shape, dtype, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale).to(dtype).cuda()


def weights(seed, shape, kind):
    """(w, w_scale) of outputs of about 1."""
    k = shape[-1]
    if kind != torch.int8:
        return normal(seed, shape, kind, k ** -0.5), None
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=gen, dtype=torch.int8).cuda(), ((torch.rand(shape[:-1], generator=gen) + 0.5) / (73 * k ** 0.5)).cuda()


def formula(x, w, scale, b, act, r):
    """(result, bound of what the sums may lose) in 64 bits."""
    x, w = x.double().cpu(), w.double().cpu()
    v, size = x @ w.T, x.abs() @ w.abs().T
    if scale is not None:
        v, size = v * scale.double().cpu(), size * scale.double().cpu()
    if b is not None:
        v, size = v + b.double().cpu(), size + b.double().cpu().abs()
    y = ACTS[act](v)
    if r is not None:
        y = y + r.double().cpu()
    return y, size


def check(y, want, size, K):
    got = y.double().cpu()
    half = y.dtype == HALF
    bound = (2.0 ** -11 if half else 2.0 ** -24) * want.abs() + (2.0 ** -25 if half else 0) + 1.2 * (K + 8) * 2.0 ** -24 * size + (4e-6 if half else 2.0 ** -20) * size
    off = (got - want).abs() - bound
    assert torch.isfinite(got).all() and off.max() <= 0, "off by %g more than the bound" % off.max()


TYPES = [(HALF, HALF), (HALF, torch.int8), (FLOAT, FLOAT)]


@pytest.mark.parametrize("kind,w_kind", TYPES)
@pytest.mark.parametrize("m,k,n", [
    (1, 1, 1), (1, 64, 16), (3, 130, 65), (16, 512, 64), (17, 63, 100), (33, 256, 33),         # few rows: one, two, four tiles of 16
    (64, 1000, 130), (65, 64, 64), (129, 96, 200), (300, 330, 17),                             # the bounds of both kernels, ragged steps
    (2000, 128, 6600),                                                                         # the large tiles
    (150, 72, 10300), (300, 130, 9000), (90, 200, 9700),                                       # tiles of 64 x 128, of 128 x 128; more than one round of few rows
    (1, 0x1200, 0x900),
])
def test_sizes(g, kind, w_kind, m, k, n):
    act = sorted(ACTS)[(m + k + n) % 5]
    x, (w, scale) = normal(1, (m, k), kind), weights(2, (n, k), w_kind)
    b, r = (normal(3, (n,), kind) if n % 2 else None), (normal(4, (m, n), kind) if m % 2 else None)
    plan = g.ops.LinearPlan(w, b=b, w_scale=scale)
    y = plan.run(x, activation=act, r=r)
    assert y.dtype == kind and y.shape == (m, n)
    check(y, *formula(x, w, scale, b, act, r), k)


@pytest.mark.parametrize("kind,w_kind", TYPES)
@pytest.mark.parametrize("act", sorted(ACTS))
def test_epilogue(g, kind, w_kind, act):
    """Every activation over a wide range of sums, with all operands; a float32 result of float16 rows."""
    m, k, n = 40, 70, 72
    x, (w, scale) = normal(5, (m, k), kind, 6.0), weights(6, (n, k), w_kind)
    b, r = normal(7, (n,), FLOAT, 3.0), normal(8, (m, n), FLOAT)
    plan = g.ops.LinearPlan(w, b=b, w_scale=scale)
    check(plan.run(x, activation=act, r=r, dtype=FLOAT), *formula(x, w, scale, b, act, r), k)
    if kind == HALF:
        check(plan.run(x, activation=act, r=r.half()), *formula(x, w, scale, b, act, r.half()), k)


def activated(g, w_kind, values, act, r=None):
    """act of each of the values as a float32 result of float16 rows: against the unit matrix the sums are the values themselves."""
    n = 64
    x = values.reshape(-1, n).cuda()
    eye = torch.eye(n)
    plan = g.ops.LinearPlan(eye.to(w_kind).cuda(), w_scale=torch.ones(n, device="cuda") if w_kind == torch.int8 else None)
    return plan.run(x, activation=act, dtype=FLOAT, r=r).cpu().reshape(-1)


@pytest.mark.parametrize("kind,w_kind", TYPES)
@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_float32_results_of_activations(g, kind, w_kind, few, act):
    """Results of 32 bits, whatever the rows are: relative bounds, for every value from -11 to 11 (float16 ones: all there are; SiLU: from -80).

    In units of 2^-24 of the result.  GELU, v erfc(-v / sqrt(2)) / 2: the argument is off by 1.5 units, which changes erfc by (v^2 + 1) times as much, erfc by 8, two
    products by 2.  By tanh, v / (1 + exp(-2 u)): u of four roundings and three constants is off by 6 units, which changes the quotient by 2 |u| times as
    much, exp by 4, a sum and a quotient by 3.  SiLU: exp 4, sum, quotient and its rounding 3.  Where exp(-2 u) is above 2^128 the quotient may be 0: it is |v| 2^-128 there, or less."""
    v = torch.arange(0, 1 << 15, dtype=torch.int32).to(torch.int16).view(HALF)
    v = v[(v <= (80 if act == "silu" else 11)) & (v >= 2.0 ** -10)]
    v = torch.cat([-v, v[v <= 11]])
    v = v[: len(v) // 64 * 64 if not few else 64 * 30]
    if few:
        v = torch.cat([v, torch.linspace(-11, 11, 64 * 2).half()])
    y = activated(g, w_kind, v.to(kind), act).double()
    x = v.double()
    want = ACTS[act](x)
    u = math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
    units = {"gelu": 1.5 * (x ** 2 + 1) + 10, "gelu_tanh": 12 * u.abs() + 7, "silu": 7.0 + 0 * x}[act]
    assert ((y - want).abs() <= units * 2.0 ** -24 * want.abs() + x.abs() * 2.0 ** -127).all()


@pytest.mark.parametrize("kind,w_kind", TYPES)
@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("act", sorted(ACTS))
def test_activations_of_infinite_sums(g, kind, w_kind, rows, act):
    """An infinite sum gives the activation's limit, in every type and in both kernels: itself, and 0 (without an activation itself) on the lower side; a NaN stays one."""
    n = 64
    x = torch.zeros(rows, n, dtype=kind)
    x[:, 0], x[1:, 0] = math.inf, -math.inf
    w = torch.zeros(n, n)
    w[:, 0] = 1
    b = torch.zeros(n, dtype=FLOAT)
    b[7] = math.nan
    plan = g.ops.LinearPlan(w.to(w_kind).cuda(), b=b.cuda(), w_scale=torch.ones(n, device="cuda") if w_kind == torch.int8 else None)
    for dtype in {kind, FLOAT}:
        y = plan.run(x.cuda(), activation=act, dtype=dtype).cpu()
        assert bool(torch.isnan(y[:, 7]).all())
        y[:, 7] = y[:, 6]
        assert bool((y[0] == math.inf).all()) and bool((y[1:] == (0 if act else -math.inf)).all()), y[:2, :2]


@pytest.mark.parametrize("kind", [HALF, FLOAT])
@pytest.mark.parametrize("m", [5, 200])
def test_layouts(g, kind, m):
    """Rows of a larger array at any alignment, columns apart, several leading axes, weights [K, N], a result of any strides; what lies
    around the operands is not used, what lies around the result not written."""
    k, n = 192, 136
    w, b = normal(9, (n, k), kind, k ** -0.5), normal(10, (n,), kind)
    want = None
    for col, gap, first in [(1, 0, 0), (1, 8, 8), (1, 3, 1), (2, 5, 1)]:
        space = torch.full((m + 2, first + k * col + gap), math.nan, dtype=kind, device="cuda")
        x = space[1: m + 1, first: first + k * col: col]
        x.copy_(normal(11, (m, k), kind))
        if want is None:
            want = formula(x, w, None, b, "gelu", x[:, :n])
        for plan_w in (w, w.T.contiguous().T):
            plan = g.ops.LinearPlan(plan_w, b=b)
            check(plan.run(x, activation="gelu", r=x[:, :n]), *want, k)
            for ycol, ygap in [(1, 0), (1, 8), (1, 3), (3, 1)]:
                out = torch.full((m + 2, n * ycol + ygap + 2), 7.0, dtype=kind, device="cuda")
                y = out[1: m + 1, 2: 2 + n * ycol: ycol]
                assert plan.run(x, activation="gelu", r=x[:, :n], out=y) is y
                check(y, *want, k)
                y.fill_(7.0)
                assert bool((out == 7.0).all())
    plan = g.ops.LinearPlan(w, b=b)
    check(plan.run(x[0]).reshape(1, n), *formula(x[:1], w, None, b, "", None), k)               # one axis
    check(plan.run(x[:1].expand(m, k)), *formula(x[:1].expand(m, k), w, None, b, "", None), k)   # one row again and again
    x3 = normal(12, (3, 4, k), kind)
    y3 = g.ops.LinearPlan(w).run(x3)
    assert y3.shape == (3, 4, n)
    check(y3.reshape(12, n), *formula(x3.reshape(12, k), w, None, None, "", None), k)


@pytest.mark.parametrize("kind,w_kind", TYPES)
@pytest.mark.parametrize("m", [3, 150])
def test_rows_stay_apart(g, kind, w_kind, m):
    """A NaN or an infinity in one row shows in that row alone, and K that is not whole steps takes nothing from the next row."""
    k, n = 77, 50
    x, (w, scale) = normal(13, (m, k), kind), weights(14, (n, k), w_kind)
    plan = g.ops.LinearPlan(w, w_scale=scale)
    clean = plan.run(x)
    x[1, :] = math.nan
    x[0, 3] = math.inf
    y = plan.run(x)
    assert bool(torch.isnan(y[1]).all()) and not bool(torch.isfinite(y[0][w[:, 3] != 0]).any())
    assert torch.equal(y[2:], clean[2:])


def test_residual_in_place_and_no_rows(g):
    x, w, r = normal(15, (90, 64), HALF), normal(16, (80, 64), HALF), normal(17, (90, 80), HALF)
    plan = g.ops.LinearPlan(w)
    want = plan.run(x, r=r)
    assert plan.run(x, r=r, out=r) is r and torch.equal(r, want)
    assert plan.run(x[:0]).shape == (0, 80)


@pytest.mark.parametrize("kind", [HALF, FLOAT])
def test_recorded_and_on_two_streams(g, kind):
    """One plan in a graph, in eager calls between its replays, and on two streams at once."""
    k, n = 512, 256
    w, (big, small) = normal(18, (n, k), kind, k ** -0.5), (normal(19, (700, k), kind), normal(20, (2, k), kind))
    plan = g.ops.LinearPlan(w)
    torch.cuda.synchronize()
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=first):
        ys = plan.run(big, activation="silu"), plan.run(small, activation="silu")
    for i in range(3):
        big.copy_(normal(30 + i, big.shape, kind))
        small.copy_(normal(40 + i, small.shape, kind))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ys[0], plan.run(big, activation="silu")) and torch.equal(ys[1], plan.run(small, activation="silu"))
    want = plan.run(big), plan.run(small)
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        got = [plan.run(big) for _ in range(5)]
    with torch.cuda.stream(second):
        also = [plan.run(small) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[0]) for y in got) and all(torch.equal(y, want[1]) for y in also)


def test_a_plan_is_not_created_inside_a_recording(g):
    w, x = normal(35, (64, 64), HALF), normal(36, (4, 64), HALF)
    plan = g.ops.LinearPlan(w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(g.capi.ChxHipError) as e:
            g.ops.LinearPlan(w)
        y = plan.run(x)
    assert e.value.code == g.capi.EUNSUPPORTED
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, plan.run(x))


def test_tensors_that_are_not_on_the_device(g):
    w, x = normal(37, (64, 64), HALF), normal(38, (4, 64), HALF)
    plan = g.ops.LinearPlan(w)
    for call in (lambda: g.ops.LinearPlan(w.cpu()), lambda: plan.run(x.cpu()), lambda: plan.run(x, r=x.cpu()), lambda: plan.run(x, out=x.cpu())):
        with pytest.raises(ValueError):
            call()
    plan.close()
    with pytest.raises(ValueError):
        plan.run(x)


# ---- experts -------------------------------------------------------------------------------------------

def routed(seed, places, experts, empty=()):
    gen = torch.Generator().manual_seed(seed)
    free = torch.tensor([e for e in range(experts) if e not in empty])
    chosen = free[(torch.rand(places, generator=gen) ** 2 * len(free)).long()]
    order = torch.sort(chosen, stable=True).indices
    offsets = torch.zeros(experts + 1, dtype=torch.int64)
    offsets[1:] = torch.bincount(chosen, minlength=experts).cumsum(0)
    return chosen, order.int().cuda(), offsets.int().cuda()


@pytest.mark.parametrize("kind,w_kind", TYPES)
@pytest.mark.parametrize("places,experts,fan,k,n", [
    (1, 1, 1, 64, 64), (8, 70, 2, 130, 48), (96, 130, 8, 64, 200),                 # a row or none to an expert, more than 64 experts
    (640, 3, 2, 100, 130), (3000, 20, 1, 64, 96), (9000, 3, 3, 128, 1100),         # tiles of 128 and of 256 rows
    (600, 18, 2, 200, 150), (700, 9, 1, 96, 90),                                   # tiles of 64 rows
    (1100, 4, 1, 96, 300), (600, 5, 1, 130, 140),                                  # an expert's rows over two tiles that they do not fill
])
def test_experts(g, kind, w_kind, places, experts, fan, k, n):
    chosen, order, offsets = routed(21, places, experts, empty=(0,) if experts > 1 else ())
    x, (w, scale) = normal(22, (places // fan, k), kind), weights(23, (experts, n, k), w_kind)
    b = normal(24, (experts, n), kind)
    y = g.ops.LinearPlan(w, b=b, w_scale=scale).run_experts(x, order, offsets, activation="silu")
    assert y.shape == (places, n)
    for e in range(experts):
        p = (chosen == e).nonzero()[:, 0].cuda()
        if len(p):
            check(y[p], *formula(x[p // fan], w[e], None if scale is None else scale[e], b[e], "silu", None), k)


@pytest.mark.parametrize("places", [40, 2000])
def test_places_that_are_not_named(g, places):
    """Rows that no place names stay as they are, also where order and offsets hold numbers outside their range."""
    experts, k, n = 5, 64, 32
    chosen, order, offsets = routed(25, places, experts)
    x, w = normal(26, (places, k), HALF), normal(27, (experts, n, k), HALF, 0.125)
    plan = g.ops.LinearPlan(w)
    want = plan.run_experts(x, order, offsets)
    torch.cuda.synchronize()
    cut = offsets.clone()
    cut[2:] = cut[1]                                              # the first two experts' alone
    broken_order = order.clone()
    broken_order[0], broken_order[3] = -1, places
    ends = offsets.clone()
    ends[0], ends[-1] = -5, places + 1000                         # taken as the ends of the order
    backwards = offsets.flip(0).contiguous()                      # no expert has a place
    for o, f, left_out in [(order, cut, chosen > 0), (broken_order, offsets, None), (order, ends, chosen < 0), (order, backwards, chosen >= 0)]:
        out = torch.full((places, n), 7.0, dtype=HALF, device="cuda")
        y = plan.run_experts(x, o, f, out=out)
        if left_out is None:
            left_out = torch.zeros(places, dtype=torch.bool)
            left_out[order[[0, 3]].cpu().long()] = True
        left_out = left_out.cuda()
        assert bool((y[left_out] == 7.0).all()) and torch.equal(y[~left_out], want[~left_out])


def test_a_feed_forward_layer_with_experts_and_its_answer(g):
    """Scores, routing, both products, their weighted sum with the residual, the head's product and the log probabilities: as one
    run, and recorded."""
    T, D, H, E, top, V = 50, 192, 320, 12, 3, 777
    x, gate = normal(28, (T, D), HALF), normal(29, (E, D), HALF, D ** -0.5)
    up, down, head = normal(30, (E, H, D), HALF, D ** -0.5), normal(31, (E, D, H), HALF, H ** -0.5), normal(32, (V, D), HALF, 2 * D ** -0.5)
    b = normal(33, (E, H), HALF, 0.3)
    bias = normal(34, (E,), FLOAT, 0.05)
    tokens = torch.arange(T).cuda() * 13
    plans = [g.ops.LinearPlan(gate), g.ops.LinearPlan(up, b=b), g.ops.LinearPlan(down), g.ops.LinearPlan(head)]

    def layer():
        scores = plans[0].run(x, dtype=FLOAT)
        experts, share, order, offsets = g.ops.ExpertRouting(scores, top, bias=bias, score="sigmoid", scale=1.25)
        h = plans[1].run_experts(x, order, offsets, activation="gelu")
        y = g.ops.ExpertCombine(plans[2].run_experts(h, order, offsets), share, r=x)
        logits = plans[3].run(y, dtype=FLOAT)
        return (scores, experts, share, h, y, logits) + g.ops.TokenLogProbs(logits, tokens, top=4)

    got = layer()
    scores, experts, share, h, y, logits, logp, entropy, best_logp, best = got
    check(scores, *formula(x, gate, None, None, "", None), D)
    p = torch.sigmoid(scores.double())
    assert torch.equal(experts.long(), (p + bias.double()).topk(top, dim=1).indices)
    w = p.gather(1, experts.long())
    assert ((share.double() - 1.25 * w / w.sum(1, keepdim=True)).abs() <= 2.0 ** -20).all()
    flat = experts.reshape(-1).long()
    for e in range(E):
        at = (flat == e).nonzero()[:, 0]
        if len(at):
            check(h[at], *formula(x[at // top], up[e], None, b[e], "gelu", None), D)
    # the second product and the sum from what the first gave: two roundings to float16, of the terms and of the sum
    terms = torch.stack([h[i].double() @ down[flat[i]].double().T for i in range(T * top)]).reshape(T, top, D)
    want = (terms * share.double()[:, :, None]).sum(1) + x.double()
    room = 2.0 ** -11 * want.abs() + ((2.0 ** -11 + 2.0 ** -14) * terms.abs() * share.double()[:, :, None]).sum(1) + 1e-4
    assert ((y.double() - want).abs() <= room).all()
    check(logits, *formula(y, head, None, None, "", None), D)
    ref = torch.log_softmax(logits.double(), 1)
    # (float32 differences and exponentials of numbers up to 16, sums of 777 of them)
    assert ((logp.double() - ref.gather(1, tokens[:, None])[:, 0]).abs() <= 1e-5).all()
    assert ((entropy.double() - torch.special.entr(ref.exp()).sum(1)).abs() <= 1e-5).all()
    assert torch.equal(best, logits.topk(4, dim=1).indices) and ((best_logp.double() - ref.gather(1, best)).abs() <= 1e-5).all()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = layer()
    for i in range(3):
        x.copy_(normal(50 + i, x.shape, HALF))
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(recorded, layer()):
            assert torch.equal(a, c)


def test_more_work_than_one_launch_has(g):
    """More than 2^31 threads' work in the launches that lay weights out and bring rows into whole pieces: what lies behind the first launch's part."""
    experts, n, k = 70, 16384, 16384
    w = normal(60, (n, k), HALF, k ** -0.5)
    x = normal(61, (2, k), HALF)
    plan = g.ops.LinearPlan(w.expand(experts, n, k))                                  # 38 GB laid out
    order = torch.arange(experts, dtype=torch.int32, device="cuda")
    offsets = torch.arange(experts + 1, dtype=torch.int32, device="cuda")
    y = plan.run_experts(x[:1].expand(experts, k).contiguous(), order, offsets)
    plan.close()
    assert torch.equal(y, y[:1].expand(experts, n))
    check(y[-1:], *formula(x[:1], w, None, None, "", None), k)
    n, k, rows = 64, 16385, (1 << 20) + 5                                              # 34 GB of pieces
    x, plan = normal(62, (1, k), HALF), g.ops.LinearPlan(normal(63, (n, k), HALF, k ** -0.5))
    y = plan.run(x.expand(rows, k))
    few = plan.run(x.expand(300, k))
    check(few[:1], *formula(x, normal(63, (n, k), HALF, k ** -0.5), None, None, "", None), k)
    assert torch.equal(y[:300], y[-300:]) and torch.equal(y[:1].expand(rows, n), y) and torch.allclose(y[:1].float(), few[:1].float(), atol=2e-2)
    del w, x, y
    torch.cuda.empty_cache()


def whole(seed, shape, dtype):
    """Whole numbers: their products' sums are exact in float32, in any order."""
    return torch.randint(-3, 4, shape, generator=torch.Generator().manual_seed(seed), dtype=torch.int8).to(dtype).cuda()


KINDS = {linear_sizes.HALF: (HALF, HALF), linear_sizes.INT8: (HALF, torch.int8), linear_sizes.FLOAT: (FLOAT, FLOAT)}


@pytest.mark.parametrize("which,kernel,m,blocks,n", linear_sizes.PLAIN)
def test_long_products(g, which, kernel, m, blocks, n):
    """Every kernel over enough of k that its rings and loops come round, number for number."""
    kind, w_kind = KINDS[which]
    k = blocks * linear_sizes.BLOCK[which]
    x, w = whole(40, (m, k), kind), whole(41, (n, k), w_kind)
    scale = torch.full((n,), 0.5, device="cuda") if w_kind == torch.int8 else None
    y = g.ops.LinearPlan(w, w_scale=scale).run(x, dtype=FLOAT)
    want = x.double() @ w.double().T
    assert torch.equal(y.double(), want if scale is None else 0.5 * want)


@pytest.mark.parametrize("which,kernel,experts,fan,m,blocks,n", linear_sizes.EXPERTS)
def test_long_products_of_experts(g, which, kernel, experts, fan, m, blocks, n):
    """Likewise, with experts of few and of many rows, so that tiles lack none, some or nearly all of theirs."""
    kind, w_kind = KINDS[which]
    k = blocks * linear_sizes.BLOCK[which]
    chosen, order, offsets = routed(42, m, experts)
    x, w = whole(43, (m // fan, k), kind), whole(44, (experts, n, k), w_kind)
    scale = torch.full((experts, n), 0.5, device="cuda") if w_kind == torch.int8 else None
    y = g.ops.LinearPlan(w, w_scale=scale).run_experts(x, order, offsets, dtype=FLOAT)
    for e in range(experts):
        p = (chosen == e).nonzero()[:, 0].cuda()
        want = x[p // fan].double() @ w[e].double().T
        assert torch.equal(y[p].double(), want if scale is None else 0.5 * want)


@pytest.mark.parametrize("k", [2 ** 22 + 64, 2 ** 22 + 3])
def test_rows_too_long_for_a_tile(g, k):
    """Rows of 8 MB and more (weights of 8 bits alone have as many columns) are left to the kernel for few rows, whatever their number."""
    rows, n = 20000, 64
    x, w, scale = whole(45, (1, k), HALF), whole(46, (n, k), torch.int8), torch.full((n,), 0.5, device="cuda")
    y = g.ops.LinearPlan(w, w_scale=scale).run(x.expand(rows, k), dtype=FLOAT)
    assert torch.equal(y.double(), 0.5 * (x.double() @ w.double().T).expand(rows, n))


@pytest.mark.parametrize("fan", [1, 2])
def test_experts_rows_over_more_than_4_GiB(g, fan):
    """Rows that 32 bits of an address do not reach: gathered from x of 4.3 GB, in a mixed order."""
    k, n, experts = 16448, 48, 3
    places = (2 ** 17 + 10) * fan
    x = torch.randint(-2, 3, (places // fan, k), generator=torch.Generator(device="cuda").manual_seed(47), dtype=torch.int8, device="cuda").half()
    assert x.numel() * 2 > 2 ** 32
    w = whole(48, (experts, n, k), HALF)
    chosen, order, offsets = routed(49, places, experts)
    y = g.ops.LinearPlan(w).run_experts(x, order, offsets, dtype=FLOAT)
    for e in range(experts):
        for p in (chosen == e).nonzero()[:, 0].cuda().split(1 << 14):
            assert torch.equal(y[p], x[p // fan].float() @ w[e].float().T)
    del x, y
    torch.cuda.empty_cache()
