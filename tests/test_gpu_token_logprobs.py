"""Log probabilities, entropy and alternatives (csrc/token_logprobs.hip) against their definitions in 64 bits.

Bounds: a difference x - m is rounded by 2^-24 of itself, so exp of it is off by 2^-24 |x - m| and two roundings; a term of the sums weighs p.  The
sums themselves add at most V numbers, a lane's 32 at a time: no more than 2^-24 (V / 256 + 64) of the sum.  With differences D = m - min x of what counts (p above
2^-24, so D < 17 + log V), a log probability is off by at most 2^-24 (2 |log p| + D + V / 256 + 64), and the entropy, a mean of log p,
by as much with |log p| < D."""
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


def check(g, logits, tokens, top):
    got = g.ops.TokenLogProbs(logits, tokens, top=top)
    x = logits.double().cpu()
    V = x.shape[-1]
    ref = torch.log_softmax(x, -1)
    none = (x == -math.inf).all(-1, keepdim=True)
    ref = torch.where(none, -math.inf, ref)
    best = x.sort(dim=-1, descending=True, stable=True).indices[..., :top]  # (NaN first, as they are asked for)
    want_top = ref.gather(-1, best)
    want_h = torch.where(none[..., 0], 0.0, torch.where(torch.isnan(ref).any(-1), math.nan, torch.special.entr(ref.exp()).sum(-1)))
    assert got[3].dtype == torch.int64 and torch.equal(got[3].cpu(), best)
    wanted = [(got[1], want_h), (got[2], want_top)]
    if tokens is None:
        assert got[0] is None
    else:
        t = tokens.long().cpu()
        want = torch.where(t < 0, 0.0, ref.gather(-1, t.clamp(0, V - 1)[..., None])[..., 0])
        wanted.append((got[0], torch.where(t >= V, math.nan, want)))
    for y, want in wanted:
        y = y.double().cpu()
        assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y == -math.inf, want == -math.inf)
        fine = torch.isfinite(want)
        room = 2.0 ** -24 * (3 * want[fine].abs() + 2 * (17 + math.log(V)) + V / 256 + 64)
        assert ((y[fine] - want[fine]).abs() <= room).all()
    return got


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("R,V,top", [(1, 1, 1), (1, 2, 0), (4, 7, 7), (3, 64, 64), (2, 65, 5), (5, 1000, 20), (300, 2048, 3), (2, 8192, 1), (7, 8193, 64),
                                     (1, 100003, 40), (1200, 9000, 6), (3, 300001, 12)])
def test_sizes(g, dtype, R, V, top):
    """One part and several, whole steps and a token over; float16 rows with many equal logits."""
    logits = normal(1, (R, V), dtype, 2.5)
    tokens = (torch.arange(R) * 7919 % V).cuda()
    tokens[R // 2] = V - 1
    check(g, logits, tokens, top)


@pytest.mark.parametrize("V", [50, 9000, 40000])
def test_equal_logits_take_the_lower_index(g, V):
    logits = torch.zeros(6, V, dtype=HALF, device="cuda")
    logits[1, V // 2:] = 1.0
    logits[2, V - 3:] = 1.0
    logits[3, ::2] = -0.0
    logits[4] = (torch.arange(V) // 16).half() / 64          # ascending, in runs: every block has better ones
    logits[5] = -(torch.arange(V) // 16).half() / 64
    check(g, logits, torch.arange(6).cuda(), 40)


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("V", [33, 20000])
def test_masked_rows(g, dtype, V):
    """Rows without a token, with one, with fewer than alternatives are asked for, with the type's lowest value, infinities and NaN."""
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    logits = normal(2, (12, V), dtype, 2.0)
    logits[0] = -math.inf
    logits[1] = -math.inf
    logits[1, V - 1] = 3.0
    logits[2, 4: V - 4] = -math.inf
    logits[3] = low
    logits[4, 1:] = low
    logits[5, V // 2] = math.inf
    logits[6, V // 3] = math.nan
    logits[7] = math.nan
    logits[8] = -math.inf
    logits[8, 7] = low
    logits[9, 3] = high
    logits[10] = high
    tokens = torch.tensor([0, V - 1, 8, 3, 0, 1, 2, 3, 7, 3, 5, -100]).cuda()
    for top in (0, 1, 20):
        check(g, logits, tokens, top)


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("R,V", [(2000, 1), (40, 60), (2100, 5000), (7, 9000), (6, 100003), (600, 9000)])
def test_a_token_that_is_certain(g, dtype, R, V):
    """The only token of a row has log probability 0 and the row entropy 0, whatever its logit is: no rounding is left of it.  Nor are log probabilities above 0 and entropies below."""
    logits = torch.full((R, V), -math.inf, dtype=dtype, device="cuda")
    tokens = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(9)).cuda()
    values = normal(10, (R,), dtype, 6.0)
    values[: R // 2] *= 4.0 ** torch.arange(R // 2, device="cuda").remainder(9).sub(2).to(dtype)
    values = values.clamp(-60000, 60000)
    logits[torch.arange(R, device="cuda"), tokens] = values
    logp, entropy, best, which = g.ops.TokenLogProbs(logits, tokens, top=1)
    assert torch.equal(which[:, 0], tokens)
    assert bool((logp == 0).all()) and bool((entropy == 0).all()) and bool((best == 0).all())
    if V > 1:
        other = (tokens + 1 + torch.arange(R, device="cuda") % (V - 1)) % V
        logits[torch.arange(R, device="cuda"), other] = values - (torch.arange(R, device="cuda") % 24).to(dtype)  # from as likely down to 4e-11
        logp, entropy, best, _ = check(g, logits, tokens, 2)
        assert bool((logp <= 0).all()) and bool((best <= 0).all()) and bool((entropy >= 0).all())


def test_tokens_outside_the_vocabulary(g):
    logits = normal(3, (6, 500), HALF)
    for dtype in (torch.int32, torch.int64):
        got = check(g, logits, torch.tensor([-1, 0, 499, 500, -2 ** 31, 2 ** 31 - 1], dtype=dtype).cuda(), 2)
        assert got[0].cpu()[0] == 0 and bool(torch.isnan(got[0][3]))


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("V", [70, 17000])
def test_strides(g, dtype, V):
    """Rows of a larger array at any alignment, columns apart, several leading axes, every other token."""
    plain, tokens = normal(4, (6, V), dtype, 2.0), torch.arange(12).cuda()[::2]
    want = check(g, plain, tokens, 9)
    for first, gap, col in [(0, 8, 1), (1, 2, 1), (3, 0, 2)]:
        space = torch.full((6, first + V * col + gap), math.nan, dtype=dtype, device="cuda")
        x = space[:, first: first + V * col: col]
        x.copy_(plain)
        for a, b in zip(g.ops.TokenLogProbs(x, tokens, top=9), want):
            assert torch.equal(a, b)
    got = g.ops.TokenLogProbs(plain.reshape(2, 3, V), None, top=9)
    assert got[0] is None and got[1].shape == (2, 3) and got[2].shape == got[3].shape == (2, 3, 9)
    assert torch.equal(got[3].reshape(6, 9), want[3])
    assert g.ops.TokenLogProbs(plain[:0], tokens[:0], top=2)[2].shape == (0, 2)


def test_tokens_and_logits_of_a_shifted_text(g):
    """What a text's scores are asked with: the tokens one place further, which is a slice of several axes; logits whose leading axes are not one run of rows are refused."""
    B, T, V = 3, 5, 900
    logits, text = normal(7, (B, T, V), HALF, 2.0), torch.randint(0, V, (B, T + 1), generator=torch.Generator().manual_seed(8)).cuda()
    got, want = g.ops.TokenLogProbs(logits, text[:, 1:], top=3), g.ops.TokenLogProbs(logits, text[:, 1:].contiguous(), top=3)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    check(g, logits, text[:, 1:], 3)
    check(g, logits[:, ::1, 5:], text[:, :T] % 800, 3)
    with pytest.raises(ValueError, match="one run of rows"):
        g.ops.TokenLogProbs(logits[:, :-1], text[:, 1:T])


def test_recorded_and_on_two_streams(g):
    """Calls that split rows, recorded side by side, replayed with eager calls in between; and on two streams at once."""
    logits = normal(5, (3, 30000), HALF, 2.0), normal(6, (2, 50000), HALF, 2.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = [g.ops.TokenLogProbs(x, None, top=5) for x in logits]
    for i in range(3):
        for j, x in enumerate(logits):
            x.copy_(normal(20 + 2 * i + j, x.shape, HALF, 2.0))
        graph.replay()
        torch.cuda.synchronize()
        for x, got in zip(logits, recorded):
            for a, b in zip(got[1:], g.ops.TokenLogProbs(x, None, top=5)[1:]):
                assert torch.equal(a, b)
    want = [g.ops.TokenLogProbs(x, None, top=5) for x in logits]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for s, x, to in zip(streams, logits, got):
            with torch.cuda.stream(s):
                to.append(g.ops.TokenLogProbs(x, None, top=5))
    torch.cuda.synchronize()
    for each, w in zip(got, want):
        for one in each:
            assert all(torch.equal(a, b) for a, b in zip(one[1:], w[1:]))
