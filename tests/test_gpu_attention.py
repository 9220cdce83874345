"""Attention over a cache and over an encoder's states (csrc/attention_kernel.h) against its formula in 64 bits.

Bounds.  A score s = scale sum q k is a sum of D products in float32: off by at most 2^-23 (D + 8) scale sum |q k|, which is E at most over the places that a row sees; its exponential by that and
2^-22 of itself (rounding of the exponent, the exponential's own).  A result sum w v / sum w is off by at most
  A (2 E' + W + S) + the result's rounding,   A = sum w |v| / sum w,  E' = E + 2^-22,
W the rounding of a weight that is multiplied (float16: 2^-11, and 2^-31 of the largest below the normal numbers), S that of the sums of L places, 2^-24 (L + 64).  A place's
mass, a sum of weights over rows, is off by 2 E' + S of itself and by the sum's own roundings, 2^-24 of it for each row."""
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


def numbers(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def attend(q, k, v, seen, scale):
    """q [T, H, D], k and v [L, G, D], seen [T, L] on the CPU, in 64 bits: (y, room for its error, weights [G, L] and room for theirs)."""
    T, H, D = q.shape
    L, G = k.shape[:2]
    half = q.dtype == HALF
    q, k, v = q.double(), k.double(), v.double()
    y, room = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    mass, mass_room = torch.zeros(G, L, dtype=torch.float64), torch.zeros(G, L, dtype=torch.float64)
    if L == 0:
        return y, room, mass, mass_room
    for h in range(H):
        group = h // (H // G)
        s = (scale * (q[:, h] @ k[:, group].T)).masked_fill(~seen, -math.inf)
        size = (scale * (q[:, h].abs() @ k[:, group].abs().T)).masked_fill(~seen, 0).amax(1, keepdim=True)
        off = 2.0 ** -23 * (D + 8) * size + 2.0 ** -22
        some = (s > -math.inf).any(1, keepdim=True)
        w = torch.where(some, torch.softmax(s.masked_fill(~some, 0.0), 1), 0.0)
        kept = (w > 0).double()
        values = torch.where(kept.amax(0)[:, None] > 0, v[:, group], 0.0)  # (what nobody sees adds nothing)
        y[:, h] = w @ values
        largest = w.amax(1, keepdim=True)
        room[:, h] = (w @ values.abs()) * (2 * off + (2.0 ** -11 if half else 2.0 ** -23) + 2.0 ** -24 * (L + 64)) + y[:, h].abs() * (2.0 ** -11 if half else 2.0 ** -23)
        if half:
            room[:, h] += largest * (kept @ values.abs()) * 2.0 ** -31 + 2.0 ** -25
        mass[group] += w.sum(0)
        mass_room[group] += (w * (2 * off + 2.0 ** -24 * (L + 64 + T * H // G))).sum(0) + 2.0 ** -126 * T
    return y, room, mass, mass_room


def close(got, want, room, slack=1.0):
    assert torch.isfinite(got.cpu()).all()
    off = (got.double().cpu() - want).abs() - slack * room
    assert (off <= 0).all(), (off.max().item(), (off > 0).sum().item(), off.numel())


class Cache:
    """Pages in an order of their own, everything that no sequence holds a NaN."""

    def __init__(self, seed, dtype, B, G, D, R, lengths, tokens, layout="prgd", gap=0):
        self.B, self.G, self.D, self.R, self.tokens = B, G, D, R, tokens
        M = max(1, -(-(max(lengths) + tokens) // R))
        P = B * M + 2
        order = {"prgd": (0, 1, 2), "pgrd": (0, 2, 1), "gprd": (2, 0, 1)}[layout]
        extents = (P, R, G)
        back = [order.index(i) for i in range(3)]

        def pool():
            space = torch.full([extents[i] for i in order] + [D + gap], math.nan, dtype=dtype, device="cuda")
            return space[..., :D].permute(*back, 3)

        self.keys, self.values = pool(), pool()
        self.tables = torch.randperm(P, generator=torch.Generator().manual_seed(seed))[: B * M].reshape(B, M).to(torch.int32).cuda()
        self.lengths = numbers(lengths)
        self.rows = []
        for b, n in enumerate(lengths):
            k, v = normal(seed + 10 + b, (n + tokens, G, D), dtype), normal(seed + 50 + b, (n + tokens, G, D), dtype)
            for p in range(n + tokens):
                page = int(self.tables[b, p // R])
                self.keys[page, p % R], self.values[page, p % R] = k[p], v[p]
            self.rows.append((k.cpu(), v.cpu()))


def fill(cache):
    """What the pages hold, read back: [(keys, values)] of the sequences."""
    got = []
    for b in range(cache.B):
        t = cache.tables[b].long()
        got.append([x[t].reshape(-1, cache.G, cache.D).cpu() for x in (cache.keys, cache.values)])
    return got


def line_of(parents, T):
    sees = torch.zeros(T, T, dtype=torch.bool)
    for t in range(T):
        if parents is None:
            sees[t, : t + 1] = True
        else:
            if 0 <= parents[t] < t:
                sees[t] = sees[parents[t]]
            sees[t, t] = True
    return sees


def tree_of(seed, B, T):
    gen = torch.Generator().manual_seed(seed)
    back = torch.randint(1, 6, (B, T), generator=gen)
    return (torch.arange(T) - back).clamp(min=-1).to(torch.int32).cuda()


def check_tree(g, cache, q, parents=None, counts=None, scale=None, mass=None, out=None):
    B, T, H, D = q.shape
    before = None if mass is None else mass.double().cpu().clone()
    got = g.ops.TreeAttention(q, cache.keys, cache.values, cache.tables, cache.lengths, parents=parents, counts=counts, scale=scale, mass=mass, out=out)
    scale = 1 / math.sqrt(D) if scale is None else scale
    for b, (k, v) in enumerate(cache.rows):
        count = T if counts is None else min(max(int(counts[b]), 0), T)
        n = len(k) - cache.tokens
        sees = torch.cat([torch.ones(T, n, dtype=torch.bool), line_of(None if parents is None else parents[b].tolist(), T)], 1)
        sees[count:] = False
        want, room, weights, weights_room = attend(q[b].cpu(), k[: n + T], v[: n + T], sees, scale)
        close(got[b], want, room)
        assert (got[b, count:] == 0).all()
        if mass is not None:
            base = before[b].clone()
            base[:, n: n + count] = 0
            L = n + count
            base[:, :L] += weights[:, :L]
            room = 2.0 ** -24 * base.abs() + 1e-30
            room[:, :L] += weights_room[:, :L]
            close(mass[b], base, room)
    return got


# one token, few, many; heads that share and that do not; sizes that fill a kernel's and that do not; pages of one place, of some that are no power of two, of more than a sequence has
SIZES = [
    (1, 1, 1, 64, 16, 1, [0]), (1, 4, 1, 64, 16, 1, [63]), (3, 8, 2, 128, 16, 1, [1, 64, 700]), (2, 4, 4, 32, 1, 3, [5, 130]), (2, 6, 2, 96, 20, 5, [77, 300]),
    (2, 14, 2, 80, 64, 19, [0, 200]), (1, 5, 5, 75, 7, 33, [31]), (2, 2, 1, 1, 5, 4, [9, 70]), (1, 8, 1, 256, 16, 9, [150]), (1, 3, 1, 129, 256, 70, [128]),
    (1, 2, 2, 192, 64, 130, [191]), (2, 16, 2, 128, 32, 24, [900, 1030]), (1, 4, 2, 64, 8, 256, [64]),
]


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("B,H,G,D,R,T,lengths", SIZES)
def test_sizes(g, dtype, tree, B, H, G, D, R, T, lengths):
    cache = Cache(1, dtype, B, G, D, R, lengths, T)
    mass = torch.rand((B, G, cache.tables.shape[1] * R), generator=torch.Generator().manual_seed(3)).cuda()
    check_tree(g, cache, normal(2, (B, T, H, D), dtype, 2.0), tree_of(4, B, T) if tree else None, mass=mass)


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("H,G,D,T,length", [(8, 1, 128, 1, 9000), (2, 1, 64, 3, 20011), (2, 2, 256, 1, 5000), (4, 1, 96, 40, 6001), (4, 1, 64, 80, 8300), (2, 2, 256, 90, 700)])
def test_long_caches_in_parts(g, dtype, H, G, D, T, length):
    cache = Cache(5, dtype, 2, G, D, 64, [length, length // 9], T)
    check_tree(g, cache, normal(6, (2, T, H, D), dtype, 2.0), tree_of(7, 2, T), mass=torch.zeros(2, G, cache.tables.shape[1] * 64, device="cuda"))


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
def test_a_prompt_in_pieces(g, dtype):
    """Chains of more rows than a work-group has, from nothing and over what is there."""
    for length, T in ((0, 300), (77, 515)):
        check_tree(g, Cache(8, dtype, 1, 2, 64, 16, [length], T), normal(9, (1, T, 6, 64), dtype, 2.0))


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
def test_counts(g, dtype):
    """Sequences with fewer tokens than the batch, down to none of either: rows without a token are 0."""
    cache = Cache(11, dtype, 5, 2, 64, 16, [40, 0, 0, 129, 3], 9)
    q = normal(12, (5, 9, 4, 64), dtype, 2.0)
    mass = torch.zeros(5, 2, cache.tables.shape[1] * 16, device="cuda")
    check_tree(g, cache, q, tree_of(13, 5, 9), numbers([9, 4, 0, -3, 100]), mass=mass)
    check_tree(g, cache, q, None, numbers([0, 9, 0, 2, 1]), mass=mass, out=torch.full_like(q, math.nan))


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("layout,gap", [("prgd", 0), ("pgrd", 0), ("gprd", 8), ("prgd", 3)])
def test_strides(g, dtype, layout, gap):
    cache = Cache(14, dtype, 2, 2, 64, 16, [50, 333], 6, layout, gap)
    wide = normal(15, (2, 8, 6, 64 + gap), dtype, 2.0)
    q = wide[:, 1:7, 1:5, :64]
    space = torch.full((4, 2, 6, 67), math.nan, dtype=dtype, device="cuda")
    out = space.permute(1, 2, 0, 3)[..., 3:] if gap == 3 else space[..., :64].permute(1, 2, 0, 3)
    parents = tree_of(16, 2, 6)
    cache.tables = torch.cat([cache.tables, torch.full_like(cache.tables, 7)], 1)[:, : cache.tables.shape[1]]
    got = check_tree(g, cache, q, parents, out=out)
    assert got is out
    outside = torch.ones_like(space, dtype=torch.bool)
    (outside.permute(1, 2, 0, 3)[..., 3:] if gap == 3 else outside[..., :64].permute(1, 2, 0, 3)).fill_(False)
    assert torch.isnan(space[outside]).all()


def test_parents_and_pages_outside_their_range(g):
    """A parent that is no token before makes a token follow the others; pages that are none hide their places."""
    T = 70
    cache = Cache(17, HALF, 1, 1, 64, 16, [100], T)
    parents = tree_of(18, 1, T)
    strange = parents.clone()
    strange[0, ::7] = numbers([-2, 0, 100, 2 ** 31 - 1, -2 ** 31, 35, 42, 69, 69, 70])
    for i in range(0, T, 7):
        if not 0 <= int(strange[0, i]) < i:
            parents[0, i] = -1
        else:
            parents[0, i] = strange[0, i]
    q = normal(19, (1, T, 2, 64), HALF, 2.0)
    a = g.ops.TreeAttention(q, cache.keys, cache.values, cache.tables, cache.lengths, parents=strange)
    assert torch.equal(a, check_tree(g, cache, q, parents))
    pages = cache.tables.clone()
    pages[0, 1], pages[0, 3], pages[0, 7] = -1, cache.keys.shape[0], 2 ** 31 - 1
    mass = torch.full((1, 1, cache.tables.shape[1] * 16), 5.0, device="cuda")
    got = g.ops.TreeAttention(q, cache.keys, cache.values, pages, cache.lengths, parents=parents, mass=mass)
    k, v = cache.rows[0]
    sees = torch.cat([torch.ones(T, 100, dtype=torch.bool), line_of(parents[0].tolist(), T)], 1)
    for i in (1, 3, 7):
        sees[:, 16 * i: 16 * i + 16] = False
        assert (mass[0, 0, 16 * i: 16 * i + 16] == 5).all()
    want, room, _, _ = attend(q[0].cpu(), k, v, sees, 1 / 8)
    close(got[0], want, room)
    nothing = torch.full_like(cache.tables, -1)
    assert (g.ops.TreeAttention(q, cache.keys, cache.values, nothing, cache.lengths, parents=parents) == 0).all()


@pytest.mark.parametrize("length", [-5, 2 ** 31 - 1, 1000])
def test_lengths_outside_their_range(g, length):
    """Negative ones as 0, ones behind the table as its end: its drafted rows are then nowhere."""
    cache = Cache(20, HALF, 1, 1, 64, 16, [60], 4)
    q = normal(21, (1, 4, 2, 64), HALF, 2.0)
    places = cache.tables.shape[1] * 16
    cache.keys.nan_to_num_(0.25), cache.values.nan_to_num_(0.5)
    k, v = fill(cache)[0]
    got = g.ops.TreeAttention(q, cache.keys, cache.values, cache.tables, numbers([length]))
    n = 0 if length < 0 else places
    sees = torch.cat([torch.ones(4, n, dtype=torch.bool), line_of(None, 4)], 1)[:, :places]
    want, room, _, _ = attend(q[0].cpu(), k[: n + 4], v[: n + 4], sees, 1 / 8)
    close(got[0], want, room)


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("T", [6, 90])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite_in_places_that_are_not_seen(g, dtype, T, value):
    """Rows of other branches and of later tokens, whatever they hold, change nothing for those that do not see them; those that do have it."""
    cache = Cache(22, dtype, 1, 2, 128, 16, [90], T)
    q = normal(23, (1, T, 4, 128), dtype)
    parents = tree_of(24, 1, T)
    for tree in (None, parents):
        clean = check_tree(g, cache, q, tree)
        bad = 3
        page, row = int(cache.tables[0, (90 + bad) // 16]), (90 + bad) % 16
        for pool, several in ((cache.values, True), (cache.values, False), (cache.keys, True)):
            kept = pool[page, row].clone()
            if several:
                pool[page, row, 1] = value
            else:
                pool[page, row, 0, 5] = value
            mass = torch.zeros(1, 2, cache.tables.shape[1] * 16, device="cuda")
            got = g.ops.TreeAttention(q, cache.keys, cache.values, cache.tables, cache.lengths, parents=tree, mass=mass)
            line = line_of(None if tree is None else tree[0].tolist(), T)
            sees = line[:, bad]
            # (places that only rows without the bad one see have weights as ever; where v is bad, all have)
            fine = torch.ones(90 + T, dtype=torch.bool)
            if pool is cache.keys:
                fine[:90] = False
                fine[90:] = ~(line & sees[:, None]).any(0)
            assert torch.isfinite(mass[0][:, : 90 + T][:, fine.cuda()]).all() and torch.isfinite(mass[0, 0]).all()
            assert torch.equal(got[0][~sees], clean[0][~sees])
            group = 1 if several else 0
            other = slice(0, 2) if group else slice(2, 4)
            assert torch.equal(got[0][:, other], clean[0][:, other])
            touched = got[0][sees][:, 2 * group: 2 * group + 2]
            if pool is cache.values:
                touched = touched if several else touched[..., 5]
                assert (torch.isnan(touched) if math.isnan(value) else touched == value).all()
            elif math.isnan(value):
                assert torch.isnan(touched).all()
            pool[page, row] = kept


def test_both_infinities_and_what_weighs_nothing(g):
    """inf and -inf together are NaN; a place whose weight is 0 adds nothing, also of the cache."""
    cache = Cache(25, FLOAT, 1, 1, 64, 16, [200], 2)
    q = torch.zeros(1, 2, 1, 64, device="cuda")
    q[..., 0] = 1.0
    cache.keys[..., 0].nan_to_num_(0.0).fill_(0.0)
    at = lambda p: (int(cache.tables[0, p // 16]), p % 16)  # noqa: E731
    cache.keys[at(150)][0, 0] = -1e6  # (exp(-125000) is 0)
    cache.values[at(150)][0] = math.inf
    got = g.ops.TreeAttention(q, cache.keys, cache.values, cache.tables, cache.lengths)
    assert torch.isfinite(got).all()
    cache.values[at(10)][0, 3] = math.inf
    cache.values[at(130)][0, 3] = -math.inf
    cache.values[at(11)][0, 4] = -math.inf
    got = g.ops.TreeAttention(q, cache.keys, cache.values, cache.tables, cache.lengths)
    assert torch.isnan(got[..., 3]).all() and (got[..., 4] == -math.inf).all() and torch.isfinite(got[..., 5:]).all()


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
def test_scores_far_apart(g, dtype):
    """Maxima that rise from place to place, the largest first, last and in between; scores that are all alike."""
    cache = Cache(26, dtype, 1, 1, 64, 64, [1500], 1)
    q = torch.zeros(1, 1, 8, 64, device="cuda", dtype=dtype)
    q[..., 0] = torch.tensor([1.0, -1.0, 8.0, -8.0, 64.0, -64.0, 0.0, 0.125]).to(dtype)
    k = cache.rows[0][0]
    k[:, 0, 0] = torch.linspace(-8, 8, 1501).to(dtype)
    k[700, 0, 0] = 12.0
    for p in range(1501):
        cache.keys[int(cache.tables[0, p // 64]), p % 64] = k[p].cuda()
    check_tree(g, cache, q, scale=1.0)
    check_tree(g, cache, q, scale=1e-6)
    check_tree(g, cache, q, scale=30.0)


def test_scores_that_are_minus_infinity(g):
    """A token that has no score above -inf has a result of 0, one that has some goes by those."""
    cache = Cache(27, FLOAT, 1, 1, 64, 16, [70], 1)
    big = torch.finfo(FLOAT).max
    cache.keys.fill_(0.0)
    for p in range(71):
        at = (int(cache.tables[0, p // 16]), p % 16)
        cache.keys[at][0, 0] = -big
        cache.keys[at][0, 1] = -big if p != 40 else 1.0
    q = torch.zeros(1, 1, 2, 64, device="cuda")
    q[0, 0, 0, 0], q[0, 0, 1, 1] = 4.0, 4.0  # products of -inf
    got = g.ops.TreeAttention(q, cache.keys, cache.values, cache.tables, cache.lengths, scale=1.0)
    assert (got[0, 0, 0] == 0).all()
    assert torch.equal(got[0, 0, 1].cpu(), cache.rows[0][1][40, 0])


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
def test_recorded_and_on_two_streams(g, dtype):
    """Calls in parts with mass, recorded side by side with appends, replayed with eager work between; the same calls on two streams at once."""
    T = 3
    caches = [Cache(30 + i, dtype, 1, 2, 64, 16, [n], T) for i, n in enumerate((1500, 900))]
    qs = [normal(32 + i, (1, T, 4, 64), dtype, 2.0) for i in range(2)]
    parents = numbers([[-1, 0, 0]])
    new = [normal(34 + i, (1, T, 2, 64), dtype) for i in range(2)]
    masses = [torch.zeros(1, 2, c.tables.shape[1] * 16, device="cuda") for c in caches]

    def step(i, mass):
        c = caches[i]
        g.ops.CacheAppend(c.keys, c.values, new[i], new[1 - i], c.tables, c.lengths)
        return g.ops.TreeAttention(qs[i], c.keys, c.values, c.tables, c.lengths, parents=parents, mass=mass)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = [step(i, masses[i]) for i in range(2)]
    for r in range(3):
        for i in range(2):
            qs[i].copy_(normal(40 + 2 * r + i, qs[i].shape, dtype, 2.0))
            new[i].copy_(normal(50 + 2 * r + i, new[i].shape, dtype))
            masses[i].zero_()
        graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            mass = torch.zeros_like(masses[i])
            assert torch.equal(step(i, mass), recorded[i]) and torch.equal(mass, masses[i])
    want = [step(i, None) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i, None))
    torch.cuda.synchronize()
    assert all(torch.equal(one, want[i]) for i in range(2) for one in got[i])


@pytest.mark.parametrize("dtype,D,T", [(HALF, 128, 200), (HALF, 256, 3), (FLOAT, 256, 2), (FLOAT, 128, 150)])
def test_recorded_before_any_other_call(g, dtype, D, T):
    """What a kernel needs, as more LDS than every one has, is asked for in a recording too; heads beside, so that many rows and few are met."""
    cache = Cache(36, dtype, 2, 2, D, 16, [70, 400], T)
    q, mass = normal(37, (2, T, 8, D), dtype, 2.0), torch.zeros(2, 2, cache.tables.shape[1] * 16, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = g.ops.TreeAttention(q, cache.keys, cache.values, cache.tables, cache.lengths, mass=mass)
    for _ in range(3):
        mass.zero_()
        q.copy_(q.flip(1))
        graph.replay()
        torch.cuda.synchronize()
        kept, again = mass.clone(), torch.zeros_like(mass)
        assert torch.equal(got, check_tree(g, cache, q, mass=again)) and torch.equal(kept, again)


def test_a_pool_of_more_than_4_gib(g):
    """Pages far apart: offsets that 32 bits do not hold."""
    P, R, G, D = 9000, 256, 8, 128  # 4.7 GB of keys
    keys = torch.zeros(P, R, G, D, dtype=HALF, device="cuda")
    values = torch.zeros(P, R, G, D, dtype=HALF, device="cuda")
    tables = numbers([[8999, 0, 8500]])
    k, v = normal(60, (1, 600, G, D), HALF), normal(61, (1, 600, G, D), HALF)
    g.ops.CacheAppend(keys, values, k, v, tables, numbers([0]))
    assert torch.equal(keys[8999], k[0, :256]) and torch.equal(values[8500, :88], v[0, 512:])
    q = normal(62, (1, 1, 16, D), HALF, 2.0)
    got = g.ops.TreeAttention(q, keys, values, tables, numbers([599]))
    want, room, _, _ = attend(q[0].cpu(), k[0].cpu(), v[0].cpu(), torch.ones(1, 600, dtype=torch.bool), D ** -0.5)
    close(got[0], want, room)


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("D,R,gap", [(80, 16, 8), (96, 8, 0), (192, 20, 16), (75, 16, 0), (75, 20, 3), (201, 64, 0), (40, 16, 8), (33, 8, 1), (3, 16, 0), (128, 1, 8)])
@pytest.mark.parametrize("B,H,G,T,lengths", [(2, 4, 2, 3, [700, 333]), (1, 4, 1, 2, [4000]), (4, 16, 8, 300, [0, 200, 333, 64])])
def test_rows_that_do_not_fill_a_tile(g, dtype, D, R, gap, B, H, G, T, lengths):
    """What lies behind a row, here NaN, is no part of it, in whole tiles as in those that a sequence ends in; and results are the same each time."""
    cache = Cache(80, dtype, B, G, D, R, lengths, T, gap=gap)
    q = normal(81, (B, T, H, D), dtype, 2.0)
    mass = torch.zeros(B, G, cache.tables.shape[1] * R, device="cuda")
    got = check_tree(g, cache, q, None if T > 256 else tree_of(82, B, T), mass=mass)
    for _ in range(3):
        again = torch.zeros_like(mass)
        assert torch.equal(got, g.ops.TreeAttention(q, cache.keys, cache.values, cache.tables, cache.lengths, parents=None if T > 256 else tree_of(82, B, T), mass=again))
        assert torch.equal(mass, again)


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("D", [64, 75, 128, 256])
@pytest.mark.parametrize("tree", [False, True])
def test_mass_of_many_rows(g, dtype, D, tree):
    """By rows where places are few, by places, in several rounds of rows, where they are many; sequences with fewer tokens than the batch."""
    for B, G, H, T, lengths, counts in ((4, 1, 2, 200, [0, 300, 31, 95], [200, 77, 0, 129]), (4, 8, 16, 90, [1100, 0, 1500, 700], [90, 90, 33, 0])):
        cache = Cache(83, dtype, B, G, D, 16, lengths, T)
        mass = torch.rand((B, G, cache.tables.shape[1] * 16), generator=torch.Generator().manual_seed(84)).cuda()
        check_tree(g, cache, normal(85, (B, T, H, D), dtype, 2.0), tree_of(86, B, T) if tree else None, numbers(counts), mass=mass)


def test_places_that_are_not_seen_weigh_nothing(g):
    """A key that no row sees, of another branch's node or of a page that is none, gets no mass, and a NaN there none."""
    cache = Cache(87, HALF, 1, 1, 64, 16, [40], 150)
    parents = torch.full((1, 150), -1, dtype=torch.int32, device="cuda")
    cache.tables[0, 1] = cache.keys.shape[0]
    mass = torch.full((1, 1, cache.tables.shape[1] * 16), 3.0, device="cuda")
    q = normal(88, (1, 150, 2, 64), HALF)
    got = g.ops.TreeAttention(q, cache.keys, cache.values, cache.tables, cache.lengths, parents=parents, mass=mass)
    assert torch.isfinite(got).all() and torch.isfinite(mass).all()
    assert (mass[0, 0, 16:32] == 3).all() and (mass[0, 0, 190:] == 3).all()
    total = (mass[0, 0, :190].sum() - 3.0 * 40).item()  # each of 300 rows weighs 1, off by 2^-11 of a weight
    assert abs(total - 300.0) < 300 * 2.0 ** -10


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("T", [1, 7, 60, 200])
def test_padding_holds_anything(g, dtype, T):
    """Queries of tokens that a sequence does not have, and keys and values in its drafted places behind them, NaN: nobody else sees them."""
    counts = [0, T // 2, T]
    cache = Cache(92, dtype, 3, 2, 64, 16, [50, 333, 0], T)
    q = normal(93, (3, T, 8, 64), dtype, 2.0)
    for b, count in enumerate(counts):
        q[b, count:] = math.nan
        n = len(cache.rows[b][0]) - T
        for p in range(n + count, n + T):
            at = (int(cache.tables[b, p // 16]), p % 16)
            cache.keys[at], cache.values[at] = math.nan, math.inf
        for rows in cache.rows[b]:
            rows[n + count:] = 0.0
    for tree in (None, tree_of(94, 3, T)):
        check_tree(g, cache, q, tree, numbers(counts), mass=torch.ones(3, 2, cache.tables.shape[1] * 16, device="cuda"))


def test_threads(g):
    """Calls of different kernels from threads at once, each on a stream of its own."""
    import threading
    calls, want, got = [], [], {}
    for i, (dtype, D, T, n) in enumerate(((HALF, 128, 1, 900), (FLOAT, 256, 2, 300), (HALF, 64, 256, 100), (FLOAT, 64, 40, 500))):
        cache = Cache(90 + i, dtype, 1, 2, D, 16, [n], T)
        calls.append((normal(95 + i, (1, T, 4, D), dtype), cache.keys, cache.values, cache.tables, cache.lengths, tree_of(99 + i, 1, T)))
        want.append(g.ops.TreeAttention(*calls[-1]))
    torch.cuda.synchronize()

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got[i] = [g.ops.TreeAttention(*calls[i]) for _ in range(20)]
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(one, want[i]) for i in range(4) for one in got[i])


@pytest.mark.parametrize("dtype,D,P", [(HALF, 96, 12000), (FLOAT, 75, 7200)])
def test_short_rows_in_a_pool_of_more_than_4_gib(g, dtype, D, P):
    keys, values = (torch.zeros(P, 256, 8, D, dtype=dtype, device="cuda") for _ in range(2))
    tables = numbers([[P - 1, 0, P - 500]])
    k, v = normal(63, (1, 600, 8, D), dtype), normal(64, (1, 600, 8, D), dtype)
    g.ops.CacheAppend(keys, values, k, v, tables, numbers([0]))
    q = normal(65, (1, 1, 16, D), dtype, 2.0)
    mass = torch.zeros(1, 8, 768, device="cuda")
    got = g.ops.TreeAttention(q, keys, values, tables, numbers([599]), mass=mass)
    want, room, weights, weights_room = attend(q[0].cpu(), k[0].cpu(), v[0].cpu(), torch.ones(1, 600, dtype=torch.bool), D ** -0.5)
    close(got[0], want, room)
    close(mass[0, :, :600], weights, weights_room + 2.0 ** -24 * weights)


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("length,M,far", [(1024, 128, False), (20, 2, False), (3000, 200, True), (40, 3, True)])
def test_scores_that_are_no_number_wherever_they_lie(g, dtype, length, M, far):
    """A token with a score that is NaN has NaN, whether its place shares a part of the cache with others (few places), is alone in one (the token's own, the first of its part), or lies in one
    whose other scores weigh nothing."""
    cache = Cache(100, dtype, 1, 8, 64, 16, [length], 1)
    more = torch.full((1, M - cache.tables.shape[1]), int(cache.tables[0, 0]), dtype=torch.int32, device="cuda")
    cache.tables = torch.cat([cache.tables, more], 1)
    q = normal(101, (1, 1, 32, 64), dtype)
    if far:  # one score that is 2^9 above all others, in the first part
        q[..., 0] = 8.0
        for p in range(length + 1):
            cache.keys[int(cache.tables[0, p // 16]), p % 16, :, 0] = 64.0 if p == 3 else 0.0
        for rows in cache.rows:
            rows[0][:, :, 0] = 0.0
            rows[0][3, :, 0] = 64.0
    mass = torch.zeros(1, 8, M * 16, device="cuda")
    clean = check_tree(g, cache, q, scale=1.0, mass=mass)
    cache.keys[int(cache.tables[0, length // 16]), length % 16, 2:4, 7] = math.nan
    mass.zero_()
    got = g.ops.TreeAttention(q, cache.keys, cache.values, cache.tables, cache.lengths, scale=1.0, mass=mass)
    touched = torch.zeros(32, dtype=torch.bool)
    touched[8:16] = True
    assert torch.isnan(got[0, 0, touched]).all() and torch.isnan(mass[0, 2:4, : length + 1]).all()
    assert torch.equal(got[0, 0, ~touched], clean[0, 0, ~touched]) and torch.isfinite(mass[0, [0, 1, 4, 5, 6, 7]]).all()
    assert (mass[0, :, length + 1:] == 0).all()


@pytest.mark.parametrize("D", [64, 128, 200])
@pytest.mark.parametrize("T,length", [(1, 300), (40, 5000), (300, 77), (1, 20000)])
def test_float32_values_next_to_the_largest(g, D, T, length):
    """Means of values up to 3e38 of either sign are what they are: sums before the division would be above float32's largest.  In the same calls small values in other elements, and an infinite one."""
    cache = Cache(110, FLOAT, 1, 2, D, 16, [length], T)
    gen = torch.Generator().manual_seed(111)
    big = (torch.rand(length + T, 2, D, generator=gen) * 2 - 1) * 3e38
    big[:, 0, : D // 2] = big[:, 0, : D // 2].abs() * 0.5 + 1.5e38  # (all of one sign: the mean is as large)
    big[:, 1, 5:9] = torch.randn(length + T, 4, generator=gen)
    place = torch.arange(length + T, device="cuda")
    cache.values[cache.tables[0].long()[place // 16], place % 16] = big.cuda()
    cache.rows[0] = (cache.rows[0][0], big)
    q = normal(112, (1, T, 4, D), FLOAT, 0.5)
    q[0, T // 2] = 0.0  # (all places weigh the same)
    mass = torch.zeros(1, 2, cache.tables.shape[1] * 16, device="cuda")
    clean = check_tree(g, cache, q, mass=mass)
    at = (int(cache.tables[0, 0]), 4)
    cache.values[at][1, 3], cache.values[at][1, 6] = math.inf, -math.inf
    got = g.ops.TreeAttention(q, cache.keys, cache.values, cache.tables, cache.lengths)
    assert (got[0, :, 2:, 3] == math.inf).all() and (got[0, :, 2:, 6] == -math.inf).all()
    others = torch.ones(4, D, dtype=torch.bool)
    others[2:, 3] = others[2:, 6] = False
    assert torch.isfinite(got[0][:, others]).all()
    # (made once with the sums as they are and once smaller: two roundings apart at most, in products of sums and weights)
    assert torch.allclose(got[0][:, others].double(), clean[0][:, others].double(), rtol=2.0 ** -20, atol=2.0 ** -100)


@pytest.mark.parametrize("T", [1, 300])
def test_float16_values_next_to_the_largest(g, T):
    """A mean of values that all are float16's largest is that one.  Weights are rounded before they are multiplied, the sum that divides is not: here nearly all of it is one weight between 2^13 and 2^14,
    whose rounding is up to 2^-11 of it, and half of that is enough for a result that rounds to infinity."""
    cache = Cache(115, HALF, 1, 1, 64, 16, [200], T)
    cache.keys.fill_(0.0)
    cache.keys[..., 0] = -60.0
    at = [(int(cache.tables[0, p // 16]), p % 16) for p in (0, 128)]
    cache.keys[at[0]][0, 0], cache.keys[at[1]][0, 0] = 0.0, 1.0
    cache.values[..., :32], cache.values[..., 32:] = 65504.0, -65504.0
    k, v = cache.rows[0]
    k.zero_()
    k[..., 0] = -60.0
    k[0, 0, 0], k[128, 0, 0] = 0.0, 1.0
    v[..., :32], v[..., 32:] = 65504.0, -65504.0
    q = torch.zeros(1, T, 64, 64, dtype=HALF, device="cuda")
    q[..., 0] = 4.859375 + torch.arange(64, device="cuda") / 256
    check_tree(g, cache, q, scale=1.0)
    cache.values[at[0]][0, 3] = math.inf
    got = g.ops.TreeAttention(q, cache.keys, cache.values, cache.tables, cache.lengths, scale=1.0)
    others = torch.arange(64) != 3
    assert (got[..., 3] == math.inf).all() and torch.isfinite(got[..., others]).all()


@pytest.mark.parametrize("dtype,gap", [(HALF, 1), (HALF, 3), (FLOAT, 1)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T", [1, 8, 200])
def test_queries_at_any_alignment(g, dtype, gap, D, T):
    """Rows that fill a kernel's size and are not at multiples of 16 bytes: the same results, number for number, as of those that are."""
    cache = Cache(120, dtype, 2, 2, D, 16, [90, 700], T)
    q = normal(121, (2, T, 4, D), dtype, 2.0)
    space = torch.full((2, T, 4, D + gap), math.nan, dtype=dtype, device="cuda")
    apart = space[..., gap:]
    apart.copy_(q)
    want = check_tree(g, cache, q)
    for _ in range(4):
        assert torch.equal(want, g.ops.TreeAttention(apart, cache.keys, cache.values, cache.tables, cache.lengths))


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("D", [64, 75, 129, 256])
@pytest.mark.parametrize("T", [1, 40, 300])
def test_values_that_are_not_finite_at_every_size(g, dtype, D, T):
    """Sums that are made again, in each kernel: infinite values and NaN are in their own elements alone, the others are what they are without them."""
    cache = Cache(130, dtype, 2, 2, D, 16, [90, 700], T)
    q = normal(131, (2, T, 4, D), dtype)
    clean = check_tree(g, cache, q)
    for b in range(2):
        at = [(int(cache.tables[b, p // 16]), p % 16) for p in (10, 60)]
        cache.values[at[0]][1, 1], cache.values[at[0]][1, 2], cache.values[at[0]][1, D - 1] = math.inf, -math.inf, math.inf
        cache.values[at[1]][1, 2], cache.values[at[1]][1, 3] = math.inf, math.nan
    for _ in range(2):
        got = g.ops.TreeAttention(q, cache.keys, cache.values, cache.tables, cache.lengths)
        assert (got[:, :, 2:, 1] == math.inf).all() and (got[:, :, 2:, D - 1] == math.inf).all() and torch.isnan(got[:, :, 2:, 2:4]).all()
        others = torch.ones(4, D, dtype=torch.bool)
        others[2:, 1:4] = others[2:, D - 1] = False
        assert torch.equal(got[:, :, others], clean[:, :, others])


# ---- an encoder's states ----------------------------------------------------------------------------

def check_cross(g, q, k, v, lengths=None, scale=None, out=None):
    got = g.ops.CrossAttention(q, k, v, lengths=lengths, scale=scale, out=out)
    B, T, H, D = q.shape
    for b in range(B):
        n = k.shape[1] if lengths is None else min(max(int(lengths[b]), 0), k.shape[1])
        want, room, _, _ = attend(q[b].cpu(), k[b, :n].cpu(), v[b, :n].cpu(), torch.ones(T, n, dtype=torch.bool), D ** -0.5 if scale is None else scale)
        close(got[b], want, room)
    return got


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("B,T,S,H,G,D", [(1, 1, 1, 1, 1, 64), (2, 1, 1500, 4, 4, 64), (3, 197, 77, 6, 6, 64), (1, 33, 129, 8, 2, 128), (2, 300, 65, 2, 1, 80), (1, 5, 2000, 7, 1, 256),
                                         (1, 128, 64, 2, 2, 75), (2, 64, 31, 4, 4, 32), (1, 257, 400, 4, 4, 192), (1, 1, 30000, 2, 1, 128)])
def test_cross_sizes(g, dtype, B, T, S, H, G, D):
    q, k, v = normal(70, (B, T, H, D), dtype, 2.0), normal(71, (B, S, G, D), dtype), normal(72, (B, S, G, D), dtype)
    check_cross(g, q, k, v)
    if B > 1:
        lengths = numbers([S // 2 + 1, 0, S][:B])
        k[0, S // 2 + 1:], v[0, S // 2 + 1:] = math.nan, math.inf
        k[1], v[1] = math.nan, math.nan
        got = check_cross(g, q, k, v, lengths)
        assert (got[1] == 0).all()


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
def test_cross_strides(g, dtype):
    """Heads in front of rows, rows of a product of queries, keys and values together, any alignment, expanded states."""
    B, T, S, H, D = 2, 40, 90, 3, 64
    together = normal(73, (B, S, 3, H, D), dtype)
    check_cross(g, together[:, :T, 0], together[:, :, 1], together[:, :, 2])
    apart = [normal(74 + i, (B, H, n, D + 5), dtype)[..., 1:65].transpose(1, 2) for i, n in enumerate((T, S, S))]
    out = torch.empty(B, H, T, D, dtype=dtype, device="cuda").transpose(1, 2)
    assert check_cross(g, *apart, lengths=numbers([90, 50]), out=out) is out
    one = normal(77, (1, S, 1, D), dtype)
    check_cross(g, together[:, :T, 0, :1], one.expand(B, S, 1, D), one.expand(B, S, 1, D))


def test_states_of_more_than_2_gib(g):
    """One sequence whose rows are further apart than 31 bits hold."""
    S = 1_100_000
    gen = torch.Generator(device="cuda").manual_seed(82)
    k, v = (torch.zeros(1, S, 8, 128, dtype=HALF, device="cuda")[:, :, 7:] for _ in range(2))
    for x in (k, v):
        x.copy_(torch.randn(x.shape, generator=gen, device="cuda").half())
    q = normal(83, (1, 2, 1, 128), HALF, 2.0)
    got = g.ops.CrossAttention(q, k, v)
    s = (q[0, :, 0].double() @ k[0, :, 0].double().T) * 128 ** -0.5
    w, values = torch.softmax(s, 1), v[0, :, 0].double()
    size = (q[0, :, 0].double().abs() @ k[0, :, 0].double().abs().T).amax(1, keepdim=True) * 128 ** -0.5
    want = w @ values
    room = (w @ values.abs()) * (2 * (2.0 ** -23 * 136 * size + 2.0 ** -22) + 2.0 ** -11 + 2.0 ** -24 * (S + 64)) + want.abs() * 2.0 ** -11 + w.amax(1, keepdim=True) * values.abs().sum(0) * 2.0 ** -31 + 2.0 ** -25
    close(got[0, :, 0], want.cpu(), room.cpu())


def test_nothing_to_attend_to(g):
    q = normal(78, (2, 3, 4, 64), HALF)
    none = torch.empty(2, 0, 4, 64, dtype=HALF, device="cuda")
    assert (g.ops.CrossAttention(q, none, none) == 0).all()
    assert g.ops.CrossAttention(q[:, :0], q, q).shape == (2, 0, 4, 64)
    assert g.ops.CrossAttention(q[:0], q[:0], q[:0]).shape == (0, 3, 4, 64)


def test_refusals_of_python_calls(g):
    q = normal(79, (1, 3, 4, 64), HALF)
    with pytest.raises(ValueError, match="not a tensor on the current device"):
        g.ops.CrossAttention(q, q.cpu(), q)
    with pytest.raises(g.capi.ChxHipError, match="overlap"):
        g.ops.CrossAttention(q, q, q, out=q)
    with pytest.raises(g.capi.ChxHipError, match="scale"):
        g.ops.CrossAttention(q, q, q, scale=0.0)
    with pytest.raises(g.capi.ChxHipError, match="do not share"):
        g.ops.CrossAttention(q, q[:, :, :3], q[:, :, :3])
    with pytest.raises(g.capi.ChxHipError, match="float16 or float32"):
        g.ops.CrossAttention(q.double(), q.double(), q.double())
