"""A cache of keys and values in pages (csrc/cache.hip) against plain loops: what moves is the same, number for number."""
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


def numbers(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Pages:
    """A pool with random rows, and tables of it."""

    def __init__(self, seed, dtype, B, M, R, G, D, layout="prgd", gap=0):
        gen = torch.Generator().manual_seed(seed)
        P = B * M + 3
        order = {"prgd": (0, 1, 2), "gprd": (2, 0, 1)}[layout]
        extents, back = (P, R, G), [order.index(i) for i in range(3)]

        def pool():
            space = torch.randn([extents[i] for i in order] + [D + gap], generator=gen).to(dtype).cuda()
            return space[..., gap:].permute(*back, 3)

        self.keys, self.values = pool(), pool()
        self.tables = torch.randperm(P, generator=gen)[: B * M].reshape(B, M).to(torch.int32).cuda()
        self.R, self.places = R, M * R
        self.mass = torch.rand(B, G, M * R, generator=gen).cuda()

    def copy(self):
        return [x.cpu().clone() for x in (self.keys, self.values, self.mass)]

    def at(self, b, p):
        """(page, row) of a place, None where it is nowhere."""
        if not 0 <= p < self.places:
            return None
        page = int(self.tables[b, p // self.R])
        return (page, p % self.R) if 0 <= page < self.keys.shape[0] else None

    def same(self, want, mass=True):
        for got, w in zip((self.keys, self.values, self.mass), want if mass else want[:2]):
            assert torch.equal(torch.nan_to_num(got.cpu(), nan=77.0), torch.nan_to_num(w, nan=77.0))


LAYOUTS = [(HALF, 16, 2, 128, "prgd", 0), (HALF, 1, 3, 80, "prgd", 0), (FLOAT, 20, 5, 75, "prgd", 0), (HALF, 64, 1, 7, "gprd", 0), (HALF, 8, 2, 64, "gprd", 1), (FLOAT, 16, 2, 256, "prgd", 2),
           (FLOAT, 3, 1, 1, "prgd", 0), (HALF, 16, 2, 256, "prgd", 4)]


@pytest.mark.parametrize("dtype,R,G,D,layout,gap", LAYOUTS)
@pytest.mark.parametrize("T", [1, 37])
def test_append(g, dtype, R, G, D, layout, gap, T):
    """Counts of none, some and too many; lengths below 0 (as 0), over and behind the table's end; pages that are none.  All else stays as it is."""
    B, M = 6, -(-60 // R)
    p = Pages(1, dtype, B, M, R, G, D, layout, gap)
    p.tables[1, 0], p.tables[1, M - 1] = -1, p.keys.shape[0]
    lengths = numbers([0, 3, p.places - 2, -4, p.places + 9, 11])
    gen = torch.Generator().manual_seed(2)
    k, v = (torch.randn(B, T, G, D + 3, generator=gen).to(dtype).cuda()[..., :D] for _ in range(2))
    for counts in (None, numbers([T, 1, T + 50, T, T, -1])):
        want = p.copy()
        for b in range(B):
            for t in range(T if counts is None else min(T, int(counts[b]))):
                at = p.at(b, max(0, min(int(lengths[b]), p.places)) + t)
                if at:
                    want[0][at], want[1][at] = k[b, t].cpu(), v[b, t].cpu()
        assert g.ops.CacheAppend(p.keys, p.values, k, v, p.tables, lengths, counts=counts) is None
        p.same(want)
    g.ops.CacheAppend(p.keys, p.values, k[:, :0], v[:, :0], p.tables, lengths)
    p.same(want)


def test_append_takes_what_is_contiguous_fast(g):
    """Whole 16-byte pieces of a longer prompt."""
    p = Pages(3, HALF, 2, 40, 16, 4, 128)
    k, v = torch.randn(2, 600, 4, 128, device="cuda").half(), torch.randn(2, 600, 4, 128, device="cuda").half()
    g.ops.CacheAppend(p.keys, p.values, k, v, p.tables, numbers([5, 40]))
    for b, n in enumerate((5, 40)):
        for pool, rows in ((p.keys, k), (p.values, v)):
            assert torch.equal(pool[p.tables[b].long()].flatten(0, 1)[n: n + 600], rows[b])


@pytest.mark.parametrize("dtype,R,G,D,layout,gap", LAYOUTS)
@pytest.mark.parametrize("with_mass", [False, True])
def test_accept(g, dtype, R, G, D, layout, gap, with_mass):
    """None, all, in any order, twice the same, up to the first negative one, from and to places that are nowhere."""
    B, M, A = 7, -(-90 // R), 12
    p = Pages(4, dtype, B, M, R, G, D, layout, gap)
    p.tables[4, 0] = -1
    lengths = numbers([0, 5, 20, p.places - 6, 0, -3, p.places + 2])
    gen = torch.Generator().manual_seed(5)
    accepted = torch.stack([torch.arange(A), torch.randperm(40, generator=gen)[:A].sort().values, torch.randint(0, 30, (A,), generator=gen), torch.arange(A) * 2, torch.randperm(40, generator=gen)[:A],
                            torch.arange(A) + 1, torch.arange(A)]).to(torch.int32)
    accepted[1, 7] = -1
    accepted[2, 3] = 2 ** 31 - 1
    accepted[5, 0] = -9
    want = p.copy()
    counts = []
    for b in range(B):
        n = min(max(int(lengths[b]), 0), p.places)
        row = accepted[b].tolist()
        row = row[: next((i for i, a in enumerate(row) if a < 0), A)]
        counts.append(min(n + len(row), p.places))
        before = [x.clone() for x in want]
        for j, a in enumerate(row):
            to, source = p.at(b, n + j), p.at(b, n + a)
            if to and source:
                want[0][to], want[1][to] = before[0][source], before[1][source]
            if n + j < p.places and n + a < p.places:
                want[2][b, :, n + j] = before[2][b, :, n + a]
    got = g.ops.CacheAccept(p.keys, p.values, p.tables, lengths, accepted.cuda(), mass=p.mass if with_mass else None)
    assert got.dtype == torch.int32 and got.tolist() == counts
    p.same(want, with_mass)
    kept = p.copy()
    assert torch.equal(g.ops.CacheAccept(p.keys, p.values, p.tables, lengths, accepted[:, :0].cuda()), lengths.clamp(0, p.places))
    p.same(kept)


def test_accept_256_rows(g):
    p = Pages(6, FLOAT, 1, 40, 16, 1, 200)
    accepted = torch.randperm(400, generator=torch.Generator().manual_seed(7))[:256].to(torch.int32)[None]
    before = p.copy()
    assert g.ops.CacheAccept(p.keys, p.values, p.tables, numbers([100]), accepted.cuda(), mass=p.mass).tolist() == [356]
    for j in range(0, 256, 5):
        to, source = p.at(0, 100 + j), p.at(0, 100 + int(accepted[0, j]))
        assert torch.equal(p.keys[to].cpu(), before[0][source]) and torch.equal(p.values[to].cpu(), before[1][source])
    assert torch.equal(p.mass[0, 0, 100: 356].cpu(), before[2][0, 0, 100 + accepted[0].long()])


def evicted(p, lengths, keep, recent):
    """What eviction leaves, by its definition: (keys, values, mass), new lengths."""
    want, counts = p.copy(), []
    for b in range(len(lengths)):
        n = min(max(int(lengths[b]), 0), p.places)
        counts.append(min(n, keep))
        if n <= keep:
            continue
        best, old = keep - recent, n - recent
        for h in range(p.mass.shape[1]):
            before = [x.clone() for x in want]
            m = before[2][b, h, :old].tolist()
            rank = sorted(range(old), key=lambda i: (0 if math.isnan(m[i]) else 1, 0 if math.isnan(m[i]) else -m[i], i))
            chosen = set(rank[:best])
            holes = [i for i in range(best) if i not in chosen]
            movers = sorted(i for i in chosen if i >= best)
            for to, source in list(zip(holes, movers)) + [(best + i, old + i) for i in range(recent)]:
                a, c = p.at(b, to), p.at(b, source)
                if a and c:
                    want[0][a][h], want[1][a][h] = before[0][c][h], before[1][c][h]
                want[2][b, h, to] = before[2][b, h, source]
            want[2][b, h, keep:n] = 0
    return want, counts


@pytest.mark.parametrize("dtype,R,G,D,layout,gap", LAYOUTS)
@pytest.mark.parametrize("keep,recent", [(40, 8), (40, 0), (40, 40), (1, 0), (1, 1), (0, 0), (69, 30), (70, 5), (10, 9)])
def test_evict(g, dtype, R, G, D, layout, gap, keep, recent):
    """Every kind of move: none, all, recent places onto themselves; sequences that are short enough already; weights that are equal, 0, NaN, infinite and negative."""
    B, M = 6, -(-70 // R)
    p = Pages(8, dtype, B, M, R, G, D, layout, gap)
    p.mass[1] = 0.0
    p.mass[2] = (p.mass[2] * 3).floor()
    p.mass[3, :, ::9], p.mass[3, :, 4], p.mass[3, :, 5], p.mass[3, :, 6] = math.nan, math.inf, -math.inf, -0.0
    p.mass[3, :, 10:30] -= 0.5
    p.tables[5, M // 2] = -1
    lengths = numbers([70, 70, 66, 61, p.places + 3, 70])
    lengths[4] = p.places + 3 if keep % 2 else 41
    want, counts = evicted(p, lengths, keep, recent)
    got = g.ops.CacheEvict(p.keys, p.values, p.tables, lengths, p.mass, keep, recent)
    assert got.tolist() == counts
    p.same(want)


@pytest.mark.parametrize("n,keep,recent", [(5000, 4990, 1000), (5000, 700, 300), (3000, 2999, 2500), (9001, 4000, 0), (20000, 19000, 64), (40001, 500, 100), (40001, 39000, 1)])
def test_evict_long(g, n, keep, recent):
    """More places than a work-group has lanes, than LDS has room for; recent ones that overlap themselves over many pieces."""
    p = Pages(9, HALF, 2, -(-n // 16), 16, 2, 64)
    p.mass[1, 1] = (p.mass[1, 1] * 50).floor()
    before = [x[p.tables[:].long()].flatten(1, 2)[:, :n].cpu() for x in (p.keys, p.values)]
    mass = p.mass.cpu().clone()
    assert g.ops.CacheEvict(p.keys, p.values, p.tables, numbers([n, n]), p.mass, keep, recent).tolist() == [keep, keep]
    after = [x[p.tables[:].long()].flatten(1, 2)[:, :n].cpu() for x in (p.keys, p.values)]
    best, old = keep - recent, n - recent
    for b in range(2):
        for h in range(2):
            chosen = torch.sort(mass[b, h, :old], descending=True, stable=True).indices[:best].sort().values
            source = torch.arange(keep)
            hole = torch.ones(best, dtype=torch.bool)
            hole[chosen[chosen < best]] = False
            source[:best][hole] = chosen[chosen >= best]
            source[best:] = torch.arange(old, n)
            for x, y in zip(before, after):
                assert torch.equal(y[b, :keep, h], x[b, source, h]) and torch.equal(y[b, keep:, h], x[b, keep:, h])
            assert torch.equal(p.mass[b, h, :keep].cpu(), mass[b, h, source]) and (p.mass[b, h, keep:n] == 0).all()


def test_recorded(g):
    """A step of a conversation recorded: rows appended, attention with mass, rows accepted, the cache cut; replayed with eager work in between, each against the eager result."""
    B, G, D, R, T = 2, 2, 64, 16, 5
    p = Pages(10, HALF, B, 8, R, G, D)
    first = [x.clone() for x in (p.keys, p.values, p.mass)]
    lengths, parents, accepted = numbers([100, 90]), numbers([[-1, 0, 0, 1, 2]] * B), numbers([[0, 2, 4], [1, 3, -1]])
    q, k, v = (torch.randn(B, T, n, D, device="cuda").half() for n in (4, G, G))

    def step():
        g.ops.CacheAppend(p.keys, p.values, k, v, p.tables, lengths)
        y = g.ops.TreeAttention(q, p.keys, p.values, p.tables, lengths, parents=parents, mass=p.mass)
        longer = g.ops.CacheAccept(p.keys, p.values, p.tables, lengths, accepted, mass=p.mass)
        return y, longer, g.ops.CacheEvict(p.keys, p.values, p.tables, longer, p.mass, 95, 20)

    def reset():
        for x, y in zip((p.keys, p.values, p.mass), first):
            x.copy_(y)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    for r in range(3):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(r)).half())
        reset()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in recorded] + [x.clone() for x in (p.keys, p.values, p.mass)]
        reset()
        want = list(step()) + [p.keys, p.values, p.mass]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert got[1].tolist() == [103, 92] and got[2].tolist() == [95, 92]


@pytest.mark.parametrize("dtype", [HALF, FLOAT])
@pytest.mark.parametrize("shape,axis", [((20, 2, 16, 3, 64), 1), ((20, 16, 2, 3, 64), 2), ((20, 16, 3, 2, 75), 3), ((20, 3, 16, 2, 128), 3), ((2, 20, 16, 3, 64), 0)])
def test_keys_and_values_in_one_allocation(g, dtype, shape, axis):
    """Pages that hold both: the same as of two pools, number for number, and nothing else is touched."""
    gen = torch.Generator().manual_seed(13)
    heads_first = shape == (20, 3, 16, 2, 128)
    pool = torch.randn(shape, generator=gen).to(dtype).cuda()
    one = [x.transpose(1, 2) if heads_first else x for x in pool.unbind(axis)]
    two = [x.clone() for x in one]
    P, R, G, D = one[0].shape
    tables = torch.randperm(P, generator=gen)[:16].reshape(2, 8).to(torch.int32).cuda()
    lengths, T = numbers([50, 100]), 7
    q, k, v = (torch.randn(2, T, n, D, generator=gen).to(dtype).cuda() for n in (2 * G, G, G))
    accepted = numbers([[0, 2, 4, 6], [1, 3, -1, 0]])
    results = []
    for keys, values in (one, two):
        mass = torch.zeros(2, G, 8 * R, device="cuda")
        g.ops.CacheAppend(keys, values, k, v, tables, lengths)
        y = g.ops.TreeAttention(q, keys, values, tables, lengths, mass=mass)
        longer = g.ops.CacheAccept(keys, values, tables, lengths, accepted, mass=mass)
        shorter = g.ops.CacheEvict(keys, values, tables, longer, mass, 60, 12)
        results.append([y, longer, shorter, mass, keys, values])
    assert results[0][1].tolist() == [54, 102] and results[0][2].tolist() == [54, 60]
    assert all(torch.equal(a, b) for a, b in zip(*results))
    with pytest.raises(g.capi.ChxHipError, match="keys and values overlap"):
        g.ops.CacheAppend(one[0], one[0], k, v, tables, lengths)


def test_a_conversation(g):
    """The operators together: a prompt in pieces, drafted trees of which some is accepted, a cache that is cut again and again; against dense caches in 64 bits, one for each
    sequence and head.  float32, so that the choice of what stays is the same (weights further apart than their errors)."""
    B, H, G, D, R, T = 2, 4, 2, 64, 16, 6
    gen = torch.Generator().manual_seed(11)
    p = Pages(12, FLOAT, B, 12, R, G, D)
    p.mass.zero_()
    lengths = numbers([0, 0])
    dense = [[dict(k=torch.zeros(0, D, dtype=torch.float64), v=torch.zeros(0, D, dtype=torch.float64), m=torch.zeros(0, dtype=torch.float64)) for _ in range(G)] for _ in range(B)]
    keep, recent = 64, 16
    for step in range(12):
        tokens = 40 if step == 0 else 33 if step == 1 else T
        tree = step > 1
        q, k, v = (torch.randn(B, tokens, n, D, generator=gen) * (2.0 if n == H else 1.0) for n in (H, G, G))
        parents = torch.stack([torch.arange(tokens) - torch.randint(1, 4, (tokens,), generator=gen) for _ in range(B)]).clamp(min=-1).to(torch.int32)
        g.ops.CacheAppend(p.keys, p.values, k.cuda(), v.cuda(), p.tables, lengths)
        y = g.ops.TreeAttention(q.cuda(), p.keys, p.values, p.tables, lengths, parents=parents.cuda() if tree else None, mass=p.mass)
        path = []
        for b in range(B):
            line = torch.zeros(tokens, tokens, dtype=torch.bool)
            for t in range(tokens):
                up = int(parents[b, t]) if tree else t - 1
                if up >= 0:
                    line[t] = line[up]
                line[t, t] = True
            path.append([i for i in range(tokens) if line[tokens - 1, i]])
            for c in range(G):
                d = dense[b][c]
                d["k"], d["v"] = torch.cat([d["k"], k[b, :, c].double()]), torch.cat([d["v"], v[b, :, c].double()])
                n = len(d["m"])
                d["m"] = torch.cat([d["m"], torch.zeros(tokens, dtype=torch.float64)])
                sees = torch.cat([torch.ones(tokens, n, dtype=torch.bool), line], 1)
                for h in range(c * H // G, (c + 1) * H // G):
                    w = torch.softmax((q[b, :, h].double() @ d["k"].T / math.sqrt(D)).masked_fill(~sees, -math.inf), 1)
                    d["m"] += w.sum(0)
                    # (scores are off by 2^-23 (D + 8) times sums of products below 100, weights by twice that; each step's keys carry no error over)
                    assert torch.allclose(y[b, :, h].double().cpu(), w @ d["v"], rtol=0, atol=2 * 2.0 ** -23 * 72 * 25 * 4)
        longest = max(map(len, path))
        accepted = torch.tensor([x + [-1] * (longest - len(x)) for x in path], dtype=torch.int32)
        longer = g.ops.CacheAccept(p.keys, p.values, p.tables, lengths, accepted.cuda(), mass=p.mass)
        shorter = g.ops.CacheEvict(p.keys, p.values, p.tables, longer, p.mass, keep, recent)
        for b in range(B):
            n = int(lengths[b])
            assert int(longer[b]) == n + len(path[b])
            for c in range(G):
                d = dense[b][c]
                rows = list(range(n)) + [n + i for i in path[b]]
                for name in "kvm":
                    d[name] = d[name][rows]
                if len(rows) > keep:
                    old, best = len(rows) - recent, keep - recent
                    order = torch.argsort(d["m"][:old], descending=True, stable=True)
                    chosen = set(order[:best].tolist())
                    source = [i if i in chosen else None for i in range(best)]
                    movers = iter(sorted(i for i in chosen if i >= best))
                    source = [next(movers) if i is None else i for i in source] + list(range(old, len(rows)))
                    for name in "kvm":
                        d[name] = d[name][source]
                assert len(d["m"]) == int(shorter[b])
                t = p.tables[b].long()
                for pool, name in ((p.keys, "k"), (p.values, "v")):
                    assert torch.equal(pool[t].flatten(0, 1)[: len(d["m"]), c].cpu().double(), d[name])
                assert torch.allclose(p.mass[b, c, : len(d["m"])].cpu().double(), d["m"], rtol=1e-3, atol=1e-5)
        lengths = shorter
