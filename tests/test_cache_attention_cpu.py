"""What the entry points of a paged cache and of attention over it refuse, the memory they ask for and the launches they make, without a GPU."""
import ctypes

import pytest

import host_hip


@pytest.fixture(scope="module")
def host_so(tmp_path_factory):
    return host_hip.build(tmp_path_factory.mktemp("host_hip"))


@pytest.mark.parametrize("case", ["caches", "append", "tree", "cross", "accept", "evict", "empty", "launches", "large", "reached"])
def test_case(host_so, case):
    host_hip.run_case(host_so, __file__, case)


def test_arrays_between_each_others_rows(host_so):
    host_hip.run_case(host_so, __file__, "interleaved")


def ref(t):
    return None if t is None else ctypes.byref(t)


def refused(host, rc, text):
    assert rc == host.capi.EINVAL, (rc, host.lib.chx_hip_last_error())
    assert text.encode() in host.lib.chx_hip_last_error(), host.lib.chx_hip_last_error()
    assert host.launches() == []


def shifted(t, by):
    d = type(t).from_buffer_copy(t)
    d.data += by
    return d


class Calls:
    """Each operator with arguments that it takes, any of which a test can replace."""

    def __init__(self, host, dtype="float16", B=2, T=3, H=4, G=2, D=64, P=9, R=16, M=4, A=5, address=None):
        T_ = self.T_ = host.tensor if address is None else lambda d, s, st=None: self.far(host, d, s, st)
        self.host, self.lib, self.next = host, host.lib, address
        self.names = dict(keys=T_(dtype, (P, R, G, D)), values=T_(dtype, (P, R, G, D)), tables=T_("int32", (B, M)), lengths=T_("int32", (B,)), counts=None, parents=None, mass=None,
                          q=T_(dtype, (B, T, H, D)), y=T_(dtype, (B, T, H, D)), k=T_(dtype, (B, T, G, D)), v=T_(dtype, (B, T, G, D)), accepted=T_("int32", (B, A)),
                          new_lengths=T_("int32", (B,)), scale=0.125, keep=20, recent=5, space=None, short=0)
        self.full_mass = T_("float32", (B, G, M * R))

    def far(self, host, dtype, shape, strides):
        """Descriptors of memory that nobody touches."""
        self.next += 1 << 44
        return host.tensor(dtype, shape, strides, base=self.next)

    def space(self, need, n):
        size = need if n["space"] is None else n["space"]
        return ctypes.c_void_p((host_space(self) if size else 0) + n["short"]), ctypes.c_size_t(size)

    def append(self, **with_):
        n = dict(self.names, **with_)
        return self.lib.chx_hip_cache_append(*[ref(n[i]) for i in ("keys", "values", "k", "v", "tables", "lengths", "counts")], None)

    def tree(self, **with_):
        n, need = dict(self.names, **with_), ctypes.c_size_t()
        self.lib.chx_hip_tree_attention_workspace(ref(n["q"]), ref(n["keys"]), ref(n["tables"]), int(n["mass"] is not None), ctypes.byref(need))
        return self.lib.chx_hip_tree_attention(*[ref(n[i]) for i in ("q", "keys", "values", "tables", "lengths", "parents", "counts")], ctypes.c_float(n["scale"]), ref(n["mass"]), ref(n["y"]),
                                               *self.space(need.value, n), None)

    def accept(self, **with_):
        n = dict(self.names, **with_)
        return self.lib.chx_hip_cache_accept(*[ref(n[i]) for i in ("keys", "values", "tables", "lengths", "accepted", "mass", "new_lengths")], None)

    def evict(self, **with_):
        n, need = dict(self.names, **dict({"mass": self.full_mass}, **with_)), ctypes.c_size_t()
        if n["keys"] is not None and n["tables"] is not None:
            self.lib.chx_hip_cache_evict_workspace(*[ctypes.c_int64(i) for i in (n["tables"].shape[0], n["keys"].shape[2], n["tables"].shape[1] * n["keys"].shape[1], n["keep"])], ctypes.byref(need))
        return self.lib.chx_hip_cache_evict(*[ref(n[i]) for i in ("keys", "values", "tables", "lengths", "mass")], ctypes.c_int64(n["keep"]), ctypes.c_int64(n["recent"]), ref(n["new_lengths"]),
                                            *self.space(need.value, n), None)

    def cross(self, **with_):
        n, need = dict(self.names, **with_), ctypes.c_size_t()
        self.lib.chx_hip_cross_attention_workspace(ref(n["q"]), ref(n["keys"]), ctypes.byref(need))
        return self.lib.chx_hip_cross_attention(*[ref(n[i]) for i in ("q", "keys", "values", "lengths")], ctypes.c_float(n["scale"]), ref(n["y"]), *self.space(need.value, n), None)


def host_space(calls):
    return 1 << 46  # (aligned, and nobody touches it)


def caches(host):
    """What every operator of a cache refuses of it."""
    T, c = host.tensor, Calls(host)
    n, page = c.names, (9, 16, 2, 64)
    for with_, text in [({"keys": None}, "null tensor"), ({"values": None}, "null tensor"), ({"tables": None}, "null tensor"), ({"lengths": None}, "null tensor"),
                        ({"keys": T("int8", page)}, "float16 or float32"), ({"values": T("float32", page)}, "must be float16"), ({"keys": T("float16", page[1:])}, "needs 4 axes"),
                        ({"values": T("float16", (9, 16, 2, 63))}, "one shape"), ({"keys": T("float16", page, [4096, 128, 64, 2])}, "has gaps"), ({"values": shifted(n["values"], 1)}, "whole elements"),
                        ({"keys": T("float16", (9, 16, 2, 257)), "values": T("float16", (9, 16, 2, 257))}, "1 to 256 elements"),
                        ({"keys": T("float16", (9, 16, 2, 0)), "values": T("float16", (9, 16, 2, 0))}, "1 to 256 elements"),
                        ({"keys": T("float16", (9, 16, 0, 64)), "values": T("float16", (9, 16, 0, 64))}, "a head"), ({"keys": T("float16", (9, 0, 2, 64)), "values": T("float16", (9, 0, 2, 64))}, "a place"),
                        ({"tables": T("float32", (2, 4))}, "int32 matrix"), ({"tables": T("int32", (2,))}, "int32 matrix"), ({"tables": T("int32", (2, 4), [8, 2])}, "row of tables must be contiguous"),
                        ({"tables": shifted(n["tables"], 2)}, "row of tables must be contiguous"), ({"lengths": T("int32", (3,))}, "another shape"), ({"lengths": T("float32", (2,))}, "must be int32"),
                        ({"lengths": T("int32", (2,), [2])}, "contiguous"), ({"lengths": T("int32", (2, 1))}, "another shape"),
                        ({"tables": T("int32", (2, 1 << 26), [0, 1], base=n["tables"].data)}, "2^30 places")]:
        for op in (c.append, c.tree, c.accept, c.evict):
            refused(host, op(**with_), text)
    odd = T("float16", page)
    odd.strides[1] = 257
    refused(host, c.tree(keys=odd), "whole elements")
    # rows of tables may lie apart, and pages in any order of axes
    apart = {"tables": T("int32", (2, 4), [9, 1]), "keys": T("float16", page, [2048, 64, 9 * 2048, 1]), "values": T("float16", page, [2048, 64, 9 * 2048, 1])}
    for op in (c.append, c.tree, c.accept, c.evict):
        host.clear()
        host.check(op(**apart))
        assert host.launches()


def append(host):
    T, c = host.tensor, Calls(host)
    n, new = c.names, (2, 3, 2, 64)
    for with_, text in [({"k": None}, "null tensor"), ({"k": T("float32", new)}, "k must be float16"), ({"v": T("float32", new)}, "v must be float16"), ({"v": T("float16", (2, 2, 2, 64))}, "k and v must be"),
                        ({"k": T("float16", (3, 3, 2, 64)), "v": T("float16", (3, 3, 2, 64))}, "k and v must be"), ({"k": T("float16", (2, 3, 4, 64)), "v": T("float16", (2, 3, 4, 64))}, "k and v must be"),
                        ({"k": T("float16", (2, 3, 2, 32)), "v": T("float16", (2, 3, 2, 32))}, "k and v must be"), ({"counts": T("int32", (3,))}, "another shape"), ({"counts": T("float32", (2,))}, "int32"),
                        ({"keys": T("float16", (9, 16, 2, 64), [0, 128, 64, 1])}, "elements of keys or values overlap"), ({"values": n["keys"]}, "keys and values overlap"),
                        ({"k": T("float16", new, base=n["keys"].data)}, "keys and k overlap"), ({"v": T("float16", new, base=n["values"].data)}, "values and v overlap"),
                        ({"lengths": T("int32", (2,), base=n["values"].data)}, "values and lengths overlap"), ({"tables": T("int32", (2, 4), base=n["keys"].data)}, "keys and tables overlap"),
                        ({"k": T("float16", (2, 1 << 30, 2, 64), [0, 0, 64, 1]), "v": T("float16", (2, 1 << 30, 2, 64), [0, 0, 64, 1])}, "2^30 tokens")]:
        refused(host, c.append(**with_), text)
    host.check(c.append(counts=T("int32", (2,))))
    host.check(c.append(k=n["v"]))  # (k and v are only read)
    assert len(host.launches()) == 2


def tree(host):
    T, c = host.tensor, Calls(host)
    n, rows, mass = c.names, (2, 3, 4, 64), c.full_mass
    inside = T("float32", (2, 2, 64), base=n["keys"].data)
    for with_, text in [({"q": None}, "null tensor"), ({"y": None}, "null tensor"), ({"q": T("float32", rows)}, "q must be float16"), ({"y": T("float32", rows)}, "y must be float16"),
                        ({"q": T("float16", (3, 3, 4, 64))}, "q has 3 sequences"), ({"q": T("float16", (2, 3, 4, 32))}, "q has 32 elements"), ({"q": T("float16", (2, 3, 3, 64))}, "do not share"),
                        ({"q": T("float16", (2, 3, 0, 64))}, "do not share"), ({"y": T("float16", (2, 3, 4, 63))}, "q's shape"), ({"y": T("float16", rows, [0, 256, 64, 1])}, "elements of y overlap"),
                        ({"y": n["q"]}, "y and q overlap"), ({"y": T("float16", rows, base=n["keys"].data)}, "y and keys overlap"), ({"y": T("float16", rows, base=n["values"].data)}, "y and values overlap"),
                        ({"parents": T("int32", (2, 4))}, "another shape"), ({"parents": T("float32", (2, 3))}, "int32"), ({"parents": T("int32", (2, 3), [4, 1])}, "contiguous"),
                        ({"counts": T("int32", (1,))}, "another shape"), ({"scale": 0.0}, "positive"), ({"scale": -1.0}, "positive"), ({"scale": float("nan")}, "positive"), ({"scale": float("inf")}, "positive"),
                        ({"scale": 3e38}, "positive"), ({"mass": T("float16", (2, 2, 64))}, "mass must be float32"), ({"mass": T("float32", (2, 64))}, "three axes"), ({"mass": T("float32", (2, 2, 63))}, "a number for each"),
                        ({"mass": T("float32", (2, 3, 64))}, "a number for each"), ({"mass": T("float32", (2, 2, 64), [0, 64, 1])}, "elements of mass overlap"), ({"mass": T("float32", (2, 2, 64), [256, 128, 2])}, "has gaps"),
                        ({"mass": inside}, "mass and keys overlap"), ({"mass": mass, "y": T("float16", rows, base=mass.data)}, "y and mass overlap"), ({"mass": mass, "space": 16}, "workspace"),
                        ({"mass": mass, "short": 4}, "workspace")]:
        refused(host, c.tree(**with_), text)
    refused(host, c.tree(q=T("float16", (2, 257, 4, 64)), y=T("float16", (2, 257, 4, 64)), parents=T("int32", (2, 257))), "at most 256 nodes")
    refused(host, c.lib.chx_hip_tree_attention_workspace(ref(n["q"]), ref(n["keys"]), ref(n["tables"]), 0, None), "null output")
    refused(host, c.lib.chx_hip_tree_attention_workspace(ref(n["q"]), ref(n["keys"]), None, 0, ctypes.byref(ctypes.c_size_t())), "null tensor")
    host.check(c.tree(parents=T("int32", (2, 3)), counts=T("int32", (2,)), mass=T("float32", (2, 2, 70))))
    host.check(c.tree(values=n["keys"]))  # (both are only read)
    assert [line.split("<")[0].split("::")[-1] for line in host.launches()] == ["attention_places_kernel", "attention_mass_kernel", "attention_places_kernel"], host.launches()


def cross(host):
    T, c = host.tensor, Calls(host)
    states, rows = (2, 50, 2, 64), (2, 3, 4, 64)
    k, v = T("float16", states), T("float16", states)
    for with_, text in [({"keys": None}, "null tensor"), ({"values": T("float32", states)}, "values must be float16"), ({"values": T("float16", (2, 49, 2, 64))}, "one shape"), ({"keys": T("int8", states)}, "float16 or float32"),
                        ({"keys": T("float16", (2, 50, 2, 257))}, "1 to 256 elements"), ({"q": T("float16", (3,) + rows[1:])}, "q has 3 sequences"), ({"q": T("float16", (2, 3, 5, 64))}, "do not share"),
                        ({"lengths": T("int32", (3,))}, "another shape"), ({"y": c.names["q"]}, "y and q overlap"), ({"y": T("float16", rows, base=v.data)}, "y and values overlap"), ({"scale": -0.5}, "positive"),
                        ({"keys": T("float16", (2, 1 << 30, 2, 64), [0, 0, 64, 1]), "values": T("float16", (2, 1 << 30, 2, 64), [0, 0, 64, 1])}, "2^30 states"), ({"y": T("float16", rows, [768, 0, 64, 1])}, "elements of y overlap")]:
        refused(host, c.cross(**dict({"keys": k, "values": v}, **with_)), text)
    long = [T("float16", (2, 5000, 2, 64)) for _ in range(2)]
    refused(host, c.cross(keys=long[0], values=long[1], space=8), "workspace")
    host.check(c.cross(keys=k, values=v, lengths=None))
    assert len(host.launches()) == 1


def accept(host):
    T, c = host.tensor, Calls(host)
    n, mass = c.names, c.full_mass
    for with_, text in [({"accepted": None}, "null tensor"), ({"accepted": T("int32", (3, 5))}, "another shape"), ({"accepted": T("int32", (2,))}, "another shape"), ({"accepted": T("float32", (2, 5))}, "int32"),
                        ({"accepted": T("int32", (2, 257))}, "at most 256"), ({"accepted": T("int32", (2, 5), [6, 1])}, "contiguous"), ({"new_lengths": None}, "null tensor"), ({"new_lengths": T("int32", (3,))}, "another shape"),
                        ({"new_lengths": n["lengths"]}, "new_lengths and lengths overlap"), ({"new_lengths": T("int32", (2,), base=n["accepted"].data)}, "new_lengths and accepted overlap"),
                        ({"values": shifted(n["keys"], 64)}, "keys and values overlap"), ({"mass": T("float32", (2, 2, 64), base=n["values"].data)}, "values and mass overlap"), ({"mass": T("float32", (2, 2, 63))}, "a number for each"),
                        ({"mass": mass, "new_lengths": T("int32", (2,), base=mass.data)}, "new_lengths and mass overlap"), ({"keys": T("float16", (9, 16, 2, 64), [2048, 128, 32, 1])}, "overlap")]:
        refused(host, c.accept(**with_), text)
    host.check(c.accept(mass=mass))
    host.check(c.accept(accepted=T("int32", (2, 0))))  # (still says how long they are)
    assert len(host.launches()) == 2


def evict(host):
    T, c = host.tensor, Calls(host)
    n, mass = c.names, c.full_mass
    for with_, text in [({"mass": None}, "null tensor"), ({"mass": T("float32", (2, 2, 63))}, "a number for each"), ({"keep": -1, "recent": 0}, "recent"), ({"recent": -1}, "recent"), ({"recent": 21}, "recent"),
                        ({"space": 4}, "workspace"), ({"short": 2}, "workspace"), ({"new_lengths": n["lengths"]}, "new_lengths and lengths overlap"), ({"mass": T("float32", (2, 2, 64), base=n["keys"].data)}, "keys and mass overlap"),
                        ({"lengths": T("int32", (2,), base=mass.data)}, "mass and lengths overlap")]:
        refused(host, c.evict(**with_), text)
    size = ctypes.c_size_t()

    def workspace(*numbers):
        return c.lib.chx_hip_cache_evict_workspace(*[ctypes.c_int64(i) for i in numbers], ctypes.byref(size))

    for numbers, text in [((-1, 2, 64, 20), "out of range"), ((2, 1 << 16, 64, 20), "out of range"), ((2, 2, 1 << 30, 20), "out of range"), ((2, 2, 64, -1), "negative"), (((1 << 24) - 1, (1 << 16) - 1, (1 << 30) - 1, 1 << 29), "one launch")]:
        refused(host, workspace(*numbers), text)
    refused(host, c.lib.chx_hip_cache_evict_workspace(*[ctypes.c_int64(1)] * 4, None), "null output")
    # a number of moves, and where they go and come from: no more than stay, nor than go
    for keep, moves in ((0, 0), (20, 20), (32, 32), (44, 20), (64, 0), (1 << 40, 0)):
        host.check(workspace(2, 3, 64, keep))
        assert size.value == 4 * 2 * 3 * (1 + 2 * moves)
    host.check(c.evict())
    assert [line.split("<")[0].split("::")[-1] for line in host.launches()] == ["cache_choose_kernel", "cache_evict_kernel"]
    host.clear()
    host.check(c.evict(keep=1 << 40, recent=1 << 40))  # nothing goes
    assert len(host.launches()) == 1


def empty(host):
    """No sequences, no tokens, no pages: nothing to do, or results without a place."""
    T = host.tensor
    for sizes, launched in (({"B": 0}, "-----"), ({"T": 0}, "--aev"), ({"P": 0}, "-taev"), ({"M": 0}, "-taev")):
        c = Calls(host, **sizes)
        for op, letter in ((c.append, "p"), (c.tree, "t"), (c.accept, "a"), (c.evict, "e")):
            host.clear()
            host.check(op())
            assert bool(host.launches()) == (letter in launched), (sizes, letter, host.launches())
    c = Calls(host)
    host.clear()
    host.check(c.cross(keys=T("float16", (2, 0, 2, 64)), values=T("float16", (2, 0, 2, 64))))  # every result is 0
    assert len(host.launches()) == 1


def launches(host):
    """Parts are joined, mass has a launch of its own, by places or, where those are few and rows many, by rows."""
    def names(dtype="float16", mass=False, **sizes):
        c = Calls(host, dtype, address=1 << 46, **sizes)
        host.clear()
        host.check(c.tree(mass=c.full_mass if mass else None))
        return [line.split("<")[0].split("::")[-1][len("attention_"):-len("_kernel")] for line in host.launches()]

    assert names(T=1, M=4, R=16) == ["places"]
    assert names(T=1, M=500, R=64) == ["places", "join"]
    assert names(T=24, M=500, R=64, H=16, mass=True) == ["places", "join", "mass"]
    assert names(B=8, T=2048, M=64, R=64, H=16) == ["rows"]
    assert names(B=1, T=600, M=4, R=64, H=16, mass=True)[-1] == "mass_rows"
    assert names(B=8, T=600, M=300, R=64, H=16, mass=True)[-1] == "mass_rows"
    assert names(B=8, T=40, M=300, R=64, H=16, mass=True)[-1] == "mass"
    # workspaces: parts' results and statistics, and the rows' sums
    size, c = ctypes.c_size_t(), Calls(host, T=1, M=500, R=64, address=1 << 46)
    n = c.names
    for mass, more in ((0, 0), (1, 4 * 2 * 2 * 2)):
        host.check(c.lib.chx_hip_tree_attention_workspace(ref(n["q"]), ref(n["keys"]), ref(n["tables"]), mass, ctypes.byref(size)))
        parts = (size.value - more) // (2 * 2 * 32 * 4 * 66)  # of 2 sequences and 2 heads: 32 rows of 64 elements and two numbers
        assert 1 < parts <= 64 and size.value == parts * 2 * 2 * 32 * 4 * 66 + more
    for rc in (c.tree(), c.tree(mass=c.full_mass)):
        host.check(rc)
    host.clear()
    refused(host, c.tree(space=size.value - more - 1), "workspace")


def large(host):
    """Launches have fewer than 2^32 threads, at the most work that is taken; more is refused before anything runs."""
    def threads():
        lines = host.launches()
        return [(line, int(line.split("grid=")[1].split(",")[0]) * int(line.split("block=")[1].split()[0])) for line in lines]

    # (numbers of tokens, sequences and heads at their bounds; descriptors of memory that nobody touches)
    c = Calls(host, B=3, T=(1 << 24) - 1, H=2, G=2, D=256, P=1 << 20, R=256, M=(1 << 22) - 1, address=1 << 46)
    host.check(c.append())
    found = threads()
    assert len(found) > 1 and all(n < 2 ** 32 for _, n in found) and sum(n for _, n in found) >= 3 * ((1 << 24) - 1) * 2 * 32
    host.clear()
    host.check(c.tree())
    assert all(0 < n < 2 ** 32 for _, n in threads())
    host.clear()
    refused(host, c.tree(q=c.T_("float16", (3, 1 << 24, 2, 256)), y=c.T_("float16", (3, 1 << 24, 2, 256))), "2^24 tokens")
    many = Calls(host, B=(1 << 24) - 1, T=1, H=8, G=8, D=64, P=64, R=16, M=1, address=1 << 46)
    refused(host, many.tree(), "more tiles than one launch has")
    refused(host, many.evict(), "more sequences and heads than one launch has")
    refused(host, many.accept(), "more sequences and heads than one launch has")
    most = Calls(host, B=(1 << 20) - 1, T=1, H=8, G=8, D=64, P=64, R=16, M=1, address=1 << 46)
    host.check(most.tree(mass=most.full_mass))
    assert len(host.launches()) == 2 and all(0 < n < 2 ** 32 for _, n in threads()), threads()
    host.clear()
    moved = Calls(host, B=(1 << 17) - 1, T=1, H=8, G=8, D=64, P=64, R=64, M=1, address=1 << 46)
    host.check(moved.evict())
    host.check(moved.accept(mass=moved.full_mass))
    assert len(host.launches()) == 3 and all(0 < n < 2 ** 32 for _, n in threads()), threads()
    host.clear()
    long = Calls(host, B=8, T=1, H=8, G=8, D=64, P=64, R=1 << 15, M=(1 << 15) - 1, address=1 << 46)
    host.check(long.tree())
    host.clear()
    refused(host, Calls(host, B=8, T=1, H=8, G=8, D=64, P=64, R=1 << 15, M=(1 << 15) - 1, address=1 << 46).tree(mass=long.full_mass), "more places than one launch has")


def reached(host):
    """Every kernel is what some call takes."""
    host.hh.hh_kernels.restype = ctypes.c_char_p
    names = {k for k in host.hh.hh_kernels().decode().splitlines() if "attention_" in k or "cache_" in k}
    taken = set()
    for dtype in ("float16", "float32"):
        for D in (1, 2, 4, 64, 75, 128, 200, 256):
            for B, T, R, M in ((1, 1, 16, 4), (2, 1, 64, 500), (8, 600, 64, 4), (1, 600, 64, 4), (8, 2048, 64, 300), (64, 24, 1024, 40)):
                c = Calls(host, dtype, B=B, T=T, H=16, G=4, D=D, R=R, M=M, address=1 << 46)
                for op, with_ in ((c.append, {}), (c.tree, {}), (c.tree, {"mass": c.full_mass}), (c.accept, {"mass": c.full_mass}), (c.evict, {"keep": R * M // 2})):
                    host.clear()
                    host.check(op(**with_))
                    taken.update(line.split(" grid=")[0] for line in host.launches())
    assert len(names) > 30 and names <= taken, sorted(names - taken)


def interleaved(host):
    """Keys and values of one allocation: taken where no byte is of both, refused where one is, whatever the order of the axes and the gaps between them."""
    import itertools
    import random
    T, rng = host.tensor, random.Random(1)
    found = {True: 0, False: 0}
    for _ in range(600):
        shape = [rng.choice([1, 2, 3]) for _ in range(3)] + [rng.choice([1, 2, 8])]
        order, strides, inside = rng.sample(range(3), 3) + [3], [0] * 4, 1
        for axis in reversed(order):
            strides[axis] = inside if axis == 3 else inside + rng.choice([0, 0, 1, 5, inside, 3 * inside])
            inside = strides[axis] * shape[axis]
        offset = rng.choice([0, rng.randrange(2 * inside + 2), rng.choice(strides) // 2, shape[3]])
        calls = Calls(host, P=shape[0], R=shape[1], G=shape[2], D=shape[3])
        keys = T("float16", shape, strides, base=1 << 50)
        values = shifted(keys, rng.choice([2, 2, 2, 1]) * offset * rng.choice([1, -1]))
        used = [{t.data + sum(i * s for i, s in zip(index, t.strides)) + byte for index in itertools.product(*map(range, shape)) for byte in (0, 1)} for t in (keys, values)]
        meet = bool(used[0] & used[1])
        host.clear()
        if values.data % 2:
            refused(host, calls.append(keys=keys, values=values), "whole elements")
            continue
        found[meet] += 1
        for op in (calls.append, calls.accept, calls.evict):
            host.clear()
            if meet:
                refused(host, op(keys=keys, values=values), "keys and values overlap")
            else:
                host.check(op(keys=keys, values=values))
    assert min(found.values()) > 100, found
    # a result between the rows of q is taken as well, one over them is not
    c = Calls(host)
    host.clear()
    both = T("float16", (2, 3, 2, 4, 64))
    q = T("float16", (2, 3, 4, 64), [3 * 2 * 256, 2 * 256, 64, 1], base=both.data)
    host.check(c.tree(q=q, y=shifted(q, 512)))
    host.clear()
    refused(host, c.tree(q=q, y=shifted(q, 510)), "y and q overlap")


if __name__ == "__main__":
    host_hip.main(globals())
