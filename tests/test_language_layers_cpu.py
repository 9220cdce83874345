"""What the entry points of the float layers of a language model refuse, and which launches they make, without a GPU."""
import ctypes

import pytest

import host_hip
import linear_sizes


@pytest.fixture(scope="module")
def host_so(tmp_path_factory):
    return host_hip.build(tmp_path_factory.mktemp("host_hip"))


@pytest.mark.parametrize("case", ["plans", "runs", "experts", "another_device", "no_memory", "routing", "combine", "logprobs", "launches"])
def test_case(host_so, case):
    host_hip.run_case(host_so, __file__, case)


def ref(t):
    return None if t is None else ctypes.byref(t)


def refused(host, rc, text, code=None):
    assert rc == (host.capi.EINVAL if code is None else code), (rc, host.lib.chx_hip_last_error())
    assert text.encode() in host.lib.chx_hip_last_error(), host.lib.chx_hip_last_error()
    assert host.launches() == []


def make(host, w, scale=None, b=None):
    plan = ctypes.c_void_p()
    rc = host.lib.chx_hip_linear_plan_create(ref(w), ref(scale), ref(b), None, ctypes.byref(plan))
    assert rc == 0 or not plan.value
    return rc, plan


def shifted(t, by):
    d = type(t).from_buffer_copy(t)
    d.data += by
    return d


def plans(host):
    T = host.tensor
    w = T("float16", (64, 32))
    for args, text in [((None,), "null tensor descriptor"), ((T("uint8", (64, 32)),), "float16, float32 or int8"), ((T("float16", (64,)),), "[N, K]"),
                       ((T("float16", (1, 2, 3, 4)),), "[N, K]"), ((T("float16", (0, 32)),), "no elements"), ((T("float16", (64, 0)),), "no elements"),
                       ((T("int8", (64, 32)),), "w_scale"), ((w, T("float32", (64,))), "w_scale"), ((T("int8", (64, 32)), T("float16", (64,))), "type of w_scale"),
                       ((w, None, T("int32", (64,))), "type of b"), ((w, None, T("float16", (63,))), "b must be"), ((T("float16", (3, 64, 32)), None, T("float16", (64,))), "b must be"),
                       ((shifted(w, 1),), "address"), ((T("float16", (1 << 25, 1), [0, 1]),), "2^24"), ((T("float16", (1, 1 << 25), [0, 0]),), "2^24")]:
        refused(host, make(host, *args)[0], text)
    assert host.lib.chx_hip_linear_plan_create(ref(w), None, None, None, None) == host.capi.EINVAL
    host.lib.chx_hip_linear_plan_destroy(None)


def runs(host):
    T, lib = host.tensor, host.lib
    half, quantized, floats = make(host, T("float16", (64, 32)))[1], make(host, T("int8", (64, 32)), T("float32", (64,)))[1], make(host, T("float32", (64, 32)))[1]
    experts = make(host, T("float16", (3, 64, 32)))[1]
    host.clear()

    def run(plan, x, y, r=None, act=0):
        return lib.chx_hip_linear_plan_run(plan, ref(x), act, ref(r), ref(y), None, ctypes.c_size_t(0), None)

    x, y = T("float16", (5, 32)), T("float16", (5, 64))
    both = T("float16", (5, 100))
    inside = T("float16", (5, 32), [100, 1], base=both.data)
    for args, text in [((None, x, y), "null plan"), ((half, None, y), "null tensor"), ((half, x, None), "null tensor"), ((half, T("float32", (5, 32)), y), "x must be float16"),
                       ((quantized, T("int8", (5, 32)), y), "x must be float16"), ((floats, x, y), "x must be float32"), ((floats, T("float32", (5, 32)), y), "y must be float32"),
                       ((half, x, T("int8", (5, 64))), "y must be"), ((half, x, y, None, 5), "activation"), ((half, x, y, None, -1), "activation"),
                       ((half, T("float16", (5, 31)), y), "last axis of x"), ((half, x, T("float16", (5, 63))), "last axis of y"), ((half, x, T("float16", (4, 64))), "differ on axis"),
                       ((half, T("float16", (1, 5, 32)), y), "number of axes"), ((half, T("float16", (5, 2, 32), [32, 320, 1]), T("float16", (5, 2, 64))), "not one run of rows"),
                       ((half, x, y, T("float16", (4, 64))), "r must have"), ((half, x, y, T("float32", (5, 64))), "r must have"), ((experts, x, y), "run_experts"),
                       ((half, shifted(x, 1), y), "address"), ((half, x, shifted(y, 1)), "address"),
                       ((half, inside, T("float16", (5, 64), [100, 1], base=both.data)), "x and y overlap"),
                       ((half, x, y, shifted(y, 2)), "r and y overlap"),
                       ((half, x, T("float16", (5, 64), [0, 1])), "elements of y overlap"), ((half, x, T("float16", (5, 64), [63, 1])), "elements of y overlap"),
                       ((half, x, T("float16", (5, 64), [1, 4])), "elements of y overlap"),
                       ((half, T("float16", (1 << 31, 32), [0, 1]), T("float16", (1 << 31, 64), [0, 1])), "2^31 rows")]:
        refused(host, run(*args), text)
    odd = T("float16", (5, 32))
    odd.strides[0] = 65
    refused(host, run(half, odd, y), "whole elements")
    host.check(run(half, x, y, y))      # r may be y
    host.check(run(half, T("float16", (0, 32)), T("float16", (0, 64))))
    assert len(host.launches()) == 1


def experts(host):
    T, lib = host.tensor, host.lib
    plain, plan = make(host, T("float16", (64, 32)))[1], make(host, T("float16", (3, 64, 32)))[1]
    host.clear()
    x, order, offsets, y = T("float16", (4, 32)), T("int32", (8,)), T("int32", (4,)), T("float16", (8, 64))

    def run(p, x, o, f, y):
        return lib.chx_hip_linear_plan_run_experts(p, ref(x), ref(o), ref(f), 0, ref(y), None, ctypes.c_size_t(0), None)

    for args, text in [((plain, x, order, offsets, y), "no experts"), ((plan, x, None, offsets, y), "null tensor"), ((plan, x, order, None, y), "null tensor"),
                       ((plan, x, T("int32", (7,)), offsets, y), "order must be"), ((plan, x, T("int32", (8,), [2]), offsets, y), "order must be"),
                       ((plan, x, T("float32", (8,)), offsets, y), "order must be"), ((plan, x, order, T("int32", (3,)), y), "offsets must be"),
                       ((plan, T("float16", (3, 32)), order, offsets, y), "multiple"), ((plan, T("float16", (0, 32)), order, offsets, y), "multiple"),
                       ((plan, T("float16", (1, 4, 32)), order, offsets, y), "matrices"), ((plan, x, shifted(order, 2), offsets, y), "address"),
                       ((plan, x, T("int32", (8,), base=y.data), offsets, y), "overlaps order")]:
        refused(host, run(*args), text)
    host.check(run(plan, x, order, offsets, y))
    host.check(run(plan, T("float16", (0, 32)), T("int32", (0,)), offsets, T("float16", (0, 64))))
    assert len(host.launches()) == 1


def another_device(host):
    T = host.tensor
    plan = make(host, T("float16", (64, 32)))[1]
    host.clear()
    host.check(host.lib.chx_hip_init(1))
    refused(host, host.lib.chx_hip_linear_plan_run(plan, ref(T("float16", (5, 32))), 0, None, ref(T("float16", (5, 64))), None, ctypes.c_size_t(0), None), "created on device 0, run on device 1")


def no_memory(host):
    w = host.tensor("float16", (64, 32))
    host.hh.hh_no_memory(ctypes.c_size_t(64 * 64 * 2))
    refused(host, make(host, w)[0], "hipMalloc", host.capi.EUNSUPPORTED)


def routing(host):
    T, lib = host.tensor, host.lib

    def run(T_, E, k, logits="float32", bias=None, groups=1, top_groups=1, best=1, space=None, order=None, weights=None):
        need = ctypes.c_size_t()
        if lib.chx_hip_expert_routing_workspace(ctypes.c_int64(T_), ctypes.c_int64(E), ctypes.byref(need)) != 0:
            need.value = 0
        have = need.value if space is None else space
        x = T(logits, (T_, E)) if isinstance(logits, str) else logits
        return lib.chx_hip_expert_routing(ref(x), ref(bias), 0, groups, top_groups, best, 1, ctypes.c_float(1), ref(T("int32", (T_, k))), ref(weights or T("float32", (T_, k))),
                                          ref(order or T("int32", (T_ * k,))), ref(T("int32", (E + 1,))), ctypes.c_void_p(host.malloc(max(have, 16))), ctypes.c_size_t(have), None)

    for args, kw, text in [((5, 16, 17), {}, "no more than there are"), ((5, 100, 65), {}, "1 to 64"), ((5, 1025, 2), {}, "1 to 1024"), ((5, 16, 2), {"logits": "int8"}, "float16 or float32"),
                           ((5, 16, 2), {"groups": 3, "top_groups": 1}, "equal size"), ((5, 128, 2), {"groups": 128}, "1 to 64 groups"), ((5, 16, 2), {"groups": 0}, "groups"),
                           ((5, 16, 2), {"groups": 4, "top_groups": 5}, "have no"), ((5, 16, 2), {"groups": 4, "top_groups": 0}, "have no"), ((5, 16, 5), {"groups": 4, "top_groups": 1}, "have no"),
                           ((5, 16, 2), {"best": 3}, "one or two"), ((5, 16, 1), {"groups": 16, "best": 2}, "one or two"), ((5, 16, 2), {"bias": T("float32", (15,))}, "bias must be"),
                           ((5, 16, 2), {"bias": T("float16", (16,))}, "bias must be"), ((1000, 16, 2), {"space": 100}, "workspace"), ((5, 16, 2), {"order": T("int32", (9,))}, "order must be"),
                           ((5, 16, 2), {"weights": T("float16", (5, 2))}, "weights must be")]:
        refused(host, run(*args, **kw), text)
    assert lib.chx_hip_expert_routing_workspace(ctypes.c_int64(5), ctypes.c_int64(0), ctypes.byref(ctypes.c_size_t())) == host.capi.EINVAL
    host.check(run(16, 16, 2))
    assert len(host.launches()) == 1
    host.clear()
    host.check(run(17, 1024, 64))
    assert len(host.launches()) == 2


def combine(host):
    T, lib = host.tensor, host.lib
    x, w, y = T("float16", (6, 32)), T("float32", (3, 2)), T("float16", (3, 32))

    def run(x, w, y, r=None):
        return lib.chx_hip_expert_combine(ref(x), ref(w), ref(r), ref(y), None)

    for args, text in [((None, w, y), "null tensor"), ((T("int8", (6, 32)), w, y), "float16 or float32"), ((x, T("float16", (3, 2)), y), "weights must be"), ((x, T("float32", (2, 2)), y), "must have 4 rows"),
                       ((x, T("float32", (3, 2), [4, 1]), y), "weights must be"), ((x, w, T("float32", (3, 32))), "of the type of x"), ((x, w, T("float16", (3, 31))), "y must be"),
                       ((x, w, y, T("float16", (2, 32))), "r must have"), ((x, w, T("float16", (3, 32), base=x.data)), "overlaps x"), ((x, w, y, shifted(y, 2)), "not the same array"),
                       ((shifted(x, 1), w, y), "whole elements"), ((x, w, T("float16", (3, 32), [0, 1])), "elements of y overlap")]:
        refused(host, run(*args), text)
    host.check(run(x, w, y, y))
    assert len(host.launches()) == 1


def logprobs(host):
    T, lib = host.tensor, host.lib

    def run(R, V, top, logits="float32", tokens="int32", space=None, entropy="float32", best=True):
        need = ctypes.c_size_t()
        if lib.chx_hip_token_logprobs_workspace(ctypes.c_int64(R), ctypes.c_int64(V), ctypes.c_int64(top), ctypes.byref(need)) != 0:
            need.value = 0
        have = need.value if space is None else space
        x = T(logits, (R, V)) if isinstance(logits, str) else logits
        long = host.capi.make_desc(host.malloc(8 * R * top + 64), host.capi.INT64, (R, top), (8 * top, 8))
        k = None if tokens is None else T(tokens, (R,)) if isinstance(tokens, str) else tokens
        return lib.chx_hip_token_logprobs(ref(x), ref(k), ref(T("float32", (R,)) if best else None), ref(T(entropy, (R,))), ref(T("float32", (R, top))), ref(long),
                                          ctypes.c_void_p(host.malloc(max(have, 16))), ctypes.c_size_t(have), None)

    for args, kw, text in [((4, 100, 65), {}, "at most 64"), ((4, 5, 6), {}, "no more than there are"), ((4, 100, 5), {"logits": "int8"}, "float16 or float32"), ((4, 0, 0), {}, "1 to 2^30"),
                           ((4, 100, 5), {"tokens": "float32"}, "int32 or int64"), ((4, 100, 5), {"tokens": T("int32", (3,))}, "a token for each row"), ((4, 100, 5), {"tokens": None}, "given together"),
                           ((4, 100, 5), {"best": False}, "given together"), ((1, 100000, 5), {"space": 32}, "workspace"), ((4, 100, 5), {"entropy": "float16"}, "entropy must be")]:
        refused(host, run(*args, **kw), text)
    host.check(run(4, 100, 5))
    assert len(host.launches()) == 1
    host.clear()
    host.check(run(1, 100000, 64, logits="float16", tokens=None, best=False))
    assert len(host.launches()) == 2


def launches(host):
    """Few rows take the kernel that streams weights, many the tiles; every type has both."""
    T, lib = host.tensor, host.lib
    for kind, w_kind in (("float16", "float16"), ("float16", "int8"), ("float32", "float32")):
        plan = make(host, T(w_kind, (256, 128)), T("float32", (256,)) if w_kind == "int8" else None)[1]
        for rows, name in ((1, "linear_rows_kernel"), (16, "linear_rows_kernel"), (20000, "linear_tile_kernel")):
            host.clear()
            host.check(lib.chx_hip_linear_plan_run(plan, ref(T(kind, (rows, 128))), 0, None, ref(T(kind, (rows, 256))), None, ctypes.c_size_t(0), None))
            assert len(host.launches()) == 1 and name in host.launches()[0], host.launches()
        # many rows that are not whole pieces are brought into such first, in the caller's memory
        x, y, size = T(kind, (20000, 128), [129, 1]), T(kind, (20000, 256)), ctypes.c_size_t()
        host.check(lib.chx_hip_linear_plan_workspace(plan, ref(x), ctypes.c_int64(20000), ctypes.byref(size)))
        assert size.value == 20000 * (512 if kind == "float32" else 256)
        host.clear()
        refused(host, lib.chx_hip_linear_plan_run(plan, ref(x), 0, None, ref(y), ctypes.c_void_p(host.malloc(size.value)), ctypes.c_size_t(size.value - 1), None), "workspace")
        host.check(lib.chx_hip_linear_plan_run(plan, ref(x), 0, None, ref(y), ctypes.c_void_p(host.malloc(size.value)), size, None))
        assert len(host.launches()) == 2 and "linear_pieces_kernel" in host.launches()[0] and "linear_tile_kernel" in host.launches()[1], host.launches()
        for few in (T(kind, (8, 128), [129, 1]), T(kind, (20000, 128))):
            host.check(lib.chx_hip_linear_plan_workspace(plan, ref(few), ctypes.c_int64(few.shape[0]), ctypes.byref(size)))
            assert size.value == 0


@pytest.mark.parametrize("case", ["large", "reached", "long_products"])
def test_sizes_at_the_bounds(host_so, case):
    host_hip.run_case(host_so, __file__, case)


def large(host):
    """Launches have fewer than 2^32 threads: more work than that goes in several, and products of more results are refused before anything runs."""
    T, lib = host.tensor, host.lib
    address = host.malloc(64)

    def threads():
        """Of each launch: name, threads."""
        lines = host.launches()
        return [(line, int(line.split("grid=")[1].split(",")[0]) * int(line.split("block=")[1].split()[0])) for line in lines]

    def some(name, least):
        found = threads()
        assert len(found) > 1 and all(name in line and n < 2 ** 32 for line, n in found) and sum(n for _, n in found) >= least, found

    # (descriptors of memory that nobody touches)
    rows, n = (1 << 20) + 3, 4099
    host.check(lib.chx_hip_expert_combine(ref(T("float16", (rows, n), base=address + (1 << 40))), ref(T("float32", (rows, 1), base=address + (1 << 45))), None, ref(T("float16", (rows, n), base=address)), None))
    some("expert_combine_kernel", rows * n)
    host.clear()
    plan = make(host, T("float16", (64, 16385)))[1]
    host.clear()
    rows = 1 << 20
    x, y, size = T("float16", (rows, 16385), [0, 1]), T("float16", (rows, 64), base=address + (1 << 40)), ctypes.c_size_t()
    host.check(lib.chx_hip_linear_plan_workspace(plan, ref(x), ctypes.c_int64(rows), ctypes.byref(size)))
    assert size.value == rows * 16448 * 2
    host.check(lib.chx_hip_linear_plan_run(plan, ref(x), 0, None, ref(y), ctypes.c_void_p((address + (1 << 45)) & ~15), size, None))
    found = threads()
    assert "linear_tile_kernel" in found.pop()[0]
    assert len(found) > 1 and all("linear_pieces_kernel" in line and n < 2 ** 32 for line, n in found) and sum(n for _, n in found) >= size.value // 16, found
    # a result of 2^31 - 1 rows, whose tiles are more than a launch has
    rows = (1 << 31) - 1
    x, y = T("float16", (rows, 16385), [0, 1]), T("float16", (rows, 64), base=address + (1 << 40))
    host.check(lib.chx_hip_linear_plan_workspace(plan, ref(x), ctypes.c_int64(rows), ctypes.byref(size)))
    host.clear()
    refused(host, lib.chx_hip_linear_plan_run(plan, ref(x), 0, None, ref(y), ctypes.c_void_p((address + (1 << 45)) & ~15), size, None), "fewer than 2^32 threads")
    for kind, columns in (("float16", 1 << 22), ("float32", 1 << 21), ("int8", 1 << 23)):
        scale = T("float32", (1,)) if kind == "int8" else None
        host.clear()
        refused(host, make(host, T(kind, (1, columns), [0, 0]), scale)[0], "too long")
        rc, longest = make(host, T(kind, (1, columns - 128), [0, 0]), scale)
        host.check(rc)
        lib.chx_hip_linear_plan_destroy(longest)
    host.clear()
    # the layout of many weights
    memory = T("int8", (64, 64, 128))
    host.check(lib.chx_hip_linear_plan_create(ref(T("int8", (16384, 16384, 128), [0, 128, 1], base=memory.data)), ref(T("float32", (16384, 16384), [0, 0], base=memory.data)), None, None, ctypes.byref(plan)))
    found = threads()
    assert len(found) > 1 and all(n < 2 ** 32 for _, n in found), found
    layout = sum(n for line, n in found if "linear_layout_kernel" in line)
    assert layout >= 16384 * 16384 * 128 // 16 and sum(n for line, n in found if "linear_vector_kernel" in line) >= 16384 * 16384


def reached(host):
    """Every kernel of the products is what some call takes: sizes over the range of each type, with rows that can be copied in whole pieces and others, small and large weights."""
    T, lib = host.tensor, host.lib
    host.hh.hh_kernels.restype = ctypes.c_char_p
    names = {k for k in host.hh.hh_kernels().decode().splitlines() if "linear_rows_kernel" in k or "linear_tile_kernel" in k}
    memory, result = T("int8", (64,)).data, T("int8", (64,)).data + (1 << 45)  # (descriptors of memory that nobody touches)
    taken = set()

    def note():
        taken.update(line.split(" grid=")[0] for line in host.launches() if line.split(" grid=")[0] in names)
        host.clear()

    for kind, w_kind in (("float16", "float16"), ("float16", "int8"), ("float32", "float32")):
        for K, columns in ((128, (16, 600, 1100, 2100, 4200, 9000, 20000)), (8192, (600, 1100, 2100, 4200, 9000))):
            for N in columns:
                scale = T("float32", (N,), [0], base=memory) if w_kind == "int8" else None
                plan = make(host, T(w_kind, (N, K), [0, 0], base=memory), scale)[1]
                for M in (1, 8, 9, 32, 33, 64, 65, 100, 150, 200, 300, 500, 700, 1000, 2000, 5000):
                    for gap in (0, 1):
                        host.check(lib.chx_hip_linear_plan_run(plan, ref(T(kind, (M, K), [K + gap, 1], base=memory)), 0, None, ref(T(kind, (M, N), base=result)),
                                                               ctypes.c_void_p(1 << 20), ctypes.c_size_t(1 << 40), None))
                        note()
                lib.chx_hip_linear_plan_destroy(plan)
        for E in (1, 8, 64):
            for K, N in ((128, 30), (128, 128), (128, 200), (128, 768), (128, 2000), (2048, 2048), (4096, 60), (4096, 128), (4096, 4096)):
                scale = T("float32", (E, N), [0, 0], base=memory) if w_kind == "int8" else None
                plan = make(host, T(w_kind, (E, N, K), [0, 0, 0], base=memory), scale)[1]
                for each in (1, 4, 6, 8, 12, 13, 24, 25, 33, 64, 100, 300, 1000, 1 << 16):
                    for pitch in (K, K + 1, 0):  # (0: one row again and again, however many)
                        M = E * each
                        host.check(lib.chx_hip_linear_plan_run_experts(plan, ref(T(kind, (M, K), [pitch, 1], base=memory)), ref(T("int32", (M,), base=memory)), ref(T("int32", (E + 1,), base=memory)), 0,
                                                                       ref(T(kind, (M, N), base=result)), ctypes.c_void_p(1 << 20), ctypes.c_size_t(1 << 40), None))
                        note()
                lib.chx_hip_linear_plan_destroy(plan)
    assert len(names) > 20 and names == taken, sorted(names - taken)


def long_products(host):
    """The sizes whose results test_gpu_linear_plan.py checks over the kernels' steady state take the kernels that they stand for."""
    T, lib = host.tensor, host.lib
    names = {linear_sizes.HALF: ("float16", "float16"), linear_sizes.INT8: ("float16", "int8"), linear_sizes.FLOAT: ("float32", "float32")}
    fragments_of = {64: "2, 2, 2", 128: "4, 2, 2", 256: "8, 2, 4"}

    def launched(which, kernel, experts, m, blocks, n, fan=1):
        kind, w_kind = names[which]
        K, lead = blocks * linear_sizes.BLOCK[which], (experts,) if experts else ()
        plan = make(host, T(w_kind, lead + (n, K)), T("float32", lead + (n,)) if w_kind == "int8" else None)[1]
        host.clear()
        x, y = T(kind, (m // fan, K)), T("float32", (m, n))
        if experts:
            host.check(lib.chx_hip_linear_plan_run_experts(plan, ref(x), ref(T("int32", (m,))), ref(T("int32", (experts + 1,))), 0, ref(y), None, ctypes.c_size_t(0), None))
        else:
            host.check(lib.chx_hip_linear_plan_run(plan, ref(x), 0, None, ref(y), None, ctypes.c_size_t(0), None))
        if kernel[0] == "rows":
            want = "linear_rows_kernel<(chx::LinearType)%d, %d, %d, true, %s" % (which, kernel[1], kernel[2], "true" if experts else "false")
        else:
            want = "linear_tile_kernel<(chx::LinearType)%d, %s, %s" % (which, fragments_of[kernel[1]], "true" if experts else "false")
        assert len(host.launches()) == 1 and want in host.launches()[0], (which, kernel, experts, m, blocks, n, host.launches())

    for which, kernel, m, blocks, n in linear_sizes.PLAIN:
        launched(which, kernel, 0, m, blocks, n)
    for which, kernel, experts, fan, m, blocks, n in linear_sizes.EXPERTS:
        launched(which, kernel, experts, m, blocks, n, fan)


if __name__ == "__main__":
    host_hip.main(globals())
