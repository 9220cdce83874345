"""Waits and registers of the attention kernels, in the code that was built: what a missing wait or a lost register does, no run shows reliably."""
import re

import pytest

import gpu_code


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    found = gpu_code.functions("attention_places_kernel", tmp_path_factory.mktemp("code"))
    return {name: f for name, f in found.items() if any(op.startswith("global_load_lds") for op, _ in f.code)}


def copies_before_reads(f):
    """Copies from memory into LDS that can start while reads of LDS are under way: those copies write it past the order of the wavefront's LDS instructions."""
    reads, todo, found = {}, [(0, 0)], set()
    while todo:
        i, n = todo.pop()
        if reads.get(i, -1) >= n:
            continue
        reads[i] = n  # at most this many instructions are under way from the earliest such read on
        op, operands = f.code[i]
        if op.startswith("global_load_lds") and n:
            found.add(i)
        if op.startswith("ds_read") or (n and op.startswith(("ds_", "s_load"))):
            n = min(n + 1, 16)
        elif op == "s_waitcnt":
            m = re.search(r"lgkmcnt\((\d+)\)", operands)
            n = min(n, int(m.group(1))) if m else n
        todo += [(j, n) for j in f.next[i]]
    return found


def test_reads_of_lds_are_waited_for_before_copies_into_it(kernels):
    assert len(kernels) >= 20, sorted(kernels)
    for name, f in kernels.items():
        assert any(op.startswith("ds_read") for op, _ in f.code)
        found = copies_before_reads(f)
        assert not found, (name, len(found))


def test_a_missing_wait_is_found(kernels):
    """The same code without its waits for LDS."""
    name, f = next((n, f) for n, f in kernels.items() if "attention_places_kernelILb1ELi128" in n)
    kept = f.code
    f.code = [("s_nop", "0") if op == "s_waitcnt" and "lgkmcnt(0)" in operands else (op, operands) for op, operands in kept]
    assert copies_before_reads(f)
    f.code = kept


def test_no_kernel_keeps_registers_in_memory(tmp_path):
    """Where registers run out the compiler moves live ones about, also inside branches that only some lanes take, where the other lanes lose theirs; so none of these kernels is over the limit."""
    found = {name: of for name, of in gpu_code.resources("attention_places_kernel", tmp_path).items() if "attention_" in name}
    assert len(found) > 20, sorted(found)
    for name, of in found.items():
        assert of["vgpr_spill_count"] == 0 and of["private_segment_fixed_size"] == 0 and of["vgpr_count"] <= 512, (name, of["vgpr_spill_count"], of["private_segment_fixed_size"])
