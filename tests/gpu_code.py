"""The instructions of the built library's kernels, as the disassembler prints them: for tests of what a run does not reliably show."""
import os
import re
import struct
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIBRARY = os.path.join(ROOT, "chainer-compiler_amd", "lib", "libchx_hip.so")
TOOLS = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")
OBJDUMP, READELF = os.path.join(TOOLS, "llvm-objdump"), os.path.join(TOOLS, "llvm-readelf")


def code_objects():
    """The library's device code, one object to a source file."""
    with open(LIBRARY, "rb") as f:
        data = f.read()
    at = data.find(b"__CLANG_OFFLOAD_BUNDLE__")
    while at >= 0:
        p = at + 32
        for _ in range(struct.unpack_from("<Q", data, at + 24)[0]):
            offset, size, length = struct.unpack_from("<QQQ", data, p)
            if size and b"gfx950" in data[p + 24: p + 24 + length]:
                yield data[at + offset: at + offset + size]
            p += 24 + length
        at = data.find(b"__CLANG_OFFLOAD_BUNDLE__", at + 24)


def files(containing, tmp_path):
    """Files with the code objects that hold a symbol with this in its name."""
    for i, data in enumerate(code_objects()):
        if containing.encode() in data:
            path = os.path.join(str(tmp_path), "%d.elf" % i)
            with open(path, "wb") as f:
                f.write(data)
            yield path


def resources(containing, tmp_path):
    """{symbol of a kernel: {what its metadata says of it}} of the code objects that hold a symbol with this in its name."""
    found = {}
    for path in files(containing, tmp_path):
        of = {}
        for line in subprocess.run([READELF, "--notes", path], capture_output=True, text=True, check=True).stdout.splitlines():
            m = re.match(r"^  (- |  )\.(\w+):\s*(\S*)", line)  # (arguments stand further in)
            if not m:
                continue
            if m.group(1) == "- ":
                of = {}
            of[m.group(2)] = int(m.group(3)) if m.group(3).isdigit() else m.group(3)
            if m.group(2) == "name":
                found[m.group(3)] = of
    return found


class Function:
    """Instructions as (name, operands), and of each the indexes of those that can follow it."""

    def __init__(self):
        self.lines, self.next = [], []

    def link(self):
        at = {address: i for i, (address, _, _, _) in enumerate(self.lines)}
        for i, (_, name, _, target) in enumerate(self.lines):
            follow = [] if name in ("s_branch", "s_endpgm", "s_setpc_b64") else [i + 1]
            if name.startswith(("s_branch", "s_cbranch")):
                follow.append(at[self.lines[0][0] + target])
            self.next.append([j for j in follow if j < len(self.lines)])
        self.code = [line[1:3] for line in self.lines]


def functions(containing, tmp_path):
    """{symbol: Function} of the code objects that hold a symbol with this in its name."""
    found = {}
    for path in files(containing, tmp_path):
        function = None
        for line in subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", path], capture_output=True, text=True, check=True).stdout.splitlines():
            start = re.match(r"^[0-9a-f]+ <(.+)>:", line)
            if start:
                function = found[start.group(1)] = Function()
                continue
            m = re.match(r"^\t(\S+)\s*(.*?)\s*// ([0-9A-F]+):", line)
            if m:
                target = re.search(r"<[^<>]+\+0x([0-9a-f]+)>$", line)
                function.lines.append((int(m.group(3), 16), m.group(1), m.group(2), int(target.group(1), 16) if target else 0))
    for f in found.values():
        f.link()
    return found
