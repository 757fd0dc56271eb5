"""The library's own device code, disassembled: what the sources rely on the compiler not to do.  No GPU."""
import os
import re
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TOOLS = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")
SHIFT64 = re.compile(r"\bv_(?:lshlrev_b64|lshrrev_b64|ashrrev_i64)(?:_e64)?\s+v\[\d+:\d+\],\s*v(\d+),")


def _code_objects(path):
    """The gfx950 code objects of a library: offload bundles are a magic, a count, and (offset, size, name) entries."""
    data, magic, out = open(path, "rb").read(), b"__CLANG_OFFLOAD_BUNDLE__", []
    at = data.find(magic)
    while at >= 0:
        n, = struct.unpack_from("<Q", data, at + 24)
        p = at + 32
        for _ in range(n):
            off, size, length = struct.unpack_from("<QQQ", data, p)
            name = data[p + 24:p + 24 + length].decode()
            p += 24 + length
            if "gfx950" in name and size:
                out.append(data[at + off:at + off + size])
        at = data.find(magic, at + 1)
    return out


def _kernels(obj):
    """(name, registers) of a code object's kernels: all vector registers, and those before the accumulation registers."""
    notes = subprocess.run([os.path.join(TOOLS, "llvm-readelf"), "--notes", obj], check=True, capture_output=True, text=True).stdout
    out = {}
    for part in notes.split("  - .agpr_count:")[1:]:
        agprs = int(part.split(None, 1)[0])
        name, total = (re.search(key + r":\s+(\S+)", part).group(1) for key in (r"\.symbol", r"\.vgpr_count"))
        out[name[:-3] if name.endswith(".kd") else name] = (int(total), int(total) - agprs)
    return out


def _last_register_shifts(text, kernels):
    bad, name = [], None
    for line in text.splitlines():
        if line.endswith(">:"):
            name = line[line.index("<") + 1:-2]
            continue
        m = SHIFT64.search(line)
        if m and name in kernels and int(m.group(1)) in [-(-n // 8) * 8 - 1 for n in kernels[name]]:  # (registers come in eights)
            bad.append((name, line.strip()))
    return bad


@pytest.mark.skipif(not os.path.exists(os.path.join(TOOLS, "llvm-objdump")), reason="no llvm-objdump")
def test_no_64_bit_shift_by_a_kernels_last_register(tmp_path):
    """Such a shift has taken a wrong amount on this hardware, in some waves of some runs."""
    from vae_amd import _lib as L
    L.lib()
    objects, seen = _code_objects(L.LIB_PATH), 0
    assert objects
    for i, code in enumerate(objects):
        path = str(tmp_path / f"{i}.o")
        with open(path, "wb") as f:
            f.write(code)
        kernels = _kernels(path)
        seen += len(kernels)
        text = subprocess.run([os.path.join(TOOLS, "llvm-objdump"), "-d", "--no-show-raw-insn", path], check=True, capture_output=True, text=True).stdout
        assert not _last_register_shifts(text, kernels)
    assert seen > 100


def test_the_check_sees_such_a_shift():
    text = "0000 <k>:\n\tv_lshrrev_b64 v[4:5], v31, v[2:3]\n\tv_lshrrev_b64 v[4:5], v30, v[2:3]\n\tv_lshlrev_b64 v[4:5], 3, v[2:3]\n"
    assert len(_last_register_shifts(text, {"k": (32, 32)})) == 1
    assert len(_last_register_shifts(text, {"k": (29, 29)})) == 1
    assert not _last_register_shifts(text, {"k": (40, 40)})
    assert len(_last_register_shifts(text, {"k": (64, 32)})) == 1


def test_inline_assembly_writes_no_register_behind_the_compilers_back():
    """m0 goes in as an operand: the compiler reserves it, so it cannot be named as overwritten."""
    src = os.path.join(ROOT, "vae_amd", "csrc")
    for name in sorted(os.listdir(src)):
        if name.endswith((".h", ".hip")):
            for text in re.findall(r'asm(?: volatile)?\("((?:[^"\\]|\\.)*)"', open(os.path.join(src, name)).read()):
                assert not re.search(r"\bs_\w+\s+m0\b", text), (name, text)
