"""What the sources' inline assembly may not do.  No GPU."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_inline_assembly_writes_no_register_behind_the_compilers_back():
    """m0 goes in as an operand: the compiler reserves it, so it cannot be named as overwritten."""
    src = os.path.join(ROOT, "vae_amd", "csrc")
    for name in sorted(os.listdir(src)):
        if name.endswith((".h", ".hip")):
            for text in re.findall(r'asm(?: volatile)?\("((?:[^"\\]|\\.)*)"', open(os.path.join(src, name)).read()):
                assert not re.search(r"\bs_\w+\s+m0\b", text), (name, text)
