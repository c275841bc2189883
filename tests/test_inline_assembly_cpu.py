"""The inline assembly of the device code names the registers that it changes."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_assembly_that_writes_m0_says_so():
    """m0 is where the compiler, too, keeps what some instructions take from there; a write that it does not know of would change that."""
    found = 0
    for path in glob.glob(os.path.join(ROOT, "paella_amd", "csrc", "**", "*"), recursive=True):
        if path.endswith((".h", ".hip", ".cpp")):
            for asm in re.findall(r"\basm\b[^;]*;", open(path, errors="replace").read()):
                if re.search(r"\bm0\s*,", asm):
                    found += 1
                    assert '"m0"' in asm.split(":")[-1], (path, asm)
    assert found
