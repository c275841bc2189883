"""What the kernels write goes through to memory (sc1): a direct queue's packets release nothing, so a line that stayed in one XCD's cache would leave it at any time later, over what others have written there
since.  By the assembly of the code objects that the library was built with."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "paella_amd", "lib", "libpaella_ops.so")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
OBJECTS = ["long_cache", "long_f32", "long_bf16", "long_f16", "decode", "attention_f32", "attention_bf16", "attention_f16"]


def output(*cmd):
    return subprocess.run(cmd, capture_output=True, text=True, check=True).stdout


def code_object(name):
    """The bytes of a code object that the library holds for direct queues."""
    symbols = {n: int(a, 16) for a, n in re.findall(r"^([0-9a-f]+) \w (paella_hsaco_\w+)$", output("nm", "-D", "--defined-only", LIB), flags=re.M)}
    begin, end = (symbols["paella_hsaco_%s_%s" % (name, which)] for which in ("begin", "end"))
    for offset, address, size in re.findall(r"^\s*LOAD\s+0x(\w+) 0x(\w+) 0x\w+ 0x(\w+)", output("readelf", "-lW", LIB), flags=re.M):
        offset, address, size = (int(x, 16) for x in (offset, address, size))
        if address <= begin and end <= address + size:
            with open(LIB, "rb") as f:
                f.seek(offset + begin - address)
                return f.read(end - begin)
    raise AssertionError(name)


@pytest.mark.parametrize("name", OBJECTS)
def test_every_store_goes_through(name, tmp_path):
    path = tmp_path / (name + ".hsaco")
    path.write_bytes(code_object(name))
    kernel, stores, kept = None, 0, []
    for line in output(OBJDUMP, "-d", str(path)).splitlines():
        label = re.match(r"[0-9a-f]+ <(.*)>:", line)
        kernel = label.group(1) if label else kernel
        if re.search(r"\b(global|buffer|flat|scratch)_store_", line):
            stores += 1
            if "sc1" not in line:
                kept.append((kernel, line.split("//")[0].strip()))
    assert stores > 10 and kept == []
