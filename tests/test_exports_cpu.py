"""What libpaella_ops.so shows to the programs that load it."""
import os
import re
import subprocess

from test_abi_cpu import ROOT


def exported():
    lib = os.path.join(ROOT, "paella_amd", "lib", "libpaella_ops.so")
    lines = subprocess.run(["nm", "-D", "--defined-only", lib], capture_output=True, text=True, check=True).stdout.splitlines()
    return [line.split()[-1] for line in lines]


def test_kernels_stay_inside():
    """A handle that a program's kernel of the same name takes the place of would have the library launch that one."""
    names = exported()
    hidden = re.compile(r"_kernelI|__device_stub__|^_ZN6paella\d+(attention_kernel|attention_join|page_attention|key_sums|key_weights|stored_weights)_?")
    assert [n for n in names if hidden.search(n)] == []


def test_the_interface_is_shown():
    """Every function that a header declares and this library has, and what the other libraries here take from it."""
    from paella_amd import _abi, _abi_decode, _abi_long, _abi_models
    names = set(exported())
    for table in (_abi.OPS_SYMBOLS, _abi.RING_SYMBOLS, _abi_models.MODEL_SYMBOLS, _abi_decode.DECODE_SYMBOLS, _abi_long.LONG_SYMBOLS):
        assert set(table) <= names
    for other in ("libpaella_serve.so", "libpaella_probes.so", "libjob_tvm_mnist.so"):
        lib = os.path.join(ROOT, "paella_amd", "lib", other)
        wanted = subprocess.run(["nm", "-D", "-u", lib], capture_output=True, text=True, check=True).stdout.split()
        assert {n for n in wanted if re.match(r"paella_|_ZN6paella", n)} <= names
