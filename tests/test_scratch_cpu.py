"""The scratch memory of systems that are composed of several launches, and of the 8-bit merger (on a stand-in runtime,
hip_stub.c): allocated ahead by lcrc_reserve, never while a stream is captured, and kept while a graph may use it."""
import os
import subprocess
import sys

import pytest

from phnrec_amd import modelgen
from tests.util import ROOT


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("stub") / "libamdhip64.so.7")
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-w", "-o", so, os.path.join(ROOT, "tests", "hip_stub.c"), "-lpthread"], check=True)
    return so


RUN = """
import ctypes as C, sys
stub = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
L = C.CDLL(sys.argv[2])
vp = C.c_void_p
L.lcrc_create_system.argtypes = [C.POINTER(vp), C.c_char_p, C.c_char_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int]
L.lcrc_posteriors_device.argtypes = [vp, vp, vp, C.c_int, C.c_int, vp, vp]
L.lcrc_set_merger_fp8.argtypes = [vp, C.c_int]
L.lcrc_reserve.argtypes = [vp, C.c_int, C.c_int, C.c_longlong]
L.lcrc_last_error.argtypes = [vp]
L.lcrc_last_error.restype = C.c_char_p
L.lcrc_destroy.argtypes = [vp]
def value(name): return C.c_int.in_dll(stub, name).value
def capturing(on): C.c_int.in_dll(stub, "stub_capturing").value = on
system, length, fp8 = sys.argv[4], int(sys.argv[5]), int(sys.argv[6])
c = vp()
assert L.lcrc_create_system(C.byref(c), sys.argv[3].encode(), system.encode(), 15, length, 1, 0, 0) == 0, L.lcrc_last_error(None)
if fp8: assert L.lcrc_set_merger_fp8(c, 1) == 0, L.lcrc_last_error(c)
P, S = vp(1 << 20), vp(1 << 12)
def run(rows): return L.lcrc_posteriors_device(c, P, None, 1, rows, P, S)
calls = value("stub_launches")
capturing(1)
assert run(100) == -6 and b"lcrc_reserve" in L.lcrc_last_error(c), L.lcrc_last_error(c)
assert value("stub_launches") == calls, "something was launched"
capturing(0)
assert L.lcrc_reserve(c, 100, 1, 0) == 0
capturing(1)
before = value("stub_mallocs")
assert run(100) == 0 and run(40) == 0
assert value("stub_mallocs") == before, "allocated inside a capture"
assert run(5000) == -6
capturing(0)
frees = value("stub_frees")
assert run(5000) == 0 and run(50000) == 0
print("freed under a graph:", value("stub_frees") - frees)
L.lcrc_destroy(c)
print("left at the end:", value("stub_mallocs") - value("stub_frees"))
"""


@pytest.mark.parametrize("system,length,fp8", [("1BT_DCT", 31, 1), ("1BT", 31, 1), ("3BT", 31, 1), ("LCRC", 21, 1), ("1BT_DCT", 21, 0), ("1BT", 21, 0),
                                               ("LCRC", 21, 0)])
def test_scratch_of_a_captured_launch(stub, tmp_path, system, length, fp8):
    d = str(tmp_path / "m")
    if system == "LCRC":
        modelgen.write_model_dir(d, 15, 64, 138, seed=3, trap_len=length)
    else:
        modelgen.write_traps_dir(d, system, 15, 64, 138, seed=3, coefs=6, trap_len=length)
    lib = os.path.join(ROOT, "phnrec_amd", "lib", "libphnrec_lcrc.so")
    p = subprocess.run([sys.executable, "-c", RUN, stub, lib, d, system, str(length), str(fp8)], capture_output=True, text=True)
    assert p.returncode == 0, p.stderr
    assert "freed under a graph: 0\n" in p.stdout and "left at the end: 0\n" in p.stdout, p.stdout
