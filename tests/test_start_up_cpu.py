"""A device's first HIP calls: the warm-up helper thread's and a context's creation take turns (a stand-in runtime, hip_stub.c,
notices a call that is inside the runtime while another thread loads a code object)."""
import os
import subprocess
import sys

import pytest

from phnrec_amd import modelgen
from tests.util import ROOT


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("stub") / "libstub.so")
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-w", "-o", so, os.path.join(ROOT, "tests", "hip_stub.c")], check=True)
    return so


RUN = """
import ctypes as C, sys, threading, time
stub = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
L = C.CDLL(sys.argv[2])
L.lcrc_create_system.argtypes = [C.POINTER(C.c_void_p), C.c_char_p, C.c_char_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int]
L.lcrc_clone.argtypes = [C.POINTER(C.c_void_p), C.c_void_p]
def value(name): return C.c_int.in_dll(stub, name).value
C.c_int.in_dll(stub, "stub_load_us").value = 150000
def make():
    c = C.c_void_p()
    assert L.lcrc_create_system(C.byref(c), sys.argv[3].encode(), sys.argv[4].encode(), 15, 31, 1, 0, 0) == 0
    return c
def warm_up():
    assert L.lcrc_device_warmup(0) == 0 and L.lcrc_device_preload(0, 3) == 0
base = make()
for wait in (0.0, 0.01, 0.05, 0.2):
    t = threading.Thread(target=warm_up)
    t.start()
    time.sleep(wait)
    make()
    other = C.c_void_p()
    assert L.lcrc_clone(C.byref(other), base) == 0
    t.join()
print("beside a load:", value("stub_beside_a_load"), "calls:", value("stub_calls"))
"""


@pytest.mark.parametrize("system", ["LCRC", "1BT_DCT"])
def test_a_context_is_not_created_beside_a_warm_up(stub, tmp_path, system):
    d = str(tmp_path / "m")
    if system == "LCRC":
        modelgen.write_model_dir(d, 15, 64, 138, seed=3)
    else:
        modelgen.write_traps_dir(d, system, 15, 64, 138, seed=3, coefs=6)
    lib = os.path.join(ROOT, "phnrec_amd", "lib", "libphnrec_lcrc.so")
    out = subprocess.check_output([sys.executable, "-c", RUN, stub, lib, d, system], text=True).split()
    assert out[:4] == ["beside", "a", "load:", "0"] and int(out[5]) > 20, out


def test_pinned_memory_is_allocated_and_never_registered():
    for name in ("libphnrec_lcrc.so", "libphnrec_lcrc_ops.so"):
        wanted = subprocess.check_output(["nm", "-D", "--undefined-only", os.path.join(ROOT, "phnrec_amd", "lib", name)], text=True)
        assert "hipLaunchKernel" in wanted and "hipHostRegister" not in wanted and "hipHostUnregister" not in wanted
