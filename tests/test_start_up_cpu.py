"""What the library and the command line do around the HIP runtime's start-up (on a stand-in runtime, hip_stub.c)."""
import os
import subprocess
import sys

import pytest

from tests.util import GOLD, ROOT, model_dir


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("stub") / "libamdhip64.so.7")
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-w", "-o", so, os.path.join(ROOT, "tests", "hip_stub.c"), "-lpthread"], check=True)
    return so


@pytest.mark.parametrize("args", [["-t", "post"], [], ["-t", "post", "-E"], ["-t", "post", "-H"], ["-F", "-D"], ["-l"], ["-l", "-E"],
                                  ["-l", "-g", "2"], ["-l", "-g", "4"], ["-l", "-F", "-D", "-g", "4"]])
def test_the_runtime_comes_up_while_there_is_one_thread(stub, tmp_path, args):
    """memory that another thread takes from the system meanwhile has been lost again before its first use"""
    raw = os.path.join(GOLD, "test.raw")
    if args[:1] == ["-l"]:
        (tmp_path / "l.scp").write_text("".join("%s %s\n" % (raw, tmp_path / ("%d.rec" % i)) for i in range(3)))
        args = ["-l", str(tmp_path / "l.scp")] + args[1:]
    else:
        args = ["-i", raw, "-o", str(tmp_path / "o")] + args
    env = dict(os.environ, STUB_START_UP="1", LD_LIBRARY_PATH=os.path.dirname(stub), PHNREC_DEVICE_MAP="0,0,0,0")
    p = subprocess.run([os.path.join(ROOT, "phnrec_amd", "bin", "phnrec"), "-c", model_dir("PHN_HU_SPDAT_LCRC_N1500")] + args, env=env,
                       capture_output=True, text=True)
    assert p.returncode == 0 and p.stderr.count("stub: ") == 1, p.stderr
    assert "stub: 1 thread(s) while the runtime comes up" in p.stderr


def test_pinned_memory_is_allocated_and_never_registered():
    for name in ("libphnrec_lcrc.so", "libphnrec_lcrc_ops.so"):
        wanted = subprocess.check_output(["nm", "-D", "--undefined-only", os.path.join(ROOT, "phnrec_amd", "lib", name)], text=True)
        assert "hipLaunchKernel" in wanted and "hipHostRegister" not in wanted and "hipHostUnregister" not in wanted


OUTSIDE = """
import ctypes as C, sys
C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
L = C.CDLL(sys.argv[2])
L.lcrc_stage_buffers.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_void_p]
c, a, b = C.c_void_p(), C.c_void_p(), C.c_void_p()
L.lcrc_debug_pinned_outside_rss.restype = C.c_longlong
assert L.lcrc_create(C.byref(c), sys.argv[3].encode(), 15, 31, 1, 0) == 0
before = L.lcrc_debug_pinned_outside_rss()
assert L.lcrc_stage_buffers(c, 100000, C.byref(a), C.byref(b)) == 0
untouched = L.lcrc_debug_pinned_outside_rss()
C.memmove(a, bytes(100000 * 15 * 4), 100000 * 15 * 4)
C.memmove(b, bytes(100000 * 4), 100000 * 4)
touched = L.lcrc_debug_pinned_outside_rss()
L.lcrc_destroy.argtypes = [C.c_void_p]
L.lcrc_destroy(c)
print(before, untouched, touched, L.lcrc_debug_pinned_outside_rss())
"""


def test_pinned_memory_that_the_resident_set_leaves_out(stub, tmp_path):
    """(memory that was never touched stands for memory that is not counted)"""
    from phnrec_amd import capi, modelgen
    modelgen.write_model_dir(str(tmp_path), 15, 64, 138, seed=3)
    out = subprocess.check_output([sys.executable, "-c", OUTSIDE, stub, capi.LIB_PATH, str(tmp_path)], text=True)
    before, untouched, touched, after = (int(v) for v in out.split())
    rows = 100000 * 15 * 4
    assert before < 1 << 20 and untouched >= rows * 0.9 and untouched - touched >= rows * 0.9 and after == 0, out
