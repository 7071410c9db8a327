"""What the library and the command line do around the HIP runtime's start-up (on a stand-in runtime, hip_stub.c)."""
import os
import subprocess

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
