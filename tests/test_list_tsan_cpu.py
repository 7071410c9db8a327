"""The list modes' host code under -fsanitize=thread (`make tsan`) on a stand-in HIP runtime (hip_stub.c: kernels do nothing, so every
posterior is 0): workers that build their contexts beside the running list, clones that wait for their base, contexts that are
left out, a launch that fails."""
import os
import shutil
import subprocess

import pytest

from tests.util import GOLD, ROOT, model_dir

HU = "PHN_HU_SPDAT_LCRC_N1500"


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("stub") / "libamdhip64.so.7")
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-w", "-o", so, os.path.join(ROOT, "tests", "hip_stub.c"), "-lpthread"], check=True)
    return so


@pytest.fixture(scope="module")
def tsan():
    csrc = os.path.join(ROOT, "phnrec_amd", "csrc")
    if subprocess.run(["make", "-s", "-C", csrc, "tsan"], capture_output=True, text=True).returncode != 0 or not shutil.which("setarch"):
        pytest.skip("no thread-sanitizer build / no setarch here")
    return os.path.join(ROOT, "phnrec_amd", "bin", "phnrec_tsan")


@pytest.mark.parametrize("gpus", [1, 4])
@pytest.mark.parametrize("flags", [[], ["-E"], ["-F"], ["-F", "-D"], ["-E", "-D"]])
@pytest.mark.parametrize("fault", [None, "4"])
def test_list_modes(stub, tsan, tmp_path, gpus, flags, fault):
    raw = open(os.path.join(GOLD, "test.raw"), "rb").read()
    names = []
    for i in range(90):                                  # (of many lengths: launches of a few files each)
        names.append(str(tmp_path / ("file_with_a_long_enough_name_for_a_long_list_%03d.raw" % i)))
        open(names[-1], "wb").write(raw[:4000 + 2 * (i * 977 % 9000)])
    lst = tmp_path / "l.scp"
    lst.write_text("\n".join(names) + "\n")
    env = dict(os.environ, LD_LIBRARY_PATH=os.path.dirname(stub), PHNREC_DEVICE_MAP="0,0,0,0",
               TSAN_OPTIONS="halt_on_error=0 exitcode=66 report_thread_leaks=0")
    if fault:
        env.update(LCRC_FAULT_INJECTION="1", PHNREC_FAIL_LAUNCH_NTH=fault)
    p = subprocess.run(["setarch", "x86_64", "-R", tsan, "-c", model_dir(HU), "-l", str(lst), "-m", str(tmp_path / "o.mlf"), "-g", str(gpus),
                        "-b", "600"] + flags, capture_output=True, text=True, env=env, timeout=200)
    if "unexpected memory mapping" in p.stderr:
        pytest.skip("the sanitizer does not start on this kernel")
    assert "WARNING: ThreadSanitizer" not in p.stderr, p.stderr[:4000]
    entries = (tmp_path / "o.mlf").read_text().count("\n.\n")
    if fault:
        assert p.returncode not in (0, 66) and p.returncode > 0 and "injected launch failure" in p.stderr and entries < 90
    else:
        assert p.returncode == 0 and entries == 90, (p.returncode, p.stderr)
