"""How the command line leaves: at once after its outputs are closed, or by the ordinary return where a preloaded tool may live
on exit handlers.  A tool that is not there -- a variable that is set but empty -- does not count."""
import os
import subprocess

import pytest

from tests.util import GOLD, ROOT, model_dir

BIN = os.path.join(ROOT, "phnrec_amd", "bin", "phnrec")


@pytest.mark.parametrize("name,value,ordinary", [(None, None, False), ("LD_PRELOAD", "", False), ("ROCP_TOOL_LIBRARIES", "", False),
                                                 ("HSA_TOOLS_LIB", "", False), ("PHNREC_CLEAN_EXIT", "", False),
                                                 ("LD_PRELOAD", "libm.so.6", True), ("PHNREC_CLEAN_EXIT", "1", True)])
def test_ordinary_exit_only_for_a_tool_that_is_named(tmp_path, name, value, ordinary):
    if os.environ.get("LD_PRELOAD"):
        pytest.skip("something is preloaded here")
    env = {k: v for k, v in os.environ.items() if k not in ("LD_PRELOAD", "ROCP_TOOL_LIBRARIES", "HSA_TOOLS_LIB", "PHNREC_CLEAN_EXIT")}
    if name:
        env[name] = value
    # the loader reports the end of every object, unless the process leaves without exit handlers
    p = subprocess.run([BIN, "-c", model_dir("PHN_HU_SPDAT_LCRC_N1500"), "-i", os.path.join(GOLD, "test.raw"), "-t", "par", "-o",
                        str(tmp_path / "o")], env=dict(env, LD_DEBUG="files"), capture_output=True, text=True)
    assert p.returncode == 0 and ("calling fini" in p.stderr) == ordinary


def test_a_crash_names_its_place(tmp_path):
    """the signal ends the process as before, behind the objects and offsets it ended in"""
    import signal
    import time
    fifo = str(tmp_path / "in.raw")
    os.mkfifo(fifo)                                          # (a file that never opens: the process waits)
    p = subprocess.Popen([BIN, "-c", model_dir("PHN_HU_SPDAT_LCRC_N1500"), "-i", fifo, "-t", "par", "-o", str(tmp_path / "o")],
                         stderr=subprocess.PIPE, text=True)
    time.sleep(0.5)
    p.send_signal(signal.SIGSEGV)
    err = p.communicate(timeout=60)[1]
    assert p.returncode == -signal.SIGSEGV and "ended by a signal" in err and "phnrec" in err.split("at\n", 1)[1], (p.returncode, err)
