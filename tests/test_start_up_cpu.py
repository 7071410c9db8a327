"""What the library and the command line do around the HIP runtime's start-up (on a stand-in runtime, hip_stub.c)."""
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


def test_pinned_memory_is_allocated_and_never_registered():
    for name in ("libphnrec_lcrc.so", "libphnrec_lcrc_ops.so"):
        wanted = subprocess.check_output(["nm", "-D", "--undefined-only", os.path.join(ROOT, "phnrec_amd", "lib", name)], text=True)
        assert "hipLaunchKernel" in wanted and "hipHostRegister" not in wanted and "hipHostUnregister" not in wanted
