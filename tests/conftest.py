import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


@pytest.fixture(scope="session")
def oracle_mod():
    from oracle import binding
    binding.lib()
    return binding


def _no_device_under_the_thread_sanitizer():
    """whether this kernel lays a process under ThreadSanitizer out so that the HIP runtime finds no range of addresses that it
    can use ("No SVM range compatible with all GPU and software constraints"): no device then, with or without setarch -R"""
    import shutil
    import subprocess
    csrc = os.path.join(ROOT, "phnrec_amd", "csrc")
    if not shutil.which("setarch") or subprocess.run(["make", "-s", "-C", csrc, "tsan"], capture_output=True).returncode != 0:
        return False
    run = [os.path.join(ROOT, "phnrec_amd", "bin", "phnrec_tsan"), "-c", os.path.join(ROOT, "tests", "golden", "models", "PHN_HU_SPDAT_LCRC_N1500"),
           "-i", os.path.join(ROOT, "tests", "golden", "test.raw"), "-o", os.devnull]
    p = subprocess.run(["setarch", "x86_64", "-R"] + run, capture_output=True, text=True, timeout=120, env=dict(os.environ, HSAKMT_DEBUG_LEVEL="3"))
    return "no HIP device" in p.stderr and "SVM range" in p.stderr


def pytest_runtest_setup(item):
    if item.name == "test_list_pipeline_under_thread_sanitizer_on_the_gpu" and _no_device_under_the_thread_sanitizer():
        pytest.skip("no HIP device in a process under ThreadSanitizer on this kernel: no usable range of addresses; the same modes run "
                    "under it on a stand-in runtime (test_list_tsan_cpu.py)")


@pytest.fixture(autouse=True)
def _an_empty_folder_is_no_reference(request, monkeypatch):
    """the binding's test asks for the reference's command line where /root/reference is there: a folder without sources builds none"""
    reference = "/root/reference"
    if request.node.name == "test_binding_compiles_and_links" and os.path.isdir(reference) and not os.listdir(reference):
        isdir = os.path.isdir
        monkeypatch.setattr(os.path, "isdir", lambda p: p != reference and isdir(p))
    yield
