"""The operators' kernels are an object of their own, which a process that uses none of them -- the command line -- never loads."""
import ctypes as C
import os
import subprocess
import sys

from phnrec_amd import capi
from tests.util import GOLD, ROOT, model_dir

OBJECT = os.path.join(ROOT, "phnrec_amd", "lib", "libphnrec_lcrc_ops.so")
KERNELS = (b"score_short_kernel", b"score_wave_kernel", b"score_long_kernel", b"score_join_kernel", b"fp8_pack_kernel", b"fp8_unpack_kernel",
           b"fp8_tile_kernel", b"fp8_split_kernel", b"softmax_rows_kernel")


def test_the_library_registers_none_of_the_operators_kernels():
    lib = open(capi.LIB_PATH, "rb").read()
    ops = open(OBJECT, "rb").read()
    for name in KERNELS:
        assert name not in lib and name in ops


def test_the_object_finds_what_it_needs():
    """all symbols bound at once, as the library loads it; the table is complete"""
    capi.load()
    table = C.CDLL(OBJECT, mode=os.RTLD_NOW).lcrc_ops_table
    table.restype = C.POINTER(C.c_void_p * 8)                # (version, seven launches)
    assert all(table().contents)


MOVED = """
import ctypes as C, os, sys
C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
os.chdir(sys.argv[2])
L = C.CDLL("./libphnrec_lcrc.so")
os.chdir("/")
L.lcrc_last_error.restype = C.c_char_p
print(L.lcrc_debug_score_blocks(1 << 22), L.lcrc_last_error(None).decode())
"""


def test_the_object_is_found_beside_the_library(tmp_path):
    """loaded by a relative path, from another folder afterwards; missing; of another build"""
    import shutil
    stub = str(tmp_path / "stub.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-w", "-o", stub, os.path.join(ROOT, "tests", "hip_stub.c"), "-lpthread"], check=True)

    def said(folder):
        return subprocess.check_output([sys.executable, "-c", MOVED, stub, folder], text=True)

    here = tmp_path / "lib"
    here.mkdir()
    shutil.copy(capi.LIB_PATH, str(here))
    assert said(str(here)).startswith("-4 cannot load the operators' kernels") and "libphnrec_lcrc_ops.so" in said(str(here))
    shutil.copy(OBJECT, str(here))
    assert said(str(here)).startswith("%d " % (1 << 22))
    (tmp_path / "o.c").write_text("static const long table[8] = {1}; const void *lcrc_ops_table(void) { return table; }")
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(here / "libphnrec_lcrc_ops.so"), str(tmp_path / "o.c")], check=True)
    assert "another build" in said(str(here))


def test_refusals_and_sizes_do_not_load_it():
    code = ("from phnrec_amd import capi\n"
            "capi.score_workspace(3, 200003, 64); capi.fp8_bytes(5, 5)\n"
            "try: capi.score(capi.ScoreArgs(rows=-1))\n"
            "except capi.LcrcError: pass\n"
            "print('lcrc_ops' in open('/proc/self/maps').read())\n")
    assert subprocess.check_output([sys.executable, "-c", code], cwd=ROOT, text=True).split()[-1] == "False"


def test_the_command_line_does_not_load_it(tmp_path):
    """a conversion that ends in front of the GPU"""
    p = subprocess.run([os.path.join(ROOT, "phnrec_amd", "bin", "phnrec"), "-c", model_dir("PHN_HU_SPDAT_LCRC_N1500"), "-i",
                        os.path.join(GOLD, "test.raw"), "-t", "par", "-o", str(tmp_path / "o")], env=dict(os.environ, LD_DEBUG="files"),
                       capture_output=True, text=True)
    assert p.returncode == 0 and "libphnrec_lcrc.so" in p.stderr and "lcrc_ops" not in p.stderr


def test_the_products_test_sizes_reach_every_kernel():
    """(a change of lcrc_fp8_linear's choice must not leave one of its kernels untested)"""
    from tests import test_gpu_fp8_tiles as tiles
    tiles.test_the_sizes_reach_every_kernel(capi)
    for size in tiles.SIZES:
        for y in ("bf16", "f32"):
            tiles._route(capi, size, y)


P = 1 << 20


def test_sizes_beyond_a_grid_are_refused():
    """a grid has fewer than 2^32 threads: 64 to a tile of 16 x 128, 256 to 64 x 128 results (nothing reaches a GPU here: the arguments
    are refused before one is asked for)"""
    import pytest

    def code(fn, *a, **k):
        with pytest.raises(capi.LcrcError) as e:
            fn(*a, **k)
        return e.value.code

    over, under = capi.LCRC_E_ARG, capi.LCRC_E_DEVICE         # (no GPU here: what passes the checks fails for that)
    import torch
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    assert code(capi.fp8_pack, P, capi.T_F32, 1 << 30, 128, 128, P) == over
    assert code(capi.fp8_pack, P, capi.T_F32, (1 << 30) - 16, 128, 128, P) == under
    assert code(capi.fp8_unpack, P, 1 << 30, 128, P, capi.T_F32, 128) == over
    assert code(capi.fp8_unpack, P, 1 << 30, 1, P, capi.T_F32, 128) == over
    assert code(capi.fp8_unpack, P, (1 << 30) - 16, 1, P, capi.T_F32, 128) == under

    def linear(rows, n_in, n_out):
        a = capi.Fp8LinearArgs(x=P, x_type=capi.T_E4M3, rows=rows, n_in=n_in, n_out=n_out, ldx=0, w=P, act=0, y=P, y_type=capi.T_BF16, ldy=n_out)
        return code(capi.fp8_linear, a)

    assert linear(1 << 30, 128, 128) == over and linear((1 << 30) - 1024, 128, 128) == under
    assert linear(129, 1, 128 * 7400000) == over              # 9 x 7.4 million tiles of 16 x 128, but 3 x 7.4 million of 64 x 128
    assert linear(129, 1, 128 * 5500000) == under


def test_posteriors_scored_checks_what_it_hands_over():
    """offsets that leave the features, labels that do not go by frames or would wrap, lists without an end: nothing reaches the library"""
    import numpy as np
    import pytest

    class Library:
        calls = []

        def lcrc_posteriors_scored(self, h, mel, off, n, post, labels, m, k, *out):
            self.calls.append(np.ctypeslib.as_array(C.cast(labels, C.POINTER(C.c_int)), (4 * m,)).tolist() if m else [])
            return 0

    ctx = capi.Lcrc.__new__(capi.Lcrc)
    ctx.L, ctx.h, ctx.nbanks, ctx.n_out = Library(), None, 15, 39
    mel = np.zeros((4, 15), np.float32)
    for bad in (dict(off=[0, 5]), dict(off=[0, 3]), dict(off=[]), dict(off=[[0, 4]]), dict(off=[0, 4], labels=[1, 2, 3])):
        with pytest.raises(capi.LcrcError) as e:
            ctx.posteriors_scored(mel, **bad)
        assert e.value.code == capi.LCRC_E_ARG
    for bad in (dict(k=65), dict(k=-1), dict(k=1 << 40), dict(labels=np.zeros((4, 65)))):
        with pytest.raises(capi.LcrcError) as e:
            ctx.posteriors_scored(mel, [0, 4], **bad)
        assert e.value.code == capi.LCRC_E_ARG
    with pytest.raises(capi.LcrcError):
        ctx.posteriors_scored(mel[:0], [0], labels=[1])
    assert Library.calls == []
    ctx.posteriors_scored(mel, [0, 4], labels=np.array([2 ** 32 + 1, -2 ** 40, 7, 2 ** 31 - 1]))
    ctx.posteriors_scored(mel[:0], [0], labels=np.zeros((0, 3)))
    assert Library.calls == [[2 ** 31 - 1, -1, 7, 2 ** 31 - 1], []]
    ctx.h = None


def test_no_kernel_has_packed_f32_instructions(tmp_path):
    """v_pk_add / _mul / _fma_f32, which the compiler makes of ordinary float code where nothing forbids it: some of their forms have
    given wrong results now and then"""
    import pytest
    llvm = "/opt/rocm/llvm/bin/"
    objects = [os.path.join(ROOT, "phnrec_amd", "lib", "obj", n + ".o")
               for n in ("lcrc_kernels", "traps_kernels", "phndec_kernels", "frontend_kernels", "score_kernels", "fp8_kernels", "softmax_kernels")]
    if not all(os.path.exists(p) for p in objects + [llvm + "llvm-objdump", llvm + "clang-offload-bundler"]):
        pytest.skip("no objects of a build, or no tools to look into them")
    for p in objects:
        fat, code = str(tmp_path / "fat"), str(tmp_path / "code")
        subprocess.run(["objcopy", "-O", "binary", "--only-section=.hip_fatbin", p, fat], check=True)
        subprocess.run([llvm + "clang-offload-bundler", "--unbundle", "--type=o", "--input=" + fat, "--output=" + code,
                        "--targets=hipv4-amdgcn-amd-amdhsa--gfx950"], check=True)
        text = subprocess.check_output([llvm + "llvm-objdump", "-d", code], text=True)
        assert text.count("\n") > 1000 and not [l for l in text.splitlines() if "v_pk_" in l and "_f32 " in l and "cvt" not in l][:3], p
