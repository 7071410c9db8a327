"""Refusals and sizes of the operators on matrices in device memory (lcrc_score, lcrc_fp8_*): nothing here reaches a GPU."""
import ctypes as C

import numpy as np
import pytest

from phnrec_amd import capi
from tests import ops_ref as ref

P = 1 << 20                                            # an address that is aligned and never followed


def _score(**kw):
    a = dict(x=P, type=capi.T_F32, form=0, rows=4, cols=138, ld=138, labels=P, n_labels=1, k=5, logp=P, entropy=P, top_index=P,
             top_logp=P, workspace=P, workspace_bytes=1 << 30)
    a.update(kw)
    return capi.ScoreArgs(**a)


def _linear(**kw):
    a = dict(x=P, x_type=capi.T_F32, rows=4, n_in=276, n_out=1500, ldx=276, w=P, bias=P, act=0, y=P, y_type=capi.T_F32, ldy=1500,
             workspace=P, workspace_bytes=1 << 30)
    a.update(kw)
    return capi.Fp8LinearArgs(**a)


def _refused(fn, *args, code=capi.LCRC_E_ARG, **kw):
    with pytest.raises(capi.LcrcError) as e:
        fn(*args, **kw)
    assert e.value.code == code and len(str(e.value)) > 20
    return str(e.value)


@pytest.mark.parametrize("kw", [
    dict(type=3), dict(type=-1), dict(form=2), dict(rows=-1), dict(cols=0), dict(cols=(1 << 30) + 1, ld=1 << 31), dict(k=-1), dict(k=65),
    dict(cols=4, k=5), dict(n_labels=-1), dict(n_labels=65), dict(x=None), dict(x=P + 2), dict(type=1, x=P + 1), dict(ld=137), dict(ld=-1),
    dict(labels=None), dict(labels=P + 1), dict(logp=P + 2), dict(entropy=P + 1), dict(top_index=P + 3), dict(top_logp=P + 2)])
def test_score_refuses(kw):
    _refused(capi.score, _score(**kw))


@pytest.mark.parametrize("kw", [
    dict(x_type=4), dict(x_type=-1), dict(y_type=4), dict(act=3), dict(act=-1), dict(rows=-1), dict(n_in=0), dict(n_out=0), dict(x=None),
    dict(x=P + 2), dict(ldx=275), dict(w=None), dict(w=P + 8), dict(bias=P + 2), dict(y=None), dict(y=P + 1), dict(ldy=1499),
    dict(y_type=3, y=P + 8), dict(x_type=3, x=P + 8), dict(x_type=3, x=None), dict(workspace=None), dict(workspace=P + 8),
    dict(workspace_bytes=capi.load().lcrc_fp8_linear_workspace(4, 276, 0) - 1)])
def test_fp8_linear_refuses(kw):
    _refused(capi.fp8_linear, _linear(**kw))


def test_fp8_pack_and_unpack_refuse():
    _refused(capi.fp8_pack, P, 4, 4, 4, 4, P)
    _refused(capi.fp8_pack, P, 0, -1, 4, 4, P)
    _refused(capi.fp8_pack, P, 0, 4, 0, 4, P)
    _refused(capi.fp8_pack, P, 0, 4, 4, 3, P)
    _refused(capi.fp8_pack, None, 0, 4, 4, 4, P)
    _refused(capi.fp8_pack, P + 1, 1, 4, 4, 4, P)
    _refused(capi.fp8_pack, P, 0, 4, 4, 4, P + 4)
    _refused(capi.fp8_pack, P, 0, 4, 4, 4, None)
    _refused(capi.fp8_pack, P, 0, 4, 4, 4, P, scales=P)
    _refused(capi.fp8_pack, P, 3, 4, 4, 4, P)
    _refused(capi.fp8_unpack, P, 4, 4, P, 3, 4)
    _refused(capi.fp8_unpack, P + 8, 4, 4, P, 0, 4)
    _refused(capi.fp8_unpack, P, 4, 4, None, 0, 4)
    _refused(capi.fp8_unpack, P, 4, 4, P, 0, 3)
    _refused(capi.fp8_unpack, P, -4, 4, P, 0, 4)


def test_null_arguments():
    L = capi.load()
    assert L.lcrc_score(0, None, None) == capi.LCRC_E_ARG
    assert L.lcrc_fp8_linear(0, None, None) == capi.LCRC_E_ARG
    assert b"lcrc_fp8_linear" in L.lcrc_last_error(None)


def test_no_rows_is_no_call():
    capi.score(_score(rows=0, x=None, workspace=None))
    capi.fp8_linear(_linear(rows=0, x=None, y=None, w=None))
    capi.fp8_pack(None, 0, 0, 4, 4, None)
    capi.fp8_unpack(None, 0, 4, None, 0, 4)


def test_without_a_gpu_the_operators_fail_loudly():
    import torch
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    assert "no CPU path" in _refused(capi.score, _score(), code=capi.LCRC_E_DEVICE)
    _refused(capi.fp8_linear, _linear(), code=capi.LCRC_E_DEVICE)
    _refused(capi.fp8_pack, P, 0, 4, 4, 4, P, code=capi.LCRC_E_DEVICE)
    _refused(capi.fp8_unpack, P, 4, 4, P, 0, 4, code=capi.LCRC_E_DEVICE)


def test_sizes():
    assert capi.fp8_bytes(0, 5) == 0 and capi.fp8_bytes(5, 0) == 0 and capi.fp8_bytes(-1, 5) == 0
    assert capi.fp8_bytes(1, 1) == 2048 + 64
    assert capi.fp8_bytes(17, 513) == 2 * (5 * 2048 + 2 * 64)
    assert capi.fp8_bytes(1 << 20, 1 << 20) == (1 << 16) * ((1 << 13) * 2048 + (1 << 11) * 64)       # beyond 32 bits
    assert capi.fp8_linear_workspace(100, 276, capi.T_E4M3) == 0
    assert capi.fp8_linear_workspace(100, 276, capi.T_BF16) <= capi.fp8_bytes(100, 276)
    assert capi.score_workspace(0, 10, 1) == 0 and capi.score_workspace(8192, 138, 5) == 0


def test_structures_match_the_header(tmp_path):
    """field offsets of the ctypes structures against the C compiler's"""
    import os
    import subprocess
    from tests.util import ROOT
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"lcrc_pipeline.h\"\nint main(void) {\n"
    for cls, name in ((capi.ScoreArgs, "lcrc_score_args"), (capi.Fp8LinearArgs, "lcrc_fp8_linear_args")):
        src += "  printf(\"%%zu\\n\", sizeof(%s));\n" % name
        for f, _ in cls._fields_:
            src += "  printf(\"%%zu\\n\", offsetof(%s, %s));\n" % (name, f)
    (tmp_path / "s.c").write_text(src + "  return 0;\n}\n")
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    said = [int(v) for v in subprocess.check_output([str(tmp_path / "s")]).split()]
    want = []
    for cls in (capi.ScoreArgs, capi.Fp8LinearArgs):
        want += [C.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    assert said == want


def test_the_reference_form_rounds_to_the_nearest():
    """ops_ref.held against a search over all e4m3 values"""
    rng = np.random.default_rng(2)
    x = np.concatenate([rng.standard_normal(120) * 5, [0.0, -0.0, 448, 447.9, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10]])[None]
    q, e = ref.held(x)
    t = ref.e4m3_table()
    t = t[np.isfinite(t)] * 2.0 ** e[0, 0]
    assert np.array_equal(np.abs(x[0] - q[0]), np.abs(x[0][:, None] - t[None]).min(1))
    assert q[0, -4] == 16.0 and q[0, -3] == 20.0 and q[0, -2] == 0.0 and q[0, -1] == 2 * 2.0 ** -9     # ties to even
