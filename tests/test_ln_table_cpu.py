"""The 16 intervals of ln() (host/veclog.cpp, frontend_kernels.hip) computed from what they are."""
import os
import re
from decimal import Decimal, getcontext

import numpy as np
import pytest

from tests.util import ROOT


def _array(path, name):
    text = open(os.path.join(ROOT, "phnrec_amd", "csrc", path)).read()
    if name == "A0":
        return [float.fromhex(re.search(r"A%d = (-?0x[0-9a-fp.+-]+)" % i, text).group(1)) for i in range(3)]
    body = re.search(r"%s\[\d+\]\s*=\s*\{(.*?)\}" % name, text, re.S).group(1)
    return [float.fromhex(v.strip()) for v in body.split(",")]


@pytest.mark.parametrize("path,names", [("host/veclog.cpp", ("kInvC", "kLogC", "kA")), ("frontend_kernels.hip", ("kLnInvC", "kLnLogC", "A0"))])
def test_table(path, names):
    getcontext().prec = 60
    inv, log, poly = (_array(path, n) for n in names)
    off = 0x3f330000                                         # the first interval's first value, in bits of an f32; 2^19 of them each
    edge = np.array([off + (k << 19) for k in range(17)], np.uint32).view(np.float32).astype(np.float64)
    for k in range(16):
        lo, hi = edge[k], edge[k + 1]
        c = 1 / inv[k]
        assert lo < c < hi
        if k == 9:
            assert inv[k] == 1.0 and lo < 1.0 < hi
        elif k != 10:
            middle = (lo + hi) / 2 - (2.0 ** -25 if hi <= 1 else 2.0 ** -24)
            assert inv[k] == 1 / middle
        assert log[k] == float(-Decimal(inv[k]).ln())        # rounded to the nearest
    # ln(1 + r) = r + A2 r^2 + A1 r^3 + A0 r^4 over the intervals: no worse than the series cut off there, r^5 / 5
    r = np.linspace(-0.0316, 0.0316, 4001)
    err = r + r ** 2 * (poly[2] + r * (poly[1] + r * poly[0])) - np.log1p(r)
    assert np.abs(err).max() < 0.0316 ** 5 / 5
