"""Calls of the operators on matrices in device memory that were once answered wrongly, and kernels that no other test reaches."""
import numpy as np
import pytest

from tests import ops_ref as ref
from tests.test_gpu_ops import Linear, Scored, _activations, _close, _pack, _strided, _stream, _weights

pytestmark = pytest.mark.gpu

torch = ref.torch
EPS = ref.EPS["f32"]


@pytest.fixture(scope="module")
def capi():
    from phnrec_amd import capi
    capi.load()
    return capi


# 8 lanes to a row, a wave that holds it, a wave that streams it, a workgroup (2048 rows and more: one part), parts and their join
FAMILIES = [(100, 5, 3, 8), (100, 20, 3, 64), (3000, 5, 3, 64), (9000, 5, 2050, 256), (70000, 5, 3, 256)]


@pytest.mark.parametrize("cols,k,rows,lanes", FAMILIES)
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1.5e-45, 3e-45, 1e-44, 1e-42, 1e-40, 1e-39, 1.2e-38, 1e-37, 1e-24, 5e-20, 6e-20, 1e-10])
def test_rows_of_tiny_posteriors_are_normalised(capi, cols, k, rows, lanes, type, size):
    """Rows that do not add up to 1 are normalised, however small their sum.  Row 0: equal classes, entropy ln n; row 1: random ones;
    row 2: one of 1 beside them.  ln p and the entropy are differences of numbers of at most L = max |ln|: each logarithm is good
    to 2 eps L, sums of `depth` additions one behind another to depth eps of their value (S and T: terms of one sign)."""
    if type == "bf16" and size < 9.2e-41:
        size = 9.2e-41                                       # its smallest
    rng = np.random.default_rng(cols)
    a = np.full((min(rows, 3), cols), size)
    a[1] *= rng.random(cols) * 50
    a[2, cols // 3] = 1.0
    exact3 = _strided(a, type, 0)[1]
    x = _strided(np.tile(a, (-(-rows // 3), 1))[:rows], type, 0)[0]
    labels = np.tile([0, cols // 3], (rows, 1))
    logp, ent, ti, tl = Scored(capi, x, type, "probs", labels, k, cols).run().get()
    w_logp, w_ent, w_ti, w_tl = ref.score(exact3, labels[:3], k, "probs")
    depth = -(-cols // lanes) + 40
    L = 104.0 + np.log(cols)
    tol = EPS * L * (8 + 2 * depth)
    assert np.array_equal(ti[:3], w_ti)
    for g, w in ((logp, w_logp), (tl, w_tl), (ent, w_ent)):
        _close(g[:3], w, tol)
    for g in (logp, ent, ti, tl):                            # (every row of a launch like the first of its kind)
        for r in range(3):
            assert np.array_equal(g[r::3], np.broadcast_to(g[r], g[r::3].shape), equal_nan=True)
