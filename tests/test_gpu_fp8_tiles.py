"""Every kernel of lcrc_fp8_linear at sizes that it makes (lcrc_debug_fp8_route), with rows, outputs and sums that end inside a tile."""
import numpy as np
import pytest

from tests import ops_ref as ref
from tests.test_gpu_ops import Linear, _activations, _pack, _strided, _weights
from tests.test_gpu_ops_context import _fexp, _held

pytestmark = pytest.mark.gpu

torch = ref.torch
EPS = ref.EPS["f32"]
EXACT = 4                                                    # of a route: sums in 32 bits throughout

# rows, n_in, n_out: the route of results in bf16 and of those that come from sums in 32 bits
SIZES = {(33, 700, 300): (0, 0), (1031, 300, 1999): (1, 1), (777, 1030, 2309): (1, 1), (2100, 1030, 4100): (2, 2), (4100, 1030, 8200): (3, 2),
         (9001, 129, 140): (1, 1), (513, 2049, 17000): (2, 2)}
IN_32_BITS = ("f32", "f16", "e4m3")


@pytest.fixture(scope="module")
def capi():
    from phnrec_amd import capi
    capi.load()
    return capi


def _route(capi, size, y_type):
    rows, n_in, n_out = size
    got = capi.load().lcrc_debug_fp8_route(rows, n_in, n_out, capi.TYPES[y_type])
    assert got == SIZES[size][y_type in IN_32_BITS] + (EXACT if y_type in IN_32_BITS else 0)


def _product(a, b):
    """a b^T in 64 bits, on the GPU"""
    return (torch.from_numpy(a).cuda() @ torch.from_numpy(np.ascontiguousarray(b.T)).cuda()).cpu().numpy()


def _whole_numbers(rng, rows, n_in, n_out):
    """Small whole numbers, and in each block of 128 two columns of 256 and -256 whose products of 2^16 cancel one another: all are
    held exactly (one scale, 4 significant bits), and sums in 32 bits are exact in any order (below 2^24).  What cuts small
    products off beside large ones (13 bits below the largest of eight) loses their last three bits."""
    x = rng.integers(-15, 16, (rows, n_in)).astype(np.float64)
    w = rng.integers(-7, 8, (n_out, n_in)).astype(np.float64)
    for k in range(0, n_in, 128):
        if k + 128 <= n_in:
            a = k + int(rng.integers(0, 64))
            x[:, a], x[:, a + 64] = 256, 256
            w[:, a] = 256 * rng.choice([-1, 1], n_out)
            w[:, a + 64] = -w[:, a]
    return x, w, rng.integers(-50, 51, n_out).astype(np.float64)


@pytest.mark.parametrize("y_type", ["f32", "f16", "e4m3", "bf16"])
@pytest.mark.parametrize("size", list(SIZES))
def test_products_of_whole_numbers(capi, size, y_type):
    rows, n_in, n_out = size
    if y_type == "e4m3" and rows * n_out > 9e6:
        rows = 2100                                          # (the same route; the reference form of so much takes its time)
        if (capi.load().lcrc_debug_fp8_route(rows, n_in, n_out, 3) & 3) != SIZES[size][1]:
            pytest.skip("another size has this route")
    else:
        _route(capi, size, y_type)
    rng = np.random.default_rng(rows + n_in)
    x, w, b = _whole_numbers(rng, rows, n_in, n_out)
    assert np.array_equal(ref.held(x[:50])[0], x[:50]) and np.array_equal(ref.held(w[:50])[0], w[:50])
    X, W = (torch.from_numpy(v.astype(np.float32)).cuda() for v in (x, w))
    got = Linear(capi, X, "f32", rows, n_in, n_out, _pack(capi, W, "f32", n_out, n_in), torch.from_numpy(b.astype(np.float32)).cuda(),
                 "none", y_type).run().get()
    want = _product(x, w) + b
    if y_type == "f32":
        assert np.array_equal(got, want)
    elif y_type == "f16":
        assert np.array_equal(got, want.astype(np.float16).astype(np.float64))
    elif y_type == "e4m3":
        assert np.array_equal(got, ref.held(want)[0])
    else:
        mag = _product(np.abs(x), np.abs(w))
        err = np.abs(got - want)
        tol = 7 * 2.0 ** -13 * mag                            # (the 8-bit instructions, test_gpu_ops._linear_tolerance)
        assert (err <= tol + (np.abs(want) + tol) * ref.EPS["bf16"]).all()


@pytest.mark.parametrize("act", ["none", "sigmoid", "fsigmoid"])
@pytest.mark.parametrize("x_type,y_type", [("bf16", "bf16"), ("f16", "f32"), ("f32", "e4m3"), ("e4m3", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("size", [s for s in SIZES if s[0] * s[2] < 2e7])
@pytest.mark.filterwarnings("ignore::RuntimeWarning")
def test_products_against_64_bits(capi, size, x_type, y_type, act):
    """activations and weights of every size of block; as test_gpu_ops holds it, but with sums in 32 bits behind results in 8 bits"""
    _route(capi, size, y_type)
    rows, n_in, n_out = size
    rng = np.random.default_rng(rows * 3 + n_out)
    a = _activations(rng, rows, n_in) * 2.0 ** rng.integers(-4, 3, (1, -(-n_in // 128))).repeat(128, 1)[:, :n_in]
    src = "f32" if x_type == "e4m3" else x_type
    x, exact = _strided(a, src, 0 if x_type == "e4m3" else 5)
    xq = ref.held(exact)[0]
    if x_type == "e4m3":
        x = _pack(capi, x, src, rows, n_in)
    w, wq = _weights(capi, rng, n_out, n_in)
    b = rng.standard_normal(n_out).astype(np.float32)
    got = Linear(capi, x, x_type, rows, n_in, n_out, w, torch.from_numpy(b).cuda(), act, y_type, ldx=0 if x_type == "e4m3" else None).run().get()
    v = _product(xq, wq) + b
    mag = _product(np.abs(xq), np.abs(wq)) + np.abs(b)
    dv = ((n_in + n_in // 128 + 2) * EPS + (7 * 2.0 ** -13 if y_type == "bf16" else 0.0)) * mag
    if act == "sigmoid":
        f, df = 1 / (1 + np.exp(-v)), dv / 4 + 4 * EPS
    elif act == "fsigmoid":                                   # monotonous, in steps of 2^-20 relative: its ends bound it
        f = 1 / (1 + _fexp(-v))
        df = np.maximum(np.abs(1 / (1 + _fexp(-(v + dv))) - f), np.abs(1 / (1 + _fexp(-(v - dv))) - f)) + 2.0 ** -19
    else:
        f, df = v, dv
    if y_type == "e4m3":
        f, tol = _held(f, df)
        tol = tol * (1 + 1e-12)
    else:
        tol = df + (np.abs(f) + df) * (ref.EPS[y_type] if y_type != "f32" else EPS)
    err = np.abs(got - f)
    bad = ~(err <= tol)
    if act == "fsigmoid":
        # FEXP is an exponential while 2^20 y / ln 2 + 1072632447 is the upper half of a positive normal double: |y| < 708.  Beyond
        # it the sum wraps, here as in the reference (lcrc_pipeline.h); not compared, nor what shares a scale with it.
        beyond = np.abs(v) + dv >= 708
        if y_type == "e4m3":
            pad = -beyond.shape[1] % 128
            block = np.pad(beyond, ((0, 0), (0, pad))).reshape(rows, -1, 128).any(2)
            beyond = block.repeat(128, 1)[:, :n_out]
        assert beyond.mean() < 0.2
        bad &= ~beyond
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:5], got[bad][:5], f[bad][:5], tol[bad][:5])


def test_the_sizes_reach_every_kernel(capi):
    seen = {capi.load().lcrc_debug_fp8_route(*size, capi.TYPES[y]) for size in SIZES for y in ("bf16", "f16", "f32")}
    assert seen == {0, 1, 2, 3, 4, 5, 6}
