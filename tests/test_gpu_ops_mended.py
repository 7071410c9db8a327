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


def _other_system(tmp_path, capi, system, nb=15, n_out=48, hidden=200):
    """a context of a system that runs from memory, its nets in 64 bits"""
    from phnrec_amd import modelgen
    d = str(tmp_path / "m")
    if system == "LCRC":                                     # a geometry of its own: trajectories of 21 frames
        nets = modelgen.write_model_dir(d, nb, hidden, n_out, seed=hidden, trap_len=21)
        return capi.Lcrc(d, nb, trap_len=21), nets
    nets = modelgen.write_traps_dir(d, system, nb, hidden, n_out, seed=hidden, coefs=6)
    return capi.Lcrc(d, nb, system=system), nets


@pytest.mark.parametrize("system", ["1BT_DCT", "1BT", "3BT", "LCRC"])
def test_a_graph_of_the_8_bit_merger_and_larger_launches_behind_it(capi, tmp_path, system):
    """captured with the memory that lcrc_reserve got, replayed behind launches that needed more; without it the capture refuses"""
    from contextlib import closing
    from phnrec_amd import modelgen
    import ctypes as C
    ctx, _ = _other_system(tmp_path, capi, system)
    with closing(ctx):
        ctx.set_merger_fp8(True)
        ctx.L.lcrc_set_timing(ctx.h, 0)
        rows, more = 70, 9000
        mel = torch.from_numpy(modelgen.synth_mel(more, 15, seed=1).reshape(more, 15).astype(np.float32)).cuda()
        post, big = torch.zeros(rows, ctx.n_out, device="cuda"), torch.zeros(more, ctx.n_out, device="cuda")

        def launch(n, out, stream):
            return ctx.L.lcrc_posteriors_device(ctx.h, C.c_void_p(mel.data_ptr()), None, 1, n, C.c_void_p(out.data_ptr()), C.c_void_p(stream))

        assert launch(5, post, _stream()) == 0                # (the kernels' code is loaded)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s = torch.cuda.current_stream().cuda_stream
            assert launch(more, big, s) == capi.LCRC_E_UNSUPPORTED
            assert b"lcrc_reserve" in ctx.L.lcrc_last_error(ctx.h)
            big.add_(1.0)                                     # (a graph of something)
        ctx.L.lcrc_reserve(ctx.h, rows, 1, 0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            assert launch(rows, post, torch.cuda.current_stream().cuda_stream) == 0
        for i in range(3):
            mel.copy_(torch.from_numpy(modelgen.synth_mel(more, 15, seed=10 + i).reshape(more, 15).astype(np.float32)))
            assert launch(more - 1000 * (2 - i), big, _stream()) == 0          # grows its memory each time
            torch.cuda.synchronize()
            filler = [torch.full((1 << 20,), 7.0, device="cuda") for _ in range(8)]      # (lands where memory was given back)
            graph.replay()
            torch.cuda.synchronize()
            got = post.cpu().numpy().copy()
            assert launch(rows, post, _stream()) == 0
            torch.cuda.synchronize()
            assert np.array_equal(got, post.cpu().numpy()) and all((t == 7.0).all() for t in filler)
