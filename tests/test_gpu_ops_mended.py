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
    else:
        nets = modelgen.write_traps_dir(d, system, nb, hidden, n_out, seed=hidden, coefs=6)
    for i, name in enumerate(sorted(n for n in nets if n.startswith("band"))):
        nets[name] = _few_terms("%s/weights/%s.nbin" % (d, name), nets[name], i)
    if system == "LCRC":
        return capi.Lcrc(d, nb, trap_len=21), nets
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


def _few_terms(path, net, seed):
    """a band net whose sums have one term each, weights that are powers of two and inputs as they come: what 32 bits compute of it
    is known to a few roundings"""
    from phnrec_amd import modelgen
    rng = np.random.default_rng(seed)
    net = {k: np.zeros_like(v) for k, v in net.items()}
    hid, n_in = net["w1"].shape
    out = net["w2"].shape[0]
    net["dev"] += 1
    net["w1"][np.arange(hid), rng.permutation(np.arange(hid) % n_in)] = rng.choice([-1, 1], hid) * 2.0 ** -rng.integers(3, 5, hid)
    net["w2"][np.arange(out), rng.permutation(np.arange(out) % hid)] = rng.choice([-1, 1], out) * 2.0 ** rng.integers(1, 3, out)
    modelgen.write_nbin(path, net)
    return net


def _net(net, x, dx, terms, hold):
    """the reference's net (Normalize, two layers, FEXP sigmoid) on x in 64 bits, x being off by at most dx: outputs before the
    softmax and how far a computation in 32 bits may be from them.  Sums of so many terms; FEXP and the sigmoid are monotonous, so
    the ends bound them.  hold: with operands in 8 bits, sums in 32"""
    from tests.test_gpu_ops_context import _fexp, _held
    mean, dev, w1, b1, w2, b2 = (np.asarray(net[n], np.float64) for n in ("mean", "dev", "w1", "b1", "w2", "b2"))
    v = (x - mean) * dev
    dv = dx * np.abs(dev) + 2 * EPS * (np.abs(x) + np.abs(mean)) * np.abs(dev) * (mean != 0)
    if hold:
        v, dv = _held(v, dv)
        w1, w2 = ref.held(w1)[0], ref.held(w2)[0]
    z = v @ w1.T + b1
    dz = dv @ np.abs(w1).T + (terms or v.shape[1] + 2) * EPS * ((np.abs(v) + dv) @ np.abs(w1).T + np.abs(b1))
    h = 1 / (1 + _fexp(-z))
    dh = np.maximum(np.abs(1 / (1 + _fexp(-(z + dz))) - h), np.abs(1 / (1 + _fexp(-(z - dz))) - h)) + 4 * EPS
    if hold:
        h, dh = _held(h, dh)
    y = h @ w2.T + b2
    return y, dh @ np.abs(w2).T + (terms or w2.shape[1] + 2) * EPS * ((h + dh) @ np.abs(w2).T + np.abs(b2))


def _softmax(y, dy):
    """posteriors with FEXP, and by what factor (minus 1) each may be off: FEXP rises by 1 / ln 2 of its argument at most, in steps of
    2^-20; a sum of n terms, a quotient"""
    from tests.test_gpu_ops_context import _fexp
    e = _fexp(y - y.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True), np.expm1(2 * 1.45 * dy.max(1, keepdims=True)) + 2 * 2.0 ** -20 + (y.shape[1] + 4) * EPS


def _merger_inputs(system, nets, mel, length):
    """the merger's input rows of 1BT, 3BT and LCRC, and how far 32 bits may be from them"""
    from phnrec_amd import modelgen
    rows, nb = mel.shape
    back = length - 1 - (length - 1) // 2
    at = np.clip(np.arange(rows)[:, None] - back + np.arange(length)[None], 0, rows - 1)
    t = mel.astype(np.float64)[at].transpose(0, 2, 1)                             # [rows][bands][length]
    cols, errs = [], []
    if system == "LCRC":
        half = (length - 1) // 2 + 1
        basis = np.stack([np.ones(half)] + [np.cos(np.pi * v / half * (np.arange(half) + 0.5)) for v in range(1, 11)])
        for i, win in enumerate(modelgen.half_windows(half)):
            win = np.array([float("%.7e" % v) for v in win], np.float32).astype(np.float64)
            part = (t[:, :, :half] if i == 0 else t[:, :, half - 1:]) * win
            f = (np.sqrt(2 / half) * (part @ basis.T)).reshape(rows, -1)
            # (window, basis value -- off by a rounding and by its argument's, 2^-22 --, product, half sums, scale)
            df = (half + 12) * EPS * (np.sqrt(2 / half) * np.abs(part).sum(2)).repeat(11, 1).reshape(rows, -1)
            p, rel = _softmax(*_net(nets["band%d" % i], f, df, 2, False))
            cols.append(np.log(p))
            errs.append(np.log1p(rel) + 4 * EPS * np.abs(np.log(p)))
    else:
        for b in range(nb - 2 if system == "3BT" else nb):
            p, rel = _softmax(*_net(nets["band%d" % b], t[:, b], np.zeros_like(t[:, b]), 2, False))
            cols.append(-np.log(p))
            errs.append(np.log1p(rel) + 4 * EPS * np.abs(np.log(p)))
    return np.concatenate(cols, 1), np.concatenate([np.broadcast_to(e, c.shape) for e, c in zip(errs, cols)], 1)


@pytest.mark.parametrize("rows", [1, 70, 401])
@pytest.mark.parametrize("system", ["1BT", "3BT", "LCRC"])
def test_merger_in_8_bits_behind_band_nets(capi, tmp_path, system, rows):
    """the whole chain in 64 bits, its bounds step by step (a held value moves by the steps that its error crosses); the f32 merger
    against the same chain without 8 bits, and the oracle's merger inputs against these"""
    from contextlib import closing
    from oracle import binding
    from phnrec_amd import modelgen
    ctx, nets = _other_system(tmp_path, capi, system)
    length = 21 if system == "LCRC" else 31
    mel = modelgen.synth_mel(rows, 15, seed=rows).astype(np.float32).reshape(rows, 15)
    off = np.array([0, rows], np.int32)
    with closing(ctx):
        full = ctx.posteriors_batch(mel, off)
        ctx.set_merger_fp8(True)
        got = ctx.posteriors_batch(mel, off)
        s = ctx.posteriors_scored(mel, off, None, 3)
        assert np.array_equal(s["post"], got)
        ctx.set_merger_fp8(False)
        assert np.array_equal(ctx.posteriors_batch(mel, off), full)
    g, dg = _merger_inputs(system, nets, mel, length)
    theirs = np.zeros(g.shape, np.float32)
    orc = binding.TrapsOracle(str(tmp_path / "m"), system, 15, trap_len=length)
    orc.L.orc_traps_posteriors_batch(orc.h, mel, off, 1, np.zeros(full.shape, np.float32), theirs.ctypes.data)
    assert (np.abs(theirs - g) <= dg).all()
    for have, hold in ((full, False), (got, True)):
        p, rel = _softmax(*_net(nets["merger"], g, dg, 0, hold))
        assert rows == 1 or np.median(rel) < 0.01      # (the bounds say something)
        assert (np.abs(have - p) <= p * rel + full.shape[1] * EPS).all(), (hold, np.abs(have - p).max(), rel.max())
    assert not np.array_equal(got, full)


@pytest.mark.parametrize("form", ["logits", "probs"])
@pytest.mark.parametrize("cols,k,type", [(9, 3, "f16"), (138, 5, "f32"), (300, 8, "bf16"), (138, 20, "f32"), (400, 64, "f16"), (3000, 16, "f16"),
                                         (3000, 5, "f32"), (20000, 64, "bf16"), (70000, 7, "f32"), (140000, 33, "f16")])
@pytest.mark.parametrize("blocks", [1, 3])
def test_rows_that_a_workgroup_takes_one_after_another(capi, cols, k, type, form, blocks):
    """few workgroups over many rows: every row as in a grid with a place for each, bit for bit, whatever the row in front of it was --
    ties, more candidates than fit, no class left, no number"""
    rows = 150 if cols < 1000 else 40 if cols < 50000 else 5
    rng = np.random.default_rng(cols + k)
    a = rng.standard_normal((rows, cols)) * 3
    a[1::7] = np.round(a[1::7])                              # ties
    a[2::7] = 1.0                                            # nothing but ties
    a[3::7] = -np.inf
    a[4::7, cols // 2] = np.nan
    a[5::7] = np.arange(cols) / cols
    if form == "probs":
        a = np.exp(np.where(np.isnan(a), 0, a)) * np.where(np.isnan(a), np.nan, 1)
        a[6::7, 0] = -1
    x, exact = _strided(a, type, 3)
    labels = rng.integers(-1, cols, (rows, 9))
    L = capi.load()
    want = Scored(capi, x, type, form, labels, k, cols).run().get()
    before = L.lcrc_debug_score_blocks(blocks)
    assert before == 1 << 22
    try:
        got = Scored(capi, x, type, form, labels, k, cols).run().get()
    finally:
        assert L.lcrc_debug_score_blocks(before) == blocks
    for g, w in zip(got, want):
        assert np.array_equal(g, w, equal_nan=True)
    w_logp, w_ent, w_ti, w_tl = ref.score(exact, labels, k, form)
    lp, en = ref.score_tolerance(np.where(np.isfinite(exact) | np.isneginf(exact), exact, 0.5) if form == "logits" else np.abs(np.nan_to_num(exact)), form)
    assert np.array_equal(got[2], w_ti)
    _close(got[0], w_logp, lp[:, None])
    _close(got[1], w_ent, en)
    assert L.lcrc_debug_score_blocks(0) == capi.LCRC_E_ARG


def test_more_short_rows_than_a_grid_has_lanes_for(capi):
    """beyond 2^27 rows a group of 8 lanes takes a second one"""
    base = 1 << 12
    rows = (1 << 27) + base
    rng = np.random.default_rng(2)
    some = torch.from_numpy(np.round(rng.standard_normal((base, 2)) * 2).astype(np.float16)).cuda()
    x = some.repeat(rows // base, 1)
    x[-1, 0] = float("nan")
    ti = torch.full((rows + 8, 2), 7, dtype=torch.int32, device="cuda")
    ent = torch.full((rows + 8,), 7.0, device="cuda")
    capi.score(capi.ScoreArgs(x=x.data_ptr(), type=capi.T_F16, form=0, rows=rows, cols=2, ld=2, k=2, entropy=ent.data_ptr(),
                              top_index=ti.data_ptr()), stream=_stream())
    torch.cuda.synchronize()
    assert (ti[rows:] == 7).all() and (ent[rows:] == 7).all()
    assert (ti[rows - 1] == -1).all() and torch.isnan(ent[rows - 1])
    for t in (ti[:rows], ent[:rows]):
        t[rows - 1] = t[base - 1]
        t = t.view(rows // base, base, -1)
        assert (t == t[0]).all()
    second = (some[:, 1] > some[:, 0]).int()
    assert (ti[:base, 0] == second).all() and (ti[:base, 1] == 1 - second).all()
    _close(ent[:base].cpu().numpy(), ref.score(some.double().cpu().numpy(), np.zeros((base, 0), int), 1, "logits")[1], 64 * EPS)


FIRST = """
import sys
import numpy as np, torch
from phnrec_amd import capi
capi.load()
rng = np.random.default_rng(1)
rows, n_in, n_out, k = 40, 300, 500, 5
f = dict(device="cuda")
x = torch.from_numpy(rng.standard_normal((rows, n_in)).astype(np.float32)).cuda()
w = torch.from_numpy(rng.standard_normal((n_out, n_in)).astype(np.float32)).cuda()
q = torch.zeros(capi.fp8_bytes(n_out, n_in), dtype=torch.uint8, **f)
y = torch.zeros(rows, n_out, **f)
ws = torch.zeros(max(capi.fp8_linear_workspace(rows, n_in, 0), 16), dtype=torch.uint8, **f)
ti, ent = torch.zeros(rows, k, dtype=torch.int32, **f), torch.zeros(rows, **f)
lin = capi.Fp8LinearArgs(x=x.data_ptr(), x_type=0, rows=rows, n_in=n_in, n_out=n_out, ldx=n_in, w=q.data_ptr(), act=0, y=y.data_ptr(), y_type=0,
                         ldy=n_out, workspace=ws.data_ptr(), workspace_bytes=ws.numel())
sc = capi.ScoreArgs(x=y.data_ptr(), type=0, form=0, rows=rows, cols=n_out, ld=n_out, k=k, entropy=ent.data_ptr(), top_index=ti.data_ptr())
def calls():
    s = torch.cuda.current_stream().cuda_stream
    capi.fp8_pack(w.data_ptr(), 0, n_out, n_in, n_in, q.data_ptr(), stream=s)
    capi.fp8_linear(lin, stream=s)
    capi.score(sc, stream=s)
assert "lcrc_ops" not in open("/proc/self/maps").read()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    calls()
assert "libphnrec_lcrc_ops.so" in open("/proc/self/maps").read()
for i in range(3):
    x.normal_(); w.normal_()
    for t in (q, y, ti, ent): t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in (q, y, ti, ent)]
    for t in (q, y, ti, ent): t.zero_()
    calls()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, (q, y, ti, ent))) and float(y.abs().sum()) > 0
print("same")
"""


def test_the_first_calls_of_a_process_may_be_captured(capi):
    """the kernels' object and their code are loaded inside the capture"""
    import subprocess
    import sys
    from tests.util import ROOT
    p = subprocess.run([sys.executable, "-c", FIRST], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert p.returncode == 0 and p.stdout.split()[-1] == "same", p.stderr[-2000:]
