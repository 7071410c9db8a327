"""The operators on a context's own nets (lcrc_posteriors_scored, lcrc_set_merger_fp8), and the operators' launches at the ends of
their ranges."""
from contextlib import closing

import numpy as np
import pytest

from phnrec_amd import modelgen
from tests import ops_ref as ref
from tests.test_gpu_ops import Linear, Scored, _activations, _close, _pack, _stream, _weights

pytestmark = pytest.mark.gpu

torch = ref.torch

EPS = ref.EPS["f32"]


@pytest.fixture(scope="module")
def capi():
    from phnrec_amd import capi
    capi.load()
    return capi


def _check_scored(ctx, mel, off, k, m, seed):
    rng = np.random.default_rng(seed)
    labels = rng.integers(-1, ctx.n_out, (mel.shape[0], m))
    s = ctx.posteriors_scored(mel, off, labels if m else None, k)
    logp, ent, ti, tl = ref.score(s["post"], labels, k, "probs")
    lp, en = ref.score_tolerance(s["post"], "probs")
    assert np.array_equal(s["top_index"], ti)
    _close(s["logp"], logp, lp[:, None])
    _close(s["top_logp"], tl, lp[:, None])
    _close(s["entropy"], ent, en)
    return s


@pytest.mark.parametrize("k,m", [(5, 1), (0, 0), (64, 3), (16, 0)])
def test_posteriors_scored(capi, tmp_path, k, m):
    """the posteriors are those of lcrc_posteriors_batch, the scores those of the posteriors; batches of other sizes in between"""
    d = str(tmp_path / "m")
    modelgen.write_model_dir(d, 15, 64, 138, seed=3)
    with closing(capi.Lcrc(d, 15)) as ctx:
        for lens in ([1], [40, 0, 7], [700], [3, 3]):
            off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
            mel = modelgen.synth_mel(int(off[-1]), 15, seed=len(lens))
            s = _check_scored(ctx, mel, off, k, m, k + m)
            assert np.array_equal(s["post"], ctx.posteriors_batch(mel, off))


def test_posteriors_scored_refuses(capi, tmp_path):
    d = str(tmp_path / "m")
    modelgen.write_model_dir(d, 15, 64, 138, seed=3)
    with closing(capi.Lcrc(d, 15)) as ctx:
        mel, off = modelgen.synth_mel(9, 15, seed=1), np.array([0, 9], np.int32)
        before = ctx.posteriors_batch(mel, off)
        for bad in (dict(k=65), dict(k=-1), dict(labels=np.zeros((9, 65)))):
            with pytest.raises(capi.LcrcError) as e:
                ctx.posteriors_scored(mel, off, **bad)
            assert e.value.code == capi.LCRC_E_ARG
        for bad_off in ([1, 9], [0, 9, 5]):
            with pytest.raises(capi.LcrcError):
                ctx.posteriors_scored(mel, np.array(bad_off, np.int32), k=1)
        ctx.configure_output(("log",))
        with pytest.raises(capi.LcrcError):
            ctx.posteriors_scored(mel, off, k=1)
        ctx.configure_output(())
        with pytest.raises(capi.LcrcError) as e:
            ctx.set_merger_fp8(True)                        # a shipped LCRC shape runs the fused kernels
        assert e.value.code == capi.LCRC_E_UNSUPPORTED
        assert np.array_equal(ctx.posteriors_batch(mel, off), before)
        assert np.array_equal(ctx.posteriors_scored(mel, off, k=1)["post"], before)


def _fexp(y):
    """FEXP (fexp.h:14-21) on arrays"""
    i = np.trunc(1048576.0 / np.log(2.0) * np.asarray(y, np.float64)).astype(np.int64)
    return ((i + 1072632447) << 32).view(np.float64)


def _held(x, dx):
    """what the 8-bit form of x stands for, and how far it may be from it when x itself is off by at most dx: rounding is
    monotonous, so the ends bound it -- unless the block's scale changes between them: then a step, 2^-3 of the value (and the
    smallest step of the larger scale)"""
    q, e = ref.held(x)
    lo, e_lo = ref.held(x - dx)
    hi, e_hi = ref.held(x + dx)
    same = ref.spread(((e == e_lo) & (e == e_hi)).astype(float) - 1, x.shape[1]) == 1          # 2^0 where it is the same
    s = ref.spread(np.maximum(np.maximum(e, e_lo), e_hi), x.shape[1])
    return q, np.where(same, np.maximum(np.abs(hi - q), np.abs(lo - q)), dx + np.abs(x) * 2.0 ** -3 + s * 2.0 ** -9)


@pytest.mark.parametrize("hidden,n_out,rows", [(50, 39, 1), (200, 48, 70), (300, 138, 401)])
def test_merger_in_8_bits(capi, tmp_path, hidden, n_out, rows):
    """1BT_DCT (one net on C0 / DCT features, here in 64 bits) with the merger's operands in 8 bits.  The features in 32 bits are off
    by at most 40 eps of the sums of their terms' sizes; what follows is bounded step by step: a held value moves by the steps
    that its error crosses, a hidden sum by its operands' errors and by 7 * 2^-13 sum |x w| (the 8-bit instructions), a sigmoid
    by a quarter of that, an output by the hidden values' errors and (n + 2) eps sum |h w|, a posterior by a factor
    exp(2 max |d output|) (FEXP is exact, its steps are 2^-20)."""
    nb, coefs = 15, 6
    d = str(tmp_path / "m")
    net = modelgen.write_traps_dir(d, "1BT_DCT", nb, hidden, n_out, seed=hidden, coefs=coefs)["merger"]
    mel = modelgen.synth_mel(rows, nb, seed=rows).astype(np.float32).reshape(rows, nb)
    off = np.array([0, rows], np.int32)
    with closing(capi.Lcrc(d, nb, system="1BT_DCT")) as ctx:
        full = ctx.posteriors_batch(mel, off)
        ctx.set_merger_fp8(True)
        got = ctx.posteriors_batch(mel, off)
        assert np.array_equal(got, ctx.posteriors_batch(mel, off))
        s = _check_scored(ctx, mel, off, 5, 1, rows)
        assert np.array_equal(s["post"], got)
        clone = ctx.clone() if hasattr(ctx, "clone") else None
        if clone is not None:
            assert np.array_equal(clone.posteriors_batch(mel, off), full)                       # a setting of the context
            clone.close()
        ctx.configure_output(("log",), big_endian=True)
        be = ctx.posteriors_batch(mel, off).view(">f4").astype(np.float64)
        ctx.configure_output(())
        ctx.set_merger_fp8(False)
        assert np.array_equal(ctx.posteriors_batch(mel, off), full)
    assert np.abs(got.sum(1) - 1).max() < n_out * 2 * EPS and not np.array_equal(got, full)
    with np.errstate(divide="ignore"):
        want = np.log(got.astype(np.float64))
    assert np.abs(be - want)[np.isfinite(want)].max() <= 4 * EPS * np.abs(want[np.isfinite(want)]).max()
    # the features
    at = np.clip(np.arange(rows)[:, None] + np.arange(-15, 16)[None], 0, rows - 1)
    t = mel.astype(np.float64)[at].transpose(0, 2, 1)                                          # [rows][bands][31]
    basis = np.stack([np.ones(31)] + [np.cos(np.pi * v / 31 * (np.arange(31) + 0.5)) for v in range(1, coefs)])
    f = np.sqrt(2 / 31) * (t @ basis.T).reshape(rows, -1)
    df = 40 * EPS * np.sqrt(2 / 31) * (np.abs(t) @ np.abs(basis).T).reshape(rows, -1) + EPS * np.abs(t).max() * 31
    mean, dev, w1, b1, w2, b2 = (np.asarray(net[n], np.float64) for n in ("mean", "dev", "w1", "b1", "w2", "b2"))
    x = (f - mean) * dev
    dx = df * np.abs(dev) + 4 * EPS * (np.abs(f) + np.abs(mean)) * np.abs(dev)
    xq, dxq = _held(x, dx)
    w1q, w2q = ref.held(w1)[0], ref.held(w2)[0]
    z = xq @ w1q.T + b1
    dz = dxq @ np.abs(w1q).T + (7 * 2.0 ** -13 + (x.shape[1] + 2) * EPS) * ((np.abs(xq) + dxq) @ np.abs(w1q).T + np.abs(b1))
    h = 1 / (1 + _fexp(-z))
    dh = np.maximum(np.abs(1 / (1 + _fexp(-(z + dz))) - h), np.abs(1 / (1 + _fexp(-(z - dz))) - h)) + 2.0 ** -19
    hq, dhq = _held(h, dh)
    y = hq @ w2q.T + b2
    dy = dhq @ np.abs(w2q).T + (hidden + 4) * EPS * ((hq + dhq) @ np.abs(w2q).T + np.abs(b2))
    e = _fexp(y - y.max(1, keepdims=True))
    p = e / e.sum(1, keepdims=True)
    tol = p * (np.exp(2 * dy.max(1, keepdims=True)) - 1 + 2.0 ** -18) + n_out * EPS
    assert (np.abs(got - p) <= tol).all(), np.abs(got - p).max()


def test_score_rows_further_apart_than_32_bits_reach(capi):
    cols, ld = 138, (1 << 30) + 5
    big = torch.empty(2 * ld + cols, dtype=torch.float32, device="cuda")
    rng = np.random.default_rng(4)
    a = rng.standard_normal((3, cols))
    for r in range(3):
        big[r * ld:r * ld + cols] = torch.from_numpy(a[r].astype(np.float32))
    exact = a.astype(np.float32).astype(np.float64)
    labels = rng.integers(0, cols, (3, 1))
    got = Scored(capi, big.view(1, -1), "f32", "logits", labels, 5, cols, ld=ld).run().get()
    want = ref.score(exact, labels, 5, "logits")
    lp, en = ref.score_tolerance(exact, "logits")
    assert np.array_equal(got[2], want[2])
    _close(got[0], want[0], lp[:, None])
    _close(got[1], want[1], en)


def test_score_more_rows_than_a_grid(capi):
    """rows of one class: certain, whatever the value"""
    rows = (1 << 26) + 1000
    x = torch.full((rows, 1), 3.0, dtype=torch.float16, device="cuda")
    ti = torch.full((rows + 8, 1), 7, dtype=torch.int32, device="cuda")
    ent = torch.full((rows + 8,), 7.0, device="cuda")
    capi.score(capi.ScoreArgs(x=x.data_ptr(), type=capi.T_F16, form=0, rows=rows, cols=1, ld=1, k=1, entropy=ent.data_ptr(),
                              top_index=ti.data_ptr()), stream=_stream())
    torch.cuda.synchronize()
    assert (ti[:rows] == 0).all() and (ti[rows:] == 7).all() and (ent[:rows] == 0).all() and (ent[rows:] == 7).all()


def test_linear_rows_further_apart_than_32_bits_reach(capi):
    rng = np.random.default_rng(6)
    n_in, n_out, ld = 300, 40, (1 << 31) + 3
    a = _activations(rng, 2, n_in).astype(np.float32)
    big = torch.empty(ld + n_in, dtype=torch.bfloat16, device="cuda")
    for r in range(2):
        big[r * ld:r * ld + n_in] = torch.from_numpy(a[r])
    w, _ = _weights(capi, rng, n_out, n_in)
    near = torch.from_numpy(a).to(torch.bfloat16).cuda()
    want = Linear(capi, near, "bf16", 2, n_in, n_out, w, None, "none", "f32").run().get()
    got = Linear(capi, big.view(1, -1), "bf16", 2, n_in, n_out, w, None, "none", "f32", ldx=ld).run().get()
    assert np.array_equal(got, want)


def test_two_graphs_replayed_side_by_side(capi):
    """each with a workspace of its own, on streams of their own, over the same input and weights"""
    rng = np.random.default_rng(8)
    rows, n_in, n_out, k = 90, 700, 20011, 20
    x = torch.from_numpy(_activations(rng, rows, n_in).astype(np.float32)).cuda()
    w, _ = _weights(capi, rng, n_out, n_in)
    labels = rng.integers(0, n_out, (rows, 1))
    runs = []
    for i in range(2):
        lin = Linear(capi, x, "f32", rows, n_in, n_out, w, None, "none", "f32", pad=0)
        sc = Scored(capi, lin.y, "f32", "logits", labels, k, n_out)
        lin.run()
        sc.run()
        want = (lin.get(),) + sc.get()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lin.run()
            sc.run()
        runs.append((lin, sc, want, graph, torch.cuda.Stream()))
    for _ in range(3):
        for lin, sc, _, _, _ in runs:
            lin.y[:rows] = 0
        torch.cuda.synchronize()
        for _, _, _, graph, stream in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for lin, sc, want, _, _ in runs:
            for a, b in zip(want, (lin.get(),) + sc.get()):
                assert np.array_equal(a, b)


@pytest.mark.parametrize("rows", [2, 20, 700])
def test_a_row_does_not_depend_on_its_neighbours(capi, rows):
    """the kernels differ by the number of rows only where the results' rounding allows it: scores are the same bits"""
    rng = np.random.default_rng(rows)
    for cols, k in ((138, 5), (1000, 20), (9000, 7)):
        a = rng.standard_normal((rows, cols)).astype(np.float32)
        labels = rng.integers(0, cols, (rows, 1))
        x = torch.from_numpy(a).cuda()
        one = Scored(capi, x[:1].clone(), "f32", "logits", labels[:1], k, cols).run().get()
        many = Scored(capi, x, "f32", "logits", labels, k, cols).run().get()
        assert np.array_equal(one[2], many[2][:1])
        if capi.score_workspace(1, cols, k) == 0:
            for p, q in zip(one, many):
                assert np.array_equal(p, q[:1])


@pytest.mark.parametrize("shape", ["rising", "falling", "equal", "clustered"])
@pytest.mark.parametrize("cols,k", [(1500, 64), (4000, 40), (70000, 64), (300000, 33)])
def test_score_rows_made_against_the_search(capi, cols, k, shape):
    """rows whose best classes lie together, with one thread or in one part, and rows of few distinct values"""
    c = np.arange(cols)
    rng = np.random.default_rng(cols)
    a = {"rising": c / cols, "falling": -c / cols, "equal": np.zeros(cols),
         "clustered": np.where((c // 4) % 64 == 5, 3.0, 0.0) + np.where(c % 2048 < 8, 1.0, 0.0) + rng.integers(0, 2, cols) * 0.5}[shape]
    x = torch.from_numpy(np.stack([a, -a]).astype(np.float32)).cuda()
    exact = x.double().cpu().numpy()
    labels = np.array([[0], [cols - 1]])
    got = Scored(capi, x, "f32", "logits", labels, k, cols).run().get()
    want = ref.score(exact, labels, k, "logits")
    assert np.array_equal(got[2], want[2])
    lp, en = ref.score_tolerance(exact, "logits")
    _close(got[3], want[3], lp[:, None])
    _close(got[1], want[1], en)


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("y_type", ["f32", "bf16", "e4m3"])
def test_a_block_whose_scale_is_no_number(capi, y_type, rows):
    """exponent byte 255 in one block of one row of W makes that output NaN, and no other"""
    rng = np.random.default_rng(9)
    n_in, n_out = 300, 70
    q = torch.from_numpy(rng.integers(1, 120, (n_out, n_in)).astype(np.uint8)).cuda()
    scales = np.full((n_out, 3), 120, np.uint8)
    scales[33, 1] = 255
    w = _pack(capi, q, "e4m3", n_out, n_in, n_in, torch.from_numpy(scales).cuda())
    x = torch.from_numpy(_activations(rng, rows, n_in).astype(np.float32)).cuda()
    got = Linear(capi, x, "f32", rows, n_in, n_out, w, None, "none", y_type).run().get()
    want = np.zeros((rows, n_out), bool)
    want[:, 33] = True
    assert np.array_equal(np.isnan(got), want)


@pytest.mark.parametrize("cols", [2, 300, 20000])
def test_posteriors_whose_sum_leaves_the_range(capi, cols):
    a = np.zeros((2, cols), np.float32)
    a[0, :2] = 3e38
    a[1, :2] = 1e38
    x = torch.from_numpy(a).cuda()
    logp, ent, ti, tl = Scored(capi, x, "f32", "probs", np.array([[0], [1]]), 2, cols).run().get()
    assert np.isnan(logp[0]).all() and np.isnan(ent[0]) and (ti[0] == -1).all() and np.isnan(tl[0]).all()
    assert abs(ent[1] - np.log(2)) < 1e-5 and ti[1].tolist() == [0, 1] and np.abs(tl[1] - np.log(0.5)).max() < 1e-4
