"""The operators on matrices in device memory (lcrc_score, lcrc_fp8_*) against plain 64-bit implementations (ops_ref.py)."""
import numpy as np
import pytest

from tests import ops_ref as ref

pytestmark = pytest.mark.gpu

torch, DT = ref.torch, ref.DT


@pytest.fixture(scope="module")
def capi():
    from phnrec_amd import capi
    capi.load()
    return capi


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _strided(a, dtype, pad, fill=float("nan")):
    """rows of a, `pad` elements of `fill` between them, on the GPU; the values as the type holds them, in 64 bits"""
    t = torch.full((a.shape[0], a.shape[1] + pad), fill, dtype=DT[dtype])
    t[:, :a.shape[1]] = torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(DT[dtype])
    return t.cuda(), t[:, :a.shape[1]].double().numpy()


class Scored:
    """one call with guard values behind every output"""

    def __init__(self, capi, x, type, form, labels, k, cols, ld=None, stream=None):
        rows, m = labels.shape
        self.capi, self.rows, self.m, self.k = capi, rows, m, k
        self.x, self.labels = x, torch.from_numpy(np.ascontiguousarray(labels, np.int32)).cuda()
        self.logp = torch.full((rows * m + 64,), 77.0, device="cuda")
        self.ent = torch.full((rows + 64,), 77.0, device="cuda")
        self.ti = torch.full((rows * k + 64,), 77, dtype=torch.int32, device="cuda")
        self.tl = torch.full((rows * k + 64,), 77.0, device="cuda")
        size = capi.score_workspace(rows, cols, k)
        self.ws = torch.full((size + 64,), 171, dtype=torch.uint8, device="cuda")
        self.args = capi.ScoreArgs(x=x.data_ptr(), type=capi.TYPES[type], form=capi.SCORE_FORMS[form], rows=rows, cols=cols,
                                   ld=ld or x.stride(0), labels=self.labels.data_ptr(), n_labels=m, k=k, logp=self.logp.data_ptr(),
                                   entropy=self.ent.data_ptr(), top_index=self.ti.data_ptr(), top_logp=self.tl.data_ptr(),
                                   workspace=self.ws.data_ptr() if size else None, workspace_bytes=size)
        self.size = size

    def run(self, stream=None):
        self.capi.score(self.args, stream=_stream() if stream is None else stream)
        return self

    def get(self):
        torch.cuda.synchronize()
        r, m, k = self.rows, self.m, self.k
        for t, n in ((self.logp, r * m), (self.ent, r), (self.ti, r * k), (self.tl, r * k)):
            assert (t[n:] == 77).all(), "written behind the last row"
        assert (self.ws[self.size:] == 171).all(), "written behind the workspace"
        return (self.logp[:r * m].view(r, m).cpu().numpy(), self.ent[:r].cpu().numpy(),
                self.ti[:r * k].view(r, k).cpu().numpy(), self.tl[:r * k].view(r, k).cpu().numpy())


def _close(got, want, tol):
    got = got.astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    ok = np.isfinite(want)
    err = np.abs(got - want)
    bad = ok & ~(err <= np.broadcast_to(tol, want.shape))
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], np.broadcast_to(tol, want.shape)[bad][:5])


def _check_scores(capi, a, type, form, labels, k, pad=0):
    x, exact = _strided(a, type, pad)
    logp, ent, ti, tl = Scored(capi, x, type, form, labels, k, a.shape[1]).run().get()
    w_logp, w_ent, w_ti, w_tl = ref.score(exact, labels, k, form)
    lp, en = ref.score_tolerance(exact, form)
    assert np.array_equal(ti, w_ti)
    _close(logp, w_logp, lp[:, None])
    _close(tl, w_tl, lp[:, None])
    _close(ent, w_ent, en)
    return logp, ent, ti, tl


def _scores(rng, rows, cols, form, spread=3.0):
    a = rng.standard_normal((rows, cols)) * spread
    if form == "probs":
        a = np.exp(a - a.max(1, keepdims=True))
        a /= a.sum(1, keepdims=True)
    return a


@pytest.mark.parametrize("form", ["probs", "logits"])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,k,m,pad", [
    (1, 1, 1, 1, 0), (1, 2, 2, 1, 3), (3, 5, 5, 2, 0), (7, 63, 3, 1, 1), (2, 64, 64, 4, 0), (9, 65, 1, 0, 0), (33, 120, 5, 1, 0),
    (257, 138, 5, 1, 0), (100, 138, 5, 1, 5), (65, 186, 3, 1, 0), (31, 159, 0, 1, 0), (5, 255, 8, 3, 1), (5, 256, 64, 1, 0),
    (5, 257, 10, 1, 0), (4, 511, 20, 1, 0), (4, 512, 33, 2, 8), (3, 1023, 7, 64, 0), (3, 1025, 2, 1, 0), (2, 2049, 31, 1, 7),
    (2, 4096, 16, 1, 0), (2, 8191, 5, 1, 1), (1, 8193, 64, 1, 0), (3, 20011, 16, 4, 2), (1, 50001, 32, 1, 0), (2, 131073, 64, 2, 0),
])
def test_score_against_64_bits(capi, rows, cols, k, m, pad, type, form):
    rng = np.random.default_rng(rows * 1000003 + cols * 31 + k)
    labels = rng.integers(-1, cols, (rows, m))
    _check_scores(capi, _scores(rng, rows, cols, form), type, form, labels, k, pad)


@pytest.mark.parametrize("form", ["probs", "logits"])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("chunks", [1, 8, 16, 24, 32, 48, 64])
def test_score_on_both_sides_of_a_rows_borders(capi, chunks, type, form):
    """rows that end just before, at and just behind so many 16-byte chunks; more labels than lanes, a row more than a workgroup's"""
    width = 4 if type == "f32" else 8
    for cols in (chunks * width - 1, chunks * width, chunks * width + 1):
        rng = np.random.default_rng(cols)
        for k in (1, 2, 3, 5, 8):
            if k <= cols:
                _check_scores(capi, _scores(rng, 33, cols, form), type, form, rng.integers(-1, cols, (33, 19)), k, pad=k % 3)


@pytest.mark.parametrize("cols", [3, 64, 138, 300, 1500, 5000, 40000])
def test_score_ties_go_to_the_lowest_index(capi, cols):
    k = min(64, cols)
    rng = np.random.default_rng(cols)
    a = rng.integers(0, 3, (6, cols)).astype(np.float64)
    a[0] = 1.0                                                   # all equal
    a[1] = np.where(rng.random(cols) < 0.5, 0.0, -0.0)           # zeros of both signs are equal
    a[2] = np.arange(cols)[::-1] // 7                            # falling
    a[3] = np.arange(cols) // 7                                  # rising
    a[4] = -np.inf
    a[4, cols // 2] = 1.0                                        # one class left: the rest follow by index
    labels = np.tile([0, cols - 1], (6, 1))
    for type in ("f32", "bf16"):
        _check_scores(capi, a, type, "logits", labels, k)
    _check_scores(capi, np.abs(np.where(np.isfinite(a), a, 0)), "f32", "probs", labels, k)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", [1, 17, 138, 600, 3001, 30000])
def test_score_rows_that_leave_nothing_and_rows_that_are_no_numbers(capi, cols, type):
    rng = np.random.default_rng(cols)
    big = {"f32": 3.4028234663852886e38, "f16": 65504.0, "bf16": 3.3895313892515355e38}[type]
    a = rng.standard_normal((11, cols))
    a[1] = -np.inf                         # nothing left
    a[2, cols // 2] = np.nan
    a[3, cols - 1] = np.inf
    a[4] = -big                            # the type's lowest value is a value like any other
    a[5, : cols // 2] = -big
    a[6, 0] = big
    a[7] = -np.inf
    a[7, cols - 1] = -big
    a[8, ::2] = -np.inf
    a[9] = -np.inf
    a[9, 0] = np.nan
    labels = np.tile([0, cols - 1, -1, cols, -5, 2 ** 31 - 1], (11, 1))
    k = min(5, cols)
    _check_scores(capi, a, type, "logits", labels, k)
    p = np.abs(rng.standard_normal((9, cols)))
    p[1] = 0.0
    p[2, cols // 2] = np.nan
    p[3, 0] = -1.0
    p[4, cols - 1] = np.inf
    p[5, : cols // 2] = 0.0
    p[6] = 0.0
    p[6, cols - 1] = 1.0
    p[7] = -0.0
    _check_scores(capi, p, type, "probs", labels[:9], k)


def test_score_outputs_that_are_not_wanted(capi):
    rng = np.random.default_rng(1)
    a = _scores(rng, 20, 138, "logits")
    x, _ = _strided(a, "f32", 0)
    labels = rng.integers(0, 138, (20, 2))
    full = Scored(capi, x, "f32", "logits", labels, 5, 138).run().get()
    for left_out in ("logp", "entropy", "top_index", "top_logp"):
        s = Scored(capi, x, "f32", "logits", labels, 5, 138)
        setattr(s.args, left_out, None)
        if left_out == "logp":
            s.args.labels = None
        got = s.run()
        torch.cuda.synchronize()
        for name, t, w in (("logp", got.logp, full[0]), ("entropy", got.ent, full[1]), ("top_index", got.ti, full[2]), ("top_logp", got.tl, full[3])):
            v = t[:w.size].cpu().numpy().reshape(w.shape)
            assert (v == 77).all() if name == left_out else np.array_equal(v, w)


def _pack(capi, x, type, rows, cols, ld=None, scales=None):
    q = torch.full((capi.fp8_bytes(rows, cols) + 64,), 171, dtype=torch.uint8, device="cuda")
    capi.fp8_pack(x.data_ptr(), capi.TYPES[type], rows, cols, ld or x.stride(0), q.data_ptr(), scales=scales.data_ptr() if scales is not None else None,
                  stream=_stream())
    torch.cuda.synchronize()
    assert (q[-64:] == 171).all(), "written behind the matrix"
    return q


def _unpack(capi, q, rows, cols, type="f32"):
    y = torch.full((rows + 1, cols + 3), 77.0, dtype=DT[type], device="cuda")
    capi.fp8_unpack(q.data_ptr(), rows, cols, y.data_ptr(), capi.TYPES[type], cols + 3, stream=_stream())
    torch.cuda.synchronize()
    assert (y[rows] == 77).all() and (y[:, cols:] == 77).all()
    return y[:rows, :cols].double().cpu().numpy()


def _activations(rng, rows, cols):
    a = rng.standard_normal((rows, cols)) * np.exp(rng.standard_normal((rows, 1)))
    a[:, rng.integers(0, cols, max(1, cols // 50))] *= 30
    return a


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (1, 127, 2), (2, 128, 0), (15, 129, 1), (16, 64, 0), (17, 276, 0), (33, 372, 4),
                                           (5, 511, 1), (64, 512, 0), (3, 1025, 0), (130, 640, 8)])
def test_fp8_pack_and_unpack(capi, rows, cols, pad, type):
    rng = np.random.default_rng(rows * 131 + cols)
    x, exact = _strided(_activations(rng, rows, cols), type, pad)
    q = _pack(capi, x, type, rows, cols)
    want, _ = ref.held(exact)
    assert np.array_equal(_unpack(capi, q, rows, cols), want)
    # what is held has 4 significant bits: f16's and bf16's ranges aside it is exact in any of the types
    assert np.array_equal(_unpack(capi, q, rows, cols, "bf16"), want)


def test_fp8_every_value_scale_and_border(capi):
    """all e4m3 values in each block scale; the largest value of a block on either side of 448 * 2^e; ties; zeros; NaN, infinities"""
    t = ref.e4m3_table()
    fin = t[np.isfinite(t)]
    rows = []
    for e in (-100, -9, 0, 1, 50, 110):
        rows.append(np.resize(fin, 256) * 2.0 ** e)
        rows.append(np.resize((fin[1:126] + fin[:125]) / 2, 256) * 2.0 ** e)             # ties, scaled by what they need
        for m in (448.0, np.nextafter(np.float32(448), np.float32(1000)), np.nextafter(np.float32(448), np.float32(0)), 256.0, 255.99998):
            v = np.linspace(-1, 1, 256) * 100
            v[7] = m
            v[200] = -m
            rows.append(v * 2.0 ** e)
    v = np.zeros(256)
    rows.append(v)
    v = np.linspace(-3, 3, 256)
    v[3], v[130], v[131] = np.nan, np.inf, -np.inf
    rows.append(v)
    rows.append(np.full(256, np.inf))
    rows.append(np.full(256, 1.4e-45))                          # subnormal f32: e stops at -127
    rows.append(np.linspace(-1, 1, 256) * 1.2e-38)
    rows.append(np.linspace(-1, 1, 256) * 3.4028234e38)
    a = np.array(rows, np.float32)
    x = torch.from_numpy(a).cuda()
    want, e = ref.held(a.astype(np.float64))
    q = _pack(capi, x, "f32", *a.shape)
    got = _unpack(capi, q, *a.shape)
    # (f32 holds what is below 2^-126 in steps of 2^-149: the unpacked value is rounded to it)
    assert np.array_equal(got, want.astype(np.float32).astype(np.float64), equal_nan=True)


@pytest.mark.parametrize("rows,cols", [(1, 1), (15, 200), (40, 513)])
def test_fp8_pack_of_held_values(capi, rows, cols):
    rng = np.random.default_rng(cols)
    b = rng.integers(0, 256, (rows, cols + 5)).astype(np.uint8)
    kb = -(-cols // 128)
    s = rng.integers(100, 150, (rows, kb)).astype(np.uint8)
    q = _pack(capi, torch.from_numpy(b).cuda(), "e4m3", rows, cols, cols + 5, torch.from_numpy(s).cuda())
    want = ref.e4m3_table()[b[:, :cols]] * ref.spread(s.astype(np.int64) - 127, cols)
    assert np.array_equal(_unpack(capi, q, rows, cols), want, equal_nan=True)


class Linear:
    def __init__(self, capi, x, x_type, rows, n_in, n_out, w, bias, act, y_type, ldx=None, pad=3):
        self.capi, self.rows, self.n_out, self.y_type, self.keep = capi, rows, n_out, y_type, (x, w, bias)
        self.ldy = n_out + pad
        if y_type == "e4m3":
            self.y = torch.full((capi.fp8_bytes(rows, n_out) + 64,), 171, dtype=torch.uint8, device="cuda")
        else:
            self.y = torch.full((rows + 1, self.ldy), 77.0, dtype=DT[y_type], device="cuda")
        self.size = capi.fp8_linear_workspace(rows, n_in, capi.TYPES[x_type])
        self.ws = torch.full((self.size + 64,), 171, dtype=torch.uint8, device="cuda")
        self.args = capi.Fp8LinearArgs(
            x=x.data_ptr(), x_type=capi.TYPES[x_type], rows=rows, n_in=n_in, n_out=n_out, ldx=ldx if ldx is not None else x.stride(0),
            w=w.data_ptr(), bias=bias.data_ptr() if bias is not None else None, act=capi.ACTS[act], y=self.y.data_ptr(),
            y_type=capi.TYPES[y_type], ldy=self.ldy, workspace=self.ws.data_ptr() if self.size else None, workspace_bytes=self.size)

    def run(self, stream=None):
        self.capi.fp8_linear(self.args, stream=_stream() if stream is None else stream)
        return self

    def get(self):
        torch.cuda.synchronize()
        assert (self.ws[self.size:] == 171).all(), "written behind the workspace"
        if self.y_type == "e4m3":
            assert (self.y[-64:] == 171).all(), "written behind the matrix"
            return _unpack(self.capi, self.y, self.rows, self.n_out)
        assert (self.y[self.rows] == 77).all() and (self.y[:, self.n_out:] == 77).all(), "written outside the matrix"
        return self.y[:self.rows, :self.n_out].double().cpu().numpy()


def _linear_tolerance(v, mag, n_in, act, y_type):
    """Products of two e4m3 values are exact; adding n_in of them, the scaled sums of the blocks and the bias in 32 bits in any
    order is off by at most (n_in + blocks + 1) eps sum|x w| + |b|; the sigmoid has a slope of 1/4 and its own 4 eps; then the
    type's rounding.  In 8 bits: half a step, 2^-4 of the value, or 2^-10 of the block's scale, which is at most
    max|v| of the row / 224.
    Results in 16 or 8 bits come from the 8-bit matrix instructions, which cut each of eight products off 13 bits below the
    power of two of the largest of the eight before they add: each of the other seven loses less than 2^-13 of that largest
    one, so a group loses less than 7 * 2^-13 of its sum |x w|."""
    eps = ref.EPS["f32"]
    tol = ((n_in + n_in // 128 + 2) * eps + (0.0 if y_type == "f32" else 7 * 2.0 ** -13)) * mag
    if act != "none":
        tol = tol / 4 + 4 * eps
    if y_type == "e4m3":
        return tol * 1.01 + np.abs(v) * 2.0 ** -4 + np.abs(v).max(1, keepdims=True) / 224 * 2.0 ** -10
    small = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}[y_type]
    return tol + (np.abs(v) + tol) * ref.EPS[y_type] + small


def _weights(capi, rng, n_out, n_in):
    w = rng.standard_normal((n_out, n_in)) * 2 / np.sqrt(n_in)
    x, exact = _strided(w, "f32", 0)
    return _pack(capi, x, "f32", n_out, n_in), ref.held(exact)[0]


SIZES = [(1, 1, 1), (1, 276, 1500), (1, 128, 128), (2, 129, 127), (5, 1000, 17), (7, 512, 300), (16, 372, 186), (17, 276, 138),
         (31, 640, 257), (33, 128, 129), (64, 1500, 138), (100, 253, 500), (130, 2049, 260), (200, 300, 1000), (257, 131, 511), (300, 1030, 260)]


@pytest.mark.parametrize("rows,n_in,n_out", SIZES)
@pytest.mark.parametrize("x_type,y_type,act,pad", [("f32", "f32", "none", 0), ("bf16", "bf16", "sigmoid", 1), ("f16", "f16", "none", 8),
                                                   ("e4m3", "f32", "sigmoid", 0), ("f32", "e4m3", "sigmoid", 3), ("bf16", "e4m3", "none", 0)])
def test_fp8_linear_against_64_bits(capi, rows, n_in, n_out, x_type, y_type, act, pad):
    rng = np.random.default_rng(rows * 7919 + n_in * 31 + n_out)
    src = "f32" if x_type == "e4m3" else x_type
    x, exact = _strided(_activations(rng, rows, n_in), src, pad, fill=0.0 if x_type == "e4m3" else float("nan"))
    xq = ref.held(exact)[0]
    if x_type == "e4m3":
        x = _pack(capi, x, src, rows, n_in)
    w, wq = _weights(capi, rng, n_out, n_in)
    b = rng.standard_normal(n_out).astype(np.float32) if n_out % 2 else None
    bias = torch.from_numpy(b).cuda() if b is not None else None
    got = Linear(capi, x, x_type, rows, n_in, n_out, w, bias, act, y_type, ldx=0 if x_type == "e4m3" else None).run().get()
    v, mag = ref.linear(xq, wq, b.astype(np.float64) if b is not None else 0.0, act)
    err = np.abs(got - v)
    tol = _linear_tolerance(v, mag, n_in, act, y_type)
    assert (err <= tol).all(), (np.argwhere(~(err <= tol))[:5], got[~(err <= tol)][:5], v[~(err <= tol)][:5])


def test_fp8_linear_carries_nan_and_only_there(capi):
    """NaN or infinity in one row of x, or one row of W, spoils that row / column of y and nothing else"""
    rng = np.random.default_rng(3)
    a = _activations(rng, 40, 300)
    a[5, 17], a[20, 299] = np.nan, np.inf
    x, _ = _strided(a, "f32", 0)
    wv = rng.standard_normal((150, 300))
    wv[77, 4] = np.nan
    w = _pack(capi, torch.from_numpy(wv.astype(np.float32)).cuda(), "f32", 150, 300)
    got = Linear(capi, x, "f32", 40, 300, 150, w, None, "none", "f32").run().get()
    want = np.zeros((40, 150), bool)
    want[[5, 20]] = True
    want[:, 77] = True
    assert np.array_equal(np.isnan(got), want)


def test_fp8_net_then_scores(capi):
    """two layers, the hidden activations in 8 bits, and the scores of the logits: the run a recogniser makes of them"""
    rng = np.random.default_rng(11)
    rows, n_in, n_hid, n_out, k = 300, 276, 1500, 138, 5
    x, exact = _strided(_activations(rng, rows, n_in), "f32", 0)
    w1, q1 = _weights(capi, rng, n_hid, n_in)
    w2, q2 = _weights(capi, rng, n_out, n_hid)
    b1, b2 = (rng.standard_normal(n).astype(np.float32) for n in (n_hid, n_out))
    B1, B2 = torch.from_numpy(b1).cuda(), torch.from_numpy(b2).cuda()
    h = Linear(capi, x, "f32", rows, n_in, n_hid, w1, B1, "sigmoid", "e4m3").run()
    y = Linear(capi, h.y, "e4m3", rows, n_hid, n_out, w2, B2, "none", "f32", ldx=0, pad=0).run()
    labels = rng.integers(0, n_out, (rows, 1))
    got = Scored(capi, y.y, "f32", "logits", labels, k, n_out).run().get()
    hv = h.get()
    v1, m1 = ref.linear(ref.held(exact)[0], q1, b1.astype(np.float64), "sigmoid")
    assert (np.abs(hv - v1) <= _linear_tolerance(v1, m1, n_in, "sigmoid", "e4m3")).all()
    v2, m2 = ref.linear(hv, q2, b2.astype(np.float64), "none")          # from the hidden values as they are held
    yv = y.get()
    assert (np.abs(yv - v2) <= _linear_tolerance(v2, m2, n_hid, "none", "f32")).all()
    want = ref.score(yv, labels, k, "logits")
    lp, en = ref.score_tolerance(yv, "logits")
    assert np.array_equal(got[2], want[2])
    _close(got[0], want[0], lp[:, None])
    _close(got[1], want[1], en)


def test_ops_on_another_stream_and_in_a_graph(capi):
    """captured and replayed with new inputs in the same buffers, eager work between the replays; and on a stream of its own"""
    rng = np.random.default_rng(5)
    rows, n_in, n_out, k = 70, 276, 1500, 5
    x, _ = _strided(_activations(rng, rows, n_in), "f32", 0)
    w, _ = _weights(capi, rng, n_out, n_in)
    labels = rng.integers(0, n_out, (rows, 1))
    lin = Linear(capi, x, "f32", rows, n_in, n_out, w, None, "none", "f32", pad=0)
    sc = Scored(capi, lin.y, "f32", "logits", labels, k, n_out)

    def eager():
        lin.run()
        return (lin.get(),) + sc.run().get()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    first = eager()
    for t in (lin.y, sc.logp, sc.ent, sc.tl):
        t[: t.shape[0] - (1 if t is lin.y else 64)] = 0
    torch.cuda.synchronize()
    lin.run(side.cuda_stream)
    sc.run(side.cuda_stream)
    side.synchronize()
    for a, b in zip(first, (lin.get(),) + sc.get()):
        assert np.array_equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = torch.cuda.current_stream().cuda_stream
        lin.run(s)
        sc.run(s)
    for i in range(4):
        x.copy_(torch.from_numpy(_activations(rng, rows, n_in).astype(np.float32)))
        want = eager()
        lin.y[:rows] = 0
        torch.cuda.synchronize()
        graph.replay()
        for a, b in zip(want, (lin.get(),) + sc.get()):
            assert np.array_equal(a, b), i
