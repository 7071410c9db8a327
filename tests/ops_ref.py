"""Plain 64-bit implementations of the operators on matrices in device memory (include/lcrc_pipeline.h), for their tests."""
import numpy as np


class _Torch:
    """torch, imported when it is first used: a test process that collects the tests without running them stays small (other
    tests measure the memory of the processes they start, which begins with their parent's)"""

    def __getattr__(self, name):
        import torch
        return getattr(torch, name)


torch = _Torch()


class _Types:
    def __getitem__(self, name):
        return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


DT = _Types()

EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}       # a rounding is off by at most this, relative


def e4m3_table():
    """the 256 values of OCP e4m3: 1 sign, 4 exponent (bias 7), 3 mantissa bits; 0x7f and 0xff are NaN"""
    t = np.empty(256)
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        v = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        t[b] = np.nan if (b & 127) == 127 else v
    t[128:] = -t[128:]
    return t


def block_exponents(x):
    """the smallest e >= -127 with max|x| <= 448 * 2^e over the finite values of each run of 128 columns; 0 for a run of zeros"""
    rows, n = x.shape
    kb = -(-n // 128)
    full = np.zeros((rows, kb * 128))
    full[:, :n] = np.where(np.isfinite(x), np.abs(x), 0)
    most = full.reshape(rows, kb, 128).max(2)
    e = np.full(most.shape, -127)
    while True:
        over = most > 448 * 2.0 ** e
        if not over.any():
            break
        e = e + over
    return np.where(most == 0, 0, e)


def spread(e, n):
    return np.repeat(2.0 ** e.astype(np.float64), 128, axis=1)[:, :n]


def held(x):
    """(what the 8-bit form of x stands for, the blocks' exponents): nearest e4m3 value, ties to the even mantissa"""
    x = np.asarray(x, np.float64)
    e = block_exponents(x)
    s = spread(e, x.shape[1])
    t = e4m3_table()[:127]                        # 0 .. 448, rising; index = bit pattern, so an even index is an even mantissa
    a = np.abs(np.where(np.isfinite(x), x, 0)) / s
    hi = np.clip(np.searchsorted(t, a), 1, 126)
    lo = hi - 1
    d = (a - t[lo]) - (t[hi] - a)
    pick = np.where((d > 0) | ((d == 0) & (hi % 2 == 0)), hi, lo)
    q = np.sign(np.where(np.isfinite(x), x, 0)) * t[pick] * s
    return np.where(np.isfinite(x), q, np.nan), e


def score(x, labels, k, form):
    """lcrc_score of x [rows][cols] (any dtype, exact in 64 bits) -> logp, entropy, top_index, top_logp"""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    logp, ent = np.zeros(labels.shape), np.zeros(rows)
    ti, tl = np.zeros((rows, k), np.int64), np.zeros((rows, k))
    for r in range(rows):
        v = x[r]
        bad = bool(np.isnan(v).any() or (v == np.inf).any() or (form == "probs" and (v < 0).any()))
        with np.errstate(divide="ignore", invalid="ignore"):
            l = np.log(v) if form == "probs" else v
        order = np.argsort(-v, kind="stable")[:k]
        if bad:
            ln, ent[r], order = np.full(cols, np.nan), np.nan, np.full(k, -1)
            tl[r] = np.nan
        elif not np.isfinite(l).any():
            ln = np.full(cols, -np.inf)
            tl[r] = -np.inf
        else:
            m = l.max()
            ln = l - m - np.log(np.exp(l - m).sum())
            p = np.exp(ln)
            ent[r] = -np.sum(p[p > 0] * ln[p > 0])
            tl[r] = ln[order]
        ti[r] = order
        for j, c in enumerate(labels[r]):
            logp[r, j] = 0.0 if c < 0 else np.nan if c >= cols else ln[c]
    return logp, ent, ti, tl


def score_tolerance(x, form):
    """Per row, for ln p and the entropy: x - m is rounded once (|x - m| eps), ln and exp are good to a few ulp of their results
    (3 eps each), a rounded argument moves an exponential by R eps relative (R: the largest |l - m| that still counts, where
    exp(l - m) > 2^-30 / cols), S and T are sums of n terms of one sign (n eps relative at the very most), T / S <= R:
        ln p: eps (|l - m| + |ln S| + 4 + R + n)       entropy: eps ((R + |ln S|) (4 + R + 2 n))"""
    eps = EPS["f32"]
    x = np.asarray(x, np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        l = np.log(x) if form == "probs" else x
    n = x.shape[1]
    lp, en = np.zeros(x.shape[0]), np.zeros(x.shape[0])
    for r in range(x.shape[0]):
        f = l[r][np.isfinite(l[r])]
        if not len(f):
            continue
        m = f.max() if form == "logits" else 0.0
        reach = np.abs(f - m).max()
        ln_s = abs(np.log(np.exp(f - m).sum()))
        R = np.abs(f - m)[np.exp(f - f.max()) > 2.0 ** -30 / n].max()
        lp[r] = eps * (reach + ln_s + 4 + R + n)
        en[r] = eps * (R + ln_s) * (4 + R + 2 * n)
    return lp, en


def linear(xq, wq, bias, act):
    """act(xq wq^T + bias) of the held values in 64 bits, and sum |x w| + |b| of each output"""
    with np.errstate(invalid="ignore", over="ignore"):
        v = xq @ wq.T + bias
        mag = np.abs(xq) @ np.abs(wq).T + np.abs(bias)
        if act == "sigmoid":
            v = 1 / (1 + np.exp(-v))
    return v, mag
