"""Cases for timing and comparing the operators that include/lcrc_pipeline.h declares.

Two operators of a recogniser's output side, and the two of them as one small net:

  score   log probabilities of given classes, the entropy and the k best classes of every row of a matrix of logits or of
          probabilities (posteriors)
  linear  y = act(x W^T + b) with x and W held in 8-bit floating point (e4m3), each run of 128 inputs of a row with its own
          power-of-two scale; x arrives in 32 or 16 bits and is put into that form by the call
  net     two such products, the hidden activations handed from one to the other in 8 bits

`run` computes them either in elementary torch operations or, with `own`, by the library's kernels.
"""
import math

import torch

own = False

SCORE_OUT = ("logp", "entropy", "top_index", "top_logp")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 128
E4M3_MAX = 448.0
LARGEST_FLOPS = 2.0 * 8192 ** 3      # linear_large, the largest listed product
LARGEST_ELEMENTS = 524288 * 186      # score_list, the largest listed matrix of scores


def listed():
    return [
        # one frame's posteriors of the 46-phoneme system (46 x 3 states): streaming, where latency is all
        dict(name="score_frame", op="score", rows=1, cols=138, type="f32", form="probs", k=5, labels=1, masked=0.0, pad=0),
        # one launch of the benchmark: 8192 frames scored against an alignment, with the 5 best states of each frame
        dict(name="score_batch", op="score", rows=8192, cols=138, type="f32", form="probs", k=5, labels=1, masked=0.0, pad=0),
        # a long list of files at once (62 phonemes x 3 states): bandwidth
        dict(name="score_list", op="score", rows=524288, cols=186, type="f32", form="logits", k=3, labels=1, masked=0.0, pad=0),
        # wide heads (word pieces, tied states): 16-bit logits of odd width, a part of the classes ruled out
        dict(name="score_wide", op="score", rows=2051, cols=50001, type="bf16", form="logits", k=16, labels=4, masked=0.3, pad=0),
        # a few positions over a very wide head, many alternatives, rows further apart than they are long
        dict(name="score_long", op="score", rows=3, cols=200003, type="f16", form="logits", k=64, labels=2, masked=0.0, pad=37),
        # the merger's hidden layer for one frame
        dict(name="linear_frame", op="linear", rows=1, n_in=276, n_out=1500, x_type="f32", y_type="f32", act="sigmoid", pad=0),
        # the same layer for one launch of frames
        dict(name="linear_batch", op="linear", rows=8192, n_in=276, n_out=1500, x_type="f32", y_type="bf16", act="sigmoid", pad=0),
        # a few rows through a wide layer: the weights' bytes are what it costs
        dict(name="linear_few", op="linear", rows=5, n_in=8192, n_out=8192, x_type="bf16", y_type="f32", act="none", pad=0),
        # sizes that fit no tile, rows further apart than they are long
        dict(name="linear_odd", op="linear", rows=777, n_in=1999, n_out=2309, x_type="f16", y_type="f16", act="none", pad=9),
        # a large product: arithmetic rate
        dict(name="linear_large", op="linear", rows=8192, n_in=8192, n_out=8192, x_type="bf16", y_type="bf16", act="none", pad=0),
        # the merger of the 62-phoneme system on one launch of frames
        dict(name="net_batch", op="net", rows=8192, n_in=372, n_hid=1500, n_out=186, x_type="f32", y_type="bf16", pad=0),
        # a wide net
        dict(name="net_wide", op="net", rows=4096, n_in=2048, n_hid=8192, n_out=2048, x_type="bf16", y_type="bf16", pad=0),
    ]


def _spread(rng, lo, hi):
    """a whole number of lo..hi, evenly over its logarithm"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["score", "linear", "net"])
    pad = rng.choice([0, 0, 0, 1, 8, 37])
    if op == "score":
        cols = _spread(rng, 39, 200003)
        rows = _spread(rng, 1, max(1, min(524288, LARGEST_ELEMENTS // cols)))
        return dict(op=op, rows=rows, cols=cols, type=rng.choice(list(TYPES)), form=rng.choice(["probs", "logits"]),
                    k=rng.choice([0, 1, 2, 3, 5, 8, 16, 20, 32]), labels=rng.choice([0, 1, 1, 2, 4]) if rng.random() < 0.9 else 8,
                    masked=rng.choice([0.0, 0.0, 0.25]), pad=pad)
    rows, n_in, n_out = _spread(rng, 1, 16384), _spread(rng, 33, 16384), _spread(rng, 33, 16384)
    x_type = rng.choice(list(TYPES))
    if op == "linear":
        while 2.0 * rows * n_in * n_out > LARGEST_FLOPS:
            rows = max(1, rows // 2)
        return dict(op=op, rows=rows, n_in=n_in, n_out=n_out, x_type=x_type, y_type=rng.choice(list(TYPES)),
                    act=rng.choice(["none", "sigmoid"]), pad=pad)
    n_hid = _spread(rng, 100, 8192)
    while 2.0 * rows * n_hid * (n_in + n_out) > LARGEST_FLOPS / 4:
        rows = max(1, rows // 2)
    return dict(op=op, rows=rows, n_in=n_in, n_hid=n_hid, n_out=n_out, x_type=x_type, y_type=rng.choice(["bf16", "f16"]), pad=pad)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _padded(x, pad):
    """the same values with `pad` more elements between the starts of two rows"""
    if not pad:
        return x
    wide = torch.zeros(x.shape[0], x.shape[1] + pad, dtype=x.dtype, device=x.device)
    wide[:, :x.shape[1]] = x
    return wide[:, :x.shape[1]]


def _activations(rows, n, dtype, pad, gen):
    """normalised inputs: unit variance, rows of different loudness, a few columns that stand out"""
    x = torch.randn(rows, n, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device="cuda"))
    x[:, torch.randint(0, n, (max(1, n // 100),), generator=gen, device="cuda")] *= 8.0
    return _padded(x.to(dtype), pad)


def _exponents(x):
    """x [rows][n] in f32 -> the power of two of each row's runs of 128 (int32 [rows][ceil(n/128)]): the smallest e with
    max|x| <= 448 * 2^e, not below -127; 0 for a run of zeros"""
    rows, n = x.shape
    blocks = -(-n // BLOCK)
    full = torch.zeros(rows, blocks * BLOCK, dtype=torch.float32, device=x.device)
    full[:, :n] = x
    most = full.view(rows, blocks, BLOCK).abs().amax(2)
    m, e = torch.frexp(most)                    # most = m * 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-127)
    return torch.where(most == 0, torch.zeros_like(e), e)


def _wide(e, n):
    return torch.ldexp(torch.ones((), device=e.device), e).repeat_interleave(BLOCK, 1)[:, :n]


def _quantised(x):
    """(e4m3 values, exponents) of x [rows][n] in f32"""
    e = _exponents(x)
    return (x * _wide(-e, x.shape[1])).to(torch.float8_e4m3fn), e


def _weights(n_out, n_in, gen):
    """weights as a checkpoint holds them: e4m3 values, one exponent byte (biased by 127) for each run of 128 inputs; f32 bias"""
    w = torch.randn(n_out, n_in, generator=gen, device="cuda") * (2.0 / math.sqrt(n_in))
    q, e = _quantised(w)
    return {"q": q, "s": (e + 127).to(torch.uint8), "bias": torch.randn(n_out, generator=gen, device="cuda"),
            "n_in": n_in, "n_out": n_out}


def _handle(capi, w):
    """the weights in the layout the kernels read, made once"""
    w["packed"] = torch.empty(capi.fp8_bytes(w["n_out"], w["n_in"]), dtype=torch.uint8, device="cuda")
    capi.fp8_pack(w["q"].data_ptr(), capi.T_E4M3, w["n_out"], w["n_in"], w["n_in"], w["packed"].data_ptr(),
                  scales=w["s"].data_ptr(), stream=torch.cuda.current_stream().cuda_stream)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if own:
        from phnrec_amd import capi
        s["capi"] = capi
    rows = case["rows"]
    if case["op"] == "score":
        cols, k, m = case["cols"], case["k"], case["labels"]
        x = torch.randn(rows, cols, generator=gen, device="cuda").mul_(3.0)
        if case["masked"]:
            out = torch.rand(rows, cols, generator=gen, device="cuda") < case["masked"]
            x.masked_fill_(out, -math.inf)
        if case["form"] == "probs":
            x = torch.softmax(x, 1)
        s["x"] = _padded(x.to(TYPES[case["type"]]), case["pad"])
        labels = torch.randint(0, cols, (rows, m), generator=gen, device="cuda", dtype=torch.int32)
        none = torch.rand(rows, m, generator=gen, device="cuda") < 0.03
        s["label"] = labels.masked_fill_(none, -1)               # frames without a label
        if own:
            size = capi.score_workspace(rows, cols, k)
            s["workspace"] = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
            f32 = dict(dtype=torch.float32, device="cuda")
            s["out"] = {"logp": torch.empty(rows, m, **f32), "entropy": torch.empty(rows, **f32),
                        "top_index": torch.empty(rows, k, dtype=torch.int32, device="cuda"), "top_logp": torch.empty(rows, k, **f32)}
            o = s["out"]
            s["args"] = capi.ScoreArgs(
                x=s["x"].data_ptr(), type=capi.TYPES[case["type"]], form=capi.SCORE_FORMS[case["form"]], rows=rows, cols=cols,
                ld=s["x"].stride(0), labels=s["label"].data_ptr(), n_labels=m, k=k, logp=o["logp"].data_ptr(),
                entropy=o["entropy"].data_ptr(), top_index=o["top_index"].data_ptr(), top_logp=o["top_logp"].data_ptr(),
                workspace=s["workspace"].data_ptr(), workspace_bytes=size)
        return s
    s["x"] = _activations(rows, case["n_in"], TYPES[case["x_type"]], case["pad"], gen)
    widths = [case["n_in"], case["n_hid"], case["n_out"]] if case["op"] == "net" else [case["n_in"], case["n_out"]]
    s["w"] = [_weights(o, i, gen) for i, o in zip(widths, widths[1:])]
    if own:
        for w in s["w"]:
            _handle(capi, w)
        x, x_type, ld = s["x"], capi.TYPES[case["x_type"]], s["x"].stride(0)
        s["args"] = []
        for n, w in enumerate(s["w"]):
            last = n == len(s["w"]) - 1
            if last:
                y = torch.empty(rows, w["n_out"], dtype=TYPES[case["y_type"]], device="cuda")
            else:
                y = torch.empty(capi.fp8_bytes(rows, w["n_out"]), dtype=torch.uint8, device="cuda")
            size = capi.fp8_linear_workspace(rows, w["n_in"], x_type)
            w["workspace"] = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
            act = case["act"] if case["op"] == "linear" else "none" if last else "sigmoid"
            s["args"].append(capi.Fp8LinearArgs(
                x=x.data_ptr(), x_type=x_type, rows=rows, n_in=w["n_in"], n_out=w["n_out"], ldx=ld, w=w["packed"].data_ptr(),
                bias=w["bias"].data_ptr(), act=capi.ACTS[act], y=y.data_ptr(),
                y_type=capi.TYPES[case["y_type"]] if last else capi.T_E4M3, ldy=w["n_out"],
                workspace=w["workspace"].data_ptr(), workspace_bytes=size))
            s["y%d" % n] = y
            x, x_type, ld = y, capi.T_E4M3, 0
        s["out"] = y
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------

def _score_plain(s):
    x, k = s["x"].float(), s["k"]
    if s["form"] == "probs":
        total = x.sum(1, keepdim=True)
        log_total = torch.log(total)
        value = torch.log(x)                                       # ln 0 = -inf
        spread = torch.where(x > 0, x * value, torch.zeros_like(x)).sum(1, keepdim=True)
    else:
        value = x - x.amax(1, keepdim=True)
        e = torch.exp(value)
        total = e.sum(1, keepdim=True)
        log_total = torch.log(total)
        spread = torch.where(e > 0, e * value, torch.zeros_like(e)).sum(1, keepdim=True)
    out = {"entropy": (log_total - spread / total)[:, 0]}
    label = s["label"].long()
    given = torch.gather(value, 1, label.clamp(min=0)) - log_total
    out["logp"] = torch.where(label < 0, torch.zeros_like(given), given)
    best, order = torch.sort(x, dim=1, descending=True, stable=True)   # equal values: the lowest index first
    out["top_index"] = order[:, :k].to(torch.int32)
    out["top_logp"] = torch.gather(value, 1, order[:, :k]) - log_total
    return out


def _linear_plain(x, w, act):
    """x [rows][n_in] in f32 -> act(x W^T + b) in f32, x and W being what their 8-bit forms stand for"""
    q, e = _quantised(x)
    x = q.float() * _wide(e, w["n_in"])
    y = x @ (w["q"].float() * _wide(w["s"].to(torch.int32) - 127, w["n_in"])).t() + w["bias"]
    return 1.0 / (1.0 + torch.exp(-y)) if act == "sigmoid" else y


def run(s):
    if own:
        capi, stream = s["capi"], torch.cuda.current_stream().cuda_stream
        if s["op"] == "score":
            capi.score(s["args"], stream=stream)
        else:
            for a in s["args"]:
                capi.fp8_linear(a, stream=stream)
        return s["out"]
    if s["op"] == "score":
        return _score_plain(s)
    y = s["x"].float()
    if s["op"] == "linear":
        y = _linear_plain(y, s["w"][0], s["act"])
    else:
        y = _linear_plain(_linear_plain(y, s["w"][0], "sigmoid"), s["w"][1], "none")
    return y.to(TYPES[s["y_type"]])


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    rows = case["rows"]
    if case["op"] == "score":
        n = rows * case["cols"]
        # a maximum, an exponential and two sums for each element (an exponential counted as one operation)
        return {"bytes": n * size[case["type"]] + rows * (8 * case["labels"] + 4 + 8 * case["k"]), "flops": 6 * n}
    widths = [case["n_in"], case["n_hid"], case["n_out"]] if case["op"] == "net" else [case["n_in"], case["n_out"]]
    b = rows * (case["n_in"] * size[case["x_type"]] + case["n_out"] * size[case["y_type"]])
    f = 0
    for i, o in zip(widths, widths[1:]):
        b += o * i + o * -(-i // BLOCK) + 4 * o
        f += 2 * rows * i * o
    return {"bytes": b, "flops": f}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def _score_exact(s):
    x, label, k = s["x"].double(), s["label"].long(), s["k"]
    ln = torch.log(x) if s["form"] == "probs" else x
    ln = ln - torch.logsumexp(ln, 1, keepdim=True)                 # ln p
    p = torch.exp(ln)
    given = torch.gather(ln, 1, label.clamp(min=0))
    return {"entropy": -torch.nansum(p * ln, 1), "logp": given.masked_fill(label < 0, 0.0), "top_index": None,
            "top_logp": torch.topk(ln, k, 1).values}


def _held(x):
    """what the 8-bit form of x [rows][n] stands for, step by step in 64 bits"""
    x = x.double()
    n = x.shape[1]
    out = torch.empty_like(x)
    for b in range(0, n, BLOCK):
        v = x[:, b:b + BLOCK]
        most = v.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(torch.clamp(most, min=1e-300) / E4M3_MAX)).clamp(min=-127.0)
        v = v * torch.exp2(-e)
        # 4 significant bits down to 2^-6, steps of 2^-9 below
        step = torch.exp2(torch.floor(torch.log2(torch.clamp(v.abs(), min=2.0 ** -6))) - 3)
        out[:, b:b + BLOCK] = torch.round(v / step) * step * torch.exp2(e)
    return out


def _layer_exact(x, w, act):
    n = w["n_in"]
    scale = torch.exp2(w["s"].double() - 127).repeat_interleave(BLOCK, 1)[:, :n]
    y = torch.matmul(_held(x), (w["q"].double() * scale).t().contiguous()) + w["bias"].double()
    return torch.sigmoid(y) if act == "sigmoid" else y


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "score":
        return _score_exact(s)
    if s["op"] == "linear":
        return _layer_exact(s["x"], s["w"][0], s["act"])
    return _layer_exact(_layer_exact(s["x"], s["w"][0], "sigmoid"), s["w"][1], "none")
