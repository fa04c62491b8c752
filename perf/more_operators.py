"""Performance cases of the operators of a packed batch of texts in 8 bits: the
residual's addition, RMS norm and quantization of a step's activations, the
product of such activations with int8 weights, attention over sequences of
different lengths packed one behind the other, and log probabilities of given
tokens with entropy and the likeliest alternatives.

`run` computes them through the dispatch library where `own` is true, and in
elementary torch operations where it is not. Operands are torch tensors in
HBM; the library launches on the null stream, torch's default stream, so its
work and torch's are ordered.
"""

from __future__ import annotations

import math

import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}
EPS = 1e-5

_lib: list = []


def lib():
    if not _lib:
        from vx_amd.runtime import DispatchLibrary
        _lib.append(DispatchLibrary())
    return _lib[0]


# ---- cases ---------------------------------------------------------------

def norm(name, dtype, rows, dim, mode, residual=True) -> dict:
    """mode: what comes of the rows: "i8" or "bf16" or "both" of the norm, or
    "quantize" (8 bits without a norm)."""
    return {"name": name, "kind": "norm", "dtype": dtype, "rows": rows, "dim": dim, "mode": mode,
            "residual": residual}


def gemm(name, dtype, tokens, rows, cols) -> dict:
    return {"name": name, "kind": "gemm", "dtype": dtype, "tokens": tokens, "rows": rows, "cols": cols}


def packed(name, sequences, longest, heads, kv_heads, head_dim, layout, causal=True, pad=0) -> dict:
    """layout: "tokens" (one projection [tokens, heads + 2 kv_heads, head_dim])
    or "heads" ([heads, tokens, head_dim], as rotation leaves them)."""
    return {"name": name, "kind": "packed", "sequences": sequences, "longest": longest, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "layout": layout, "causal": causal, "pad": pad}


def logprobs(name, dtype, rows, vocab, given, top) -> dict:
    return {"name": name, "kind": "logprobs", "dtype": dtype, "rows": rows, "vocab": vocab, "given": given,
            "top": top}


def listed() -> list[dict]:
    return [
        # One token's f32 residual stream at the decoder's width: latency.
        norm("norm_1x768", "f32", 1, 768, "both"),
        # A long prompt's step between two layers, a 16-bit stream.
        norm("norm_4096x4096", "bf16", 4096, 4096, "i8"),
        # Feed-forward activations before their second product: no norm, rows
        # of another width than the stream's, an odd number of them.
        norm("quantize_777x11008", "bf16", 777, 11008, "quantize", False),
        # One token's logits from the decoder's int8 classifier.
        gemm("gemm_i8_1x32000x768", "f32", 1, 32000, 768),
        # A serving batch against one feed-forward matrix: weights from HBM.
        gemm("gemm_i8_48x11008x4096", "bf16", 48, 11008, 4096),
        # An odd chunk of prompts, a projection of grouped heads.
        gemm("gemm_i8_777x6144x4096", "bf16", 777, 6144, 4096),
        # Packed prompts filling the matrix cores.
        gemm("gemm_i8_4096x11008x4096", "bf16", 4096, 11008, 4096),
        # Five short texts with the decoder's heads.
        packed("packed_5x200_h12", 5, 200, 12, 12, 64, "heads"),
        # 64 prompts of 1 to 1024 tokens, empty slots and padding rows behind
        # them, straight from the fused projection.
        packed("packed_64x1024_h32", 64, 1024, 32, 8, 128, "tokens", pad=29),
        # A document and a shorter one: the largest.
        packed("packed_2x8192_h32", 2, 8192, 32, 8, 128, "heads"),
        # The next token's alternatives for one user.
        logprobs("logprobs_1x32000", "f32", 1, 32000, 1, 5),
        # Texts scored at a large vocabulary of odd size, 16-bit logits.
        logprobs("logprobs_512x131071", "bf16", 512, 131071, 1, 20),
    ]


def _log(rng, lo, hi) -> int:
    """A size spread over the logarithm of its range."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "gemm", "gemm", "packed", "packed", "logprobs"])
    if kind == "norm":
        while True:
            rows, dim = _log(rng, 1, 16384), _log(rng, 64, 16384)
            if rng.random() < 0.7:
                dim = (dim + 15) // 16 * 16
            if rows * dim <= 4096 * 4096:
                break
        mode = rng.choice(["i8", "bf16", "both", "quantize"])
        c = norm("", rng.choice(["f32", "bf16"]), rows, dim, mode, mode != "quantize" and rng.random() < 0.7)
    elif kind == "gemm":
        while True:
            tokens, rows, cols = _log(rng, 1, 4096), _log(rng, 64, 32000), 16 * _log(rng, 4, 688)
            if tokens * rows * cols <= 4096 * 11008 * 4096 and rows * cols <= 2 ** 27:
                break
        c = gemm("", rng.choice(["f32", "bf16"]), tokens, rows, cols)
    elif kind == "packed":
        while True:
            head_dim, kv_heads = rng.choice([64, 128]), rng.choice([1, 2, 3, 4, 8, 12])
            heads = kv_heads * rng.choice([1, 1, 3, 4, 7, 8])
            sequences, longest = _log(rng, 1, 256), _log(rng, 1, 8192)
            if heads <= 64 and sequences * heads * longest ** 2 <= 2 ** 32 and (
                    sum(_lens(sequences, longest)) * heads * head_dim <= 2 ** 26):
                break
        c = packed("", sequences, longest, heads, kv_heads, head_dim, rng.choice(["tokens", "heads"]),
                   rng.random() < 0.9, rng.choice([0, 0, rng.randint(1, 200)]))
    else:
        while True:
            rows, vocab = _log(rng, 1, 4096), _log(rng, 1000, 262144)
            if rows * vocab <= 512 * 131071:
                break
        c = logprobs("", rng.choice(["f32", "bf16"]), rows, vocab, rng.choice([1, 1, 2, 4]),
                     rng.choice([0, 1, 5, 20, rng.randint(1, 64)]))
    c.pop("name")
    return c


# ---- inputs --------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _norm_inputs(case, seed):
    """A residual stream: normal, some channels many times the others' size,
    rows of different sizes."""
    g, rows, dim = _gen(seed), case["rows"], case["dim"]
    channel = 1.0 + 15.0 * (torch.rand(dim, generator=g, device="cuda") < 0.01)
    size = torch.exp(_randn(g, rows, 1) * 0.5)
    x = (_randn(g, rows, dim) * channel * size).to(TORCH[case["dtype"]])
    residual = (_randn(g, rows, dim) * channel).to(TORCH[case["dtype"]]) if case["residual"] else None
    weight = 1.0 + 0.2 * _randn(g, dim)
    return x, residual, weight


def _rows_i8(g, rows, cols):
    """Normal rows in 8 bits, each by its largest value, and their scales."""
    x = _randn(g, rows, cols)
    unit = x.abs().amax(dim=1) / 127.0
    return torch.round(x / unit[:, None]).clamp_(-127, 127).to(torch.int8), unit


def _gemm_inputs(case, seed):
    g = _gen(seed)
    x, x_scale = _rows_i8(g, case["tokens"], case["cols"])
    w, w_scale = _rows_i8(g, case["rows"], case["cols"])
    return x, x_scale, w, w_scale * case["cols"] ** -0.5


def _lens(sequences, longest) -> list[int]:
    """Lengths up to `longest`, spread over their logarithm; every 16th slot is
    empty."""
    lens = [round(longest ** ((i + 1) / sequences)) for i in range(sequences)]
    return [0 if i % 16 == 7 else n for i, n in enumerate(lens)]


def _packed_inputs(case, seed):
    g = _gen(seed)
    h, kv, d = (case[x] for x in ("heads", "kv_heads", "head_dim"))
    lens = torch.tensor(_lens(case["sequences"], case["longest"]), device="cuda")
    lens = lens[torch.randperm(len(lens), generator=g, device="cuda")]
    offsets = torch.cat((lens.new_zeros(1), torch.cumsum(lens, dim=0))).to(torch.int32)
    total = sum(_lens(case["sequences"], case["longest"])) + case["pad"]
    if case["layout"] == "tokens":
        qkv = _randn(g, total, h + 2 * kv, d).to(torch.bfloat16)
        q, k, v = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
    else:  # seen as [tokens, heads, head_dim] too
        q, k, v = (_randn(g, n, total, d).to(torch.bfloat16).transpose(0, 1) for n in (h, kv, kv))
    return q, k, v, offsets


def _logprobs_inputs(case, seed):
    """Logits as a trained classifier gives them (a broad bulk and a few dozen
    likely tokens a row); the given tokens mostly likely ones."""
    g, rows, vocab, given = _gen(seed), case["rows"], case["vocab"], case["given"]
    logits = _randn(g, rows, vocab) * 2.0
    step = vocab // 40
    at = torch.randint(0, step, (rows, 40), generator=g, device="cuda") + torch.arange(40, device="cuda") * step
    logits.scatter_(1, at, _randn(g, rows, 40) * 2.5 + 11.0)
    logits = logits.to(TORCH[case["dtype"]])
    likely = at.gather(1, torch.randint(0, 40, (rows, given), generator=g, device="cuda"))
    any_ = torch.randint(0, vocab, (rows, given), generator=g, device="cuda")
    pick = torch.rand((rows, given), generator=g, device="cuda") < 0.8
    return logits, torch.where(pick, likely, any_).to(torch.int32)


def prepare(case, seed):
    st = {"case": case}
    if case["kind"] == "norm":
        rows, dim, mode = case["rows"], case["dim"], case["mode"]
        st["x"], st["residual"], st["weight"] = _norm_inputs(case, seed)
        st["sum"] = torch.empty_like(st["x"]) if case["residual"] else None
        st["y"] = torch.empty((rows, dim), device="cuda", dtype=torch.bfloat16) if mode in ("bf16", "both") else None
        st["q"], st["q_scale"] = None, None
        if mode != "bf16":
            st["q"] = torch.empty((rows, dim), device="cuda", dtype=torch.int8)
            st["q_scale"] = torch.empty(rows, device="cuda")
    elif case["kind"] == "gemm":
        for name, t in zip(("x", "x_scale", "w", "w_scale"), _gemm_inputs(case, seed)):
            st[name] = t
        st["y"] = torch.empty((case["tokens"], case["rows"]), device="cuda", dtype=TORCH[case["dtype"]])
    elif case["kind"] == "packed":
        for name, t in zip(("q", "k", "v", "offsets"), _packed_inputs(case, seed)):
            st[name] = t
        total, h, d = st["q"].shape
        st["o"] = torch.zeros((total, h, d), device="cuda", dtype=torch.bfloat16)
        st["lse"] = torch.zeros((h, total), device="cuda")
    else:
        st["logits"], st["given"] = _logprobs_inputs(case, seed)
        rows, top = case["rows"], case["top"]
        st["logprob"] = torch.empty((rows, case["given"]), device="cuda")
        st["entropy"] = torch.empty(rows, device="cuda")
        st["top_tokens"] = torch.empty((rows, top), device="cuda", dtype=torch.int32)
        st["top_logprob"] = torch.empty((rows, top), device="cuda")
    return st


# ---- one pass ------------------------------------------------------------

def run(st):
    return {"norm": _run_norm, "gemm": _run_gemm, "packed": _run_packed,
            "logprobs": _run_logprobs}[st["case"]["kind"]](st)


def _ptr(t):
    return t.data_ptr() if t is not None and t.numel() else None


def _ok(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what} returned {rc}")


def _run_norm(st):
    c = st["case"]
    if own:
        if c["mode"] == "quantize":
            from vx_amd.runtime import quantize_i8 as call
            _ok(call(lib(), c["dtype"], _ptr(st["x"]), _ptr(st["q"]), _ptr(st["q_scale"]), c["rows"], c["dim"]),
                "quantize_i8")
        else:
            from vx_amd.runtime import rms_norm as call
            _ok(call(lib(), c["dtype"], _ptr(st["x"]), _ptr(st["residual"]), _ptr(st["weight"]), _ptr(st["sum"]),
                     _ptr(st["y"]), _ptr(st["q"]), _ptr(st["q_scale"]), c["rows"], c["dim"], EPS), "rms_norm")
        return {name: st[name] for name in ("sum", "y", "q", "q_scale")}
    out = dict.fromkeys(("sum", "y", "q", "q_scale"))
    s = st["x"].float()
    if st["residual"] is not None:
        s = s + st["residual"].float()
        out["sum"] = s.to(st["x"].dtype)
    t, r = s, None
    if c["mode"] != "quantize":
        # squares of 16384 elements: their sum in 64 bits
        r = torch.rsqrt(s.double().square().mean(dim=1) + EPS).float()
        t = s * st["weight"]
    if c["mode"] in ("bf16", "both"):
        out["y"] = (s * r[:, None] * st["weight"]).to(torch.bfloat16)
    if c["mode"] != "bf16":
        # 127 as a tensor: by a plain number, torch multiplies by its reciprocal
        unit = t.abs().amax(dim=1) / torch.full((), 127.0, device="cuda").expand(c["rows"])
        unit = torch.where(unit > 0, unit, 1.0)
        out["q"] = torch.round(t / unit[:, None]).to(torch.int8)
        out["q_scale"] = unit if r is None else unit * r
    return out


def _run_gemm(st):
    c = st["case"]
    if own:
        from vx_amd.runtime import gemm_i8 as call
        _ok(call(lib(), c["dtype"], _ptr(st["x"]), _ptr(st["x_scale"]), _ptr(st["w"]), _ptr(st["w_scale"]),
                 _ptr(st["y"]), c["tokens"], c["rows"], c["cols"]), "gemm_i8")
        return {"y": st["y"]}
    y = torch.matmul(st["x"].float(), st["w"].float().T)
    return {"y": (y * st["x_scale"][:, None] * st["w_scale"][None, :]).to(st["y"].dtype)}


def _run_packed(st):
    c = st["case"]
    h, kv, d, n, length = (c[x] for x in ("heads", "kv_heads", "head_dim", "sequences", "longest"))
    total = st["q"].shape[0]
    if own:
        from vx_amd.runtime import flash_attention_packed as call
        _ok(call(lib(), _ptr(st["q"]), _ptr(st["k"]), _ptr(st["v"]), _ptr(st["offsets"]), _ptr(st["o"]),
                 _ptr(st["lse"]), total, n, h, kv, d, d ** -0.5, c["causal"], q_strides=st["q"].stride()[:2],
                 kv_strides=st["k"].stride()[:2], o_strides=st["o"].stride()[:2]), "flash_attention_packed")
        return {"o": st["o"], "lse": st["lse"]}
    # padded to the longest: [sequence, kv head, query head of it and position, d]
    begin = st["offsets"][:-1].long()
    lens = (st["offsets"][1:] - st["offsets"][:-1]).long()
    place = torch.arange(length, device="cuda")
    row = (begin[:, None] + place[None, :]).clamp_(max=total - 1)
    q = st["q"].float()[row].view(n, length, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, d)
    k, v = (st[x].float()[row].transpose(1, 2).contiguous() for x in ("k", "v"))
    s = torch.matmul(q * d ** -0.5, k.transpose(2, 3))
    hide = (place[None, :] >= lens[:, None])[:, None, None, None, :]
    if c["causal"]:
        hide = hide | (place[None, :] > place[:, None])[None, None, None]
    s.view(n, kv, h // kv, length, length).masked_fill_(hide, -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    s = s.sub_(top).exp_()
    weight = s.sum(dim=-1, keepdim=True)
    o = (torch.matmul(s, v) / weight).view(n, kv, h // kv, length, d).permute(0, 3, 1, 2, 4).reshape(n, length, h, d)
    lse = (top + torch.log(weight)).view(n, h, length)
    # back to packed rows; those behind the last sequence stay as they were
    token = torch.arange(total, device="cuda")
    seq = torch.searchsorted(st["offsets"][1:].long(), token, right=True)
    live = seq < n
    seq = seq.clamp(max=n - 1)
    at = torch.where(live, token - begin[seq], 0)
    o = torch.where(live[:, None, None], o[seq, at], st["o"].float()).to(torch.bfloat16)
    return {"o": o, "lse": torch.where(live[None, :], lse[seq, :, at].T, st["lse"])}


def _run_logprobs(st):
    c = st["case"]
    if own:
        from vx_amd.runtime import token_logprobs as call
        _ok(call(lib(), c["dtype"], _ptr(st["logits"]), _ptr(st["given"]), _ptr(st["logprob"]), _ptr(st["entropy"]),
                 _ptr(st["top_tokens"]), _ptr(st["top_logprob"]), c["rows"], c["vocab"], c["given"], c["top"]),
            "token_logprobs")
        return {name: st[name] for name in ("logprob", "entropy", "top_tokens", "top_logprob")}
    x = st["logits"].float()
    t = x - x.amax(dim=1, keepdim=True)
    w = torch.exp(t)
    total = w.sum(dim=1, keepdim=True)
    norm_ = torch.log(total)
    logprob = t.gather(1, st["given"].long()) - norm_
    entropy = (norm_ - (w * t).sum(dim=1, keepdim=True) / total)[:, 0]
    index = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :c["top"]]
    return {"logprob": logprob, "entropy": entropy, "top_tokens": index.to(torch.int32),
            "top_logprob": t.gather(1, index) - norm_}


# ---- what a pass cannot do without ---------------------------------------

def work(case) -> dict:
    if case["kind"] == "norm":
        size, n = BYTES[case["dtype"]], case["rows"] * case["dim"]
        each = size * (3 if case["residual"] else 1)
        each += {"i8": 1, "bf16": 2, "both": 3, "quantize": 1}[case["mode"]]
        return {"bytes": n * each + case["dim"] * 4 + case["rows"] * 4, "flops": 5.0 * n}
    if case["kind"] == "gemm":
        t, r, k = case["tokens"], case["rows"], case["cols"]
        return {"bytes": t * k + r * k + t * r * BYTES[case["dtype"]] + 4 * (t + r), "flops": 2.0 * t * r * k}
    if case["kind"] == "packed":
        h, kv, d = (case[x] for x in ("heads", "kv_heads", "head_dim"))
        lens = _lens(case["sequences"], case["longest"])
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        return {"bytes": sum(lens) * ((2 * h + 2 * kv) * d * 2 + 4 * h), "flops": 4.0 * d * h * pairs}
    r, v = case["rows"], case["vocab"]
    return {"bytes": r * v * BYTES[case["dtype"]] + r * (case["given"] * 8 + 4 + case["top"] * 8),
            "flops": 4.0 * r * v}


# ---- the definition in 64 bits -------------------------------------------

def exact(case, seed):
    return {"norm": _exact_norm, "gemm": _exact_gemm, "packed": _exact_packed,
            "logprobs": _exact_logprobs}[case["kind"]](case, seed)


def _exact_norm(case, seed):
    """Quantized values have no 64-bit counterpart: None in their place."""
    x, residual, weight = _norm_inputs(case, seed)
    out = dict.fromkeys(("sum", "y", "q", "q_scale"))
    x = x.double()
    if residual is not None:
        x += residual.double()
        out["sum"] = x
    gain = torch.ones((), device="cuda", dtype=torch.float64)
    if case["mode"] != "quantize":
        root = torch.sqrt((x * x).sum(dim=1) / case["dim"] + EPS)
        gain = weight.double()[None, :] / root[:, None]
    y = x * gain
    if case["mode"] in ("bf16", "both"):
        out["y"] = y
    if case["mode"] != "bf16":
        out["q_scale"] = torch.maximum(y.amax(dim=1), -y.amin(dim=1)) / 127.0
    return out


def _exact_gemm(case, seed):
    x, x_scale, w, w_scale = _gemm_inputs(case, seed)
    x = x.double() * x_scale.double()[:, None]
    y = torch.empty((case["tokens"], case["rows"]), device="cuda", dtype=torch.float64)
    for r in range(0, case["rows"], 4096):  # 4096 rows of weights at a time
        part = w[r:r + 4096].double() * w_scale[r:r + 4096].double()[:, None]
        y[:, r:r + 4096] = x @ part.T.contiguous()
    return {"y": y}


def _exact_packed(case, seed):
    q, k, v, offsets = _packed_inputs(case, seed)
    group = case["heads"] // case["kv_heads"]
    o = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    lse = torch.zeros((q.shape[1], q.shape[0]), device="cuda", dtype=torch.float64)
    bounds = offsets.tolist()
    for first, last in zip(bounds, bounds[1:]):
        for g in range(case["kv_heads"] if last > first else 0):
            keys, values = k[first:last, g].double(), v[first:last, g].double()
            for h in range(g * group, (g + 1) * group):
                s = (q[first:last, h].double() @ keys.T.contiguous()) * case["head_dim"] ** -0.5
                if case["causal"]:
                    s = s.masked_fill_(torch.ones_like(s, dtype=torch.bool).triu_(1), -math.inf)
                norm_ = torch.logsumexp(s, dim=-1, keepdim=True)
                o[first:last, h] = torch.exp(s - norm_) @ values
                lse[h, first:last] = norm_[:, 0]
    return {"o": o, "lse": lse}


def _exact_logprobs(case, seed):
    logits, given = _logprobs_inputs(case, seed)
    rows, top = case["rows"], case["top"]
    out = {"logprob": torch.empty((rows, case["given"]), dtype=torch.float64, device="cuda"),
           "entropy": torch.empty(rows, dtype=torch.float64, device="cuda"),
           "top_tokens": torch.empty((rows, top), dtype=torch.int32, device="cuda"),
           "top_logprob": torch.empty((rows, top), dtype=torch.float64, device="cuda")}
    for r in range(0, rows, 64):  # 64 rows at a time
        x = logits[r:r + 64].double()
        logp = x - torch.logsumexp(x, dim=1, keepdim=True)
        out["logprob"][r:r + 64] = logp.gather(1, given[r:r + 64].long())
        out["entropy"][r:r + 64] = -(torch.exp(logp) * logp).sum(dim=1)
        order = torch.argsort(x, dim=1, descending=True, stable=True)[:, :top]
        out["top_tokens"][r:r + 64] = order
        out["top_logprob"][r:r + 64] = logp.gather(1, order)
    return out
