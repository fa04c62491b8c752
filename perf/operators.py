"""Performance cases of the operators behind many answers to one prompt: the
rotation of a fused projection and its append to each sequence's own cache,
attention over a prefix that all sequences share and their own caches, and
sampling of the next tokens from logits and given uniform numbers.

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

_lib: list = []


def lib():
    if not _lib:
        from vx_amd.runtime import DispatchLibrary
        _lib.append(DispatchLibrary())
    return _lib[0]


# ---- cases ---------------------------------------------------------------

def sample(name, dtype, rows, vocab, mode) -> dict:
    return {"name": name, "kind": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "mode": mode}


def shared(name, batch, heads, kv_heads, head_dim, seq_q, shared_len, capacity, causal=True) -> dict:
    return {"name": name, "kind": "shared", "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "seq_q": seq_q, "shared_len": shared_len, "capacity": capacity,
            "causal": causal}


def rope(name, dtype, batch, heads, kv_heads, head_dim, seq_q, shared_len, capacity) -> dict:
    return {"name": name, "kind": "rope", "dtype": dtype, "batch": batch, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "seq_q": seq_q, "shared_len": shared_len,
            "capacity": capacity}


def listed() -> list[dict]:
    return [
        # One user's next token at the decoder's vocabulary: top-k and a
        # temperature, where latency counts.
        sample("sample_1x32000_topk", "f32", 1, 32000, "topk"),
        # A serving batch whose requests bring their own settings, greedy ones
        # among them.
        sample("sample_48x32000_mixed", "f32", 48, 32000, "mixed"),
        # A few answers at a large vocabulary, logits in bf16 as a 16-bit
        # classifier leaves them (many ties), nucleus sampling.
        sample("sample_8x131072_topp", "bf16", 8, 131072, "topp"),
        # The largest batch, temperature alone, a vocabulary of odd size.
        sample("sample_256x131071_plain", "f32", 256, 131071, "plain"),
        # Four answers to a short prompt with the decoder's heads: the
        # smallest call of a step.
        shared("shared_4x1_at500", 4, 12, 12, 64, 1, 500, 64),
        # 64 requests behind one system prompt, 32 query heads on 4 KV heads
        # as in the chunk-attention benchmark.
        shared("shared_64x1_at8192", 64, 32, 4, 128, 1, 8192, 512),
        # 16 answers about one long document.
        shared("shared_16x1_at65536", 16, 32, 8, 128, 1, 65536, 1024),
        # Five drafted tokens a sequence; odd batch, heads and lengths.
        shared("shared_33x5_at2047", 33, 21, 3, 64, 5, 2047, 333),
        # The questions of eight users after one prompt, prefilled together.
        shared("shared_8x256_at4096", 8, 32, 8, 128, 256, 4096, 300),
        # The projections of those steps: a few sequences, a batch, a chunk.
        rope("rope_4x1_h12", "bf16", 4, 12, 12, 64, 1, 500, 64),
        rope("rope_64x1_h32", "f32", 64, 32, 4, 128, 1, 8192, 512),
        rope("rope_8x256_h32", "bf16", 8, 32, 8, 128, 256, 4096, 300),
    ]


def _log(rng, lo, hi) -> int:
    """A size spread over the logarithm of its range."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["sample", "sample", "shared", "shared", "shared", "rope"])
    if kind == "sample":
        while True:
            rows, vocab = _log(rng, 1, 256), _log(rng, 1000, 262144)
            if rows * vocab <= 256 * 131071:
                break
        c = sample("", rng.choice(["f32", "bf16"]), rows, vocab,
                   rng.choice(["plain", "topk", "topp", "minp", "mixed"]))
    else:
        while True:
            head_dim, kv_heads = rng.choice([64, 128]), rng.choice([1, 2, 3, 4, 8, 12])
            heads = kv_heads * rng.choice([1, 1, 3, 4, 7, 8])
            batch = _log(rng, 1, 256)
            seq_q = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 256)])
            shared_len = _log(rng, 16, 65536)
            capacity = seq_q + _log(rng, 1, 1024)
            flops = 4.0 * batch * heads * seq_q * (shared_len + capacity) * head_dim
            scores = batch * heads * seq_q * (shared_len + capacity)
            if (heads <= 64 and flops <= 1.4e11 and scores <= 2 ** 28 and
                    batch * kv_heads * capacity * head_dim <= 2 ** 26):
                break
        if kind == "shared":
            c = shared("", batch, heads, kv_heads, head_dim, seq_q, shared_len, capacity, rng.random() < 0.9)
        else:
            c = rope("", rng.choice(["f32", "bf16"]), batch, heads, kv_heads, head_dim, seq_q, shared_len,
                     capacity)
    c.pop("name")
    return c


# ---- inputs --------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _sample_inputs(case, seed):
    """Logits as a trained classifier gives them (a broad bulk and a few dozen
    likely tokens a row), each row's settings, and its uniform number."""
    g, rows, vocab, mode = _gen(seed), case["rows"], case["vocab"], case["mode"]

    def uniform(lo, hi):
        return torch.rand(rows, generator=g, device="cuda") * (hi - lo) + lo

    logits = torch.randn((rows, vocab), generator=g, device="cuda") * 2.0
    step = vocab // 40
    at = torch.randint(0, step, (rows, 40), generator=g, device="cuda") + torch.arange(40, device="cuda") * step
    logits.scatter_(1, at, torch.randn((rows, 40), generator=g, device="cuda") * 2.5 + 11.0)
    logits = logits.to(TORCH[case["dtype"]])
    temperature, top_k, top_p, min_p = uniform(0.6, 1.2), None, None, None
    if mode in ("topk", "mixed"):
        top_k = torch.randint(1, 100, (rows,), generator=g, device="cuda", dtype=torch.int32)
    if mode in ("topp", "mixed"):
        top_p = uniform(0.5, 0.99)
    if mode in ("minp", "mixed"):
        min_p = uniform(0.01, 0.2)
    if mode == "mixed":  # each setting off in some rows, and every eighth row greedy
        row = torch.arange(rows, device="cuda")
        temperature[row % 8 == 3] = 0.0
        top_k[row % 3 == 0] = 0
        top_p[row % 4 == 1] = 1.0
        min_p[row % 2 == 0] = 0.0
    u = torch.rand(rows, generator=g, device="cuda")
    return logits, temperature, top_k, top_p, min_p, u


def _lens(case, g):
    """How many of its own keys each sequence has, the new ones among them:
    spread evenly from the fewest to the most, in random order; one slot of
    every 16 holds no sequence (-1)."""
    b, n, cap = case["batch"], case["seq_q"], case["capacity"]
    i = torch.arange(b, device="cuda")
    lens = n + (i * (cap - n)) // max(b - 1, 1)
    lens[i % 16 == 15] = -1
    return lens[torch.randperm(b, generator=g, device="cuda")].to(torch.int32)


def _lens_sum(case) -> tuple[int, int]:
    """The sequences of a case and their keys in all."""
    b, n, cap = case["batch"], case["seq_q"], case["capacity"]
    lens = [n + (i * (cap - n)) // max(b - 1, 1) for i in range(b) if i % 16 != 15]
    return len(lens), sum(lens)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def _shared_inputs(case, seed):
    g = _gen(seed)
    b, h, kv, d = (case[x] for x in ("batch", "heads", "kv_heads", "head_dim"))
    lens = _lens(case, g)
    q = _normal(g, b, h, case["seq_q"], d)
    ks, vs = _normal(g, kv, case["shared_len"], d), _normal(g, kv, case["shared_len"], d)
    k, v = _normal(g, b, kv, case["capacity"], d), _normal(g, b, kv, case["capacity"], d)
    return q, ks, vs, k, v, lens


def _rope_inputs(case, seed):
    g = _gen(seed)
    b, h, kv, d = (case[x] for x in ("batch", "heads", "kv_heads", "head_dim"))
    lens = _lens(case, g)
    qkv = torch.randn((b, case["seq_q"], h + 2 * kv, d), generator=g, device="cuda").to(TORCH[case["dtype"]])
    k, v = _normal(g, b, kv, case["capacity"], d), _normal(g, b, kv, case["capacity"], d)
    pos = torch.arange(case["shared_len"] + case["capacity"], device="cuda", dtype=torch.float64)
    inv = 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    ang = pos[:, None] * inv[None, :]
    return qkv, torch.stack((torch.cos(ang), torch.sin(ang)), dim=-1).float(), lens, k, v


def prepare(case, seed):
    st = {"case": case}
    if case["kind"] == "sample":
        for name, t in zip(("logits", "temperature", "top_k", "top_p", "min_p", "u"), _sample_inputs(case, seed)):
            st[name] = t
        st["tokens"] = torch.empty(case["rows"], device="cuda", dtype=torch.int32)
        st["logprob"] = torch.empty(case["rows"], device="cuda")
    elif case["kind"] == "shared":
        for name, t in zip(("q", "ks", "vs", "k", "v", "lens"), _shared_inputs(case, seed)):
            st[name] = t
        st["o"] = torch.zeros_like(st["q"])
        st["lse"] = torch.zeros(st["q"].shape[:3], device="cuda")
    else:
        for name, t in zip(("qkv", "table", "lens", "k", "v"), _rope_inputs(case, seed)):
            st[name] = t
        st["q"] = torch.zeros((case["batch"], case["heads"], case["seq_q"], case["head_dim"]), device="cuda",
                              dtype=torch.bfloat16)
    return st


# ---- one pass ------------------------------------------------------------

def run(st):
    return {"sample": _run_sample, "shared": _run_shared, "rope": _run_rope}[st["case"]["kind"]](st)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _ok(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what} returned {rc}")


def _run_sample(st):
    if own:
        from vx_amd.runtime import sample as call
        c = st["case"]
        _ok(call(lib(), c["dtype"], _ptr(st["logits"]), _ptr(st["temperature"]), _ptr(st["top_k"]),
                 _ptr(st["top_p"]), _ptr(st["min_p"]), _ptr(st["u"]), _ptr(st["tokens"]), _ptr(st["logprob"]),
                 c["rows"], c["vocab"]), "sample")
        return {"tokens": st["tokens"], "logprob": st["logprob"]}
    rows, vocab = st["logits"].shape
    logits = st["logits"].double()
    greedy = st["temperature"] <= 0
    t = logits / torch.where(greedy, 1.0, st["temperature"].double())[:, None]
    if st["top_k"] is None and st["top_p"] is None and st["min_p"] is None:
        top = t.amax(dim=1, keepdim=True)
        index = torch.arange(vocab, device=t.device)[None, :]
        best = torch.where(t == top, index, vocab).amin(dim=1, keepdim=True)
        by_index = torch.where(greedy[:, None] & (index != best), 0.0, torch.exp(t - top))
    else:
        by_index = _filtered(st, t, greedy)
    cum = torch.cumsum(by_index, dim=1)
    total = cum[:, -1:]
    token = (cum <= st["u"].double()[:, None] * total).sum(dim=1, keepdim=True)
    logprob = torch.log(by_index.gather(1, token) / total)
    return {"tokens": token[:, 0].to(torch.int32), "logprob": logprob[:, 0].float()}


def _filtered(st, t, greedy):
    """The weights of the tokens that the settings keep, 0 for the others."""
    t, order = torch.sort(t, dim=1, descending=True, stable=True)
    w = torch.exp(t - t[:, :1])
    rank = torch.arange(t.shape[1], device=w.device)[None, :]
    keep = ~greedy[:, None] | (rank == 0)
    if st["top_k"] is not None:
        keep &= (rank < st["top_k"][:, None]) | (st["top_k"][:, None] <= 0)
    if st["top_p"] is not None:
        kept = torch.where(keep, w, 0.0)
        before = torch.cumsum(kept, dim=1) - kept
        p = st["top_p"].double()[:, None]
        keep = keep & ((before < p * kept.sum(dim=1, keepdim=True)) | (p >= 1))
    if st["min_p"] is not None:
        keep = keep & (w >= st["min_p"].double()[:, None])
    keep |= rank == 0
    return torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))


def _run_shared(st):
    c = st["case"]
    if own:
        from vx_amd.runtime import flash_attention_shared as call
        _ok(call(lib(), _ptr(st["q"]), _ptr(st["ks"]), _ptr(st["vs"]), _ptr(st["k"]), _ptr(st["v"]),
                 _ptr(st["lens"]), _ptr(st["o"]), _ptr(st["lse"]), c["batch"], c["heads"], c["kv_heads"],
                 c["seq_q"], c["shared_len"], c["capacity"], c["head_dim"], c["head_dim"] ** -0.5, c["causal"]),
            "flash_attention_shared")
        return {"o": st["o"], "lse": st["lse"]}
    b, h, kv, n, d = (c[x] for x in ("batch", "heads", "kv_heads", "seq_q", "head_dim"))
    p, cap, rows = c["shared_len"], c["capacity"], h // kv * n
    q = st["q"].float().view(b, kv, rows, d) * d ** -0.5
    ks, vs, k, v = (st[x].float() for x in ("ks", "vs", "k", "v"))
    s = torch.empty((b, kv, rows, p + cap), device=q.device)
    by_kv = q.transpose(0, 1).reshape(kv, b * rows, d)
    s[..., :p] = torch.matmul(by_kv, ks.transpose(1, 2)).view(kv, b, rows, p).transpose(0, 1)
    s[..., p:] = torch.matmul(q, k.transpose(2, 3))
    lens = st["lens"].long()[:, None]
    key = torch.arange(cap, device=q.device)
    last = lens - 1
    if c["causal"]:
        last = last - (n - 1) + torch.arange(n, device=q.device)[None, :]
    hide = key[None, None, :] > last[:, :, None]
    s.view(b, kv, h // kv, n, p + cap)[..., p:].masked_fill_(hide[:, None, None], -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    s = torch.exp(s - top)
    total = s.sum(dim=-1, keepdim=True)
    o = torch.matmul(s[..., :p].transpose(0, 1).reshape(kv, b * rows, p), vs).view(kv, b, rows, d).transpose(0, 1)
    o = (o + torch.matmul(s[..., p:], v)) / total
    live = (st["lens"] >= 0)[:, None, None]
    o = torch.where(live[..., None], o.reshape(b, h, n, d), 0.0).to(torch.bfloat16)
    return {"o": o, "lse": torch.where(live, (top + torch.log(total)).view(b, h, n), 0.0)}


def _run_rope(st):
    c = st["case"]
    b, h, kv, n, d = (c[x] for x in ("batch", "heads", "kv_heads", "seq_q", "head_dim"))
    if own:
        from vx_amd.runtime import rope_append as call
        _ok(call(lib(), c["dtype"], _ptr(st["qkv"]), _ptr(st["table"]), _ptr(st["lens"]), _ptr(st["q"]),
                 _ptr(st["k"]), _ptr(st["v"]), b, n, h, kv, d, c["shared_len"], c["capacity"],
                 st["table"].shape[0]), "rope_append")
        return {"q": st["q"], "k": st["k"], "v": st["v"]}
    x = st["qkv"].float()
    at = st["lens"].long()[:, None] - n + torch.arange(n, device=x.device)[None, :]
    live = (st["lens"] >= 0)[:, None].expand(b, n)
    turn = st["table"][torch.where(live, at, 0) + c["shared_len"]][:, :, None]
    cos, sin = turn[..., 0], turn[..., 1]
    qk = x[:, :, :h + kv]
    even, odd = qk[..., 0::2], qk[..., 1::2]
    qk = torch.stack((even * cos - odd * sin, even * sin + odd * cos), dim=-1).flatten(-2).to(torch.bfloat16)
    q = torch.where(live[:, None, :, None], qk[:, :, :h].transpose(1, 2), 0.0)
    seq = torch.arange(b, device=x.device)[:, None].expand(b, n)[live]
    st["k"][seq, :, at[live]] = qk[:, :, h:][live]
    st["v"][seq, :, at[live]] = x[:, :, h + kv:][live].to(torch.bfloat16)
    return {"q": q, "k": st["k"], "v": st["v"]}


# ---- what a pass cannot do without ---------------------------------------

def work(case) -> dict:
    if case["kind"] == "sample":
        r, v = case["rows"], case["vocab"]
        # a weight for each logit, and its sum
        return {"bytes": r * v * BYTES[case["dtype"]] + r * 28, "flops": 2.0 * r * v}
    h, kv, d, n, p = (case[x] for x in ("heads", "kv_heads", "head_dim", "seq_q", "shared_len"))
    seqs, keys = _lens_sum(case)
    if case["kind"] == "rope":
        tokens = seqs * n
        return {"bytes": tokens * d * ((h + 2 * kv) * (BYTES[case["dtype"]] + 2) + 4), "flops": 3.0 * tokens * d * (h + kv)}
    hidden = seqs * n * (n - 1) // 2 if case["causal"] else 0
    return {"bytes": 4 * kv * d * (p + keys) + seqs * h * n * (4 * d + 4),
            "flops": 4.0 * d * h * (n * (seqs * p + keys) - hidden)}


# ---- the definition in 64 bits -------------------------------------------

def exact(case, seed):
    return {"sample": _exact_sample, "shared": _exact_shared, "rope": _exact_rope}[case["kind"]](case, seed)


def _exact_sample(case, seed):
    """Row by row: the kept tokens are a prefix of the order by falling
    logit and rising index, the draw goes over them by rising index."""
    logits, temperature, top_k, top_p, min_p, u = _sample_inputs(case, seed)
    tokens, logprob = [], []
    for r in range(case["rows"]):
        x = logits[r].double()
        heat = float(temperature[r])
        if heat <= 0:
            tokens.append(int((x == x.max()).nonzero()[0, 0]))
            logprob.append(0.0)
            continue
        value, index = torch.sort(x, descending=True, stable=True)
        weight = torch.exp((value - value[0]) / heat)
        count = case["vocab"]
        if top_k is not None and int(top_k[r]) > 0:
            count = min(count, int(top_k[r]))
        if top_p is not None and float(top_p[r]) < 1:
            running = weight[:count].cumsum(0)
            first = int(torch.searchsorted(running, float(top_p[r]) * running[-1]))
            count = min(count, first + 1)
        if min_p is not None:
            count = min(count, int((weight >= float(min_p[r])).sum()))
        index, by = torch.sort(index[:max(count, 1)])
        running = weight[by].cumsum(0)
        pick = int(torch.searchsorted(running, float(u[r]) * running[-1], right=True))
        tokens.append(int(index[pick]))
        logprob.append(math.log(float(weight[by[pick]]) / float(running[-1])))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "logprob": torch.tensor(logprob, dtype=torch.float64)}


def _exact_shared(case, seed):
    q, ks, vs, k, v, lens = _shared_inputs(case, seed)
    n, group = case["seq_q"], case["heads"] // case["kv_heads"]
    o = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    lse = torch.zeros(q.shape[:3], device="cuda", dtype=torch.float64)
    lens = lens.tolist()
    shared_kv = [(ks[g].double(), vs[g].double()) for g in range(case["kv_heads"])]
    for b in range(case["batch"]):
        if lens[b] < 0:
            continue
        hide = None
        total = case["shared_len"] + lens[b]
        if case["causal"]:
            row = torch.arange(n, device="cuda").repeat(group)[:, None]
            hide = torch.arange(total, device="cuda")[None, :] > row + (total - n)
        for g, (k0, v0) in enumerate(shared_kv):
            keys = torch.cat((k0, k[b, g, :lens[b]].double()))
            values = torch.cat((v0, v[b, g, :lens[b]].double()))
            heads = slice(g * group, (g + 1) * group)
            s = (q[b, heads].reshape(group * n, -1).double() @ keys.T.contiguous()) * case["head_dim"] ** -0.5
            if hide is not None:
                s.masked_fill_(hide, -math.inf)
            norm = torch.logsumexp(s, dim=-1, keepdim=True)
            o[b, heads] = (torch.exp(s - norm) @ values).view(group, n, -1)
            lse[b, heads] = norm.view(group, n)
    return {"o": o, "lse": lse}


def _exact_rope(case, seed):
    qkv, table, lens, k, v = _rope_inputs(case, seed)
    h, kv, n, d = (case[x] for x in ("heads", "kv_heads", "seq_q", "head_dim"))
    q = torch.zeros((case["batch"], h, n, d), device="cuda", dtype=torch.float64)
    k, v = k.double(), v.double()
    for b, length in enumerate(lens.tolist()):
        if length < 0:
            continue
        x = torch.view_as_complex(qkv[b, :, :h + kv].double().reshape(n, h + kv, d // 2, 2))
        first = case["shared_len"] + length - n
        turn = torch.view_as_complex(table[first:first + n].double())
        x = torch.view_as_real(x * turn[:, None]).reshape(n, h + kv, d).transpose(0, 1)
        q[b] = x[:h]
        k[b, :, length - n:length] = x[h:]
        v[b, :, length - n:length] = qkv[b, :, h + kv:].double().transpose(0, 1)
    return {"q": q, "k": k, "v": v}
