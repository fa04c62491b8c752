"""Plain implementations in 64 bits of the ops of a batch that shares a prompt
(include/vx_hip_ops.h), and what their results may be off by.

A rounding to bf16 is off by at most 2^-8 of the value, one to f32 by 2^-24.
"""

from __future__ import annotations

import numpy as np

from vx_amd.abi import bf16_to_f32

BF16, F32 = 2.0 ** -8, 2.0 ** -24


def rope_table(rows: int, head_dim: int, base: float = 10000.0) -> np.ndarray:
    ang = np.arange(rows)[:, None] * base ** (-np.arange(0, head_dim, 2) / head_dim)[None, :]
    return np.stack([np.cos(ang), np.sin(ang)], axis=-1).astype(np.float32)


def rope_append(qkv, table, lens, q, k, v, shared_len):
    """float64 q, k, v after the call, and the bound of each, from qkv [batch, n,
    heads + 2 kv, d] and what q, k, v held (float64)."""
    b, n, _, d = qkv.shape
    h, kv = q.shape[1], k.shape[1]
    cap = k.shape[2]
    q, k, v = q.copy(), k.copy(), v.copy()
    tol = [np.zeros_like(x) for x in (q, k, v)]
    x = qkv.astype(np.float64)
    for s in range(b):
        length = cap if lens is None else int(lens[s])
        if length < 0 or length > cap:
            continue
        for i in range(n):
            at = length - n + i
            pos = shared_len + at
            y = x[s, i].copy()
            bound = BF16 * np.abs(y)
            if pos < 0:
                y[:] = 0
            elif table is not None:
                c, sn = table[pos, :, 0].astype(np.float64), table[pos, :, 1].astype(np.float64)
                e, o = x[s, i, :h + kv, 0::2], x[s, i, :h + kv, 1::2]
                y[:h + kv, 0::2] = e * c - o * sn
                y[:h + kv, 1::2] = e * sn + o * c
                # two products and a sum in f32, then one rounding
                size = np.repeat(np.abs(e) + np.abs(o), 2, axis=-1)
                bound[:h + kv] = BF16 * np.abs(y[:h + kv]) + 4 * F32 * size
            q[s, :, i], tol[0][s, :, i] = y[:h], bound[:h]
            if at >= 0:
                k[s, :, at], tol[1][s, :, at] = y[h:h + kv], bound[h:h + kv]
                v[s, :, at], tol[2][s, :, at] = y[h + kv:], bound[h + kv:]
    return (q, k, v), tol


def shared_attention(q16, ks16, vs16, k16, v16, lens, shared_len, scale, causal):
    """float64 o and lse (NaN where the slot holds no sequence), and the bounds
    of both. Scores are sums of head_dim f32 products, weights are rounded to
    bf16 for their product with v, sums and statistics are f32."""
    b, h, n, d = q16.shape
    kv = (k16 if k16 is not None else ks16).shape[-3]
    cap = k16.shape[2] if k16 is not None else 0
    group = h // kv
    o, lse = np.full((b, h, n, d), np.nan), np.full((b, h, n), np.nan)
    o_tol, lse_tol = np.zeros((b, h, n, d)), np.zeros((b, h, n))
    for s in range(b):
        length = cap if lens is None else int(lens[s])
        if length < 0 or length > cap:
            continue
        for g in range(kv):
            keys, values = np.zeros((0, d)), np.zeros((0, d))
            if shared_len:
                keys = bf16_to_f32(ks16[g, :shared_len]).astype(np.float64)
                values = bf16_to_f32(vs16[g, :shared_len]).astype(np.float64)
            if length:
                keys = np.concatenate([keys, bf16_to_f32(k16[s, g, :length]).astype(np.float64)])
                values = np.concatenate([values, bf16_to_f32(v16[s, g, :length]).astype(np.float64)])
            for hh in range(g * group, (g + 1) * group):
                x = bf16_to_f32(q16[s, hh]).astype(np.float64)
                for i in range(n):
                    end = len(keys) - (n - 1 - i) if causal else len(keys)
                    if end <= 0:
                        o[s, hh, i], lse[s, hh, i] = 0, -np.inf
                        continue
                    kk, vv = keys[:end], values[:end]
                    sc = (kk @ x[i]) * scale
                    top = sc.max()
                    w = np.exp(sc - top)
                    total = w.sum()
                    o[s, hh, i] = w @ vv / total
                    lse[s, hh, i] = top + np.log(total)
                    size = w @ np.abs(vv) / total
                    # a score, its exponent's argument (in base 2, against a
                    # maximum up to 8 away) and the exponential
                    delta = (F32 * ((d + 4) * (np.abs(kk) @ np.abs(x[i])).max() * abs(scale) +
                                    4 * (np.abs(top) + 12)) + 4 * F32)
                    sums = (end + 16) * F32
                    o_tol[s, hh, i] = BF16 * (np.abs(o[s, hh, i]) * 1.01 + size) + size * 2 * (delta + sums)
                    lse_tol[s, hh, i] = delta + sums + 4 * F32 * abs(lse[s, hh, i])
    return (o, lse), (o_tol, lse_tol)


def sample(logits, temperature, top_k, top_p, min_p, u):
    """(tokens, logprob) of float logits [rows, vocab] by the definition; the
    settings are arrays of a value per row, or None."""
    rows, vocab = logits.shape
    tokens, logprob = np.full(rows, -1, np.int32), np.full(rows, -np.inf)
    for r in range(rows):
        x = logits[r].astype(np.float64)
        x = np.where(np.isnan(x), -np.inf, x)
        order = np.lexsort((np.arange(vocab), -x))
        order = order[x[order] > -np.inf]
        if not len(order):
            continue
        heat = 1.0 if temperature is None else float(temperature[r])
        if not heat > 0:
            tokens[r], logprob[r] = order[0], 0.0
            continue
        if np.isposinf(x[order[0]]):
            w = np.isposinf(x[order]).astype(np.float64)
        else:
            w = np.exp(x[order] / heat - x[order[0]] / heat)
        keep = len(order)
        if top_k is not None and top_k[r] > 0:
            keep = min(keep, int(top_k[r]))
        p = 1.0 if top_p is None else float(top_p[r])
        if p < 1:
            before = np.concatenate([[0.0], np.cumsum(w[:keep])])
            keep = max(1, int(np.sum(before[:-1] < p * before[-1])))
        m = 0.0 if min_p is None else float(min_p[r])
        if m > 0:
            keep = max(1, min(keep, int(np.sum(w >= min(m, 1.0)))))
        kept = np.sort(order[:keep])
        weight = dict(zip(order[:keep].tolist(), w[:keep].tolist()))
        w = np.array([weight[int(i)] for i in kept])
        cum = np.cumsum(w)
        at = float(u[r])
        at = 0.0 if not at > 0 else min(at, 1 - 2.0 ** -24)
        pick = min(int(np.searchsorted(cum, at * cum[-1], side="right")), len(kept) - 1)
        tokens[r], logprob[r] = kept[pick], np.log(w[pick] / cum[-1])
    return tokens, logprob


def logprob_tol(want):
    """One rounding to f32, and weights to 2^-40 of the sum."""
    return F32 * np.abs(np.where(np.isfinite(want), want, 0)) + 2.0 ** -30
