"""Plain implementations in 64 bits of the ops of a packed batch in 8 bits
(include/vx_hip_ops.h), and what their results may be off by.

A rounding to bf16 is off by at most 2^-8 of the value, one to f32 by 2^-24.
"""

from __future__ import annotations

import numpy as np

BF16, F32 = 2.0 ** -8, 2.0 ** -24


def rms_norm(x, residual, weight, eps, rounding):
    """float64 (sum, y, q_scale) and their bounds, and q, of f32 values. q is
    defined by f32 operations, so it has no bound: s = x + residual, t = s w, u =
    max |t| / 127, q = rint(t / u). rounding: of the sum's type."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        s32 = x + residual if residual is not None else x
        t = s32 * (weight if weight is not None else np.float32(1.0))
        top = np.abs(t).max(axis=1)
        unit = top / np.float32(127.0)
        unit = np.where(unit > 0, unit, np.float32(1.0)).astype(np.float32)
        finite = np.isfinite(t).all(axis=1)
        q = np.rint(t / unit[:, None]).clip(-127, 127)
        q = np.where(finite[:, None], q, 0).astype(np.int8)
        s = x.astype(np.float64) + (residual.astype(np.float64) if residual is not None else 0.0)
        w = weight.astype(np.float64) if weight is not None else np.ones(x.shape[1])
        r = 1.0 / np.sqrt((s * s).mean(axis=1) + np.float64(np.float32(eps)))
        y = s * r[:, None] * w
        scale = np.where(finite, unit.astype(np.float64) * r, np.nan)
        # past the largest f32 (max |t| below 2^-143 and no eps), it is infinite
        scale = np.where(scale < 2.0 ** 128, scale, scale * np.inf)
    # s, r, and two products in f32, then the rounding to bf16
    tol_y = np.abs(y) * (BF16 + 5 * F32) + 2.0 ** -133
    # one sum in f32, then the rounding of the type (none more for f32)
    tol_sum = np.abs(s) * (F32 + rounding * 1.01)
    # u is the definition's own; s may differ from s32 by 2^-24, r and the
    # product are rounded
    tol_scale = np.abs(scale) * 4 * F32 + 2.0 ** -149
    return (s, y, scale, q), (tol_sum, tol_y, tol_scale)


def gemm_i8(x, x_scale, w, w_scale, bf16):
    """float64 y and its bound: the exact sum, rounded to f32, and two products."""
    total = x.astype(np.int64) @ w.astype(np.int64).T
    y = total * x_scale.astype(np.float64)[:, None] * w_scale.astype(np.float64)[None, :]
    return y, np.abs(y) * (4 * F32 + (BF16 if bf16 else 0.0))


def packed_attention(q, k, v, offsets, scale, causal):
    """float64 o [heads, total, d] and lse [heads, total] (NaN: rows of no
    sequence), and the bounds of both, of q [heads, total, d] and k, v [kv, total,
    d]. Scores are sums of d f32 products, weights are rounded to bf16 for their
    product with v, sums and statistics are f32."""
    h, total, d = q.shape
    group = h // k.shape[0]
    o, lse = np.full((h, total, d), np.nan), np.full((h, total), np.nan)
    o_tol, lse_tol = np.zeros((h, total, d)), np.zeros((h, total))
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    for a, b in zip(offsets, offsets[1:]):
        n = b - a
        if n <= 0:
            continue
        see = np.tril(np.ones((n, n), bool)) if causal else np.ones((n, n), bool)
        for hh in range(h):
            qq, kk, vv = q[hh, a:b], k[hh // group, a:b], v[hh // group, a:b]
            with np.errstate(invalid="ignore"):
                s = np.where(see, (qq @ kk.T) * scale, -np.inf)
                size_s = np.where(see, np.abs(qq) @ np.abs(kk).T, 0.0).max(axis=1)
            top = s.max(axis=1)
            w = np.exp(s - top[:, None])
            z = w.sum(axis=1)
            p = w / z[:, None]
            o[hh, a:b] = p @ vv
            lse[hh, a:b] = top + np.log(z)
            size = p @ np.abs(vv)
            # a score, its exponent's argument (in base 2, against a maximum up
            # to 8 away) and the exponential
            delta = F32 * ((d + 4) * size_s * abs(scale) + 4 * (np.abs(top) + 12)) + 4 * F32
            sums = (see.sum(axis=1) + 16) * F32
            o_tol[hh, a:b] = (BF16 * (np.abs(o[hh, a:b]) * 1.01 + size) +
                              size * 2 * (delta + sums)[:, None])
            lse_tol[hh, a:b] = delta + sums + 4 * F32 * np.abs(lse[hh, a:b])
    return (o, lse), (o_tol, lse_tol)


def token_logprobs(logits, given, n_top):
    """float64 (logprob, entropy, top_tokens, top_logprob) of float logits, and
    the bounds of the three that are computed.

    A thread sums up to e = max(96, vocab / 1024) + 8 weights in f32 (rows of up to
    2048, 4096, 12288 and 49152 have 64, 128, 256 and 512 threads, longer ones
    1024), each e^d off by 2^-23 (|d| + 2), against a reference up to 8 below its
    logits, and some 40 roundings join the threads' sums."""
    x = logits.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    rows, vocab = x.shape
    logprob, entropy = np.full(given.shape, -np.inf), np.zeros(rows)
    top_tokens, top_logprob = np.full((rows, n_top), -1, np.int32), np.full((rows, n_top), -np.inf)
    tol = [np.zeros(a.shape) for a in (logprob, entropy, top_logprob)]
    each = max(96, vocab / 1024) + 8 + 40
    for r in range(rows):
        top = x[r].max()
        if top == -np.inf:
            continue
        if top == np.inf:
            d = np.where(x[r] == np.inf, 0.0, -np.inf)
        else:
            d = x[r] - top
        w = np.exp(d)
        z = w.sum()
        norm = np.log(z)
        p = w / z
        lp = d - norm
        some = d > -np.inf
        a1, a2 = (p[some] * -d[some]).sum(), (p[some] * d[some] ** 2).sum()
        entropy[r] = norm + a1
        dz = 2 * F32 * (each + a1 + 8)
        tol[1][r] = dz * (2 + a1) + 2 * F32 * (a2 + (each + 8) * (a1 + 8)) + 4 * F32 * (norm + a1)
        with np.errstate(invalid="ignore"):
            bound = np.where(some, dz + 2 * F32 * (np.abs(d) + np.abs(lp) + norm), 0.0)
        for j in range(given.shape[1]):
            t = given[r, j]
            if 0 <= t < vocab:
                logprob[r, j], tol[0][r, j] = lp[t], bound[t]
        order = np.lexsort((np.arange(vocab), -x[r]))
        order = order[x[r][order] > -np.inf][:n_top]
        top_tokens[r, :len(order)] = order
        top_logprob[r, :len(order)], tol[2][r, :len(order)] = lp[order], bound[order]
    return (logprob, entropy, top_tokens, top_logprob), tol


def close(got, want, tol):
    """Whether `got` is within `tol` of `want`, and infinite or NaN where that is."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fine = np.isfinite(want)
    same = np.where(np.isnan(want), np.isnan(got), got == want)
    with np.errstate(invalid="ignore"):
        return bool(np.all(np.where(fine, np.abs(got - want) <= tol, same)))
