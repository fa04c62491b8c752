"""vx_nn_sample_* on the GPU: tokens equal to the definition's in 64 bits,
log-probabilities to a rounding."""

import numpy as np
import pytest

from tests import batch_reference as ref
from tests.conftest import announce
from vx_amd import abi
from vx_amd.abi import bf16_to_f32, f32_to_bf16
from vx_amd.runtime import DeviceArray, HipTimer, sample

pytestmark = pytest.mark.gpu

INF, NAN = np.inf, np.nan
LOWEST = np.finfo(np.float32).min


class Call:
    """One call's operands; rows lie `pad` elements apart that hold NaN and the
    largest numbers, which must not be looked at."""

    def __init__(self, lib, logits, u, temperature=None, top_k=None, top_p=None, min_p=None,
                 dtype="f32", pad=0, logprob=True):
        rows, vocab = logits.shape
        self.lib, self.dtype, self.rows, self.vocab, self.stride = lib, dtype, rows, vocab, vocab + pad
        logits = np.asarray(logits, np.float32)
        if dtype == "bf16":
            with np.errstate(all="ignore"):
                logits = bf16_to_f32(f32_to_bf16(logits))
        self.logits = logits
        full = np.full((rows, self.stride), 3e38, np.float32)
        full[:, vocab + 1::2] = NAN
        full[:, :vocab] = logits
        self.settings = [None if x is None else np.broadcast_to(np.asarray(x, t), (rows,)).copy()
                         for x, t in ((temperature, np.float32), (top_k, np.int32), (top_p, np.float32),
                                      (min_p, np.float32))]
        self.u = np.broadcast_to(np.asarray(u, np.float32), (rows,)).copy()
        host = f32_to_bf16(full) if dtype == "bf16" else full
        self.d = [DeviceArray.of(lib, host, abi.DTYPE_BF16 if dtype == "bf16" else abi.DTYPE_F32)]
        for x, t in zip(self.settings, (abi.DTYPE_F32, abi.DTYPE_I32, abi.DTYPE_F32, abi.DTYPE_F32)):
            self.d.append(DeviceArray.of(lib, x, t) if x is not None else None)
        self.d.append(DeviceArray.of(lib, self.u, abi.DTYPE_F32))
        self.d.append(DeviceArray.of(lib, np.full(rows + 8, 77, np.int32), abi.DTYPE_I32))
        self.d.append(DeviceArray.of(lib, np.full(rows + 8, 77, np.float32), abi.DTYPE_F32) if logprob else None)

    def __call__(self, workspace=None, workspace_bytes=0):
        assert sample(self.lib, self.dtype, *(x.ptr if x is not None else None for x in self.d), self.rows,
                      self.vocab, self.stride, workspace, workspace_bytes) == 0

    def results(self):
        tokens = self.d[6].numpy()
        assert np.all(tokens[self.rows:] == 77)
        logprob = self.d[7].numpy() if self.d[7] is not None else None
        assert logprob is None or np.all(logprob[self.rows:] == 77)
        return tokens[:self.rows], logprob[:self.rows] if logprob is not None else None

    def want(self):
        return ref.sample(self.logits, *self.settings, self.u)

    def check(self, want):
        tokens, logprob = self.results()
        bad = np.flatnonzero(tokens != want[0])
        assert not len(bad), [(int(r), int(tokens[r]), int(want[0][r])) for r in bad[:4]]
        if logprob is not None:
            none = want[1] == -np.inf
            assert np.all(logprob[none] == -np.inf)
            assert np.all(np.abs(logprob - want[1])[~none] <= ref.logprob_tol(want[1])[~none])

    def free(self):
        for x in self.d:
            if x is not None:
                x.free()


def check(lib, logits, u, **kw):
    c = Call(lib, logits, u, **kw)
    want = c.want()
    c()
    c.check(want)
    # undivided, as a captured call without a workspace is
    t = HipTimer()
    stream = t.stream_create()
    lib.lib.vx_hip_set_stream(stream)
    try:
        g = t.capture(stream, c)
        t.graph_launch(g, stream)
        t.sync()
        c.check(want)
        t.graph_destroy(g)
    finally:
        lib.lib.vx_hip_set_stream(None)
        t.stream_destroy(stream)
    n = lib.lib.vx_nn_sample_workspace(c.rows, c.vocab)
    if n:
        ws = DeviceArray.of(lib, np.full(n + 256, -1, np.int8), abi.DTYPE_I8)
        c(ws.ptr, n)
        c.check(want)
        assert np.all(ws.numpy()[n:] == -1), "written past the workspace"
        ws.free()
    c.free()
    return want


def likely(rng, rows, vocab, spread=2.0, top=11.0):
    x = rng.standard_normal((rows, vocab)).astype(np.float32) * spread
    for r in range(rows):
        at = rng.choice(vocab, min(vocab, 40), replace=False)
        x[r, at] = rng.standard_normal(len(at)) * 2.5 + top
    return x


MODES = {
    "plain": {}, "hot": dict(temperature=1.7), "cold": dict(temperature=0.05),
    "top_k": dict(top_k=40, temperature=0.8), "top_k_deep": dict(top_k=700),
    "top_p": dict(top_p=0.9), "top_p_wide": dict(top_p=0.9999, temperature=1.5),
    "min_p": dict(min_p=0.05), "min_p_deep": dict(min_p=1e-6),
    "all": dict(temperature=0.9, top_k=60, top_p=0.95, min_p=0.01),
    "top_k_p": dict(top_k=900, top_p=0.7, temperature=1.3),
}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 32000), (5, 1000), (3, 4099), (2, 131071), (9, 257)])
@pytest.mark.parametrize("mode", list(MODES))
def test_modes(hiplib, mode, rows, vocab, dtype):
    announce(f"sample {mode} {rows}x{vocab} {dtype}")
    rng = np.random.default_rng([rows, vocab, len(mode)])
    check(hiplib, likely(rng, rows, vocab), rng.random(rows, dtype=np.float32), dtype=dtype,
          pad=vocab % 3, **MODES[mode])


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 127, 1023, 1024, 1025, 2049, 8191, 8193, 16385, 32769,
                                   65537, 262144])
def test_vocabularies(hiplib, vocab):
    announce(f"sample vocabulary {vocab}")
    rng = np.random.default_rng(vocab)
    rows = 4
    check(hiplib, likely(rng, rows, vocab, top=4.0), rng.random(rows, dtype=np.float32),
          temperature=[1.0, 0.7, 0.0, 1.3], top_k=[0, 50, 0, vocab], top_p=[1.0, 0.9, 0.5, 0.97], min_p=[0, 0, 0.1, 1e-4])


@pytest.mark.parametrize("rows", [1, 2, 31, 64, 200, 300, 1000])
def test_batches(hiplib, rows):
    """Many rows, each with settings of its own."""
    announce(f"sample batch {rows}")
    rng = np.random.default_rng(rows)
    r = np.arange(rows)
    check(hiplib, likely(rng, rows, 5003, top=7.0), rng.random(rows, dtype=np.float32),
          temperature=np.where(r % 5 == 4, 0, 0.5 + rng.random(rows)), top_k=np.where(r % 3 == 0, 0, r % 90 + 1),
          top_p=np.where(r % 4 == 1, 1, rng.random(rows)), min_p=np.where(r % 2 == 0, 0, rng.random(rows) * 0.3))


@pytest.mark.parametrize("vocab", [8, 1000, 40000])
def test_equal_logits(hiplib, vocab):
    """All equal: exact shares, ties kept from the lowest index on. top_p of half
    keeps half, u = j / n draws token j and the number below it token j - 1."""
    announce(f"sample equal {vocab}")
    half = vocab // 2
    u = np.array([0.0, 0.5, np.nextafter(np.float32(0.5), np.float32(0)), 1 - 2.0 ** -24, 0.25, 0.999, 0.0, 0.75],
                 np.float32)
    want = check(hiplib, np.full((8, vocab), 2.5), u)
    assert want[0][1] == half and want[0][2] == half - 1 and want[0][3] == vocab - 1
    want = check(hiplib, np.full((8, vocab), -3.0), u, top_p=0.5)
    assert want[0][3] == half - 1
    want = check(hiplib, np.zeros((8, vocab)), u, top_k=5)
    assert want[0][3] == 4 and np.all(want[0] < 5)
    check(hiplib, np.zeros((8, vocab)), u, top_k=7, top_p=0.5, min_p=1.0)
    check(hiplib, np.where(np.arange(vocab) % 2 == 0, -0.0, 0.0)[None].repeat(8, 0), u, top_k=3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masks_and_infinities(hiplib, dtype):
    announce(f"sample masks {dtype}")
    rng = np.random.default_rng(4)
    vocab, rows = 6000, 16
    x = likely(rng, rows, vocab)
    x[0] = -INF
    x[1] = NAN
    x[2, 1:] = -INF
    x[3, :-1] = NAN
    x[4, 100:] = -INF
    x[5, ::2] = NAN
    x[6, [17, 4000]] = INF
    x[7, :] = LOWEST
    x[8, 3:] = LOWEST
    x[9, 50] = INF
    x[10] = np.where(np.arange(vocab) < 10, 1e30, -1e30)
    x[11] = 1e-30
    x[12, :] = -INF
    x[12, 5990:] = [1, 2, 3, NAN, -INF, 4, 4, 4, LOWEST, 3]
    x[13, ::3] = INF
    u = rng.random(rows, dtype=np.float32)
    for kw in ({}, dict(top_k=7), dict(top_p=0.8), dict(min_p=0.1), dict(top_k=4000, top_p=0.6, min_p=1e-3),
               dict(temperature=0), dict(temperature=1e-3, top_k=50), dict(temperature=30.0, top_p=0.99)):
        want = check(hiplib, x, u, dtype=dtype, pad=5, **kw)
        assert want[0][0] == want[0][1] == -1


def test_extreme_settings(hiplib):
    announce("sample extreme settings")
    rng = np.random.default_rng(8)
    big, tiny = 3.4e38, 1e-45
    temperature = [0, -1, NAN, INF, big, tiny, 1e-30, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1]
    top_k = [0] * 7 + [-3, 2 ** 31 - 1, 1, 2999, 3000, 0, 0, 0, 0, 0, 0, 0, 0]
    top_p = [1] * 12 + [NAN, 0, -1, 1e-30, 2, 1, 1, 1]
    min_p = [0] * 17 + [NAN, 2, -1]
    rows = len(temperature)
    x = likely(rng, rows, 3000)
    for u in (rng.random(rows, dtype=np.float32), 0.0, 1.0, 7.0, -1.0, NAN, INF, 1e-40, 1 - 2.0 ** -24):
        with np.errstate(all="ignore"):
            check(hiplib, x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


def test_shares(hiplib):
    """A grid of u over one distribution: each token's count is its share."""
    announce("sample shares")
    rows, vocab = 1024, 40
    x = np.random.default_rng(2).standard_normal(vocab).astype(np.float32)
    u = (np.arange(rows) + 0.5) / rows
    c = Call(hiplib, np.broadcast_to(x, (rows, vocab)), u, temperature=0.9, top_k=30)
    want = c.want()
    c()
    c.check(want)
    tokens, _ = c.results()
    assert np.all(np.diff(tokens) >= 0)
    order = np.argsort(-x.astype(np.float64), kind="stable")[:30]
    p = np.zeros(vocab)
    p[order] = np.exp(x[order].astype(np.float64) / np.float32(0.9))
    p /= p.sum()
    assert np.all(np.abs(np.bincount(tokens, minlength=vocab) - p * rows) <= 1)
    c.free()


def test_without_logprob_and_back_to_back(hiplib):
    """Calls one after another without a wait, twice each: the same bits."""
    announce("sample back to back")
    rng = np.random.default_rng(6)
    calls = [Call(hiplib, likely(rng, r, v), rng.random(r, dtype=np.float32), logprob=i % 2 == 0, dtype=d,
                  **MODES[m]) for i, (r, v, m, d) in enumerate(
                      [(1, 32000, "all", "f32"), (64, 2000, "top_p", "bf16"), (2, 100000, "plain", "f32"),
                       (1, 50, "top_k", "bf16"), (300, 1500, "min_p", "f32"), (3, 50000, "top_p_wide", "f32")])]
    wants = [c.want() for c in calls]
    for _ in range(2):
        for c in calls:
            c()
        for c, w in zip(calls, wants):
            c.check(w)
    for c in calls:
        c.free()


def test_many_rows_of_a_large_vocabulary(hiplib):
    """More rows than workgroups share one of: with and without borders."""
    announce("sample many rows")
    rng = np.random.default_rng(12)
    for rows, vocab in ((130, 40000), (1030, 33000)):
        x = likely(rng, rows, vocab, top=9.0)
        u = rng.random(rows, dtype=np.float32)
        check(hiplib, x, u, dtype="bf16")
        check(hiplib, x, u, top_p=np.where(np.arange(rows) % 2 == 0, 0.9, 1), top_k=np.where(np.arange(rows) % 3 == 0, 30, 0))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [5000, 70000])
def test_wide_borders(hiplib, vocab, dtype):
    """Borders with more tokens above them, in their bin and at their logit than a
    list holds."""
    announce(f"sample wide borders {vocab} {dtype}")
    rng = np.random.default_rng(vocab)
    rows = 10
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    x[0] = 0
    x[1] = np.round(x[1])
    x[2] = x[2] * 1e-3 + 5
    x[3, ::2] = 1.25
    x[4] = np.where(rng.random(vocab) < 0.5, 3.0, x[4])
    x[5] *= 30
    u = rng.random(rows, dtype=np.float32)
    for kw in (dict(top_p=0.5), dict(top_p=0.999), dict(top_k=vocab // 2), dict(top_k=vocab - 1, top_p=0.7),
               dict(top_k=1500, top_p=0.99, min_p=0.5), dict(min_p=0.4), dict(top_p=0.9, min_p=1e-3, temperature=3.0)):
        check(hiplib, x, u, dtype=dtype, **kw)


@pytest.mark.parametrize("vocab", [6000, 70000])
@pytest.mark.parametrize("kept", [30, 200, 300, 900, 1500])
def test_min_p_before_the_other_border(hiplib, vocab, kept):
    """min_p keeps `kept` tokens, of which top_k and top_p would each keep all and
    more."""
    announce(f"sample min_p keeps {kept} of {vocab}")
    rng = np.random.default_rng([vocab, kept])
    rows = 6
    x = (-4 - 0.5 * rng.random((rows, vocab))).astype(np.float32)
    for r in range(rows):
        x[r, rng.choice(vocab, kept, replace=False)] = 2 * rng.random(kept, dtype=np.float32)
        x[r, rng.integers(vocab)] = 2
    u = rng.random(rows, dtype=np.float32)
    for kw in (dict(top_k=kept + 700), dict(top_k=kept + 2), dict(top_p=0.9999), dict(top_p=0.97),
               dict(top_k=kept + 1000, top_p=0.9999)):
        check(hiplib, x, u, min_p=0.1, **kw)


@pytest.mark.parametrize("vocab", [1200, 9000, 70000])
def test_top_p_within_what_top_k_keeps_of_equals(hiplib, vocab):
    """top_k ends among many equal logits, and top_p keeps nearly or quite all that
    it leaves."""
    announce(f"sample equals by top_k and top_p {vocab}")
    rng = np.random.default_rng(vocab)
    x = np.zeros((8, vocab), np.float32)
    x[4:, ::3] = 0.5
    u = rng.random(8, dtype=np.float32)
    for k in (2, 22, vocab // 3, vocab - 7):
        want = check(hiplib, x, u, top_k=k, top_p=1 - 2.0 ** -20)
        assert np.all(want[0][:4] < k)
        check(hiplib, x, u, top_k=k, top_p=0.999)
        check(hiplib, x, u, top_k=k, top_p=0.6, dtype="bf16")


def test_two_streams_at_once(hiplib):
    announce("sample on two streams")
    t = HipTimer()
    rng = np.random.default_rng(3)
    streams = [t.stream_create() for _ in range(2)]
    calls = [Call(hiplib, likely(rng, 20, 50000 + i), rng.random(20, dtype=np.float32), top_p=0.95,
                  temperature=0.9 + i) for i in range(2)]
    wants = [c.want() for c in calls]
    t.sync()
    try:
        for _ in range(10):
            for s, c in zip(streams, calls):
                hiplib.lib.vx_hip_set_stream(s)
                c()
        t.sync()
        hiplib.lib.vx_hip_set_stream(None)
        for c, w in zip(calls, wants):
            c.check(w)
    finally:
        hiplib.lib.vx_hip_set_stream(None)
        t.sync()
        for c in calls:
            c.free()
        for s in streams:
            t.stream_destroy(s)
