"""vx_nn_token_logprobs_* on the GPU against the definition in 64 bits."""

import numpy as np
import pytest

from tests import packed_reference as ref
from tests.conftest import announce
from vx_amd import abi
from vx_amd.abi import bf16_to_f32, f32_to_bf16
from vx_amd.runtime import DeviceArray, HipTimer, token_logprobs

pytestmark = pytest.mark.gpu

TYPE = {"f32": abi.DTYPE_F32, "bf16": abi.DTYPE_BF16}


class Call:
    def __init__(self, lib, dtype, logits, given, n_top, pad=0, skip=0, entropy=True, top_logprob=True):
        self.lib, self.dtype, self.n_top = lib, dtype, n_top
        self.rows, self.vocab = logits.shape
        self.stride = self.vocab + pad
        wide = np.full((self.rows, self.stride), np.nan if pad % 2 else 1e30, np.float32)
        wide[:, :self.vocab] = logits
        host = f32_to_bf16(wide) if dtype == "bf16" else wide
        self.logits = (bf16_to_f32(host) if dtype == "bf16" else host)[:, :self.vocab]
        flat = np.concatenate([np.zeros(skip, host.dtype), host.reshape(-1)])
        self.x = DeviceArray.of(lib, flat, TYPE[dtype])
        self.at = self.x.ptr + skip * abi.DTYPE_BYTES[TYPE[dtype]]
        self.given = given.astype(np.int32)
        self.g = DeviceArray.of(lib, self.given, abi.DTYPE_I32) if given.size else None
        self.out = {}
        for name, n, t, on in (("logprob", given.size, abi.DTYPE_F32, given.size > 0),
                               ("entropy", self.rows, abi.DTYPE_F32, entropy),
                               ("top_tokens", self.rows * n_top, abi.DTYPE_I32, n_top > 0),
                               ("top_logprob", self.rows * n_top, abi.DTYPE_F32, n_top > 0 and top_logprob)):
            if on:
                host = np.full(n + 64, 77, DeviceArray.NP[t])
                self.out[name] = (DeviceArray.of(lib, host, t), n)

    def ptr(self, name):
        return self.out[name][0].ptr if name in self.out else None

    def __call__(self, workspace=None, workspace_bytes=0):
        assert token_logprobs(self.lib, self.dtype, self.at, self.g.ptr if self.g else None,
                              *map(self.ptr, ("logprob", "entropy", "top_tokens", "top_logprob")), self.rows,
                              self.vocab, self.given.shape[1], self.n_top, self.stride, workspace,
                              workspace_bytes) == 0

    def got(self):
        out = {}
        for name, (a, n) in self.out.items():
            x = a.numpy()
            assert np.all(x[n:] == 77), f"{name}: written past its end"
            out[name] = x[:n]
        return out

    def check(self):
        want, tol = ref.token_logprobs(self.logits, self.given, self.n_top)
        got = self.got()
        for i, name, t in ((0, "logprob", tol[0]), (1, "entropy", tol[1]), (3, "top_logprob", tol[2])):
            if name in got:
                assert ref.close(got[name].reshape(want[i].shape), want[i], t), name
        if "top_tokens" in got:
            assert np.array_equal(got["top_tokens"].reshape(want[2].shape), want[2]), "top_tokens"
        return got

    def free(self):
        for a in (self.x, self.g, *(a for a, _ in self.out.values())):
            if a is not None:
                a.free()


def logits_of(rng, rows, vocab):
    """A broad bulk and a few likely tokens."""
    x = rng.standard_normal((rows, vocab)) * 2
    for r in range(rows):
        at = rng.integers(0, vocab, min(40, vocab))
        x[r, at] = rng.standard_normal(len(at)) * 2.5 + 11
    return x


def one(lib, dtype, x, n_given=2, n_top=5, seed=0, **kw):
    announce(f"token_logprobs {x.shape} {dtype} given {n_given} top {n_top} {kw}")
    rng = np.random.default_rng(seed)
    given = rng.integers(0, x.shape[1], (x.shape[0], n_given))
    c = Call(lib, dtype, x, given, n_top, **kw)
    c()
    c.check()
    c.free()


VOCABS = [1, 2, 7, 8, 9, 63, 100, 1000, 1031, 8192, 8193, 9001, 32000, 32768, 50257, 131071]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("n_top", [1, 20, 64])
def test_sizes(hiplib, dtype, vocab, n_top):
    one(hiplib, dtype, logits_of(np.random.default_rng(vocab), 3, vocab), n_top=n_top)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(300, 1500), (260, 20000), (1, 262145), (40, 70000)])
def test_many_rows_and_long_ones(hiplib, dtype, rows, vocab):
    one(hiplib, dtype, logits_of(np.random.default_rng(rows), rows, vocab))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,skip", [(0, 1), (1, 0), (3, 5), (8, 8), (2, 7)])
@pytest.mark.parametrize("vocab", [501, 33333])
def test_strides_and_alignment(hiplib, dtype, pad, skip, vocab):
    one(hiplib, dtype, logits_of(np.random.default_rng(3), 4, vocab), pad=pad, skip=skip)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [900, 40000])
def test_outputs_that_may_be_missing(hiplib, dtype, vocab):
    x = logits_of(np.random.default_rng(4), 3, vocab)
    one(hiplib, dtype, x, n_given=0)
    one(hiplib, dtype, x, n_top=0)
    one(hiplib, dtype, x, n_given=0, n_top=0)
    one(hiplib, dtype, x, entropy=False, top_logprob=False)
    one(hiplib, dtype, x, n_given=1500, n_top=3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [70, 5000, 40000, 200001])
def test_ties(hiplib, dtype, vocab):
    """The lower index first: all equal, few values, zeros of both signs, and more
    equal largest logits in one place than fit a list."""
    rng = np.random.default_rng(5)
    x = np.zeros((6, vocab))
    x[1] = rng.integers(-3, 4, vocab)
    x[2] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
    x[3] = -np.arange(vocab) % 5
    x[4, :vocab // 2] = 2.0
    x[5, ::1024] = 3.0  # the elements of a few threads
    x[5, 1::1024] = 3.0
    one(hiplib, dtype, x, n_top=64)
    one(hiplib, dtype, x, n_top=7, skip=3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_near_the_border_than_a_list_holds(hiplib, dtype):
    """Two threads own all of the largest logits: thousands above what the others
    have."""
    vocab, rng = 1 << 22, np.random.default_rng(6)
    x = rng.standard_normal((1, vocab)) * 0.1
    vec = 8 if dtype == "bf16" else 4
    for t in (5, 700):
        at = (np.arange(0, vocab // vec, 1024)[:, None] + t) * vec + np.arange(vec)[None, :]
        at = at.reshape(-1)
        x[0, at[at < vocab]] = 5 + rng.standard_normal(np.sum(at < vocab))
    announce(f"token_logprobs list {dtype}")
    given = np.array([[int(np.argmax(x[0])), 0]])
    for ws in (False, True):  # without one, one workgroup has the row
        c = Call(hiplib, dtype, x, given, 64)
        t = HipTimer()
        if ws:
            c()
        else:
            s = t.stream_create()
            hiplib.lib.vx_hip_set_stream(s)
            try:
                ex = t.capture(s, c)
                t.graph_launch(ex, s)
                t.sync()
                t.graph_destroy(ex)
            finally:
                hiplib.lib.vx_hip_set_stream(None)
                t.stream_destroy(s)
        # 4096 sums a thread there
        want, tol = ref.token_logprobs(c.logits, c.given, 64)
        got = c.got()
        assert np.array_equal(got["top_tokens"].reshape(1, 64), want[2])
        assert ref.close(got["top_logprob"].reshape(1, 64), want[3], tol[2])
        assert ref.close(got["logprob"].reshape(1, 2), want[0], tol[0])
        assert ref.close(got["entropy"], want[1], tol[1])
        c.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [5, 3000, 40000, 150000])
def test_masks_infinities_and_nans(hiplib, dtype, vocab):
    rng = np.random.default_rng(7)
    x = rng.standard_normal((12, vocab)) * 3
    low = -3.4028234663852886e38 if dtype == "f32" else -3.3895313892515355e38
    x[0] = -np.inf
    x[1] = np.nan
    x[2] = low  # the type's lowest value throughout
    x[3, :] = -np.inf
    x[3, vocab // 2] = -7.0
    x[4, 1:] = low
    x[5, vocab // 3] = np.nan
    x[6, [0, vocab - 1]] = np.inf
    x[7, ::2] = -np.inf
    x[7, 1::2] = np.nan
    x[8, vocab - 1] = np.inf
    x[8, 0] = np.nan
    x[9] = -low  # the largest value throughout
    x[10, :vocab - 2] = -np.inf
    x[11] = np.where(np.arange(vocab) % 3 == 0, 1e4, -1e4)
    announce(f"token_logprobs masks {vocab} {dtype}")
    given = np.stack([np.zeros(12, int), np.full(12, vocab - 1), np.full(12, vocab // 2), np.full(12, -1),
                      np.full(12, vocab), np.full(12, 2 ** 31 - 1)], axis=1)
    c = Call(hiplib, dtype, x, given, 9)
    c()
    c.check()
    c.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_certain_and_even_rows(hiplib, dtype):
    """Entropy near 0 and at its largest."""
    x = np.zeros((3, 30000))
    x[0, 17] = 60.0
    x[1, 17] = 20.0
    one(hiplib, dtype, x)


@pytest.mark.parametrize("rows,vocab", [(1, 32000), (2, 131071), (30, 40000), (300, 9000)])
def test_from_a_graph_with_and_without_a_workspace(hiplib, rows, vocab):
    """Captured without a workspace and with one full of other numbers: the same
    tokens, and logarithms within their bounds; each replay the same bits."""
    announce(f"token_logprobs from a graph {rows} x {vocab}")
    t = HipTimer()
    x = logits_of(np.random.default_rng(8), rows, vocab)
    given = np.random.default_rng(9).integers(0, vocab, (rows, 2))
    c = Call(hiplib, "f32", x, given, 10)
    need = hiplib.lib.vx_nn_token_logprobs_workspace(rows, vocab, 10)
    ws = DeviceArray.of(hiplib, np.full(max(need, 16), 0x7f, np.int8), abi.DTYPE_I8)
    s = t.stream_create()
    hiplib.lib.vx_hip_set_stream(s)
    try:
        graphs = [t.capture(s, c), t.capture(s, lambda: c(ws.ptr, ws.nbytes))]
        first = [None, None]
        for _ in range(3):
            for i, ex in enumerate(graphs):
                t.graph_launch(ex, s)
                t.sync()
                got = c.check()
                first[i] = first[i] or got
                assert all(np.array_equal(got[n], first[i][n]) for n in got)
            c()
            t.sync()
            c.check()
        for ex in graphs:
            t.graph_destroy(ex)
    finally:
        hiplib.lib.vx_hip_set_stream(None)
        t.stream_destroy(s)
    ws.free()
    c.free()
