"""The ops of a packed batch in 8 bits from several threads and streams at once,
and with operands whose offsets pass 32 bits."""

import ctypes
import threading

import numpy as np
import pytest

from tests.conftest import announce
from tests.test_gpu_flash_packed import Call as Attention
from tests.test_gpu_gemm_i8 import Call as Gemm
from tests.test_gpu_token_logprobs import Call as Logprobs
from tests.test_gpu_token_logprobs import logits_of
from vx_amd import abi
from vx_amd.abi import f32_to_bf16
from vx_amd.runtime import (DeviceArray, HipTimer, flash_attention_packed, gemm_i8, quantize_i8, rms_norm,
                            token_logprobs)

pytestmark = pytest.mark.gpu

PER_THREAD = 2  # hipStreamPerThread: one handle, a stream of each thread


def held(lib):
    """The workspaces that the library keeps, and their bytes."""
    out = (ctypes.c_int64 * 2)()
    assert lib.control(abi.HIP_CTRL_OP_WORKSPACES, out) == 1
    return tuple(out)


def calls(lib, seed):
    """Products and log probabilities that divide their work, and attention."""
    rng = np.random.default_rng(seed)
    return [Gemm(lib, "bf16", 80, 500, 4096, seed=seed), Gemm(lib, "f32", 256, 1024, 4096, seed=seed),
            Logprobs(lib, "f32", logits_of(rng, 2, 131071), rng.integers(0, 131071, (2, 3)), 5),
            Logprobs(lib, "bf16", logits_of(rng, 16, 50257), rng.integers(0, 50257, (16, 1)), 20),
            Attention(lib, [70, 0, 5, 130], 8, 2, 64, seed=seed)]


@pytest.mark.parametrize("per_thread", [False, True])
def test_from_threads_at_once(hiplib, per_thread):
    announce(f"packed ops from three threads, hipStreamPerThread {per_thread}")
    t = HipTimer()
    sets = [calls(hiplib, i) for i in range(3)]
    t.sync()
    before, errors = held(hiplib), []

    def work(i):
        s = PER_THREAD if per_thread else t.stream_create()
        try:
            hiplib.lib.vx_hip_set_stream(s)
            for turn in range(4):
                for j in range(len(sets[i])):
                    sets[i][(j + i + turn) % len(sets[i])]()
        except BaseException as e:  # noqa: BLE001 - reported below
            errors.append((i, repr(e)))
        finally:
            hiplib.lib.vx_hip_set_stream(None)
            t.sync()
            if not per_thread:
                t.stream_destroy(s)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
    for x in threads:
        x.start()
    for x in threads:
        x.join(timeout=60)
    assert not any(x.is_alive() for x in threads) and not errors, errors
    t.sync()
    assert held(hiplib) == before
    for c in sum(sets, []):
        c.check()
        c.free()


def test_two_graphs_with_workspaces_of_their_own_at_once(hiplib):
    announce("two graphs of divided products and log probabilities")
    t = HipTimer()
    streams, graphs, kept = [], [], []
    for i in range(2):
        s = t.stream_create()
        hiplib.lib.vx_hip_set_stream(s)
        try:
            for c in calls(hiplib, 10 + i)[:4]:
                ext = (c.rows, c.vocab, c.n_top) if isinstance(c, Logprobs) else c.ext
                need = (hiplib.lib.vx_nn_token_logprobs_workspace if isinstance(c, Logprobs)
                        else hiplib.lib.vx_nn_gemm_i8_workspace)(*ext)
                assert need > 0
                ws = DeviceArray(hiplib, (need,), abi.DTYPE_I8)
                graphs.append((t.capture(s, lambda c=c, ws=ws: c(ws.ptr, ws.nbytes)), s))
                kept.append((c, ws))
        finally:
            hiplib.lib.vx_hip_set_stream(None)
        streams.append(s)
    for _ in range(3):
        for ex, s in graphs[0::2] + graphs[1::2]:
            t.graph_launch(ex, s)
    t.sync()
    for c, ws in kept:
        c.check()
        c.free()
        ws.free()
    for ex, _ in graphs:
        t.graph_destroy(ex)
    for s in streams:
        t.stream_destroy(s)


class Far:
    """Memory of 8.5 GiB, in which elements lie anywhere."""

    def __init__(self, lib):
        self.t = HipTimer()
        self.a = DeviceArray(lib, (17 << 29,), abi.DTYPE_I8)
        self.t.sync()

    def put(self, at, host):
        host = np.ascontiguousarray(host)
        assert 0 <= at and at + host.nbytes <= self.a.nbytes
        assert self.t.hip.hipMemcpy(ctypes.c_void_p(self.a.ptr + at), host.ctypes.data_as(ctypes.c_void_p),
                                    host.nbytes, 1) == 0

    def get(self, at, n, dtype):
        host = np.empty(n, dtype)
        assert 0 <= at and at + host.nbytes <= self.a.nbytes
        self.t.sync()
        assert self.t.hip.hipMemcpy(host.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(self.a.ptr + at),
                                    host.nbytes, 2) == 0
        return host


@pytest.fixture(scope="module")
def far(hiplib):
    f = Far(hiplib)
    yield f
    f.a.free()


def test_norm_of_rows_far_apart(hiplib, far):
    """Row 2 begins 2^31 elements from row 0."""
    announce("rms_norm rows far apart")
    stride, dim = 2 ** 30, 96
    x = f32_to_bf16(np.random.default_rng(0).standard_normal((3, dim)).astype(np.float32))
    for r in range(3):
        far.put(2 * r * stride, x[r])
    near = DeviceArray.of(hiplib, x, abi.DTYPE_BF16)
    outs = [[DeviceArray(hiplib, (3, dim), abi.DTYPE_BF16), DeviceArray(hiplib, (3, dim), abi.DTYPE_I8),
             DeviceArray(hiplib, (3,), abi.DTYPE_F32)] for _ in range(2)]
    for (y, q, u), (ptr, step) in zip(outs, ((far.a.ptr, stride), (near.ptr, dim))):
        assert rms_norm(hiplib, "bf16", ptr, None, None, None, y.ptr, q.ptr, u.ptr, 3, dim, 1e-5, step) == 0
    for a, b in zip(*outs):
        assert np.array_equal(a.numpy(), b.numpy())
    for (_, q, u), (ptr, step) in zip(outs, ((far.a.ptr, stride), (near.ptr, dim))):
        assert quantize_i8(hiplib, "bf16", ptr, q.ptr, u.ptr, 3, dim, step) == 0
    for a, b in zip(*(o[1:] for o in outs)):
        assert np.array_equal(a.numpy(), b.numpy())
    for a in (near, *outs[0], *outs[1]):
        a.free()


@pytest.mark.parametrize("tokens,rows,stride", [(3, 40, 2 ** 30), (40, 700, 2 ** 26 + 24), (70, 130, 2 ** 25 + 1)])
def test_product_into_rows_far_apart(hiplib, far, tokens, rows, stride):
    announce(f"gemm_i8 rows far apart {tokens} {stride}")
    c = Gemm(hiplib, "bf16", tokens, rows, 144)
    assert gemm_i8(hiplib, "bf16", c.x.ptr, c.xs.ptr, c.w.ptr, c.ws.ptr, far.a.ptr, tokens, rows, 144, stride) == 0
    c()
    want = c.check()
    got = np.stack([far.get(2 * i * stride, rows, np.uint16) for i in range(tokens)])
    assert np.array_equal(got, want)
    c.free()


def test_logits_far_apart(hiplib, far):
    announce("token_logprobs rows far apart")
    rng = np.random.default_rng(1)
    stride, vocab = 2 ** 30, 1000
    c = Logprobs(hiplib, "bf16", logits_of(rng, 3, vocab), rng.integers(0, vocab, (3, 2)), 5)
    for r in range(3):
        far.put(2 * r * stride, f32_to_bf16(c.logits[r]))
    assert token_logprobs(hiplib, "bf16", far.a.ptr, c.g.ptr,
                          *map(c.ptr, ("logprob", "entropy", "top_tokens", "top_logprob")), 3, vocab, 2, 5,
                          stride) == 0
    c.check()
    c.free()


@pytest.mark.parametrize("which", ["keys", "queries", "outputs"])
def test_attention_of_rows_far_apart(hiplib, far, which):
    """Keys 2^22 elements apart, the last 2^31 from the first; or heads 2^30
    apart."""
    announce(f"flash_packed {which} far apart")
    lens, heads, kv, d = [500, 0, 200], 3, 1, 64
    c = Attention(hiplib, lens, heads, kv, d)
    total = c.total
    c()
    want, lse = c.outputs()
    x = f32_to_bf16(c.qkv)  # [heads + 2 kv, total, d]
    rows = dict(q_strides=(d, total * d), kv_strides=(d, total * d), o_strides=(d, total * d))
    at = list(c.at)
    o = DeviceArray(hiplib, (heads, total, d), abi.DTYPE_BF16)
    op = o.ptr
    if which == "keys":
        rows["kv_strides"] = (2 ** 22, 2 * d)
        at[1:] = far.a.ptr, far.a.ptr + 2 * d
        for i in range(total):
            far.put(2 * i * 2 ** 22, x[heads:, i])
    elif which == "queries":
        rows["q_strides"] = (d, 2 ** 30)
        at[0] = far.a.ptr
        for h in range(heads):
            far.put(2 * h * 2 ** 30, x[h])
    else:
        rows["o_strides"] = (d, 2 ** 30)
        op = far.a.ptr
    assert flash_attention_packed(hiplib, *at, c.off.ptr, op, c.lse.ptr, total, len(lens), heads, kv, d, c.scale, True,
                                  **rows) == 0
    if which == "outputs":
        got = np.stack([far.get(2 * h * 2 ** 30, total * d, np.uint16).reshape(total, d) for h in range(heads)])
    else:
        got = o.numpy()
    assert np.array_equal(got, want) and np.array_equal(c.outputs()[1], lse)
    o.free()
    c.free()


@pytest.mark.parametrize("tokens,rows", [(1, 270000), (16, 270000), (70, 270000), (270000, 20)])
def test_product_of_operands_past_32_bits(hiplib, far, tokens, rows):
    """The last rows of the larger operand, which begin past 2^32 bytes."""
    announce(f"gemm_i8 operands past 32 bits {tokens} {rows}")
    cols, last = 16384, 20
    rng = np.random.default_rng(tokens)
    c = Gemm(hiplib, "f32", min(tokens, last) if tokens > rows else tokens, rows if tokens > rows else last, cols)
    c()
    want = c.check()
    large = max(tokens, rows)
    far.put((large - last) * cols, c.hx if tokens > rows else c.hw)
    scale = rng.uniform(0.001, 0.1, large).astype(np.float32)
    scale[-last:] = c.hxs if tokens > rows else c.hws
    s = DeviceArray.of(hiplib, scale, abi.DTYPE_F32)
    y = DeviceArray(hiplib, (tokens, rows), abi.DTYPE_F32)
    if tokens > rows:
        args = far.a.ptr, s.ptr, c.w.ptr, c.ws.ptr
    else:
        args = c.x.ptr, c.xs.ptr, far.a.ptr, s.ptr
    assert gemm_i8(hiplib, "f32", *args, y.ptr, tokens, rows, cols) == 0
    got = y.numpy()
    assert np.array_equal(got[-last:] if tokens > rows else got[:, -last:], want)
    for a in (s, y):
        a.free()
    c.free()
