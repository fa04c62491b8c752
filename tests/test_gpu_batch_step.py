"""Several answers to one prompt, as a program makes them: a prompt's keys and
values stored once, then per step the projection (routed GEMM), rope-append,
attention over the shared prefix and the own caches, the classifier (routed
GEMM) and sampling. Every stage is checked on what the stage before left on the
GPU; then the step runs from a captured graph and draws the same tokens."""

import ctypes

import numpy as np
import pytest

from tests import batch_reference as ref
from tests.conftest import announce
from vx_amd import abi
from vx_amd.abi import bf16_to_f32, f32_to_bf16
from vx_amd.runtime import (DeviceArray, HipTimer, flash_attention_fwd, flash_attention_shared, matmul,
                            rope_append, sample)

pytestmark = pytest.mark.gpu

BF, F32, I32 = abi.DTYPE_BF16, abi.DTYPE_F32, abi.DTYPE_I32


class Answers:
    """One attention layer with a classifier on its output, for `batch` answers."""

    def __init__(self, lib, batch, heads, kv, d, vocab, prompt_len, capacity, seed=0):
        rng = np.random.default_rng(seed)
        self.lib, self.ext = lib, (batch, heads, kv, d, vocab, prompt_len, capacity)
        dim, width = heads * d, (heads + 2 * kv) * d

        def normal(scale, *shape):
            return f32_to_bf16((rng.standard_normal(shape) * scale).astype(np.float32))

        self.emb = normal(1.0, vocab, dim)
        self.wqkv, self.wout = normal(dim ** -0.5, dim, width), normal(6.0 * dim ** -0.5, dim, vocab)
        self.table = ref.rope_table(prompt_len + capacity, d)
        self.prompt = rng.integers(0, vocab, prompt_len)
        self.u = rng.random((capacity, batch), dtype=np.float32)
        r = np.arange(batch)
        self.how = (np.where(r % 4 == 3, 0, 0.8 + 0.1 * r).astype(np.float32),
                    np.where(r % 2 == 0, 20, 0).astype(np.int32), np.full(batch, 0.9, np.float32),
                    np.where(r % 3 == 1, 0.02, 0).astype(np.float32))
        dev = self.dev = {}
        for name, x, t in (("wqkv", self.wqkv, BF), ("wout", self.wout, BF), ("table", self.table, F32),
                           ("temperature", self.how[0], F32), ("top_k", self.how[1], I32),
                           ("top_p", self.how[2], F32), ("min_p", self.how[3], F32)):
            dev[name] = DeviceArray.of(lib, x, t)
        for name, shape, t in (("x", (batch, dim), BF), ("qkv", (batch, width), BF), ("q", (batch, heads, 1, d), BF),
                               ("ks", (kv, prompt_len, d), BF), ("vs", (kv, prompt_len, d), BF),
                               ("k", (batch, kv, capacity, d), BF), ("v", (batch, kv, capacity, d), BF),
                               ("o", (batch, heads, 1, d), BF), ("logits", (batch, vocab), F32),
                               ("lens", (batch,), I32), ("u", (batch,), F32), ("tokens", (batch,), I32),
                               ("logprob", (batch,), F32)):
            dev[name] = DeviceArray(lib, shape, t)

    def prefill(self):
        """The prompt as one sequence: its rotated keys and values become the
        shared ones, its last output the first logits of all answers."""
        b, h, kv, d, vocab, n, cap = self.ext
        lib, dev = self.lib, self.dev
        x = DeviceArray.of(lib, self.emb[self.prompt], BF)
        qkv, q, o = (DeviceArray(lib, s, BF) for s in ((n, (h + 2 * kv) * d), (1, h, n, d), (1, h, n, d)))
        matmul(lib, x.descriptor(), BF, dev["wqkv"].descriptor(), BF, qkv.descriptor(), BF)
        # the prompt's own positions: a cache of n rows behind an empty prefix
        assert rope_append(lib, "bf16", qkv.ptr, dev["table"].ptr, None, q.ptr, dev["ks"].ptr, dev["vs"].ptr, 1, n, h,
                           kv, d, 0, n, self.table.shape[0]) == 0
        assert flash_attention_fwd(lib, q.ptr, dev["ks"].ptr, dev["vs"].ptr, o.ptr, None, 1, h, kv, n, n, d,
                                   d ** -0.5, True) == 0
        last = o.numpy()[0, :, -1].reshape(1, h * d)
        for a in (x, qkv, q, o):
            a.free()
        return last

    def put(self, name, host, stream=None):
        src = DeviceArray.of(self.lib, np.ascontiguousarray(host), self.dev[name].dtype)
        t = HipTimer()
        t.sync()
        assert t.hip.hipMemcpy(ctypes.c_void_p(self.dev[name].ptr), ctypes.c_void_p(src.ptr), src.nbytes, 3) == 0
        t.sync()
        src.free()

    def classify_and_draw(self, workspace=(None, 0)):
        b, h, kv, d, vocab, n, cap = self.ext
        lib, dev = self.lib, self.dev
        o = abi.Descriptor(dev["o"].ptr, (b, h * d))
        matmul(lib, o, BF, dev["wout"].descriptor(), BF, dev["logits"].descriptor(), F32)
        assert sample(lib, "f32", dev["logits"].ptr, dev["temperature"].ptr, dev["top_k"].ptr, dev["top_p"].ptr,
                      dev["min_p"].ptr, dev["u"].ptr, dev["tokens"].ptr, dev["logprob"].ptr, b, vocab, None,
                      *workspace) == 0

    def step(self, workspace=(None, 0), sample_ws=(None, 0)):
        b, h, kv, d, vocab, n, cap = self.ext
        lib, dev = self.lib, self.dev
        matmul(lib, dev["x"].descriptor(), BF, dev["wqkv"].descriptor(), BF, dev["qkv"].descriptor(), BF)
        assert rope_append(lib, "bf16", dev["qkv"].ptr, dev["table"].ptr, dev["lens"].ptr, dev["q"].ptr, dev["k"].ptr,
                           dev["v"].ptr, b, 1, h, kv, d, n, cap, self.table.shape[0]) == 0
        assert flash_attention_shared(lib, dev["q"].ptr, dev["ks"].ptr, dev["vs"].ptr, dev["k"].ptr, dev["v"].ptr,
                                      dev["lens"].ptr, dev["o"].ptr, None, b, h, kv, 1, n, cap, d, d ** -0.5, True,
                                      workspace=workspace[0], workspace_bytes=workspace[1]) == 0
        self.classify_and_draw(sample_ws)

    def free(self):
        for a in self.dev.values():
            a.free()


def run(a, steps, step, check=False):
    b, h, kv, d, vocab, n, cap = a.ext
    dev = a.dev
    last = a.prefill()
    if check:
        x = a.emb[a.prompt]
        qkv = bf16_to_f32(f32_to_bf16(bf16_to_f32(x) @ bf16_to_f32(a.wqkv))).reshape(1, n, h + 2 * kv, d)
        held = [np.zeros((1, h, n, d))] + [np.zeros((1, kv, n, d))] * 2
        (_, wk, wv), _ = ref.rope_append(qkv, a.table, None, *held, 0)
        # the GEMM's bf16 rounding may fall the other way than the plain product's
        for name, w in (("ks", wk), ("vs", wv)):
            assert np.all(np.abs(bf16_to_f32(dev[name].numpy()) - w[0]) <= 2.0 ** -6 * np.abs(w[0]) + 2.0 ** -6)
    a.put("o", np.broadcast_to(last.reshape(1, h, 1, d), (b, h, 1, d)))
    a.put("u", a.u[0])
    a.classify_and_draw()
    out = [dev["tokens"].numpy().copy()]
    for s in range(1, steps):
        # answer 1 has ended: its slot holds no sequence any more
        lens = np.where((np.arange(b) == 1) & (s > 3), -1, s).astype(np.int32)
        a.put("x", a.emb[out[-1]])
        a.put("lens", lens)
        a.put("u", a.u[s])
        before = [dev[x].numpy().copy() for x in ("q", "k", "v")] if check else None
        o_before = dev["o"].numpy().copy() if check else None
        step()
        tokens = dev["tokens"].numpy().copy()
        if check:
            qkv = bf16_to_f32(dev["qkv"].numpy()).reshape(b, 1, h + 2 * kv, d)
            # what memory held before, whatever it was, stays as it was
            held = [np.zeros(x.shape) for x in before]
            want, tol = ref.rope_append(qkv, a.table, lens, *held, n)
            touched, _ = ref.rope_append(np.ones_like(qkv), None, lens, *held, n)
            for name, w, t, b16, new in zip(("q", "k", "v"), want, tol, before, touched):
                got = dev[name].numpy()
                assert np.array_equal(got[new == 0], b16[new == 0]), (s, name)
                assert np.all(np.abs(bf16_to_f32(got) - w)[new == 1] <= t[new == 1]), (s, name)
            (wo, _), (to, _) = ref.shared_attention(dev["q"].numpy(), dev["ks"].numpy(), dev["vs"].numpy(),
                                                    dev["k"].numpy(), dev["v"].numpy(), lens, n, d ** -0.5, True)
            o = dev["o"].numpy()
            live = lens >= 0
            assert np.all(np.abs(bf16_to_f32(o)[live] - wo[live]) <= to[live]), s
            assert np.array_equal(o[~live], o_before[~live]), s
            logits = dev["logits"].numpy()
            plain = bf16_to_f32(o).reshape(b, h * d).astype(np.float64) @ bf16_to_f32(a.wout).astype(np.float64)
            assert np.all(np.abs(logits - plain) <= 1e-4 * np.maximum(1, np.abs(plain)))
            wt, wl = ref.sample(logits, *a.how, a.u[s])
            assert np.array_equal(tokens, wt), s
            assert np.all(np.abs(dev["logprob"].numpy() - wl) <= ref.logprob_tol(wl))
        out.append(tokens)
    return np.array(out)


@pytest.mark.parametrize("shape", [(6, 4, 2, 64, 500, 37, 12), (20, 8, 1, 128, 40000, 1100, 9)])
def test_answers_to_one_prompt(hiplib, shape):
    announce(f"answers to one prompt {shape}")
    a = Answers(hiplib, *shape)
    steps = 8
    t = HipTimer()
    stream = t.stream_create()
    spaces, graph = [], None
    try:
        eager = run(a, steps, a.step, check=True)
        assert len({tuple(c) for c in eager.T}) > 1, "the answers differ"
        b, h, kv, d, vocab, n, cap = a.ext
        sizes = (hiplib.lib.vx_nn_flash_attention_shared_workspace(b, h, kv, 1, n, cap, d),
                 hiplib.lib.vx_nn_sample_workspace(b, vocab))
        spaces = [DeviceArray(hiplib, (max(s, 16),), abi.DTYPE_I8) for s in sizes]
        hiplib.lib.vx_hip_set_stream(stream)
        graph = t.capture(stream, lambda: a.step((spaces[0].ptr, sizes[0]), (spaces[1].ptr, sizes[1])))
        hiplib.lib.vx_hip_set_stream(None)

        def replay():
            t.graph_launch(graph, stream)
            t.sync()

        # captured products may round differently than eager ones: each replayed
        # run draws the same as the other
        first = run(a, steps, replay)
        assert np.array_equal(run(a, steps, replay), first)
        assert np.mean(first == eager) > 0.5
    finally:
        hiplib.lib.vx_hip_set_stream(None)
        if graph is not None:
            t.graph_destroy(graph)
        for s in spaces:
            s.free()
        t.stream_destroy(stream)
        a.free()
