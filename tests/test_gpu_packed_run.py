"""Texts of different lengths scored in one packed run, as a program makes it: norm
and 8 bits, the projection, rotation by each token's position, packed attention, 8
bits again and the second projection, the residual's norm, the classifier, and the
log probabilities of each text's next tokens. Every stage is checked on what the
stage before left on the GPU; a text's results do not depend on the others, and the
whole run from a captured graph gives the same bits."""

import ctypes

import numpy as np
import pytest

from tests import batch_reference, packed_reference as ref
from tests.conftest import announce
from vx_amd import abi
from vx_amd.abi import bf16_to_f32, f32_to_bf16
from vx_amd.llama import quantize_rows
from vx_amd.runtime import (DeviceArray, HipTimer, flash_attention_packed, gemm_i8, quantize_i8, rms_norm,
                            rope_append, token_logprobs)

pytestmark = pytest.mark.gpu

BF, F32, I32, I8 = abi.DTYPE_BF16, abi.DTYPE_F32, abi.DTYPE_I32, abi.DTYPE_I8
EPS = 1e-5
TOP = 4


class Scorer:
    def __init__(self, lib, lens, heads, kv, d, vocab, seed=0):
        rng = np.random.default_rng(seed)
        self.lib, self.ext = lib, (heads, kv, d, vocab)
        self.dim, self.width = heads * d, (heads + 2 * kv) * d
        self.offsets = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        self.total = n = int(self.offsets[-1])
        self.texts = [rng.integers(0, vocab, k) for k in lens]
        self.emb = f32_to_bf16(rng.standard_normal((vocab, self.dim)).astype(np.float32))
        self.norms = [(1 + 0.2 * rng.standard_normal(self.dim)).astype(np.float32) for _ in range(2)]
        self.w = {}
        for name, rows in (("qkv", self.width), ("out", self.dim), ("cls", vocab)):
            self.w[name] = quantize_rows(rng.standard_normal((rows, self.dim)).astype(np.float32) * self.dim ** -0.5)
        positions = np.concatenate([np.arange(k) for k in lens])
        self.table = batch_reference.rope_table(max(lens), d)[positions]  # a row a token
        dev = self.dev = {}
        for name, (q, s) in self.w.items():
            dev[name + "_q"], dev[name + "_s"] = DeviceArray.of(lib, q, I8), DeviceArray.of(lib, s, F32)
        for name, x, t in (("n0", self.norms[0], F32), ("n1", self.norms[1], F32), ("table", self.table, F32),
                           ("offsets", self.offsets, I32)):
            dev[name] = DeviceArray.of(lib, x, t)
        for name, shape, t in (("x", (n, self.dim), BF), ("x8", (n, self.dim), I8), ("x_s", (n,), F32),
                               ("qkv", (1, n, heads + 2 * kv, d), BF), ("q", (1, heads, n, d), BF),
                               ("k", (1, kv, n, d), BF), ("v", (1, kv, n, d), BF), ("o", (n, heads, d), BF),
                               ("lse", (heads, n), F32), ("o8", (n, self.dim), I8), ("o_s", (n,), F32),
                               ("y", (n, self.dim), BF), ("sum", (n, self.dim), BF), ("h8", (n, self.dim), I8),
                               ("h_s", (n,), F32), ("logits", (n, vocab), F32), ("given", (n, 1), I32),
                               ("logprob", (n, 1), F32), ("entropy", (n,), F32), ("top", (n, TOP), I32),
                               ("top_lp", (n, TOP), F32)):
            dev[name] = DeviceArray(lib, shape, t)
        self.feed()

    def put(self, name, host):
        src, t = DeviceArray.of(self.lib, np.ascontiguousarray(host), self.dev[name].dtype), HipTimer()
        t.sync()
        assert t.hip.hipMemcpy(ctypes.c_void_p(self.dev[name].ptr), ctypes.c_void_p(src.ptr), src.nbytes, 3) == 0
        t.sync()
        src.free()

    def feed(self):
        self.put("x", self.emb[np.concatenate(self.texts)])
        # the last token of a text has none behind it
        self.put("given", np.concatenate([np.append(t[1:], -1) for t in self.texts]).astype(np.int32)[:, None])

    def __call__(self):
        heads, kv, d, vocab = self.ext
        lib, n, dim = self.lib, self.total, self.dim
        p = {name: a.ptr for name, a in self.dev.items()}
        calls = [
            rms_norm(lib, "bf16", p["x"], None, p["n0"], None, None, p["x8"], p["x_s"], n, dim, EPS),
            gemm_i8(lib, "bf16", p["x8"], p["x_s"], p["qkv_q"], p["qkv_s"], p["qkv"], n, self.width, dim),
            rope_append(lib, "bf16", p["qkv"], p["table"], None, p["q"], p["k"], p["v"], 1, n, heads, kv, d, 0, n, n),
            flash_attention_packed(lib, p["q"], p["k"], p["v"], p["offsets"], p["o"], p["lse"], n, len(self.texts),
                                   heads, kv, d, d ** -0.5, True, o_strides=(dim, d)),
            quantize_i8(lib, "bf16", p["o"], p["o8"], p["o_s"], n, dim),
            gemm_i8(lib, "bf16", p["o8"], p["o_s"], p["out_q"], p["out_s"], p["y"], n, dim, dim),
            rms_norm(lib, "bf16", p["y"], p["x"], p["n1"], p["sum"], None, p["h8"], p["h_s"], n, dim, EPS),
            gemm_i8(lib, "f32", p["h8"], p["h_s"], p["cls_q"], p["cls_s"], p["logits"], n, vocab, dim),
            token_logprobs(lib, "f32", p["logits"], p["given"], p["logprob"], p["entropy"], p["top"], p["top_lp"], n,
                           vocab, 1, TOP)]
        assert calls == [0] * len(calls)

    def results(self):
        return {name: self.dev[name].numpy() for name in ("sum", "logits", "logprob", "entropy", "top", "top_lp")}

    def check(self):
        heads, kv, d, vocab = self.ext
        g = {name: a.numpy() for name, a in self.dev.items()}
        n = self.total

        def norm(x, residual, weight, q, scale, total=None):
            want, tol = ref.rms_norm(bf16_to_f32(x), None if residual is None else bf16_to_f32(residual), weight, EPS,
                                     ref.BF16)
            assert np.array_equal(q, want[3]) and ref.close(scale, want[2], tol[2])
            if total is not None:
                assert ref.close(bf16_to_f32(total), want[0], tol[0])

        def product(x, scale, w, y, bf16):
            want, tol = ref.gemm_i8(x, scale, *self.w[w], bf16)
            assert ref.close((bf16_to_f32(y) if bf16 else y).reshape(want.shape), want, tol), w

        norm(g["x"], None, self.norms[0], g["x8"], g["x_s"])
        product(g["x8"], g["x_s"], "qkv", g["qkv"], True)
        zeros = [np.zeros((1, h, n, d)) for h in (heads, kv, kv)]
        want, tol = batch_reference.rope_append(bf16_to_f32(g["qkv"]), self.table, None, *zeros, 0)
        for name, w, t in zip("qkv", want, tol):
            assert ref.close(bf16_to_f32(g[name]), w, t), name
        want, tol = ref.packed_attention(*(bf16_to_f32(g[x])[0] for x in "qkv"), self.offsets, d ** -0.5, True)
        assert ref.close(bf16_to_f32(g["o"]).transpose(1, 0, 2), want[0], tol[0])
        assert ref.close(g["lse"], want[1], tol[1])
        q, s = quantize_rows(bf16_to_f32(g["o"]).reshape(n, -1))
        assert np.array_equal(g["o8"], q) and np.array_equal(g["o_s"], s)
        product(g["o8"], g["o_s"], "out", g["y"], True)
        norm(g["y"], g["x"], self.norms[1], g["h8"], g["h_s"], g["sum"])
        product(g["h8"], g["h_s"], "cls", g["logits"], False)
        want, tol = ref.token_logprobs(g["logits"], g["given"], TOP)
        assert ref.close(g["logprob"], want[0], tol[0]) and ref.close(g["entropy"], want[1], tol[1])
        assert np.array_equal(g["top"], want[2]) and ref.close(g["top_lp"], want[3], tol[2])

    def free(self):
        for a in self.dev.values():
            a.free()


EXTENTS = [([5, 1, 33, 12], 4, 2, 64, 300), ([70, 3, 129, 64, 1, 40], 4, 1, 128, 1001), ([200, 90], 12, 12, 64, 2500)]


@pytest.mark.parametrize("lens,heads,kv,d,vocab", EXTENTS)
def test_stage_by_stage(hiplib, lens, heads, kv, d, vocab):
    announce(f"packed run {lens} {heads} {kv} {d} {vocab}")
    s = Scorer(hiplib, lens, heads, kv, d, vocab)
    s()
    s.check()
    s.free()


def test_texts_do_not_see_each_other(hiplib):
    announce("packed run, another text changed")
    s = Scorer(hiplib, [40, 77, 20], 4, 2, 64, 500)
    s()
    before = s.results()
    s.texts[1] = (s.texts[1] + 1) % 500
    s.feed()
    s()
    after = s.results()
    others = np.r_[0:40, 117:137]
    for name in before:
        assert np.array_equal(before[name][others], after[name][others]), name
        assert not np.array_equal(before[name][40:117], after[name][40:117]), name
    s.free()


def test_from_a_graph(hiplib):
    announce("packed run from a graph")
    s = Scorer(hiplib, [30, 64, 5, 101], 4, 2, 128, 700)
    s()
    want = s.results()
    t = HipTimer()
    stream = t.stream_create()
    hiplib.lib.vx_hip_set_stream(stream)
    try:
        ex = t.capture(stream, s)
        for turn in range(4):
            if turn == 2:  # other texts of the same lengths, the eager result first
                s.texts = [(x + 3) % 700 for x in s.texts]
                s.feed()
                s()
                t.sync()
                want = s.results()
            s.put("logits", np.zeros((s.total, 700), np.float32))
            t.graph_launch(ex, stream)
            t.sync()
            got = s.results()
            assert all(np.array_equal(got[name], want[name]) for name in want)
        s.check()
        t.graph_destroy(ex)
    finally:
        hiplib.lib.vx_hip_set_stream(None)
        t.stream_destroy(stream)
    s.free()
