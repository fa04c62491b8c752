"""vx_nn_flash_attention_packed_bf16 on the GPU against the definition in 64
bits."""

import ctypes

import numpy as np
import pytest

from tests import packed_reference as ref
from tests.conftest import announce
from vx_amd import abi
from vx_amd.abi import bf16_to_f32, f32_to_bf16
from vx_amd.runtime import DeviceArray, HipTimer, flash_attention_packed

pytestmark = pytest.mark.gpu

NAN, INF = 0x7FC0, 0x7F80


class Call:
    """layout "heads": [heads, total, d]; "tokens": slices of a projection
    [total, heads + 2 kv, d], o [total, heads, d] with `gap` elements between
    rows. Rows of no sequence hold NaN and infinities."""

    def __init__(self, lib, lens, heads, kv, d, causal=True, layout="heads", scale=None, lead=0, tail=0, gap=0,
                 lse=True, seed=0, put=None):
        rng = np.random.default_rng(seed)
        self.lib, self.heads, self.kv, self.d, self.causal, self.layout = lib, heads, kv, d, causal, layout
        self.scale = d ** -0.5 if scale is None else scale
        self.offsets = np.concatenate([[lead], lead + np.cumsum(lens)]).astype(np.int32)
        self.total = total = int(self.offsets[-1]) + tail
        x = f32_to_bf16(rng.standard_normal((total, heads + 2 * kv, d)).astype(np.float32))
        x[:lead], x[self.offsets[-1]:] = NAN, INF
        if put:
            put(x)
        self.qkv = bf16_to_f32(x).transpose(1, 0, 2)
        self.n_seq = len(lens)
        row = (heads + 2 * kv) * d
        if layout == "tokens":
            self.x = DeviceArray.of(lib, x, abi.DTYPE_BF16)
            self.strides = dict(q_strides=(row, d), kv_strides=(row, d), o_strides=(heads * d + gap, d))
            self.at = [self.x.ptr + 2 * d * n for n in (0, heads, heads + kv)]
            size = total * (heads * d + gap)
        else:
            self.x = DeviceArray.of(lib, np.ascontiguousarray(x.transpose(1, 0, 2)), abi.DTYPE_BF16)
            self.strides = {}
            self.at = [self.x.ptr + 2 * d * total * n for n in (0, heads, heads + kv)]
            size = total * heads * d
        self.off = DeviceArray.of(lib, self.offsets, abi.DTYPE_I32)
        self.gap = gap
        self.o = DeviceArray.of(lib, np.full(size + 64, 0x5a5a, np.uint16), abi.DTYPE_BF16)
        self.lse = DeviceArray.of(lib, np.full(heads * total + 16, 77.5, np.float32), abi.DTYPE_F32) if lse else None

    def __call__(self):
        assert flash_attention_packed(self.lib, *self.at, self.off.ptr, self.o.ptr,
                                      self.lse.ptr if self.lse else None, self.total, self.n_seq, self.heads, self.kv,
                                      self.d, self.scale, self.causal, **self.strides) == 0

    def outputs(self):
        h, total, d = self.heads, self.total, self.d
        o = self.o.numpy()
        assert np.all(o[-64:] == 0x5a5a)
        if self.layout == "tokens":
            o = o[:-64].reshape(total, h * d + self.gap)
            assert np.all(o[:, h * d:] == 0x5a5a)
            o = o[:, :h * d].reshape(total, h, d).transpose(1, 0, 2)
        else:
            o = o[:-64].reshape(h, total, d)
        lse = None
        if self.lse:
            lse = self.lse.numpy()
            assert np.all(lse[-16:] == 77.5)
            lse = lse[:-16].reshape(h, total)
        return o, lse

    def check(self, offsets=None):
        h, kv = self.heads, self.kv
        x = self.qkv
        want, tol = ref.packed_attention(x[:h], x[h:h + kv], x[h + kv:], self.offsets if offsets is None else offsets,
                                         self.scale, self.causal)
        o, lse = self.outputs()
        none = np.isnan(want[1])
        assert np.all(o[none] == 0x5a5a), "rows of no sequence"
        assert ref.close(bf16_to_f32(o)[~none], want[0][~none], tol[0][~none]), "o"
        if lse is not None:
            assert np.all(lse[none] == 77.5)
            assert ref.close(lse[~none], want[1][~none], tol[1][~none]), "lse"

    def free(self):
        for a in (self.x, self.off, self.o, self.lse):
            if a is not None:
                a.free()


def one(lib, *args, **kw):
    announce(f"flash_packed {args} {kw}")
    c = Call(lib, *args, **kw)
    c()
    c.check()
    c.free()


LENS = [[1], [2], [63], [64], [65], [127], [129], [200], [1, 1, 1], [0, 5, 0], [0, 0], [3, 8, 24, 69, 0, 200],
        [130, 1, 64, 33], [257, 256]]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(hiplib, lens, d, causal):
    one(hiplib, lens, 4, 2, d, causal, tail=4)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (7, 7), (12, 12), (21, 3), (8, 8), (16, 8), (32, 4), (40, 1)])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_heads_and_layouts(hiplib, heads, kv, d, layout):
    one(hiplib, [37, 0, 70, 5], heads, kv, d, layout=layout, lead=3, tail=9, gap=8 if layout == "tokens" else 0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_tiles_of_128_rows(hiplib, d, causal):
    """Enough tiles that they are of 128 rows, several of a sequence."""
    one(hiplib, [300, 17, 0, 128, 400, 64, 1], 64, 32, d, causal, tail=5)


@pytest.mark.parametrize("n", [64, 65, 255, 256, 257, 300, 1000, 5000])
def test_many_sequences(hiplib, n):
    """Sequences are searched 64 at a time."""
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 6, n)
    lens[n // 2], lens[n - 1] = 150, 70
    one(hiplib, lens, 3, 1, 64, tail=2, layout="tokens")


@pytest.mark.parametrize("heads,kv,d", [(5, 1, 128), (32, 8, 64), (16, 8, 128)])
def test_many_sequences_of_several_heads(hiplib, heads, kv, d):
    """Rows before the first sequence, empty ones at both ends, tiles of both
    sizes."""
    rng = np.random.default_rng(heads)
    lens = rng.integers(0, 12, 700)
    lens[:3], lens[300], lens[-3:] = 0, 190, 0
    one(hiplib, lens, heads, kv, d, lead=137, tail=40)


def test_one_long_sequence_of_one_head(hiplib):
    one(hiplib, [2500], 1, 1, 128)
    one(hiplib, [40, 2100, 30], 2, 1, 64, causal=False)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.5, 1e-30])
def test_scales(hiplib, scale):
    one(hiplib, [100, 30], 4, 2, 64, scale=scale)
    one(hiplib, [90, 30], 64, 16, 128, scale=scale)


def test_without_lse(hiplib):
    one(hiplib, [77, 12], 4, 4, 128, lse=False)


@pytest.mark.parametrize("value", [NAN, INF, 0xFF80, 0x7F7F])
@pytest.mark.parametrize("d,heads,kv", [(64, 4, 2), (128, 4, 1), (128, 64, 64), (64, 64, 32)])
def test_a_key_that_is_not_seen_does_not_reach_a_query(hiplib, value, d, heads, kv):
    """The last three tokens' keys and values of a sequence are NaN, infinities or
    the largest number: the queries before them do not change by a bit, nor the
    sequences beside."""
    announce(f"flash_packed hidden {value:x} {d} {heads} {kv}")
    lens, bad = [90, 150, 40], [237, 238, 239]

    def put(x):
        x[bad, heads:] = value

    plain, c = Call(hiplib, lens, heads, kv, d), Call(hiplib, lens, heads, kv, d, put=put)
    plain()
    c()
    (o, lse), (po, plse) = c.outputs(), plain.outputs()
    rows = [r for r in range(280) if r not in bad]
    assert np.array_equal(o[:, rows], po[:, rows]) and np.array_equal(lse[:, rows], plse[:, rows])
    if value == NAN:
        assert np.all(np.isnan(bf16_to_f32(o)[:, bad]))
    plain.free()
    c.free()


def test_offsets_that_fall_or_lie_outside_touch_nothing_else(hiplib):
    """Sequences whose offsets are in order come out all the same where others'
    lie past the end or before the begin (those are cut)."""
    announce("flash_packed offsets outside")
    c = Call(hiplib, [20, 30, 10], 4, 2, 64)
    c.off.free()
    c.off = DeviceArray.of(hiplib, np.array([-5, 20, 50, 1000], np.int32), abi.DTYPE_I32)
    c()
    c.check(offsets=[0, 20, 50, 60])
    c.free()


def test_many_offsets_that_fall_touch_nothing_else(hiplib):
    """In any order: rows of no sequence stay."""
    announce("flash_packed many offsets that fall")
    n = 900
    c = Call(hiplib, [2] * n, 4, 2, 64, tail=50)
    rng = np.random.default_rng(1)
    for offsets in (rng.permutation(c.offsets), c.offsets[::-1].copy(),
                    rng.integers(-2 ** 31, 2 * n, n + 1).astype(np.int32)):
        c.off.free()
        c.off = DeviceArray.of(hiplib, offsets, abi.DTYPE_I32)
        c()
        o, lse = c.outputs()
        assert np.all(o[:, 2 * n:] == 0x5a5a) and np.all(lse[:, 2 * n:] == 77.5)
    c.free()


def test_from_a_graph_that_follows_the_offsets(hiplib):
    announce("flash_packed from a graph")
    t = HipTimer()
    c = Call(hiplib, [50, 70, 0, 9], 8, 4, 128, layout="tokens")
    s = t.stream_create()
    hiplib.lib.vx_hip_set_stream(s)
    try:
        ex = t.capture(s, c)
        for lens in ([50, 70, 0, 9], [129, 0, 0, 0], [1, 2, 3, 4], [30, 30, 30, 39]):
            offsets = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
            for dst, host in ((c.off, offsets), (c.o, np.full(c.o.shape, 0x5a5a, np.uint16)),
                              (c.lse, np.full(c.lse.shape, 77.5, np.float32))):
                src = DeviceArray.of(hiplib, host, dst.dtype)
                t.sync()
                assert t.hip.hipMemcpy(ctypes.c_void_p(dst.ptr), ctypes.c_void_p(src.ptr), src.nbytes, 3) == 0
                t.sync()
                src.free()
            t.graph_launch(ex, s)
            t.sync()
            c.check(offsets=offsets)
        t.graph_destroy(ex)
    finally:
        hiplib.lib.vx_hip_set_stream(None)
        t.stream_destroy(s)
    c.free()

