"""vx_nn_gemm_i8_* on the GPU against the exact sum."""

import numpy as np
import pytest

from tests import packed_reference as ref
from tests.conftest import announce
from vx_amd import abi
from vx_amd.abi import bf16_to_f32
from vx_amd.runtime import DeviceArray, HipTimer, gemm_i8

pytestmark = pytest.mark.gpu

OUT = {"f32": abi.DTYPE_F32, "bf16": abi.DTYPE_BF16}
GUARD = 96


class Call:
    def __init__(self, lib, dtype, tokens, rows, cols, pad=0, skip=0, seed=0, x=None, w=None):
        rng = np.random.default_rng(seed)
        self.lib, self.dtype, self.ext, self.stride, self.skip = lib, dtype, (tokens, rows, cols), rows + pad, skip
        self.hx = rng.integers(-128, 128, (tokens, cols)).astype(np.int8) if x is None else x
        self.hw = rng.integers(-128, 128, (rows, cols)).astype(np.int8) if w is None else w
        self.hxs = rng.uniform(0.001, 0.1, tokens).astype(np.float32)
        self.hws = rng.uniform(0.001, 0.1, rows).astype(np.float32)
        self.x, self.w = DeviceArray.of(lib, self.hx, abi.DTYPE_I8), DeviceArray.of(lib, self.hw, abi.DTYPE_I8)
        self.xs, self.ws = DeviceArray.of(lib, self.hxs, abi.DTYPE_F32), DeviceArray.of(lib, self.hws, abi.DTYPE_F32)
        size = skip + tokens * self.stride + GUARD
        t = OUT[dtype]
        self.y = DeviceArray.of(lib, np.frombuffer(b"\x5a" * (size * abi.DTYPE_BYTES[t]), DeviceArray.NP[t]), t)

    def __call__(self, workspace=None, workspace_bytes=0):
        t = OUT[self.dtype]
        assert gemm_i8(self.lib, self.dtype, self.x.ptr, self.xs.ptr, self.w.ptr, self.ws.ptr,
                       self.y.ptr + self.skip * abi.DTYPE_BYTES[t], *self.ext, self.stride, workspace,
                       workspace_bytes) == 0

    def check(self):
        tokens, rows, _ = self.ext
        got = self.y.numpy()
        body = got[self.skip:self.skip + tokens * self.stride].reshape(tokens, self.stride)
        for rest in (got[:self.skip], got[self.skip + tokens * self.stride:], body[:, rows:]):
            assert np.all(np.ascontiguousarray(rest).view(np.uint8) == 0x5a), "written outside"
        want, tol = ref.gemm_i8(self.hx, self.hxs, self.hw, self.hws, self.dtype == "bf16")
        y = body[:, :rows]
        assert ref.close(bf16_to_f32(y) if self.dtype == "bf16" else y, want, tol)
        return body[:, :rows].copy()

    def free(self):
        for a in (self.x, self.w, self.xs, self.ws, self.y):
            a.free()


def one(lib, *args, **kw):
    announce(f"gemm_i8 {args} {kw}")
    c = Call(lib, *args, **kw)
    c()
    y = c.check()
    c.free()
    return y


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [16, 48, 64, 80, 1040])
@pytest.mark.parametrize("rows", [1, 3, 16, 17, 130])
@pytest.mark.parametrize("tokens", [1, 2, 16, 17, 33, 64])
def test_few_tokens(hiplib, dtype, tokens, rows, cols):
    one(hiplib, dtype, tokens, rows, cols)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [16, 64, 80, 320, 336, 1040])
@pytest.mark.parametrize("rows", [1, 127, 128, 261])
@pytest.mark.parametrize("tokens", [65, 128, 129, 300])
def test_tiles(hiplib, dtype, tokens, rows, cols):
    one(hiplib, dtype, tokens, rows, cols)


# sizes at which launches of every kind are chosen
LARGE = [(1, 9000, 768), (1, 100, 11008), (5, 2000, 4096), (24, 5000, 2048), (64, 4100, 1024), (80, 500, 4096),
         (100, 5000, 4096), (256, 1024, 4096), (300, 2100, 2048), (520, 3000, 1040), (777, 1300, 528), (1000, 5000, 512),
         (2100, 4400, 272)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("ext", LARGE)
def test_larger(hiplib, dtype, ext):
    one(hiplib, dtype, *ext)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,skip", [(4, 0), (1, 0), (3, 1), (8, 2), (0, 3)])
@pytest.mark.parametrize("tokens", [3, 40, 130])
def test_strides_and_alignment(hiplib, dtype, tokens, pad, skip):
    one(hiplib, dtype, tokens, 132, 96, pad=pad, skip=skip)


@pytest.mark.parametrize("tokens", [1, 20, 70])
def test_the_largest_sums(hiplib, tokens):
    """-128 throughout at the most columns: 131056 x 2^14, below 2^31."""
    x, w = np.full((tokens, 131056), -128, np.int8), np.full((19, 131056), -128, np.int8)
    w[1] = 127
    w[2, ::2] = 127
    one(hiplib, "f32", tokens, 19, 131056, x=x, w=w)


def test_scales_that_are_not_finite_stay_with_their_token_and_row(hiplib):
    announce("gemm_i8 scales that are not finite")
    for tokens in (7, 90):
        c = Call(hiplib, "f32", tokens, 40, 128)
        c.hxs[3], c.hws[5] = np.nan, np.inf
        c.xs.free(), c.ws.free()
        c.xs, c.ws = (DeviceArray.of(hiplib, h, abi.DTYPE_F32) for h in (c.hxs, c.hws))
        c()
        y = c.y.numpy()[:tokens * 40].reshape(tokens, 40)
        bad = np.zeros((tokens, 40), bool)
        bad[3], bad[:, 5] = True, True
        assert np.array_equal(~np.isfinite(y), bad)
        c.free()


@pytest.mark.parametrize("ext", [(1, 300, 4096), (80, 500, 4096), (256, 1024, 4096), (520, 600, 1040)])
def test_from_a_graph_with_and_without_a_workspace(hiplib, ext):
    """The same bits eager, captured without a workspace, and captured with one
    that is full of other numbers."""
    announce(f"gemm_i8 from a graph {ext}")
    t = HipTimer()
    c = Call(hiplib, "f32", *ext)
    c()
    want = c.check()
    need = hiplib.lib.vx_nn_gemm_i8_workspace(*ext)
    ws = DeviceArray.of(hiplib, np.full(max(need, 16), 0x7f, np.int8), abi.DTYPE_I8)
    s = t.stream_create()
    hiplib.lib.vx_hip_set_stream(s)
    try:
        graphs = [t.capture(s, c), t.capture(s, lambda: c(ws.ptr, ws.nbytes))]
        for _ in range(3):
            for ex in graphs:
                t.graph_launch(ex, s)
                t.sync()
                assert np.array_equal(c.check(), want)
            c()  # eager, on the same stream
            t.sync()
            assert np.array_equal(c.check(), want)
        for ex in graphs:
            t.graph_destroy(ex)
    finally:
        hiplib.lib.vx_hip_set_stream(None)
        t.stream_destroy(s)
    ws.free()
    c.free()
