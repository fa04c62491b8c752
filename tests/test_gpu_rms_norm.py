"""vx_nn_rms_norm_* and vx_nn_quantize_i8_* on the GPU against the definition:
the computed values in 64 bits, the 8-bit ones bit for bit."""

import numpy as np
import pytest

from tests import packed_reference as ref
from tests.conftest import announce
from vx_amd import abi
from vx_amd.abi import bf16_to_f32, f32_to_bf16
from vx_amd.llama import quantize_rows
from vx_amd.runtime import DeviceArray, HipTimer, quantize_i8, rms_norm

pytestmark = pytest.mark.gpu

TYPE = {"f32": abi.DTYPE_F32, "bf16": abi.DTYPE_BF16}
GUARD = 96  # elements behind an output, which stay as they were


def held(x, dtype):
    """x as the stream's type holds it: what goes to the GPU, and as f32."""
    if dtype == "f32":
        return x.astype(np.float32), x.astype(np.float32)
    h = f32_to_bf16(x.astype(np.float32))
    return h, bf16_to_f32(h)


def fresh(lib, n, dtype):
    """An output of n elements and a guard, every byte 0x5a."""
    host = np.frombuffer(b"\x5a" * ((n + GUARD) * abi.DTYPE_BYTES[dtype]), DeviceArray.NP[dtype])
    return DeviceArray.of(lib, host, dtype)


def taken(a, n):
    got = a.numpy()
    assert np.all(got[n:].view(np.uint8) == 0x5a), "written past its end"
    return got[:n]


class Call:
    """One call with outputs of its own; `skip` elements shift every operand off
    its allocation's alignment."""

    def __init__(self, lib, dtype, x, residual, weight, outputs, eps=1e-5, pad=0, skip=0):
        self.lib, self.dtype, self.eps, self.outputs = lib, dtype, eps, outputs
        self.rows, self.dim = x.shape
        self.stride, self.skip = self.dim + pad, skip
        wide = np.full((self.rows, self.stride), 3e4)
        wide[:, :self.dim] = x
        host, as_f32 = held(wide, dtype)
        self.x = as_f32[:, :self.dim]
        self.residual = self.weight = None
        self.dev = {"x": self._put(host, TYPE[dtype])}
        if residual is not None:
            host, self.residual = held(residual, dtype)
            self.dev["residual"] = self._put(host, TYPE[dtype])
        if weight is not None:
            self.weight = weight.astype(np.float32)
            self.dev["weight"] = self._put(self.weight, abi.DTYPE_F32)
        self.out = {}
        n = self.rows * self.dim
        for name, size, t in (("sum", n, TYPE[dtype]), ("y", n, abi.DTYPE_BF16), ("q", n, abi.DTYPE_I8),
                              ("q_scale", self.rows, abi.DTYPE_F32)):
            if name in outputs or (name == "q_scale" and "q" in outputs):
                self.out[name] = (fresh(lib, size + skip, t), size, t)

    def _put(self, host, t):
        flat = np.concatenate([np.zeros(self.skip, host.dtype), host.reshape(-1)])
        return DeviceArray.of(self.lib, flat, t), t

    def ptr(self, name):
        if name in self.dev:
            a, t = self.dev[name]
        elif name in self.out:
            a, _, t = self.out[name]
        else:
            return None
        return a.ptr + self.skip * abi.DTYPE_BYTES[t]

    def __call__(self):
        names = ("x", "residual", "weight", "sum", "y", "q", "q_scale")
        assert rms_norm(self.lib, self.dtype, *map(self.ptr, names), self.rows, self.dim, self.eps,
                        self.stride) == 0

    def got(self, name):
        a, size, _ = self.out[name]
        whole = taken(a, size + self.skip)
        return whole[self.skip:]

    def check(self):
        want, tol = ref.rms_norm(self.x, self.residual, self.weight, self.eps,
                                 ref.BF16 if self.dtype == "bf16" else 0.0)
        shape = (self.rows, self.dim)
        if "sum" in self.out:
            s = self.got("sum").reshape(shape)
            assert ref.close(bf16_to_f32(s) if self.dtype == "bf16" else s, want[0], tol[0]), "sum"
        if "y" in self.out:
            assert ref.close(bf16_to_f32(self.got("y").reshape(shape)), want[1], tol[1]), "y"
        if "q" in self.out:
            assert ref.close(self.got("q_scale"), want[2], tol[2]), "q_scale"
            assert np.array_equal(self.got("q").reshape(shape), want[3]), "q"

    def free(self):
        for a, *_ in [*self.dev.values(), *self.out.values()]:
            a.free()


def stream(rng, rows, dim):
    return rng.standard_normal((rows, dim)) * np.where(rng.random(dim) < 0.02, 20.0, 1.0)


# every way to hold a row, at both ends of its range, and odd sizes
DIMS = [1, 7, 8, 64, 500, 512, 513, 768, 1000, 1024, 1032, 2048, 2056, 4095, 4096, 4104, 8192, 8200, 11008, 16384,
        16392, 20001, 32768]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", DIMS)
def test_sizes(hiplib, dim, dtype):
    announce(f"rms_norm 3 x {dim} {dtype}")
    rng = np.random.default_rng(dim)
    c = Call(hiplib, dtype, stream(rng, 3, dim), stream(rng, 3, dim), 1 + 0.2 * rng.standard_normal(dim),
             ("sum", "y", "q"))
    c()
    c.check()
    c.free()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("outputs", [("y",), ("q",), ("sum", "q"), ("sum", "y"), ("y", "q")])
@pytest.mark.parametrize("residual,weight", [(False, False), (True, False), (False, True)])
def test_operands_that_may_be_missing(hiplib, dtype, outputs, residual, weight):
    announce(f"rms_norm {outputs} {residual} {weight} {dtype}")
    rng = np.random.default_rng(5)
    x = stream(rng, 5, 320)
    c = Call(hiplib, dtype, x, stream(rng, 5, 320) if residual else None,
             rng.standard_normal(320) if weight else None, outputs)
    c()
    c.check()
    c.free()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pad,skip", [(8, 0), (3, 0), (0, 1), (5, 3), (24, 8)])
def test_strides_and_alignment(hiplib, dtype, pad, skip):
    announce(f"rms_norm pad {pad} skip {skip} {dtype}")
    rng = np.random.default_rng(6)
    c = Call(hiplib, dtype, stream(rng, 4, 1000), stream(rng, 4, 1000), rng.standard_normal(1000),
             ("sum", "y", "q"), pad=pad, skip=skip)
    c()
    c.check()
    c.free()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("over", ["x", "residual"])
@pytest.mark.parametrize("dim", [768, 1001, 20000])
def test_the_sum_in_place(hiplib, dtype, over, dim):
    announce(f"rms_norm sum over {over} {dim} {dtype}")
    rng = np.random.default_rng(7)
    c = Call(hiplib, dtype, stream(rng, 6, dim), stream(rng, 6, dim), rng.standard_normal(dim), ("y", "q"))
    names = ["x", "residual", "weight", over, "y", "q", "q_scale"]
    assert rms_norm(hiplib, dtype, *map(c.ptr, names), 6, dim, 1e-5) == 0
    c.check()
    want, tol = ref.rms_norm(c.x, c.residual, c.weight, 1e-5, ref.BF16 if dtype == "bf16" else 0.0)
    s = c.dev[over][0].numpy().reshape(6, dim)
    assert ref.close(bf16_to_f32(s) if dtype == "bf16" else s, want[0], tol[0])
    c.free()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("eps", [0.0, 1e-5, 1.0])
def test_rows_at_the_ends_of_the_range(hiplib, dtype, eps):
    """Zeros, numbers near the smallest and the largest, one number alone, and
    rows with infinities and NaNs beside ordinary ones."""
    announce(f"rms_norm ends of the range eps {eps} {dtype}")
    rng = np.random.default_rng(8)
    x = stream(rng, 12, 264)
    x[1] = 0.0
    x[2] *= 1e-38
    x[3] = 0.0
    x[3, 5] = 1e-44 if dtype == "f32" else 1e-40
    x[4] *= 1e35
    x[5] = 0.0
    x[5, 263] = -2.5
    x[6, 100] = np.inf
    x[7, 0] = np.nan
    x[8, 3], x[8, 4] = -np.inf, np.inf
    x[9] = 1e-42 * np.arange(264)
    x[10] = 3e38 * np.where(np.arange(264) % 2, 1, -1)
    c = Call(hiplib, dtype, x, None, None, ("sum", "y", "q"), eps=eps)
    c()
    if eps == 0.0:  # 0 * inf of the row of zeros
        assert np.all(np.isnan(bf16_to_f32(c.got("y").reshape(12, 264)))[1])
    rows = [r for r in range(12) if not (eps == 0.0 and r == 1)]
    with np.errstate(all="ignore"):
        want, tol = ref.rms_norm(c.x, None, None, eps, ref.BF16 if dtype == "bf16" else 0.0)
    y = bf16_to_f32(c.got("y").reshape(12, 264))
    assert np.array_equal(c.got("q").reshape(12, 264), want[3])
    finite = [r for r in rows if r not in (6, 7, 8)]
    # s r below the smallest normal f32 may lose its last bits
    assert ref.close(y[finite], want[1][finite], tol[1][finite] + 2.0 ** -126)
    assert ref.close(c.got("q_scale")[finite], want[2][finite], tol[2][finite])
    assert np.all(np.isnan(c.got("q_scale")[[6, 7, 8]])) and np.all(np.isnan(y[7]))
    c.free()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,dim", [(1, 1), (4, 64), (3, 1001), (2, 11008), (1, 32768), (300, 40)])
def test_quantize(hiplib, dtype, rows, dim):
    """As the weights are quantized, halves among them."""
    announce(f"quantize_i8 {rows} x {dim} {dtype}")
    rng = np.random.default_rng(9)
    x = stream(rng, rows, dim)
    x[rows // 2] = (rng.integers(-254, 255, dim) / 2) * (1.0 if dim > 1 else 0.0)  # unit 1 if 127 is there
    x[rows // 2, 0] = 127.0
    host, f32 = held(x, dtype)
    dx = DeviceArray.of(hiplib, host, TYPE[dtype])
    q, s = fresh(hiplib, rows * dim, abi.DTYPE_I8), fresh(hiplib, rows, abi.DTYPE_F32)
    assert quantize_i8(hiplib, dtype, dx.ptr, q.ptr, s.ptr, rows, dim) == 0
    want, scale = quantize_rows(f32)
    assert np.array_equal(taken(s, rows), scale)
    assert np.array_equal(taken(q, rows * dim).reshape(rows, dim), want)
    for a in (dx, q, s):
        a.free()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_every_half_and_its_neighbours(hiplib, dtype):
    """Quotients at k + 1/2, and the numbers next to them."""
    announce(f"quantize_i8 halves {dtype}")
    rng = np.random.default_rng(10)
    rows = []
    for top in (127.0, 126.9, 1.0, 0.3, 3e-5, 77.7, 1e30, 6e-30):
        unit = np.float32(np.float32(top) / np.float32(127.0))
        half = (np.arange(-126, 127) + 0.5).astype(np.float32) * unit
        row = np.concatenate([half, np.nextafter(half, np.float32(np.inf)), np.nextafter(half, np.float32(-np.inf))])
        rows.append(np.concatenate([[np.float32(top)], np.clip(row, -top, top)]))
    x = np.array(rows, np.float32)
    x[:, 1:] = x[:, 1:][:, rng.permutation(x.shape[1] - 1)]
    host, f32 = held(x, dtype)
    dx = DeviceArray.of(hiplib, host, TYPE[dtype])
    q, s = fresh(hiplib, x.size, abi.DTYPE_I8), fresh(hiplib, len(x), abi.DTYPE_F32)
    assert quantize_i8(hiplib, dtype, dx.ptr, q.ptr, s.ptr, *x.shape) == 0
    want, scale = quantize_rows(f32)
    assert np.array_equal(taken(s, len(x)), scale)
    assert np.array_equal(taken(q, x.size).reshape(x.shape), want)
    for a in (dx, q, s):
        a.free()


def test_from_a_graph_on_another_stream(hiplib):
    """Captured, replayed with the inputs changed in between, the sum in place."""
    announce("rms_norm from a graph")
    rng = np.random.default_rng(11)
    t = HipTimer()
    c = Call(hiplib, "bf16", stream(rng, 40, 768), stream(rng, 40, 768), rng.standard_normal(768), ("sum", "y", "q"))
    c()
    t.sync()
    eager = [c.got(n).copy() for n in ("sum", "y", "q", "q_scale")]
    stream_ = t.stream_create()
    hiplib.lib.vx_hip_set_stream(stream_)
    try:
        ex = t.capture(stream_, c)
        for _ in range(3):
            t.graph_launch(ex, stream_)
            t.sync()
            assert all(np.array_equal(c.got(n), e) for n, e in zip(("sum", "y", "q", "q_scale"), eager))
            c()  # eager on the same stream in between
            t.sync()
        t.graph_destroy(ex)
    finally:
        hiplib.lib.vx_hip_set_stream(None)
        t.stream_destroy(stream_)
    c.check()
    c.free()


@pytest.mark.parametrize("dtype,rows,dim", [("bf16", 2100, 4096), ("f32", 1100, 4096), ("bf16", 5000, 3600)])
def test_inputs_past_the_caches(hiplib, dtype, rows, dim):
    announce(f"rms_norm past the caches {rows} x {dim} {dtype}")
    rng = np.random.default_rng(12)
    c = Call(hiplib, dtype, stream(rng, rows, dim), stream(rng, rows, dim), rng.standard_normal(dim), ("sum", "y", "q"))
    c()
    c.check()
    c.free()
