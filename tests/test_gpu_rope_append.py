"""vx_nn_rope_append_* on the GPU against the definition in 64 bits."""

import numpy as np
import pytest

from tests import batch_reference as ref
from tests.conftest import announce
from vx_amd import abi
from vx_amd.abi import bf16_to_f32, f32_to_bf16
from vx_amd.runtime import DeviceArray, HipTimer, rope_append

pytestmark = pytest.mark.gpu

# batch, seq_q, heads, kv_heads, head_dim, shared_len, capacity, lens
CASES = [
    (1, 1, 1, 1, 8, 0, 1, [1]),
    (4, 1, 12, 12, 64, 500, 64, [1, 7, 63, 64]),
    (3, 5, 6, 2, 128, 17, 9, [5, 9, 7]),
    # more new tokens than the cache holds of one, a slot without a sequence,
    # one past its capacity, queries inside the prefix and before its begin
    (6, 4, 7, 1, 72, 2, 6, [4, 2, -1, 7, 0, 6]),
    (2, 3, 2, 2, 512, 1, 3, [3, 0]),
    (5, 33, 3, 3, 24, 100, 40, [33, 40, 12, 39, -5]),
    (2, 2, 4, 4, 64, 3, 5, None),
]


def inputs(case, dtype, seed=3):
    b, n, h, kv, d, shared, cap, lens = case
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((b, n, h + 2 * kv, d)).astype(np.float32)
    x16 = f32_to_bf16(x)
    return (x, x) if dtype == "f32" else (x16, bf16_to_f32(x16))


class Call:
    def __init__(self, lib, case, dtype, table=True, seed=3):
        b, n, h, kv, d, shared, cap, lens = case
        self.case, self.dtype, self.lib = case, dtype, lib
        host, self.x = inputs(case, dtype, seed)
        self.table = ref.rope_table(shared + cap, d) if table else None
        rng = np.random.default_rng(99)
        self.before = [f32_to_bf16(rng.standard_normal((np.prod(s) + 64,)).astype(np.float32))
                       for s in ((b, h, n, d), (b, kv, cap, d), (b, kv, cap, d))]
        self.shapes = [(b, h, n, d), (b, kv, cap, d), (b, kv, cap, d)]
        self.qkv = DeviceArray.of(lib, host, abi.DTYPE_F32 if dtype == "f32" else abi.DTYPE_BF16)
        self.rope = DeviceArray.of(lib, self.table, abi.DTYPE_F32) if table else None
        self.lens = DeviceArray.of(lib, np.array(lens, np.int32), abi.DTYPE_I32) if lens else None
        self.out = [DeviceArray.of(lib, x, abi.DTYPE_BF16) for x in self.before]

    def __call__(self):
        b, n, h, kv, d, shared, cap, lens = self.case
        rc = rope_append(self.lib, self.dtype, self.qkv.ptr, self.rope.ptr if self.rope else None,
                         self.lens.ptr if self.lens else None, *(o.ptr for o in self.out), b, n, h, kv,
                         d, shared, cap, shared + cap if self.rope else 0)
        assert rc == 0

    def check(self):
        b, n, h, kv, d, shared, cap, lens = self.case
        sizes = [int(np.prod(s)) for s in self.shapes]
        held = [bf16_to_f32(x[:m]).astype(np.float64).reshape(s)
                for x, m, s in zip(self.before, sizes, self.shapes)]
        want, tol = ref.rope_append(self.x, self.table, lens, *held, shared)
        for name, o, before, m, s, w, t in zip("qkv", self.out, self.before, sizes, self.shapes, want, tol):
            got = o.numpy()
            assert np.array_equal(got[m:], before[m:]), f"{name}: written past its end"
            got = bf16_to_f32(got[:m]).astype(np.float64).reshape(s)
            assert np.all(np.abs(got - w) <= t), name

    def free(self):
        for a in (self.qkv, self.rope, self.lens, *self.out):
            if a is not None:
                a.free()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", CASES)
def test_cases(hiplib, case, dtype):
    announce(f"rope_append {case} {dtype}")
    c = Call(hiplib, case, dtype)
    c()
    c.check()
    c.free()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_without_a_table(hiplib, dtype):
    announce(f"rope_append without a table {dtype}")
    c = Call(hiplib, CASES[3], dtype, table=False)
    c()
    c.check()
    c.free()


def test_captured_follows_the_lengths(hiplib):
    """A replayed graph reads lens as it is then; eager calls in between."""
    announce("rope_append captured")
    case = (3, 2, 4, 2, 64, 5, 16, [2, 3, 4])
    c = Call(hiplib, case, "bf16")
    t = HipTimer()
    stream = t.stream_create()
    hiplib.lib.vx_hip_set_stream(stream)
    graph = None
    try:
        graph = t.capture(stream, c)
        for step in range(3):
            lens = [2 + step, 9 + step, -1 if step == 1 else 16]
            new = DeviceArray.of(hiplib, np.array(lens, np.int32), abi.DTYPE_I32)
            assert t.hip.hipMemcpy(abi_ptr(c.lens.ptr), abi_ptr(new.ptr), 12, 3) == 0
            for o, before in zip(c.out, c.before):
                src = DeviceArray.of(hiplib, before, abi.DTYPE_BF16)
                t.sync()
                assert t.hip.hipMemcpy(abi_ptr(o.ptr), abi_ptr(src.ptr), o.nbytes, 3) == 0
                src.free()
            new.free()
            t.sync()
            t.graph_launch(graph, stream)
            t.sync()
            c.case = case[:7] + (lens,)
            c.check()
    finally:
        hiplib.lib.vx_hip_set_stream(None)
        if graph is not None:
            t.graph_destroy(graph)
        t.stream_destroy(stream)
        c.free()


def abi_ptr(p):
    import ctypes
    return ctypes.c_void_p(p)
