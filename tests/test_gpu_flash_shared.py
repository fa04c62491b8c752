"""vx_nn_flash_attention_shared_bf16 on the GPU against the definition in 64
bits, with bounds from the arithmetic (tests/batch_reference.py)."""

import numpy as np
import pytest

from tests import batch_reference as ref
from tests.conftest import announce
from vx_amd import abi
from vx_amd.abi import bf16_to_f32, f32_to_bf16
from vx_amd.runtime import DeviceArray, HipTimer, flash_attention_shared

pytestmark = pytest.mark.gpu

HELD = 0x4248  # 50.0: what outputs hold before a call
NAN, INF = 0x7FC0, 0x7F80


class Call:
    """One call's operands. Rows that do not count (of the caches beyond lens,
    of the shared buffers beyond shared_len) hold NaN and infinities."""

    def __init__(self, lib, batch, heads, kv_heads, seq_q, shared_len, capacity, head_dim, lens,
                 causal=True, scale=None, extra=0, lse=True, seed=5, ones=False):
        rng = np.random.default_rng(seed)
        self.lib, self.lens, self.causal = lib, lens, causal
        self.ext = (batch, heads, kv_heads, seq_q, shared_len, capacity, head_dim)
        self.scale = head_dim ** -0.5 if scale is None else scale
        self.extra = extra

        def normal(*shape):
            return f32_to_bf16(rng.standard_normal(shape).astype(np.float32))

        self.q = normal(batch, heads, seq_q, head_dim)
        self.ks, self.vs = (normal(kv_heads, shared_len + extra, head_dim) for _ in range(2))
        self.k, self.v = (normal(batch, kv_heads, capacity, head_dim) for _ in range(2))
        for x in (self.ks, self.vs):
            x[:, shared_len:] = NAN
            x[:, shared_len:, ::3] = INF
        if lens is not None:
            for s, n in enumerate(lens):
                for x in (self.k, self.v):
                    x[s, :, max(n, 0) if n <= capacity else 0:] = NAN
                    x[s, :, max(n, 0) if n <= capacity else 0:, ::2] = INF
        bf, i32, f32 = abi.DTYPE_BF16, abi.DTYPE_I32, abi.DTYPE_F32
        self.d = {n: DeviceArray.of(lib, getattr(self, n), bf) if getattr(self, n).size else None
                  for n in ("q", "ks", "vs", "k", "v")}
        self.d["lens"] = DeviceArray.of(lib, np.array(lens, np.int32), i32) if lens is not None else None
        self.d["o"] = DeviceArray.of(lib, np.full(self.q.size + 64, HELD, np.uint16), bf)
        self.d["lse"] = (DeviceArray.of(lib, np.full(batch * heads * seq_q + 16, 50, np.float32), f32)
                         if lse else None)

    def ptr(self, name):
        return self.d[name].ptr if self.d[name] is not None else None

    def __call__(self, workspace=None, workspace_bytes=0):
        b, h, kv, n, p, cap, d = self.ext
        rc = flash_attention_shared(
            self.lib, *(self.ptr(x) for x in ("q", "ks", "vs", "k", "v", "lens", "o", "lse")), b, h, kv, n,
            p, cap, d, self.scale, self.causal, shared_capacity=p + self.extra, workspace=workspace,
            workspace_bytes=workspace_bytes)
        assert rc == 0

    def workspace_bytes(self):
        return self.lib.lib.vx_nn_flash_attention_shared_workspace(*self.ext)

    def results(self):
        return self.d["o"].numpy(), self.d["lse"].numpy() if self.d["lse"] else None

    def want(self):
        b, h, kv, n, p, cap, d = self.ext
        return ref.shared_attention(self.q, self.ks if p else None, self.vs if p else None,
                                    self.k if cap else None, self.v if cap else None, self.lens, p,
                                    self.scale, self.causal)

    def check(self, want=None):
        b, h, kv, n, p, cap, d = self.ext
        (wo, wl), (to, tl) = want or self.want()
        o, lse = self.results()
        size = b * h * n * d
        assert np.all(o[size:] == HELD), "o: written past its end"
        got = bf16_to_f32(o[:size]).astype(np.float64).reshape(wo.shape)
        held = np.isnan(wo)
        assert np.all(got[held] == 50), "a slot without a sequence was written"
        bad = ~(np.abs(got - wo) <= to) & ~held
        assert not bad.any(), (np.argwhere(bad)[0], got[bad][:4], wo[bad][:4], to[bad][:4], bad.sum())
        if lse is None:
            return
        assert np.all(lse[b * h * n:] == 50), "lse: written past its end"
        got = lse[:b * h * n].astype(np.float64).reshape(wl.shape)
        held = np.isnan(wl)
        assert np.all(got[held] == 50)
        none = wl == -np.inf
        assert np.all(got[none] == -np.inf)
        see = ~held & ~none
        bad = np.zeros_like(see)
        bad[see] = ~(np.abs(got[see] - wl[see]) <= tl[see])
        assert not bad.any(), (np.argwhere(bad)[0], got[bad][:4], wl[bad][:4], tl[bad][:4], bad.sum())

    def free(self):
        for a in self.d.values():
            if a is not None:
                a.free()


def both(lib, *args, **kw):
    """The call with the library's own workspace, and with one of the caller's."""
    c = Call(lib, *args, **kw)
    want = c.want()
    c()
    c.check(want)
    n = c.workspace_bytes()
    if n:
        ws = DeviceArray.of(lib, np.full(n + 256, 0xFF, np.uint8).view(np.int8), abi.DTYPE_I8)
        c()
        first = [x.copy() if x is not None else None for x in c.results()]
        c(ws.ptr, n)
        c.check(want)
        for a, b in zip(first, c.results()):
            assert a is None or np.array_equal(a, b), "the caller's workspace changes the result"
        assert np.all(ws.numpy()[n:] == -1), "written past the workspace"
        ws.free()
    c.free()


# batch, heads, kv_heads, seq_q, shared_len, capacity, head_dim, lens
CASES = [
    (1, 1, 1, 1, 0, 1, 64, [1]),
    (1, 1, 1, 1, 1, 0, 64, None),
    (1, 1, 1, 1, 1, 1, 128, [0]),
    (4, 12, 12, 1, 500, 64, 64, [1, 7, 63, 64]),
    (6, 8, 2, 1, 63, 100, 128, [1, 0, -1, 101, 100, 33]),
    (5, 4, 4, 1, 64, 65, 64, [65, 64, 32, 31, 2]),
    (3, 6, 2, 5, 65, 40, 128, [5, 40, 17]),
    # fewer own keys than queries: the first queries lie inside the prefix,
    # and before its begin where that is short too
    (4, 3, 1, 4, 2, 6, 64, [4, 2, 0, 6]),
    (3, 4, 2, 8, 3, 12, 128, [1, 0, 12]),
    (33, 21, 3, 5, 127, 33, 64, [(7 * i) % 29 + 5 for i in range(33)]),
    (17, 32, 4, 1, 1025, 130, 128, [(11 * i) % 131 for i in range(17)]),
    (9, 16, 2, 1, 4097, 5, 64, [(i % 7) - 1 for i in range(9)]),
    (3, 8, 2, 33, 129, 50, 64, [33, 50, 40]),
    (2, 8, 1, 70, 200, 150, 128, [70, 149]),
    (2, 4, 2, 130, 0, 200, 128, [130, 199]),
    (3, 4, 4, 128, 300, 128, 64, [128, 1, 90]),
    (1, 7, 1, 300, 1000, 310, 128, [310]),
    (70, 2, 2, 1, 96, 3, 128, [i % 4 for i in range(70)]),
    (130, 4, 1, 1, 640, 0, 64, None),
    (2, 2, 2, 3, 31, 7, 128, None),
    (64, 8, 1, 2, 2111, 70, 128, [2 + (5 * i) % 69 for i in range(64)]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", CASES)
def test_cases(hiplib, case, causal):
    announce(f"flash_shared {case[:7]} causal {causal}")
    both(hiplib, *case, causal=causal, extra=3 * (case[4] % 2))


@pytest.mark.parametrize("scale", [0.0, -0.125, 2.0])
def test_scales(hiplib, scale):
    announce(f"flash_shared scale {scale}")
    both(hiplib, 5, 8, 2, 3, 150, 40, 64, [3, 40, 20, 2, -1], scale=scale)


def test_without_lse(hiplib):
    announce("flash_shared without lse")
    both(hiplib, 6, 8, 2, 1, 300, 40, 128, [1, 40, 20, 2, -1, 0], lse=False)
    both(hiplib, 2, 8, 2, 64, 300, 70, 128, [64, 70], lse=False)


@pytest.mark.parametrize("value", [NAN, INF, 0xFF80, 0x7F7F])
@pytest.mark.parametrize("case", [(3, 4, 2, 5, 40, 60), (2, 8, 2, 40, 70, 70), (2, 4, 4, 130, 100, 260)])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_hidden_keys_do_not_reach_a_query(hiplib, case, head_dim, value):
    """The last key of each sequence is NaN, an infinity or the largest number:
    only its own query may see it."""
    announce(f"flash_shared hidden {case} {head_dim} {value:#x}")
    b, h, kv, n, p, cap = case
    lens = [cap - 3 - s for s in range(b)]
    clean = Call(hiplib, b, h, kv, n, p, cap, head_dim, lens)
    clean()
    o, lse = (x.copy() for x in clean.results())
    clean.free()
    for name in ("k", "v"):
        c = Call(hiplib, b, h, kv, n, p, cap, head_dim, lens)
        x = getattr(c, name)
        for s, m in enumerate(lens):
            x[s, :, m - 1] = value
        c.d[name].free()
        c.d[name] = DeviceArray.of(hiplib, x, abi.DTYPE_BF16)
        c()
        o2, lse2 = c.results()
        got = o2[:c.q.size].reshape(c.q.shape)[:, :, :-1]
        assert np.array_equal(got, o[:c.q.size].reshape(c.q.shape)[:, :, :-1]), name
        assert np.array_equal(lse2[:b * h * n].reshape(b, h, n)[:, :, :-1],
                              lse[:b * h * n].reshape(b, h, n)[:, :, :-1]), name
        c.free()


def test_as_the_attention_over_the_joined_cache(hiplib):
    """One sequence whose prefix and cache are dense and joined: the framework's
    attention gives the same up to rounding."""
    from vx_amd.runtime import flash_attention_fwd
    announce("flash_shared against flash_attention_fwd")
    c = Call(hiplib, 1, 8, 2, 7, 200, 56, 128, [56])
    c()
    joined = [DeviceArray.of(hiplib, np.concatenate([s, o[0]], axis=1)[None], abi.DTYPE_BF16)
              for s, o in ((c.ks, c.k), (c.vs, c.v))]
    o = DeviceArray(hiplib, c.q.shape, abi.DTYPE_BF16)
    lse = DeviceArray(hiplib, c.q.shape[:3], abi.DTYPE_F32)
    assert flash_attention_fwd(hiplib, c.d["q"].ptr, joined[0].ptr, joined[1].ptr, o.ptr, lse.ptr, 1, 8,
                               2, 7, 256, 128, c.scale, True) == 0
    (wo, wl), (to, tl) = c.want()
    got_o, got_lse = c.results()
    a = bf16_to_f32(got_o[:c.q.size]).reshape(wo.shape).astype(np.float64)
    b = bf16_to_f32(o.numpy()).astype(np.float64)
    assert np.all(np.abs(a - b) <= 2 * to)
    assert np.all(np.abs(got_lse[:56].reshape(wl.shape) - lse.numpy()) <= 2 * tl)
    for x in (*joined, o, lse):
        x.free()
    c.free()


@pytest.mark.parametrize("case", [(6, 8, 2, 1, 700, 40, 64, [1, 40, 20, 2, -1, 0]),
                                  (64, 8, 2, 1, 1500, 40, 128, [i % 41 for i in range(64)]),
                                  (2, 8, 2, 70, 300, 90, 128, [70, 88])])
def test_captured(hiplib, case):
    """Captured without a workspace and with one each, replayed with eager calls
    in between: every result within the bounds, and replays bit for bit."""
    announce(f"flash_shared captured {case[:7]}")
    t = HipTimer()
    stream = t.stream_create()
    hiplib.lib.vx_hip_set_stream(stream)
    c = Call(hiplib, *case)
    want = c.want()
    n = c.workspace_bytes()
    spaces = [DeviceArray(hiplib, (max(n, 16),), abi.DTYPE_I8) for _ in range(2)]
    graphs = []
    try:
        calls = [lambda: c(), lambda: c(spaces[0].ptr, n), lambda: c(spaces[1].ptr, n)]
        graphs = [t.capture(stream, f) for f in calls]
        first = {}
        for rep in range(3):
            c()
            t.sync()
            c.check(want)
            for i, g in enumerate(graphs):
                t.graph_launch(g, stream)
                t.sync()
                c.check(want)
                got = c.results()[0].copy()
                assert np.array_equal(first.setdefault(i, got), got), f"replay {rep} of graph {i}"
        assert np.array_equal(first[1], first[2])
    finally:
        for g in graphs:
            t.graph_destroy(g)
        for a in spaces:
            a.free()
        c.free()
        hiplib.lib.vx_hip_set_stream(None)
        t.stream_destroy(stream)


def test_two_streams_at_once(hiplib):
    """Calls on two streams, nothing waiting between them: each has a workspace
    of its own."""
    announce("flash_shared on two streams")
    t = HipTimer()
    streams = [t.stream_create() for _ in range(2)]
    calls, wants = [], []
    for i in range(2):
        calls.append(Call(hiplib, 48, 16, 2, 1, 3000 + 77 * i, 64, 128, [(3 * j + i) % 65 for j in range(48)],
                          seed=i))
        wants.append(calls[i].want())
    try:
        for s in streams:
            hiplib.lib.vx_hip_set_stream(s)
            calls[streams.index(s)]()
        t.sync()
        for _ in range(10):
            for s, c in zip(streams, calls):
                # a set stream keeps its workspace until the next is set
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


def test_per_thread_stream(hiplib):
    """hipStreamPerThread names a stream per thread: calls under it take no
    workspace of the library's, and two threads' calls run at once."""
    import threading
    announce("flash_shared under hipStreamPerThread")
    t = HipTimer()
    case = (40, 8, 2, 1, 1200, 40, 64, [i % 41 for i in range(40)])
    calls = [Call(hiplib, *case, seed=i) for i in range(2)]
    wants = [c.want() for c in calls]
    t.sync()
    failed = []

    def work(c):
        try:
            hiplib.lib.vx_hip_set_stream(2)  # hipStreamPerThread
            for _ in range(5):
                c()
            hiplib.lib.vx_hip_set_stream(None)
        except BaseException as e:  # noqa: BLE001 - reported below
            failed.append(e)

    before = held(hiplib)
    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    t.sync()
    assert not failed
    assert held(hiplib) == before
    for c, w in zip(calls, wants):
        c.check(w)
        c.free()


def held(lib):
    """The workspaces that the library keeps, and their bytes."""
    import ctypes
    out = (ctypes.c_int64 * 2)()
    assert lib.control(abi.HIP_CTRL_OP_WORKSPACES, out) == 1
    return tuple(out)


def test_a_streams_workspace_goes_with_it(hiplib):
    announce("flash_shared workspace of a stream")
    t = HipTimer()
    stream = t.stream_create()
    c = Call(hiplib, 64, 8, 2, 1, 1500, 40, 128, [i % 41 for i in range(64)])
    before = held(hiplib)
    try:
        hiplib.lib.vx_hip_set_stream(stream)
        c()
        assert held(hiplib)[0] == before[0] + 1
        assert held(hiplib)[1] >= before[1] + c.workspace_bytes() > before[1]
        c(), t.sync()
        assert held(hiplib)[0] == before[0] + 1
    finally:
        hiplib.lib.vx_hip_set_stream(None)
    assert held(hiplib) == before
    t.sync()
    c.check()
    c.free()
    t.stream_destroy(stream)


@pytest.mark.parametrize("case", [
    (33, 21, 3, 5, 2047, 60, 64, [(7 * i) % 56 + 5 for i in range(33)]),
    (33, 3, 3, 1, 2100, 9, 128, [i % 10 for i in range(33)]),
    (5, 5, 1, 1, 4000, 30, 128, [1, 30, 0, -1, 17]),
    (1, 7, 7, 1, 3000, 200, 64, [177])])
def test_odd_rows_in_parts(hiplib, case):
    """An odd number of queries in all, several parts of the keys."""
    announce(f"flash_shared odd rows {case[:7]}")
    assert case[0] * case[1] * case[3] % 2 == 1
    assert hiplib.lib.vx_nn_flash_attention_shared_workspace(*case[:7]) > 0
    both(hiplib, *case)


def test_a_large_workspace_is_not_kept(hiplib):
    """A call whose parts take more than the library keeps for a stream has them
    for itself: what is held stays within the limit, here and on the default
    stream, and smaller calls before and after keep their block."""
    announce("flash_shared large workspace")
    limit = 128 << 20
    lens = [i % 3 if i % 61 == 0 else -1 for i in range(4096)]
    large = Call(hiplib, 4096, 32, 1, 1, 130, 2, 128, lens, lse=False)
    small = Call(hiplib, 64, 8, 2, 1, 1500, 40, 128, [i % 41 for i in range(64)])
    assert large.workspace_bytes() > limit > small.workspace_bytes() > 0
    wants = large.want(), small.want()
    t = HipTimer()
    stream = t.stream_create()
    try:
        for s in (stream, None):
            hiplib.lib.vx_hip_set_stream(s)
            small()
            before = held(hiplib)
            for _ in range(2):
                large()
                small()
                assert held(hiplib) == before
            assert before[1] <= 2 * limit
            t.sync()
            large.check(wants[0])
            small.check(wants[1])
    finally:
        hiplib.lib.vx_hip_set_stream(None)
        t.sync()
        large.free()
        small.free()
        t.stream_destroy(stream)


# batch, heads, kv_heads, seq_q, shared_len, capacity; lens; and how the call is
# divided: one tile walks shared and own keys, 16-row tiles of shared and of own
# keys, rows of a wide tile, workgroups that divide a tile's shared and own keys
# (tests/test_batch_plans.py holds the rules to it)
PLANNED = [
    ((1, 2, 1, 1, 1500, 700), [699], (1, 0, 1, 64, 0, 2)),
    ((1, 2, 2, 3, 9000, 300), [300], (1, 0, 1, 64, 0, 9)),
    # no more than 16
    ((1, 2, 1, 1, 33000, 300), [300], (1, 0, 1, 64, 0, 16)),
    ((1, 4, 1, 8, 17000, 100), [77], (1, 0, 0, 64, 0, 16)),
    ((1, 1, 1, 1, 0, 270000), [269999], (1, 0, 1, 64, 0, 16)),
    ((3, 8, 2, 5, 200, 60), [60, 5, 33], (1, 0, 0, 64, 0, 1)),
    ((1, 4, 1, 6, 3000, 1300), [1201], (1, 0, 0, 64, 0, 8)),
    ((1, 8, 1, 5, 5100, 70), [70], (1, 0, 0, 64, 0, 10)),
    ((2, 4, 1, 40, 200, 900), [900, 41], (1, 0, 0, 128, 0, 2)),
    ((1, 4, 1, 30, 5000, 100), [87], (1, 0, 0, 128, 0, 9)),
    ((4, 12, 12, 1, 1000, 64), [64, 1, 0, 33], (0, 1, 1, 64, 4, 1)),
    ((16, 8, 8, 1, 4096, 256), [(19 * i) % 257 for i in range(16)], (0, 1, 1, 64, 16, 1)),
    ((3, 4, 2, 1, 1300, 1030), [1030, 600, -1], (0, 1, 1, 64, 5, 2)),
    ((4, 4, 2, 8, 700, 12), [12, 3, 8, 9], (0, 0, 1, 64, 2, 1)),
    ((8, 32, 8, 1, 3000, 1100), [(157 * i) % 1101 for i in range(8)], (0, 0, 1, 64, 11, 2)),
    ((16, 4, 2, 8, 700, 12), [i % 13 for i in range(16)], (0, 0, 1, 128, 2, 1)),
    ((20, 8, 1, 1, 1100, 1030), [1030 if i == 3 else 51 * i for i in range(20)], (0, 0, 1, 128, 4, 2)),
    ((64, 8, 2, 1, 4600, 40), [i % 41 if i % 4 else -1 for i in range(64)], (0, 0, 1, 128, 18, 1)),
    ((33, 21, 3, 5, 2047, 90), [(7 * i) % 86 + 5 if i % 3 else -1 for i in range(33)], (0, 0, 0, 64, 4, 1)),
    ((12, 16, 1, 2, 4000, 1100), [1100, 2, 0, 600] + [40] * 8, (0, 0, 0, 64, 15, 2)),
    ((64, 32, 8, 8, 600, 20), [i % 21 if i % 4 == 0 else -1 for i in range(64)], (0, 0, 0, 128, 1, 1)),
    ((32, 64, 2, 2, 4200, 1030), [1030 if i == 8 else 31 * i if i % 4 == 0 else -1 for i in range(32)],
     (0, 0, 0, 128, 8, 2)),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("case", PLANNED, ids=lambda c: "-".join(map(str, c[0])))
def test_each_way_of_dividing(hiplib, case, head_dim, causal):
    announce(f"flash_shared divided {case[0]} {head_dim} causal {causal}")
    both(hiplib, *case[0], head_dim, case[1], causal=causal, extra=case[0][4] % 2)


# fewer own keys than queries, tiles of shared keys alone: 16 rows, 64 and 128
# rows with 16-row tiles of own keys and without
SHORT = [((2, 2, 2, 8, 700, 12), (0, 1, 1, 64, 2, 1)), ((4, 4, 2, 8, 700, 12), (0, 0, 1, 64, 2, 1)),
         ((16, 4, 2, 8, 700, 12), (0, 0, 1, 128, 2, 1)), ((3, 4, 2, 20, 1000, 30), (0, 0, 0, 64, 4, 1)),
         ((64, 32, 8, 8, 600, 20), (0, 0, 0, 128, 1, 1))]


@pytest.mark.parametrize("value", [NAN, INF, 0xFF80, 0x7F7F])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("case", SHORT, ids=lambda c: "-".join(map(str, c[0])))
def test_hidden_shared_keys_do_not_reach_a_query(hiplib, case, head_dim, value):
    """The last three shared keys are NaN, infinities or the largest number: a
    query that ends before them gets its result all the same, and one that sees
    them gets NaN where they are NaN."""
    announce(f"flash_shared hidden shared {case[0]} {head_dim} {value:#x}")
    b, h, kv, n, p, cap = case[0]
    # few sequences, so that the plain result is quick
    lens = [s % n if s % (b // 4 + 1) == 0 or b < 17 else -1 for s in range(b)]
    clean = Call(hiplib, *case[0], head_dim, lens)
    (wo, wl), (to, tl) = clean.want()
    clean.free()
    last = np.array([[p + m - n + i for i in range(n)] for m in lens])
    before = np.broadcast_to(((last < p - 3) & (np.array(lens) >= 0)[:, None])[:, None], (b, h, n))
    after = np.broadcast_to(((last >= p - 1) & (np.array(lens) >= 0)[:, None])[:, None], (b, h, n))
    assert before.any() and after.any()
    for name in ("ks", "vs"):
        c = Call(hiplib, *case[0], head_dim, lens)
        getattr(c, name)[:, p - 3:p] = value
        c.d[name].free()
        c.d[name] = DeviceArray.of(hiplib, getattr(c, name), abi.DTYPE_BF16)
        c()
        o, lse = c.results()
        o = bf16_to_f32(o[:c.q.size]).astype(np.float64).reshape(wo.shape)
        lse = lse[:b * h * n].astype(np.float64).reshape(wl.shape)
        assert np.all(np.abs(o - wo)[before] <= to[before]), name
        assert np.all(np.abs(lse - wl)[before] <= tl[before]), name
        assert value != NAN or np.all(np.isnan(o[after])), name
        c.free()
