"""vx_nn_token_logprobs_* where several tokens are likely and the others hold a
large negative number, as masks do: entropy, log probabilities and the likeliest
tokens against the definition in 64 bits."""

import numpy as np
import pytest

from tests import packed_reference as ref
from tests.conftest import announce
from tests.test_gpu_token_logprobs import Call
from vx_amd.runtime import HipTimer

pytestmark = pytest.mark.gpu

LOWEST = {"f32": -3.4028234663852886e38, "bf16": -3.3895313892515355e38}
MASKS = [None, -1e38, -1e37, -1e30, -1e9, -1e4]  # None: the type's lowest


def live_of(place, vocab):
    """Which tokens are not masked."""
    i = np.arange(vocab)
    return {"last": i >= vocab - 12, "first": i < 12, "middle": np.abs(i - vocab // 2) < 6,
            "odd": i % 2 == 1, "even": i % 2 == 0, "second half": i >= vocab // 2,
            "spread": i % (vocab // 11) == 2, "ends": (i < 3) | (i >= vocab - 3)}[place]


def check_divided_and_not(lib, c):
    """Eagerly, where long rows are divided, and captured without a workspace, where
    one workgroup has a row; the likeliest tokens and each logarithm."""
    t = HipTimer()
    c()
    c.check()
    s = t.stream_create()
    lib.lib.vx_hip_set_stream(s)
    try:
        ex = t.capture(s, c)
        for _ in range(2):
            t.graph_launch(ex, s)
            t.sync()
            c.check()
        t.graph_destroy(ex)
    finally:
        lib.lib.vx_hip_set_stream(None)
        t.stream_destroy(s)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [37, 3000, 40000, 150001])
@pytest.mark.parametrize("place", ["last", "first", "middle", "odd", "even", "second half", "spread", "ends"])
def test_several_likely_tokens_among_masked_ones(hiplib, dtype, vocab, place):
    """A thread, a wave or a slice whose logits are all masked adds nothing: times
    its count, the distance of its reference to the row's largest logit is past
    the range of f32."""
    announce(f"token_logprobs masked {place} {vocab} {dtype}")
    rng = np.random.default_rng(11)
    live = live_of(place, vocab)
    x = np.stack([np.where(live, 3 + rng.standard_normal(vocab), LOWEST[dtype] if m is None else m)
                  for m in MASKS])
    n = len(MASKS)
    given = np.stack([np.zeros(n, int), np.full(n, vocab - 1), np.full(n, vocab // 2),
                      np.full(n, np.flatnonzero(live)[1])], axis=1)
    c = Call(hiplib, dtype, x, given, 9)
    want, _ = ref.token_logprobs(c.logits, c.given, 9)
    assert want[1].min() > 0.3  # what a row of one token could not show
    check_divided_and_not(hiplib, c)
    c.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [37, 3000, 40000, 150001])
@pytest.mark.parametrize("place", ["last", "first", "odd", "spread"])
def test_distances_past_the_largest_number(hiplib, dtype, vocab, place):
    """Likely logits so large that a masked one's distance to them is infinite, and
    equal ones, whose entropy is the logarithm of their number."""
    announce(f"token_logprobs far apart {place} {vocab} {dtype}")
    live = live_of(place, vocab)
    x = np.stack([np.where(live, high, LOWEST[dtype] * part) for high in (3e38, 1e38, 0.0) for part in (1.0, 0.5)])
    at = np.flatnonzero(live)
    given = np.tile(at[[0, -1, len(at) // 2]], (len(x), 1))
    c = Call(hiplib, dtype, x, given, 5)
    check_divided_and_not(hiplib, c)
    c.free()
