"""What the ops of a batch that shares a prompt refuse, and the workspaces they
name: checked on the host before a GPU is looked for, so without one too."""

import ctypes

import pytest

from vx_amd.runtime import LIB_PATH, DispatchLibrary, flash_attention_shared, rope_append, sample

EINVAL, ENODEV, ENOTDEV, EUNSUPP = -1, -2, -3, -4


@pytest.fixture(scope="module")
def lib():
    if not LIB_PATH.exists():
        from vx_amd.build import build
        build()
    return DispatchLibrary()


@pytest.fixture(scope="module")
def p():
    """An aligned host address: what no op accepts as an operand."""
    buf = ctypes.create_string_buffer(4096 + 64)
    _keep.append(buf)
    return (ctypes.addressof(buf) + 63) // 64 * 64


_keep: list = []

ROPE = dict(dtype="bf16", batch=2, seq_q=1, heads=4, kv_heads=2, head_dim=64, shared_len=10,
            capacity=8, rope_len=18)


def rope(lib, p, **kw):
    a = dict(qkv=p, rope=p, lens=p, q=p, k_cache=p, v_cache=p, **ROPE)
    a.update(kw)
    return rope_append(lib, **a)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kw,code", [
    (dict(qkv=None), EINVAL), (dict(q=None), EINVAL), (dict(k_cache=None), EINVAL),
    (dict(v_cache=None), EINVAL), (dict(batch=0), EINVAL), (dict(seq_q=0), EINVAL),
    (dict(heads=-4), EINVAL), (dict(kv_heads=0), EINVAL), (dict(head_dim=0), EINVAL),
    (dict(capacity=0), EINVAL), (dict(shared_len=-1), EINVAL), (dict(rope_len=17), EINVAL),
    (dict(head_dim=60), EUNSUPP), (dict(head_dim=520), EUNSUPP), (dict(batch=2 ** 41), EINVAL),
    (dict(batch=2 ** 40, seq_q=2 ** 20), EUNSUPP), (dict(batch=2 ** 26), EUNSUPP), (dict(heads=2 ** 33), EUNSUPP),
    (dict(capacity=2 ** 40, rope=None), EUNSUPP)])
def test_rope_append_refuses(lib, p, dtype, kw, code):
    assert rope(lib, p, **{"dtype": dtype, **kw}) == code


def test_rope_append_refuses_alignment(lib, p):
    for name in ("qkv", "rope", "q", "k_cache", "v_cache"):
        assert rope(lib, p, **{name: p + 8}) == EUNSUPP, name
    assert rope(lib, p, lens=p + 2) == EUNSUPP
    # good arguments, memory that is not a GPU's (or no GPU)
    assert rope(lib, p) == (ENOTDEV if lib.device_count() > 0 else ENODEV)
    assert rope(lib, p, rope=None, rope_len=0, lens=None) in (ENOTDEV, ENODEV)


SHARED = dict(batch=2, heads=4, kv_heads=2, seq_q=1, shared_len=10, capacity=8, head_dim=64,
              scale=0.125, causal=True)


def shared(lib, p, **kw):
    a = dict(q=p, k_shared=p, v_shared=p, k=p, v=p, lens=p, o=p, lse=p, **SHARED)
    a.update(kw)
    return flash_attention_shared(lib, **a)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), EINVAL), (dict(o=None), EINVAL), (dict(k_shared=None), EINVAL),
    (dict(v_shared=None), EINVAL), (dict(k=None), EINVAL), (dict(v=None), EINVAL),
    (dict(batch=0), EINVAL), (dict(heads=0), EINVAL), (dict(kv_heads=0), EINVAL),
    (dict(heads=5), EINVAL), (dict(seq_q=0), EINVAL), (dict(shared_len=-1), EINVAL),
    (dict(capacity=-1), EINVAL), (dict(shared_len=0, capacity=0), EINVAL),
    (dict(head_dim=96), EUNSUPP), (dict(head_dim=256), EUNSUPP), (dict(scale=float("nan")), EINVAL),
    (dict(scale=float("inf")), EINVAL), (dict(shared_capacity=9), EINVAL),
    (dict(shared_capacity=2 ** 23), EINVAL), (dict(shared_len=2 ** 23), EUNSUPP),
    (dict(capacity=2 ** 23), EUNSUPP), (dict(seq_q=2 ** 22), EUNSUPP),
    (dict(batch=2 ** 40, seq_q=2 ** 39), EUNSUPP)])
def test_shared_attention_refuses(lib, p, kw, code):
    assert shared(lib, p, **kw) == code


@pytest.mark.parametrize("scale", [3e38, -3e38])
def test_shared_attention_refuses_a_scale_past_base_2(lib, p, scale):
    assert shared(lib, p, scale=scale) == EINVAL


def test_shared_attention_refuses_alignment(lib, p):
    for name in ("q", "k_shared", "v_shared", "k", "v", "o"):
        assert shared(lib, p, **{name: p + 8}) == EUNSUPP, name
    assert shared(lib, p, lens=p + 1) == EUNSUPP and shared(lib, p, lse=p + 2) == EUNSUPP
    assert shared(lib, p, workspace=p + 8, workspace_bytes=1 << 40) == EUNSUPP
    away = ENOTDEV if lib.device_count() > 0 else ENODEV
    assert shared(lib, p) == away
    assert shared(lib, p, shared_len=0, k_shared=None, v_shared=None) == away
    assert shared(lib, p, capacity=0, k=None, v=None, lens=None, lse=None) == away


def test_shared_attention_workspace(lib, p):
    size = lib.lib.vx_nn_flash_attention_shared_workspace
    assert size(0, 4, 2, 1, 10, 8, 64) == EINVAL and size(1, 4, 2, 1, 10, 8, 80) == EUNSUPP
    for ext in ((2, 4, 2, 1, 10, 8, 64), (64, 32, 4, 1, 8192, 512, 128), (8, 32, 8, 256, 4096, 300, 128)):
        n = size(*ext)
        assert n >= 0
        if n:
            b, h, kv, sq, sl, cap, d = ext
            kw = dict(batch=b, heads=h, kv_heads=kv, seq_q=sq, shared_len=sl, capacity=cap, head_dim=d)
            assert shared(lib, p, workspace=p, workspace_bytes=n - 1, **kw) == EINVAL


@pytest.mark.parametrize("ext", [(33, 21, 3, 5, 2047, 333, 64), (33, 21, 3, 5, 2047, 333, 128), (65, 3, 3, 1, 2100, 9, 64),
                                 (5, 5, 1, 1, 4000, 30, 128), (1, 7, 7, 1, 3000, 200, 64)])
def test_shared_attention_parts_are_aligned(lib, ext):
    """Parts of an odd number of rows, 8 bytes past a multiple of 16 each, begin
    on 16 bytes all the same."""
    b, h, kv, n, p, cap, d = ext
    rows = b * h * n
    assert rows % 2 == 1
    size = lib.lib.vx_nn_flash_attention_shared_workspace(*ext)
    part = (rows * (d + 2) * 4 + 15) // 16 * 16
    assert size >= 2 * part and size % part == 0


def draw(lib, p, **kw):
    a = dict(dtype="f32", logits=p, temperature=p, top_k=p, top_p=p, min_p=p, u=p, tokens=p,
             logprob=p, rows=4, vocab=100)
    a.update(kw)
    return sample(lib, **a)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kw,code", [
    (dict(logits=None), EINVAL), (dict(u=None), EINVAL), (dict(tokens=None), EINVAL),
    (dict(rows=0), EINVAL), (dict(rows=2 ** 21 + 1), EINVAL), (dict(vocab=0), EINVAL),
    (dict(vocab=2 ** 30 + 1), EINVAL), (dict(stride=99), EINVAL), (dict(stride=2 ** 50), EINVAL)])
def test_sample_refuses(lib, p, dtype, kw, code):
    assert draw(lib, p, **{"dtype": dtype, **kw}) == code


def test_sample_refuses_alignment(lib, p):
    for name in ("logits", "temperature", "top_k", "top_p", "min_p", "u", "tokens", "logprob"):
        assert draw(lib, p, **{name: p + 1}) == EUNSUPP, name
    assert draw(lib, p, logits=p + 2) == EUNSUPP
    away = ENOTDEV if lib.device_count() > 0 else ENODEV
    assert draw(lib, p, dtype="bf16", logits=p + 2) == away  # bf16 needs no more
    assert draw(lib, p, temperature=None, top_k=None, top_p=None, min_p=None, logprob=None) == away
    assert draw(lib, p, workspace=p + 4, workspace_bytes=1 << 40) == EUNSUPP


def test_sample_workspace(lib, p):
    size = lib.lib.vx_nn_sample_workspace
    assert size(0, 10) == EINVAL and size(1, 0) == EINVAL and size(1, 2 ** 30 + 1) == EINVAL
    for rows, vocab in ((1, 1), (1, 32000), (48, 32000), (8, 131072), (256, 131071), (1, 2 ** 30)):
        n = size(rows, vocab)
        assert n >= 0
        if n:
            assert draw(lib, p, rows=rows, vocab=vocab, workspace=p, workspace_bytes=n - 1) == EINVAL


def test_sample_workspace_stays_within_what_is_said(lib):
    """1024 x (45 KiB + 8.2 KiB per begun 32768 logits), also just past a multiple."""
    size = lib.lib.vx_nn_sample_workspace
    for vocab in (32768, 32769, 33000, 36865, 50000, 65536, 65537, 98305, 131071, 131073, 262144, 262145,
                  2 ** 25 - 1, 2 ** 25, 2 ** 25 + 1):
        bound = 1024 * (45 * 1024 + 8.2 * 1024 * -(-vocab // 32768))
        for rows in (1, 2, 7, 15, 16, 56, 57, 63, 113, 114, 255, 256, 511, 512, 1000, 1023, 1024, 1025):
            assert 0 <= size(rows, vocab) <= bound, (rows, vocab)
    # without the rounding up it takes more
    assert size(1024, 33000) > 1024 * (45 * 1024 + 8.2 * 1024 * 33000 / 32768)
