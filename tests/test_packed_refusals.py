"""What the ops of a packed batch in 8 bits refuse, and the workspaces they
name: checked on the host before a GPU is looked for, so without one too."""

import ctypes

import pytest

from vx_amd.runtime import (LIB_PATH, DispatchLibrary, flash_attention_packed, gemm_i8, quantize_i8, rms_norm,
                            token_logprobs)

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


def away(lib):
    return ENOTDEV if lib.device_count() > 0 else ENODEV


def norm(lib, p, **kw):
    a = dict(dtype="bf16", x=p, residual=p, weight=p, sum=p, y=p, q=p, q_scale=p, rows=3, dim=64, eps=1e-5)
    a.update(kw)
    return rms_norm(lib, **a)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kw,code", [
    (dict(x=None), EINVAL), (dict(y=None, q=None, q_scale=None), EINVAL), (dict(q=None), EINVAL),
    (dict(q_scale=None), EINVAL), (dict(rows=0), EINVAL), (dict(rows=-1), EINVAL), (dict(dim=0), EINVAL),
    (dict(stride=63), EINVAL), (dict(stride=2 ** 41), EINVAL), (dict(eps=-1e-9), EINVAL),
    (dict(eps=float("nan")), EINVAL), (dict(eps=float("inf")), EINVAL), (dict(rows=2 ** 21 + 1), EUNSUPP),
    (dict(dim=32769), EUNSUPP), (dict(dim=2 ** 32 + 64, stride=2 ** 33), EUNSUPP), (dict(dim=2 ** 41), EINVAL)])
def test_rms_norm_refuses(lib, p, dtype, kw, code):
    assert norm(lib, p, **{"dtype": dtype, **kw}) == code


def test_rms_norm_refuses_alignment(lib, p):
    for name in ("x", "residual", "sum", "y", "weight", "q_scale"):
        assert norm(lib, p, **{name: p + 1}) == EUNSUPP, name
    for name in ("x", "residual", "sum", "weight", "q_scale"):
        assert norm(lib, p, dtype="f32", **{name: p + 2}) == EUNSUPP, name
    # good arguments, memory that is not a GPU's (or no GPU)
    assert norm(lib, p) == away(lib)
    assert norm(lib, p, q=p + 1, x=p + 2) == away(lib)
    assert norm(lib, p, residual=None, weight=None, sum=None, y=None) == away(lib)
    assert norm(lib, p, residual=None, weight=None, sum=None, q=None, q_scale=None) == away(lib)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kw,code", [
    (dict(x=None), EINVAL), (dict(q=None), EINVAL), (dict(q_scale=None), EINVAL),
    (dict(q=None, q_scale=None), EINVAL), (dict(rows=0), EINVAL), (dict(dim=-5), EINVAL), (dict(stride=63), EINVAL),
    (dict(rows=2 ** 22), EUNSUPP), (dict(dim=40000), EUNSUPP)])
def test_quantize_refuses(lib, p, dtype, kw, code):
    a = dict(dtype=dtype, x=p, q=p, q_scale=p, rows=3, dim=64)
    a.update(kw)
    assert quantize_i8(lib, **a) == code


def gemm(lib, p, **kw):
    a = dict(dtype="bf16", x=p, x_scale=p, w=p, w_scale=p, y=p, tokens=5, rows=7, cols=64)
    a.update(kw)
    return gemm_i8(lib, **a)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kw,code", [
    (dict(x=None), EINVAL), (dict(x_scale=None), EINVAL), (dict(w=None), EINVAL), (dict(w_scale=None), EINVAL),
    (dict(y=None), EINVAL), (dict(tokens=0), EINVAL), (dict(rows=0), EINVAL), (dict(cols=0), EINVAL),
    (dict(cols=-16), EINVAL), (dict(cols=72), EUNSUPP), (dict(cols=131072), EUNSUPP),
    (dict(cols=2 ** 32 + 16), EUNSUPP), (dict(stride=6), EINVAL), (dict(stride=2 ** 50), EINVAL),
    (dict(tokens=2 ** 24 + 1), EUNSUPP), (dict(rows=2 ** 24 + 1), EUNSUPP), (dict(tokens=2 ** 20, rows=2 ** 20), EUNSUPP),
    (dict(tokens=2 ** 41), EINVAL)])
def test_gemm_refuses(lib, p, dtype, kw, code):
    assert gemm(lib, p, **{"dtype": dtype, **kw}) == code


def test_gemm_refuses_alignment(lib, p):
    for name in ("x", "w"):
        assert gemm(lib, p, **{name: p + 8}) == EUNSUPP, name
    assert gemm(lib, p, x_scale=p + 2) == EUNSUPP and gemm(lib, p, w_scale=p + 1) == EUNSUPP
    assert gemm(lib, p, y=p + 1) == EUNSUPP and gemm(lib, p, dtype="f32", y=p + 2) == EUNSUPP
    assert gemm(lib, p, workspace=p + 4, workspace_bytes=2 ** 40) == EUNSUPP
    assert gemm(lib, p, y=p + 2) == away(lib)
    assert gemm(lib, p, cols=131056) == away(lib)


def test_gemm_workspace(lib, p):
    size = lib.lib.vx_nn_gemm_i8_workspace
    assert size(0, 4, 16) == EINVAL and size(4, 4, 17) == EUNSUPP
    for ext in ((1, 32000, 768), (48, 11008, 4096), (65, 64, 11008), (200, 500, 4096), (777, 6144, 4096),
                (4096, 11008, 4096), (2 ** 20, 64, 64), (100, 100, 131056)):
        n = size(*ext)
        assert 0 <= n <= 128 << 20
        if n:
            t, r, c = ext
            assert gemm(lib, p, tokens=t, rows=r, cols=c, workspace=p, workspace_bytes=n - 1) == EINVAL


def packed(lib, p, **kw):
    a = dict(q=p, k=p, v=p, offsets=p, o=p, lse=p, total=10, sequences=2, heads=4, kv_heads=2, head_dim=64,
             scale=0.125, causal=True)
    a.update(kw)
    return flash_attention_packed(lib, **a)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), EINVAL), (dict(k=None), EINVAL), (dict(v=None), EINVAL), (dict(offsets=None), EINVAL),
    (dict(o=None), EINVAL), (dict(total=0), EINVAL), (dict(sequences=0), EINVAL), (dict(heads=0), EINVAL),
    (dict(kv_heads=0), EINVAL), (dict(heads=3), EINVAL), (dict(head_dim=96), EUNSUPP), (dict(head_dim=256), EUNSUPP),
    (dict(scale=float("nan")), EINVAL), (dict(scale=3e38), EINVAL), (dict(q_strides=(63, 640)), EINVAL),
    (dict(kv_strides=(64, 0)), EINVAL), (dict(o_strides=(-64, 640)), EINVAL), (dict(o_strides=(68, 680)), EUNSUPP),
    (dict(kv_strides=(2 ** 22 + 8, 64)), EUNSUPP), (dict(q_strides=(2 ** 41, 64)), EINVAL),
    (dict(total=2 ** 29), EUNSUPP), (dict(sequences=65537), EUNSUPP), (dict(total=2 ** 30, heads=2 ** 32, kv_heads=2 ** 32), EUNSUPP),
    (dict(total=1, heads=2 ** 24, kv_heads=2 ** 24), EUNSUPP)])
def test_packed_attention_refuses(lib, p, kw, code):
    assert packed(lib, p, **kw) == code


def test_packed_attention_refuses_alignment(lib, p):
    for name in ("q", "k", "v", "o"):
        assert packed(lib, p, **{name: p + 8}) == EUNSUPP, name
    assert packed(lib, p, offsets=p + 1) == EUNSUPP and packed(lib, p, lse=p + 2) == EUNSUPP
    assert packed(lib, p) == away(lib)
    assert packed(lib, p, lse=None, scale=0.0, causal=False, q_strides=(512, 64), kv_strides=(2 ** 22, 64)) == away(lib)


def logprobs(lib, p, **kw):
    a = dict(dtype="f32", logits=p, given=p, logprob=p, entropy=p, top_tokens=p, top_logprob=p, rows=3, vocab=100,
             n_given=2, n_top=5)
    a.update(kw)
    return token_logprobs(lib, **a)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kw,code", [
    (dict(logits=None), EINVAL), (dict(given=None), EINVAL), (dict(logprob=None), EINVAL),
    (dict(top_tokens=None), EINVAL), (dict(n_given=0, n_top=0, entropy=None), EINVAL), (dict(n_given=-1), EINVAL),
    (dict(n_top=-1), EINVAL), (dict(n_top=65), EINVAL), (dict(n_given=2 ** 20 + 1), EINVAL), (dict(rows=0), EINVAL),
    (dict(rows=2 ** 21 + 1), EINVAL), (dict(vocab=0), EINVAL), (dict(vocab=2 ** 30 + 1), EINVAL),
    (dict(stride=99), EINVAL), (dict(stride=2 ** 50), EINVAL)])
def test_logprobs_refuses(lib, p, dtype, kw, code):
    assert logprobs(lib, p, **{"dtype": dtype, **kw}) == code


def test_logprobs_refuses_alignment(lib, p):
    for name in ("logits", "given", "logprob", "entropy", "top_tokens", "top_logprob"):
        assert logprobs(lib, p, **{name: p + 1}) == EUNSUPP, name
    assert logprobs(lib, p, logits=p + 2) == EUNSUPP
    assert logprobs(lib, p, workspace=p + 4, workspace_bytes=2 ** 40) == EUNSUPP
    assert logprobs(lib, p, dtype="bf16", logits=p + 2) == away(lib)  # bf16 needs no more
    assert logprobs(lib, p, entropy=None, top_logprob=None) == away(lib)
    assert logprobs(lib, p, n_given=0, given=None, logprob=None) == away(lib)
    assert logprobs(lib, p, n_top=0, top_tokens=None, top_logprob=None) == away(lib)


def test_logprobs_workspace(lib, p):
    size = lib.lib.vx_nn_token_logprobs_workspace
    assert size(0, 10, 1) == EINVAL and size(1, 0, 1) == EINVAL and size(1, 10, 65) == EINVAL
    for rows, vocab in ((1, 1), (1, 32000), (3, 131072), (48, 32000), (100, 262144), (512, 131071), (1, 2 ** 30)):
        n = size(rows, vocab, 20)
        assert 0 <= n <= 256 * 128 * 1024
        if n:
            assert logprobs(lib, p, rows=rows, vocab=vocab, n_top=20, workspace=p, workspace_bytes=n - 1) == EINVAL
