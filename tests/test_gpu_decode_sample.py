"""vx_llama_i8_sample on the GPU: greedy settings give vx_llama_i8_generate's
tokens, every drawn token is the one whose share of the decoder's own logits the
uniform number falls in, and graphs and stream launches agree."""

import numpy as np
import pytest

from tests import batch_reference as ref
from tests.conftest import announce
from vx_amd.decode import LlamaI8
from vx_amd.llama import CONFIG_TINY, LlamaConfig, make_model, make_prompt

pytestmark = pytest.mark.gpu

# head size 64 and a vocabulary that several workgroups sample
WIDE = LlamaConfig(dim=64, hidden_dim=128, n_layers=1, n_heads=1, n_kv_heads=1, vocab_size=40000, seq_len=64)


def scaled(cfg, seed):
    """A tiny model whose logits are spread as a trained one's."""
    w = make_model(cfg, seed=seed)
    w["rms_final"] = w["rms_final"] * np.float32(12.0)
    return w


@pytest.fixture(scope="module", params=[CONFIG_TINY, WIDE], ids=["tiny", "wide"])
def model(request, hiplib):
    m = LlamaI8(hiplib, request.param, scaled(request.param, 3))
    yield m
    m.close()


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=12), dict(top_p=0.8, temperature=1.2), dict(min_p=0.3),
            dict(temperature=0.9, top_k=40, top_p=0.9, min_p=0.02)]


@pytest.mark.parametrize("n_prompt", [1, 2, 5])
def test_greedy_settings(model, n_prompt):
    announce(f"sample decode greedy {n_prompt}")
    prompt = make_prompt(model.cfg, n=n_prompt, seed=5)
    want, _ = model.generate(prompt, 9)
    for kw in (dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0)):
        got, logprob = model.sample(prompt, np.full(9, 0.9, np.float32), **kw)
        assert np.array_equal(got, want), kw
        assert np.all(logprob == 0)


@pytest.mark.parametrize("n_prompt", [1, 2, 5])
@pytest.mark.parametrize("how", SETTINGS)
def test_tokens_are_the_logits_shares(model, how, n_prompt):
    announce(f"sample decode {how} {n_prompt}")
    steps = 19
    prompt = make_prompt(model.cfg, n=n_prompt, seed=7)
    u = np.random.default_rng(n_prompt).random(steps, dtype=np.float32)
    tokens, logprob = model.sample(prompt, u, **how)
    eager, logprob_eager = model.sample(prompt, u, graph=False, **how)
    assert np.array_equal(tokens, eager) and np.array_equal(logprob, logprob_eager)
    again, _ = model.sample(prompt, u, **how)
    assert np.array_equal(tokens, again)
    logits = model.logits(np.concatenate([prompt, tokens[:-1]]))[n_prompt - 1:]

    def arrays(t=1.0, k=0, p=1.0, m=0.0):
        return (np.full(steps, t), np.full(steps, k), np.full(steps, p), np.full(steps, m))

    settings = arrays(how.get("temperature", 1.0), how.get("top_k", 0), how.get("top_p", 1.0), how.get("min_p", 0.0))
    # the logits of texts fed together differ by f32 rounding: a token next to a
    # border may fall on its other side
    want = [ref.sample(logits, *settings, np.clip(u + d, 0, 1 - 2.0 ** -24)) for d in (-2e-4, 0.0, 2e-4)]
    ok = np.any([w[0] == tokens for w in want], axis=0)
    assert ok.all(), (np.flatnonzero(~ok), tokens, want[1][0])
    same = want[1][0] == tokens
    assert np.all(np.abs(logprob - want[1][1])[same] < 1e-3)
    assert same.sum() >= steps - 2


def test_another_call_in_between(model):
    """Greedy and sampled calls in turn, other settings and lengths: each as if
    alone."""
    announce("sample decode in turn")
    prompt = make_prompt(model.cfg, n=4, seed=9)
    u = np.random.default_rng(1).random(17, dtype=np.float32)
    greedy, margin = model.generate(prompt, 12)
    first = model.sample(prompt, u[:12], temperature=0.8)
    assert np.array_equal(model.generate(prompt, 12)[0], greedy)
    model.sample(prompt[:2], u, top_k=3)
    second = model.sample(prompt, u[:12], temperature=0.8)
    assert np.array_equal(first[0], second[0]) and np.array_equal(first[1], second[1])
    longer = model.sample(prompt, u, temperature=0.8)
    assert np.array_equal(longer[0][:12], first[0])
    got, m = model.generate(prompt, 12)
    assert np.array_equal(got, greedy) and np.array_equal(m, margin)


def test_refusals(model, hiplib):
    announce("sample decode refusals")
    prompt = make_prompt(model.cfg, n=3, seed=9)
    for n in (0, model.cfg.seq_len - 1):
        with pytest.raises(RuntimeError):
            model.sample(prompt, np.zeros(n, np.float32))
    toks = np.zeros(4, np.int32)
    fn = hiplib.lib.vx_llama_i8_sample
    how = np.array([1, 0, 1, 0], np.float32)
    u = np.zeros(4, np.float32)
    assert fn(None, prompt.ctypes.data, 3, 4, how.ctypes.data, u.ctypes.data, toks.ctypes.data, None, 0) == -1
    assert fn(model.handle, prompt.ctypes.data, 3, 4, None, u.ctypes.data, toks.ctypes.data, None, 0) == -1
    assert fn(model.handle, prompt.ctypes.data, 3, 4, how.ctypes.data, None, toks.ctypes.data, None, 0) == -1
    assert fn(model.handle, prompt.ctypes.data, 3, 4, how.ctypes.data, u.ctypes.data, toks.ctypes.data, None, 0) == 0


@pytest.mark.parametrize("vocab", [256, 40000])
@pytest.mark.parametrize("n_prompt", [1, 2, 5])
def test_logits_that_are_all_nan(hiplib, vocab, n_prompt):
    """The prompt's last token alone overflows behind the last layer's cache
    writes: all its logits are NaN, its successor is -1, and generation goes on
    as after token 0."""
    announce(f"sample decode all NaN {vocab} {n_prompt}")
    cfg = LlamaConfig(dim=64, hidden_dim=128, n_layers=1, n_heads=1, n_kv_heads=1, vocab_size=vocab, seq_len=64)
    w, bad = scaled(cfg, 11), 77
    # x[0] is 0 but for that token, whose feed-forward squares it, and x[1] takes
    # the square times 1e40
    w["tok_q"][:, 0] = 0
    w["tok_q"][bad, 0] = 127
    w["wo_q"][0, 0] = 0
    w["w2_q"][0, 0] = 0
    for name in ("w1", "w3"):
        w[f"{name}_q"][0, 0] = 0
        w[f"{name}_q"][0, 0, 0] = 127
        w[f"{name}_s"][0, 0] = 1.0
    w["w2_q"][0, 1] = 0
    w["w2_q"][0, 1, 0] = 127
    w["w2_s"][0, 1] = 3e38
    w["w2_q"][0, 2:, 0] = 0
    steps = 12
    prompt = np.concatenate([make_prompt(cfg, n=n_prompt - 1, seed=2) % 70, [bad]]).astype(np.int32)
    u = np.random.default_rng(n_prompt).random(steps, dtype=np.float32) * np.float32(0.9)
    model = LlamaI8(hiplib, cfg, w)
    try:
        for how in (dict(temperature=0.8), dict(top_k=9), dict(top_p=0.9, min_p=0.01), dict(temperature=0.0)):
            tokens, logprob = model.sample(prompt, u, **how)
            eager = model.sample(prompt, u, graph=False, **how)
            assert np.array_equal(tokens, eager[0]) and np.array_equal(logprob, eager[1]), how
            assert tokens[0] == -1 and logprob[0] == -np.inf, how
            text = np.concatenate([prompt, [0], tokens[1:-1]])
            logits = model.logits(text)
            where = np.isnan(logits)
            assert where[n_prompt - 1].all() and not where[text != bad].any()
            rows = [a if a is None else np.full(steps - 1, a) for a in
                    (how.get("temperature"), how.get("top_k"), how.get("top_p"), how.get("min_p"))]
            ok = np.zeros(steps - 1, bool)
            for d in (-2e-4, 0.0, 2e-4):  # as above
                want = ref.sample(logits[n_prompt:], *rows, np.clip(u[1:] + d, 0, 1))[0]
                # a token after an overflowing one is again -1
                ok |= np.where(text[n_prompt:] == bad, -1, want) == tokens[1:]
            assert ok.all(), (how, tokens)
    finally:
        model.close()
