"""Sessions sample among what top-k, top-p and min-p leave (l2b_session_sample, sample_next, sample)."""
import ctypes as C
import io

import numpy as np
import pytest

from test_gpu_sampling import reference

pytestmark = pytest.mark.gpu


class Tokenizer:
    bos_token_id, eos_token_id = 1, 2

    def __init__(self, n):
        self.id_to_token = [f"<{i}>" for i in range(n)]


@pytest.fixture(scope="module")
def model(pkg, synth):
    cfg = pkg.ModelConfig(64, 96, 2, 4, 4, 700, 48, 10000.0, False)
    m = pkg.LanguageModel(cfg, Tokenizer(700), synth.model_weights(cfg, dict.fromkeys(("wq", "wk", "wv", "wo", "w1", "w2", "w3", "token_embd", "output"), 0), seed=3))
    yield m
    m.close()


@pytest.mark.parametrize("cuts", [dict(), dict(top_k=5), dict(top_p=0.4), dict(min_p=0.6), dict(top_k=50, top_p=0.7, min_p=0.1)])
def test_tokens_of_a_session(pkg, model, cuts):
    s = pkg.RunState(model)
    rng = np.random.default_rng(1)
    short = dict(top_k="k", top_p="p", min_p="m")
    for pos in range(6):
        pkg.transformer_(int(rng.integers(700)), pos, model.config, s)
        for t in (0.3, 1.7):
            u = float(rng.random())
            want, _ = reference(s.logits.astype(np.float64), t=float(np.float32(t)), u=u, **{short[n]: float(np.float32(v)) if n != "top_k" else v for n, v in cuts.items()})
            assert pkg.sample_next(s, t, uniform=u, **cuts) == want
        assert pkg.sample_next(s, 0.0, **cuts) == int(s.logits.argmax())
        before = s.logits.copy()
        L = pkg.lib()
        assert L.l2b_session_logits(s.session, s.logits.ctypes.data) == 0 and np.array_equal(before, s.logits)  # the logits are as they were


def test_sample_with_one_choice_is_greedy(pkg, model, monkeypatch):
    """The whole loop: top_k = 1 prints what temperature 0 prints; without cuts nothing changes."""
    from llama2_jl_b200 import tokenizer
    monkeypatch.setattr(tokenizer, "encode", lambda text, tok: [5, 9, 33])
    import random

    def text(**k):
        out = io.StringIO()
        pkg.sample(model, "x", stop_on_special_token=False, max_seq_len=20, out=out, rng=random.Random(4), **k)
        return out.getvalue().split("\n")[0]
    greedy = text(temperature=0.0)
    assert text(temperature=0.8, top_k=1) == greedy and text(temperature=0.8, top_p=1e-9) == greedy and text(temperature=0.8, min_p=1.0) == greedy
    assert text(temperature=0.0, top_k=7) == greedy
    assert text(temperature=1.5, top_k=40, top_p=0.9) == text(temperature=1.5, top_k=40, top_p=0.9)


def test_refusals(pkg, model):
    s = pkg.RunState(model)
    lib, n = pkg.lib(), C.c_int32()
    assert lib.l2b_session_sample(None, 1.0, 0, 1.0, 0.0, 0.5, C.byref(n)) == 1
    assert lib.l2b_session_sample(s.session, 1.0, 0, 1.0, 0.0, 0.5, None) == 1
    assert lib.l2b_session_sample(s.session, -1.0, 0, 1.0, 0.0, 0.5, C.byref(n)) == 1
    assert lib.l2b_session_sample(s.session, float("nan"), 0, 1.0, 0.0, 0.5, C.byref(n)) == 1
    for u in (-0.1, 1.0, float("nan")):
        assert lib.l2b_session_sample(s.session, 1.0, 0, 1.0, 0.0, u, C.byref(n)) == 1


def test_no_token_without_logits(pkg, synth):
    """A session that holds no logits of its last position refuses to sample: new, reset, after a call that failed, after a prompt that was cut inside."""
    lib, n = pkg.lib(), C.c_int32()
    cfg = pkg.ModelConfig(64, 96, 2, 4, 4, 700, 48, 10000.0, False)
    m = pkg.LanguageModel(cfg, Tokenizer(700), synth.model_weights(cfg, dict.fromkeys(("wq", "wk", "wv", "wo", "w1", "w2", "w3", "token_embd", "output"), 0), seed=3))
    s = pkg.RunState(m)

    def status():
        return lib.l2b_session_sample(s.session, 0.0, 0, 1.0, 0.0, 0.5, C.byref(n))
    assert status() == 7 and b"logits" in lib.l2b_last_error_string()
    pkg.transformer_(5, 0, cfg, s)
    assert status() == 0 and n.value == int(s.logits.argmax())
    s.reset()
    assert status() == 7
    first = pkg.prefill(s, [5, 9, 33])
    assert status() == 0 and n.value == first
    assert lib.l2b_forward(s.session, 700, 3, None) == 1  # (refused before anything has changed)
    assert status() == 0 and n.value == first
    got, _ = pkg.generate(m, np.array([5, 9, 33], np.int32), 6)
    assert status() == 0 and n.value == got[5]
    pkg.generate(m, np.array([5, 9, 33, 7, 8], np.int32), 3)
    assert status() == 7
    nxt = C.c_int32()
    assert lib.l2b_decode_next(s.session, 8, 3, 0.7, 0.3, C.byref(nxt)) == 0 and status() == 0
    m.close()
    # one rank of two that has not been connected to the other: nothing can have been computed
    from tp_worker import tiny_config
    cfg = tiny_config(pkg)
    m = pkg.LanguageModel(cfg, None, synth.model_weights(cfg, synth.ALL(synth.Q4), seed=3), tp_size=2, tp_rank=0)
    s = pkg.RunState(m)
    assert status() == 7 and lib.l2b_forward(s.session, 1, 0, None) == 7 and status() == 7
    m.close()


@pytest.mark.parametrize("compute", ["float32", "bfloat16"])
def test_layer_stack_sessions(pkg, compute):
    """The same on a layer-stack model, token by token and after prompts; a portion of several tokens keeps no logits in the session."""
    import savozen_cases as sc
    from stack_common import build
    cfg = sc.CASES["all"]
    model = build(pkg, cfg, sc.weights(cfg, 5), 40, compute)
    s, t = pkg.RunState(model), sc.tokens(cfg, 12, 6)
    lib, n, rng = pkg.lib(), C.c_int32(), np.random.default_rng(2)

    def status():
        return lib.l2b_session_sample(s.session, 1.0, 5, 1.0, 0.0, 0.5, C.byref(n))

    def tokens_agree():
        L_logits = np.zeros_like(s.logits)
        assert lib.l2b_session_logits(s.session, L_logits.ctypes.data) == 0
        for cuts, short in ((dict(top_k=5), dict(k=5)), (dict(top_p=0.5), dict(p=0.5)), (dict(), dict())):
            u = float(rng.random())
            assert pkg.sample_next(s, 0.75, uniform=u, **cuts) == reference(L_logits.astype(np.float64), t=0.75, u=u, **short)[0]
    assert status() == 7
    for pos in range(3):
        pkg.transformer_(int(t[pos]), pos, model.config, s)
        tokens_agree()
    assert pkg.prefill(s, t[3:8], 3) >= 0
    tokens_agree()
    pkg.extend(s, t[8:11], 8, [2])
    assert status() == 7
    pkg.extend(s, t[11:12], 11, [0])
    tokens_agree()
    model.close()
