"""Rules on tokens that are no good, or that come to grief inside a step: the requests beside them go on, and no set of rules is lost."""
import random
from fractions import Fraction

import numpy as np
import pytest
import torch

from k8s_llm_monitor_amd.models.llama import PRESETS, LlamaModel
from k8s_llm_monitor_amd.serving import Engine, EngineConfig, TokenRules


@pytest.fixture(scope="module")
def model():
    return LlamaModel(PRESETS["tiny"], "cpu", seed=1, dtype=torch.float32)


def engine(model, **kw):
    kw = {"max_num_seqs": 2, "max_model_len": 128, "kv_blocks": 32, "max_num_batched_tokens": 64, **kw}
    return Engine(EngineConfig(model="tiny", device="cpu", use_graphs=False, **kw), model=model)


def drain(eng):
    for _ in range(500):
        if eng.idle():
            return
        eng.step()
    raise AssertionError("engine did not drain")


PROMPT = list(range(1, 12))


@pytest.mark.parametrize("bad", [dict(allowed=(1.5,)), dict(allowed=(True,)), dict(allowed=(2.0,)), dict(allowed=("3",)), dict(allowed=((3,),)), dict(allowed=5),
                                 dict(allowed=(None,)), dict(bias={1.5: 1.0}), dict(bias={True: 1.0}), dict(bias={"3": 1.0}), dict(bias=[3]), dict(bias=None),
                                 dict(bias={3: "1"}), dict(bias={3: None}), dict(bias={3: True}), dict(bias={3: 10 ** 400}), dict(repetition="1"),
                                 dict(repetition=None), dict(repetition=True), dict(repetition=10 ** 400), dict(presence=1j), dict(frequency=[1.0])])
def test_submit_refuses_what_is_no_number_and_no_token(model, bad):
    eng = engine(model)
    beside = eng.submit(PROMPT, 8, TokenRules(repetition=1.5))
    eng.step()
    with pytest.raises(ValueError):
        eng.submit(PROMPT, 8, TokenRules(**bad))
    drain(eng)
    assert beside.error is None and len(beside.out) == 8 and sorted(eng._store._free) == [0, 1]


def test_numbers_of_other_kinds_are_numbers(model):
    eng = engine(model, max_num_seqs=4)
    plain = TokenRules(repetition=1.5, bias={7: 2.0, 9: -1.0}, allowed=(3, 7, 9, 400))
    rng = random.Random(0)
    for allowed in ([3, 7, 9, 400], np.array([3, 7, 9, 400]), {3, 7, 9, 400}, tuple(np.int32(t) for t in (3, 7, 9, 400)), range(3, 401)):
        prompt = [rng.randrange(512) for _ in range(9)]
        want = TokenRules(plain.repetition, bias=plain.bias, allowed=tuple(range(3, 401))) if isinstance(allowed, range) else plain
        a = eng.submit(prompt, 6, want)
        b = eng.submit(prompt, 6, TokenRules(np.float32(1.5), bias={np.int64(7): Fraction(2), 9: np.float64(-1)}, allowed=allowed))
        drain(eng)
        assert a.out == b.out and len(a.out) == 6 and b.error is None


def test_what_was_submitted_is_what_holds(model):
    """A caller that changes its dict afterwards changes nothing: not the tokens, and not a step that others are in."""
    eng = engine(model)
    mine = TokenRules(bias={7: 2.0})
    a, beside = eng.submit(PROMPT, 6, mine), eng.submit(PROMPT, 6)
    mine.bias.update({9999: 1.0, 9: 1e6, **{i: 0.0 for i in range(300)}})
    drain(eng)
    b = eng.submit(PROMPT, 6, TokenRules(bias={7: 2.0}))
    drain(eng)
    assert a.error is None and beside.error is None and a.out == b.out and len(beside.out) == 6


@pytest.mark.parametrize("bias", [[], 0, False, "", [1], 1.5])
def test_a_request_whose_biases_are_no_map_is_refused(bias):
    with pytest.raises(ValueError):
        TokenRules.from_request({"logit_bias": bias}, 512)


def test_a_request_without_rules_has_none():
    assert TokenRules.from_request({"prompt": [1], "logit_bias": None, "allowed_token_ids": None}, 512) is None
    assert TokenRules.from_request({"logit_bias": {}}, 512) == TokenRules()


def test_a_set_of_rules_comes_back_from_a_step_that_failed_to_fill_it(model, monkeypatch):
    eng = engine(model)
    one = eng.submit(PROMPT, 3, TokenRules(repetition=1.5))
    drain(eng)
    store, rules = eng._store, TokenRules(repetition=1.5, allowed=(1, 2, 3))
    for what in ("history", "bias_ids", "bias_values", "penalties", "prompt_lens", "mask", "mask_rows"):
        tensor = getattr(store, what)
        if what != "history":                            # (`follow` writes it, after the set has been taken)
            monkeypatch.setattr(store, what, None)
            with pytest.raises((TypeError, AttributeError)):
                store.take(rules, 3)
            assert sorted(store._free) == [0, 1], what
        monkeypatch.setattr(store, what, None)
        r = eng.submit(PROMPT, 3, rules)
        with pytest.raises((TypeError, AttributeError)):
            eng.step()
        eng._fail_all("for the test")
        assert r.error and sorted(store._free) == [0, 1], what
        monkeypatch.setattr(store, what, tensor)
    again = eng.submit(PROMPT, 3, TokenRules(repetition=1.5))
    drain(eng)
    assert again.error is None and again.out == one.out


def test_an_engine_whose_first_step_with_rules_failed_serves_the_next(model, monkeypatch):
    eng = engine(model)
    full = torch.full

    def no_memory(*a, **kw):
        raise RuntimeError("out of memory")

    eng.submit(PROMPT, 3, TokenRules(repetition=1.5))
    monkeypatch.setattr(torch, "full", no_memory)
    with pytest.raises(RuntimeError):
        eng.step()
    monkeypatch.setattr(torch, "full", full)
    eng._fail_all("for the test")
    r = eng.submit(PROMPT, 3, TokenRules(repetition=1.5))
    drain(eng)
    assert r.error is None and len(r.out) == 3
