"""The serving engine with a sliding window, with rules on the choice of tokens and with a cache that changes its size, on CPU (tiny
model, fp32): it must generate exactly the tokens of a dense forward that is written without cache, pages or batches."""
import json
import math
import os
import random
import socket
import subprocess
import sys
import urllib.error
import urllib.request
from dataclasses import replace

import pytest
import torch

from k8s_llm_monitor_amd.models.llama import PRESETS, LlamaModel
from k8s_llm_monitor_amd.ops import ref
from k8s_llm_monitor_amd.serving import Engine, EngineConfig, TokenRules
from k8s_llm_monitor_amd.serving.server import LlmServer

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TINY = PRESETS["tiny"]
WINDOW, SINKS = 37, 5


@pytest.fixture(scope="module", autouse=True)
def two_threads():
    """The products here are small: more threads only add to the machine's load, which other tests look at."""
    n = torch.get_num_threads()
    torch.set_num_threads(min(n, 2))
    yield
    torch.set_num_threads(n)


@pytest.fixture(scope="module")
def model():
    torch.manual_seed(0)
    return LlamaModel(TINY, "cpu", seed=1, dtype=torch.float32)


@pytest.fixture(scope="module")
def windowed():
    torch.manual_seed(0)
    return LlamaModel(replace(TINY, window=WINDOW, sinks=SINKS), "cpu", seed=1, dtype=torch.float32)


def dense_logits(model, seq):
    cfg, T = model.cfg, len(seq)
    h, pos = model.embed[torch.tensor(seq)], torch.arange(T)
    hidden = pos[None] > pos[:, None]
    if cfg.window:
        hidden = hidden | ((pos[None] <= pos[:, None] - cfg.window) & (pos[None] >= cfg.sinks))
    for L in model.layers:
        x = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + cfg.eps)
        qkv = ref.rope(x @ L["wqkv"].t(), model.cos_sin, pos, cfg.n_q, cfg.n_kv).view(T, -1, 128)
        q, k, v = qkv[:, :cfg.n_q], qkv[:, cfg.n_q:cfg.n_q + cfg.n_kv], qkv[:, cfg.n_q + cfg.n_kv:]
        k, v = k.repeat_interleave(cfg.n_q // cfg.n_kv, 1), v.repeat_interleave(cfg.n_q // cfg.n_kv, 1)
        s = (torch.einsum("thd,chd->htc", q, k) / math.sqrt(128)).masked_fill(hidden[None], float("-inf"))
        h = h + torch.einsum("htc,chd->thd", torch.softmax(s, -1), v).reshape(T, -1) @ L["wo"].t()
        x = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + cfg.eps)
        gu = (x @ L["w_gate_up"].t()).view(T, cfg.ffn // 8, 2, 8)
        h = h + (torch.nn.functional.silu(gu[:, :, 0]) * gu[:, :, 1]).reshape(T, cfg.ffn) @ L["w_down"].t()
    x = h[-1] * torch.rsqrt(h[-1].pow(2).mean(-1, keepdim=True) + cfg.eps)
    return x @ model.lm_head.t()


def dense_generate(model, prompt, n, rules=None):
    seq = list(prompt)
    for _ in range(n):
        x = dense_logits(model, seq)
        if rules is not None:
            out = seq[len(prompt):]
            for t in set(seq):
                x[t] = x[t] / rules.repetition if x[t] > 0 else x[t] * rules.repetition
                x[t] = x[t] - rules.frequency * out.count(t) - (rules.presence if t in out else 0.0)
            for t, b in rules.bias.items():
                x[t] = x[t] + b
            if rules.allowed is not None:
                keep = torch.zeros(len(x), dtype=torch.bool)
                keep[list(rules.allowed)] = True
                x = x.masked_fill(~keep, float("-inf"))
        seq.append(int(x.argmax()))
    return seq[len(prompt):]


def engine(model, **kw):
    kw = {"max_num_seqs": 8, "max_model_len": 256, "kv_blocks": 64, "max_num_batched_tokens": 512, **kw}
    return Engine(EngineConfig(model="tiny", device="cpu", use_graphs=False, **kw), model=model)


def drain(eng, after_step=lambda: None):
    for _ in range(3000):
        if eng.idle():
            return
        eng.step()
        after_step()
    raise AssertionError("engine did not drain")


RULES = [TokenRules(repetition=1.7), TokenRules(frequency=0.4, presence=0.3), TokenRules(repetition=0.8, frequency=-0.1, bias={7: 2.5, 400: -1.0}),
         TokenRules(allowed=tuple(range(3, 512, 9))), TokenRules(repetition=3.0, presence=5.0, bias={5: 9.0}, allowed=(0, 5, 31, 32, 511))]


# ------------------------------------------------------------------ window
@pytest.mark.parametrize("budget,mixed", [(512, True), (24, True), (24, False)])
def test_a_window_gives_the_tokens_of_the_dense_forward(windowed, budget, mixed):
    eng = engine(windowed, max_num_batched_tokens=budget, mixed_batches=mixed)
    rng = random.Random(5)
    prompts = [[rng.randrange(512) for _ in range(n)] for n in (1, 16, 36, 37, 38, 90, 120)]
    reqs = [eng.submit(p, 40) for p in prompts]
    drain(eng)
    for p, r in zip(prompts, reqs):
        assert r.error is None and r.out == dense_generate(windowed, p, 40), len(p)
    assert eng.alloc.free == eng.alloc.total


def test_blocks_behind_the_window_are_given_back_and_never_read_again(windowed):
    """Whatever is free, or was never given out, holds NaN: one value of it in a token's attention would spread to the logits."""
    eng = engine(windowed, kv_blocks=40, max_num_batched_tokens=48)
    rng = random.Random(9)
    prompts = [[rng.randrange(512) for _ in range(n)] for n in (100, 5, 70)]
    most = []

    def poison():
        for r in eng.running:
            held = [b for b in r.blocks if b >= 0]
            most.append(len(held))
            assert len(set(held)) == len(held)
            for i, b in enumerate(r.blocks):             # what a token from here on sees is held, nothing behind it
                seen = i * 16 < SINKS or i * 16 + 15 > r.n_tokens - 1 - WINDOW
                assert (b >= 0) == seen, (i, r.n_tokens)
        for b in eng.alloc._free:
            eng.cache.k[:, b] = float("nan")
            eng.cache.v[:, b] = float("nan")

    poison()
    # the slots of a block behind its sequence's last token are read and masked: a block is handed out with NaN in them
    reqs = [eng.submit(p, 100) for p in prompts]
    drain(eng, poison)
    for p, r in zip(prompts, reqs):
        assert r.error is None and r.out == dense_generate(windowed, p, 100)
    # window 37: at most 4 blocks touch it, one holds the sinks, one is for the next token
    assert max(most) <= 6 and eng.alloc.free == 40


def test_a_window_under_preemption(windowed):
    eng = engine(windowed, kv_blocks=16, max_num_seqs=5, max_num_batched_tokens=24, max_model_len=200)
    rng = random.Random(3)
    prompts = [[rng.randrange(512) for _ in range(rng.randint(20, 70))] for _ in range(8)]
    reqs = [eng.submit(p, 60) for p in prompts]

    def whole():
        held = [b for r in eng.running + eng.prefilling for b in r.blocks if b >= 0]
        assert len(held) == len(set(held)) and len(held) + eng.alloc.free == eng.alloc.total

    drain(eng, whole)
    assert eng.metrics.preemptions > 0
    for p, r in zip(prompts, reqs):
        assert r.out == dense_generate(windowed, p, len(r.out)) and len(r.out) == 60


def test_the_engine_configures_the_window():
    eng = Engine(EngineConfig(model="tiny", device="cpu", kv_blocks=32, window=20, sinks=3, use_graphs=False, max_model_len=128))
    assert (eng.model.cfg.window, eng.model.cfg.sinks) == (20, 3) == (eng.describe()["window"], eng.describe()["sinks"])
    assert eng.mcfg.flops_per_token(1000) == eng.mcfg.flops_per_token(23) > PRESETS["tiny"].flops_per_token(22)
    for kw in ({"window": -1}, {"sinks": 2}, {"window": 4, "sinks": -1}):
        with pytest.raises(ValueError):
            Engine(EngineConfig(model="tiny", device="cpu", kv_blocks=8, **kw))
    with pytest.raises(ValueError):
        Engine(EngineConfig(model="tiny", device="cpu", kv_blocks=8, window=21, sinks=3), model=eng.model)


# ------------------------------------------------------------------ rules
@pytest.mark.parametrize("budget,mixed,blocks", [(512, True, 64), (20, True, 64), (20, False, 12)])
def test_rules_give_the_tokens_of_the_formulas(model, budget, mixed, blocks):
    eng = engine(model, max_num_batched_tokens=budget, mixed_batches=mixed, kv_blocks=blocks, max_num_seqs=4, max_model_len=120)
    rng = random.Random(11)
    work = [([rng.randrange(512) for _ in range(rng.randint(1, 50))], rules, rng.randint(1, 25)) for rules in [*RULES, None, *RULES, None]]
    reqs = [eng.submit(p, n, rules) for p, rules, n in work]
    drain(eng)
    for (p, rules, n), r in zip(work, reqs):
        assert r.error is None and r.out == dense_generate(model, p, n, rules), rules
    assert blocks > 12 or eng.metrics.preemptions > 0
    assert sorted(eng._store._free) == list(range(4))                # every set of rules came back


def test_requests_without_rules_make_no_store(model):
    eng = engine(model)
    eng.submit([1, 2, 3], 4)
    drain(eng)
    assert eng._store is None


def test_a_failed_step_gives_the_sets_of_rules_back(model):
    eng = engine(model)
    r = eng.submit([1, 2, 3], 9, RULES[0])
    eng.step()
    eng._fail_all("for the test")
    assert r.error and sorted(eng._store._free) == list(range(8)) and eng.alloc.free == eng.alloc.total
    again = eng.submit([1, 2, 3], 9, RULES[1])                       # the set that was used before starts anew
    drain(eng)
    assert again.out == dense_generate(model, [1, 2, 3], 9, RULES[1])


@pytest.mark.parametrize("bad", [dict(repetition=0.0), dict(repetition=-2.0), dict(repetition=float("nan")), dict(frequency=float("inf")),
                                 dict(bias={512: 1.0}), dict(bias={-1: 1.0}), dict(bias={3: float("nan")}), dict(allowed=()),
                                 dict(allowed=(3, 512)), dict(bias={i: 1.0 for i in range(257)})])
def test_rules_that_do_not_fit_are_refused(model, bad):
    with pytest.raises(ValueError):
        engine(model).submit([1], 2, TokenRules(**bad))


def test_rules_over_http(model):
    def post(srv, **body):
        req = urllib.request.Request(srv.url + "/v1/completions", data=json.dumps({"prompt": [1, 2, 3], "max_tokens": 6, **body}).encode())
        return json.load(urllib.request.urlopen(req, timeout=60))["choices"][0]["token_ids"]

    eng = engine(model).start()
    try:
        with LlmServer(eng) as srv:
            assert post(srv) == dense_generate(model, [1, 2, 3], 6)
            assert post(srv, repetition_penalty=1.7) == dense_generate(model, [1, 2, 3], 6, RULES[0])
            assert post(srv, frequency_penalty=0.4, presence_penalty=0.3) == dense_generate(model, [1, 2, 3], 6, RULES[1])
            assert post(srv, allowed_token_ids=[77]) == [77] * 6
            assert post(srv, logit_bias={"9": 1e6}, frequency_penalty=0) == [9] * 6
            for bad in ({"repetition_penalty": 0}, {"presence_penalty": "x"}, {"logit_bias": {"x": 1}}, {"logit_bias": [1]}, {"logit_bias": {"1": True}},
                        {"allowed_token_ids": []}, {"allowed_token_ids": [512]}, {"allowed_token_ids": 3}, {"frequency_penalty": 10 ** 400}):
                with pytest.raises(urllib.error.HTTPError) as e:
                    post(srv, **bad)
                assert e.value.code == 400, bad
    finally:
        eng.stop()


# ------------------------------------------------------------------ another number of blocks
@pytest.mark.parametrize("which", ["model", "windowed"])
def test_the_cache_changes_its_size_between_steps(which, request):
    m = request.getfixturevalue(which)
    eng = engine(m, kv_blocks=64, max_num_batched_tokens=40)
    rng = random.Random(2)
    prompts = [[rng.randrange(512) for _ in range(n)] for n in (60, 9, 33, 80)]
    reqs = [eng.submit(p, 40, RULES[0]) for p in prompts]
    sizes, steps = [33, 200, 35, 64], [0]

    def resize():
        steps[0] += 1
        if steps[0] % 5 == 2 and sizes:
            eng.resize_cache(sizes.pop(0))
        held = [b for r in eng.running + eng.prefilling for b in r.blocks if b >= 0]
        assert len(held) == len(set(held)) and len(held) + eng.alloc.free == eng.alloc.total == eng.cache.num_blocks
        for b in eng.alloc._free:
            eng.cache.k[:, b] = 1e4 if which == "model" else float("nan")      # stale: masked wherever it is read

    drain(eng, resize)
    assert not sizes
    for p, r in zip(prompts, reqs):
        assert r.error is None and r.out == dense_generate(m, p, 40, RULES[0])


def test_the_size_changes_while_the_engine_thread_runs(model):
    eng = engine(model, kv_blocks=64).start()
    try:
        reqs = [eng.submit(list(range(1, 30)), 60) for _ in range(4)]
        for n in (40, 64, 50):
            eng.resize_cache(n)                           # between two steps of the other thread, however busy it is
        for r in reqs:
            assert r.done.wait(60) and r.error is None and r.out == reqs[0].out
        assert eng.alloc.total == 50 and reqs[0].out == dense_generate(model, list(range(1, 30)), 60)
    finally:
        eng.stop()


def test_a_cache_too_small_for_what_is_in_flight_is_refused(model):
    eng = engine(model)
    r = eng.submit(list(range(40)), 60)                   # 100 tokens: 7 blocks
    eng.step()
    before = (eng.cache, eng.alloc, list(r.blocks))
    for n in (0, 2, 6):
        with pytest.raises(ValueError):
            eng.resize_cache(n)
    assert (eng.cache, eng.alloc, r.blocks) == before
    eng.resize_cache(7)
    drain(eng)
    assert r.out == dense_generate(model, list(range(40)), 60)
    eng.resize_cache(1)                                   # nothing is in flight
    assert eng.submit(list(range(40)), 4).error           # and now too long a prompt


# ------------------------------------------------------------------ two ranks
@pytest.mark.timeout(300)
def test_two_ranks_choose_as_one():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    procs = [subprocess.Popen([sys.executable, "-u", os.path.join(ROOT, "tests", "tp_rules_worker.py")], cwd=ROOT,
                              env=dict(os.environ, RANK=str(r), WORLD_SIZE="2", MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port),
                                       PYTHONPATH=ROOT, OMP_NUM_THREADS="2"), stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
             for r in range(2)]
    try:
        outs = [p.communicate(timeout=240) for p in procs]
    finally:
        for p in procs:
            if p.poll() is None:
                p.kill()
    assert all(p.returncode == 0 for p in procs), outs
    res = [json.loads([l for l in so.splitlines() if l.startswith("RESULT ")][-1][7:]) for so, _ in outs]
    assert res[0]["match"] and res[0]["lowest_rank_of_a_tie"] and res[1]["steps"] == res[0]["steps"]
