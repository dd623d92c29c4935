"""The Llama decoder and the serving engine on a GPU with a sliding window, with rules on the choice of tokens and with a cache
that changes its size: against the fp32 CPU model, and graph replay against eager launches."""
from dataclasses import replace

import pytest
import torch

pytestmark = pytest.mark.gpu

from k8s_llm_monitor_amd.models.llama import PRESETS, DecodeMeta, LlamaModel, PrefillMeta  # noqa: E402
from k8s_llm_monitor_amd.serving import Engine, EngineConfig, TokenRules  # noqa: E402

CFG = replace(PRESETS["small"], window=50, sinks=4)
RULES = [TokenRules(repetition=1.6), None, TokenRules(frequency=0.3, presence=0.2, bias={17: 1.5, 31000: -2.0}), TokenRules(allowed=tuple(range(5, 32000, 7))),
         TokenRules(repetition=1.2, bias={3: 4.0}, allowed=(3, 4, 31999))]


@pytest.fixture(scope="module")
def model():
    return LlamaModel(CFG, "cuda", seed=3)


def prompts_of(seed, lens):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, CFG.vocab, (n,), generator=g).tolist() for n in lens]


def run(eng, prompts, n, rules=None, each=lambda: None):
    reqs = [eng.submit(p, n, r) for p, r in zip(prompts, rules or [None] * len(prompts))]
    for _ in range(3000):
        if eng.idle():
            break
        eng.step()
        each()
    assert all(r.error is None and len(r.out) == n for r in reqs) and eng.alloc.free == eng.alloc.total
    return [r.out for r in reqs]


def engine(model, **kw):
    return Engine(EngineConfig(**{"model": "small", "max_num_seqs": 32, "max_model_len": 512, "kv_blocks": 256, "max_num_batched_tokens": 200, **kw}), model=model)


@pytest.mark.parametrize("n_seqs", [3, 20])           # decode on the skinny kernel (no fused RoPE with a window) and on the mid-batch one
def test_logits_with_a_window_match_the_fp32_cpu_model(model, n_seqs):
    cpu = LlamaModel(CFG, "cpu", seed=0, dtype=torch.float32).load_from(model)
    g = torch.Generator().manual_seed(n_seqs)
    lens = [int(x) for x in torch.randint(5, 120, (n_seqs,), generator=g)]
    prompts = prompts_of(n_seqs, lens)
    table = torch.arange(n_seqs * 8, dtype=torch.int32).view(n_seqs, 8)
    out = []
    for m in (cpu, model):
        dev = m.device
        cache, bt = m.new_cache(n_seqs * 8), table.to(dev)
        at = [sum(lens[:i]) for i in range(n_seqs + 1)]
        slots = torch.cat([table[i].repeat_interleave(16)[:n] * 16 + torch.arange(n) % 16 for i, n in enumerate(lens)]).to(torch.int32)
        info = torch.tensor([[a, n, n] for a, n in zip(at, lens)], dtype=torch.int32, device=dev)
        last = torch.tensor([a - 1 for a in at[1:]], dtype=torch.int64, device=dev)
        pre = m.prefill(torch.tensor(sum(prompts, []), device=dev), torch.cat([torch.arange(n) for n in lens]).to(torch.int32).to(dev), slots.to(dev), cache,
                        PrefillMeta.build(CFG, lens, bt, info, last, dev), logits=True)
        n = torch.tensor(lens, dtype=torch.int32)
        nxt = (out[0][0] if out else pre.cpu()).argmax(-1)
        slot = table.gather(1, (n // 16).long()[:, None])[:, 0] * 16 + n % 16
        dec = m.decode(nxt.to(dev), n.to(dev), slot.to(torch.int32).to(dev), cache, DecodeMeta(bt, (n + 1).to(dev)), logits=True)
        out.append((pre.float().cpu(), dec.float().cpu()))
    for a, b in zip(*out):                             # the bound that the model without a window has against its fp32 twin
        assert float((a - b).abs().max() / a.abs().max()) < 0.03


def test_graphs_eager_launches_and_stale_blocks_give_the_same_tokens(model):
    prompts, outs = prompts_of(11, (7, 33, 64, 130, 16)), []
    for graphs, poison in ((True, False), (False, False), (True, True)):
        eng = engine(model, use_graphs=graphs)

        def stale():
            if poison:
                free = torch.tensor(eng.alloc._free, device="cuda")
                eng.cache.k[:, free] = float("nan")
                eng.cache.v[:, free] = float("nan")
            for r in eng.running:
                assert sum(b >= 0 for b in r.blocks) <= 6

        stale()
        outs.append(run(eng, prompts, 60, each=stale))
    assert outs[0] == outs[1] == outs[2]


def test_rules_from_a_graph_are_those_of_eager_launches(model):
    prompts, outs = prompts_of(12, (7, 33, 64, 100, 16)), []
    for graphs in (True, False):
        eng = engine(model, use_graphs=graphs)
        outs.append(run(eng, prompts, 40, RULES))
        if graphs:
            assert eng._rule_graphs and run(eng, prompts[:2], 40) != outs[0][:2]       # and without rules again
            assert run(eng, prompts, 40, RULES) == outs[0]
    assert outs[0] == outs[1]
    assert all(t % 7 == 5 for t in outs[0][3]) and set(outs[0][4]) <= {3, 4, 31999}
    assert run(engine(model), prompts, 40)[1] == outs[0][1]           # a request without rules beside others is as it was


@pytest.mark.parametrize("fp8", [False, True])
def test_the_cache_changes_its_size_under_running_graphs(model, fp8):
    prompts, kw = prompts_of(13, (60, 9, 130, 80)), {"kv_cache_dtype": "fp8" if fp8 else "bf16"}
    want = run(engine(model, **kw), prompts, 40, RULES[:4])
    eng, sizes, step = engine(model, **kw), [60, 400, 61], [0]

    def resize():
        step[0] += 1
        if step[0] % 6 == 3 and sizes:
            eng.resize_cache(sizes.pop())

    assert run(eng, prompts, 40, RULES[:4], resize) == want and not sizes


def test_a_window_beyond_the_context_is_no_window(model):
    whole = LlamaModel(PRESETS["small"], "cuda", seed=3)
    wide = LlamaModel(replace(CFG, window=4096, sinks=0), "cuda", seed=3)
    prompts = prompts_of(14, (30, 5, 77))
    a, b = run(engine(whole), prompts, 8), run(engine(wide), prompts, 8)
    assert sum(x[:2] == y[:2] for x, y in zip(a, b)) >= 2             # two kernels: near-ties aside the same text
