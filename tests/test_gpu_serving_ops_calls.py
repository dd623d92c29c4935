"""Calls of the serving operators that tests/test_gpu_serving_ops.py does not make, on the GPU: see tests/test_serving_ops_calls.py."""
from dataclasses import replace

import pytest
import torch

pytestmark = pytest.mark.gpu

from k8s_llm_monitor_amd.models.llama import PRESETS, LlamaModel  # noqa: E402
from k8s_llm_monitor_amd.ops import KlmOpsError, llm  # noqa: E402
from k8s_llm_monitor_amd.serving import Engine, EngineConfig, TokenRules  # noqa: E402

from window_oracle import SCALE, make  # noqa: E402

DEV = "cuda"


# ------------------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("kind,seqs", [("decode", [20, 3, 400, 0]), ("decode", [4000]), ("prefill", [(0, 70, 200), (70, 1, 3), (71, 30, 31)]), ("prefill", [(0, 16, 3000)])])
def test_attention_in_place_of_q(dtype, kind, seqs):
    """Same bits as into memory of its own, split and not; part of q's memory is refused."""
    q, k, v, table = make(kind, seqs, 8, 2, 150 if len(seqs) > 1 else 3000, 2, dtype)
    rows = len(seqs) if kind == "decode" else sum(n for _, n, _ in seqs)
    q, k, v, table = q[:rows].contiguous().to(DEV), k.to(DEV), v.to(DEV), table.to(DEV)
    lens = torch.tensor(seqs, dtype=torch.int32, device=DEV)

    def call(q, out=None):
        f = llm.paged_attn_decode_window if kind == "decode" else llm.paged_attn_prefill_window
        return f(q, k, v, table, lens, SCALE, 8, 150 if len(seqs) > 1 else 3000, 2, out=out)

    want = call(q)
    room = torch.empty(2 * rows + 1, 1024, dtype=torch.bfloat16, device=DEV)
    mine = room[:rows].copy_(q)
    with pytest.raises(KlmOpsError):
        call(mine, room.view(-1)[512:512 + rows * 1024].view(rows, 1024))
    assert torch.equal(call(mine, room[rows:2 * rows]), want) and torch.equal(mine, q)
    assert call(mine, mine) is mine and torch.equal(mine, want)


# ---------------------------------------------------------------------------------------------------------------- pages
def test_pairs_as_tensors_and_pairs_of_one_page():
    k = torch.randn(3, 9, 2, 16, 128, device=DEV).to(torch.bfloat16)
    v = torch.randn(3, 9, 2, 128, 16, device=DEV).to(torch.bfloat16)
    k0, v0 = k.clone(), v.clone()
    for bad in ([[0, 1], [2, 1]], [[0, 1], [1, 2]]):
        t = torch.tensor(bad)
        for form in (t, list(t), [tuple(row) for row in t], list(t.to(DEV))):
            with pytest.raises(KlmOpsError):
                llm.copy_pages(k, v, form)
    torch.cuda.synchronize()
    assert torch.equal(k, k0) and torch.equal(v, v0)
    llm.copy_pages(k, v, [(3, 3), (3, 4), (8, 8)])
    llm.copy_pages(k, v, list(torch.tensor([[0, 5], [0, 6]])))
    at = [0, 1, 2, 3, 3, 0, 0, 7, 8]
    assert torch.equal(k, k0[:, at]) and torch.equal(v, v0[:, at])


# ------------------------------------------------------------------------------------------------------- rules on logits
def test_out_beside_and_between_rows_of_logits():
    B, V = 5, 5000
    flat = torch.zeros(2 * B * V, device=DEV)
    with pytest.raises(KlmOpsError):
        llm.choose_tokens(flat.view(B, 2 * V)[:, :V], out=flat[B * V:].view(B, V))
    room = torch.empty(B * 7 * V, device=DEV)
    logits, out = room.view(B, 7 * V)[:, :V], room[V:V + B * V].view(B, V)
    x = torch.randn(B, V, device=DEV)
    logits.copy_(x)
    ids, best = llm.choose_tokens(logits, out=out)
    assert torch.equal(out, x) and torch.equal(logits, x) and torch.equal(ids, x.argmax(-1)) and torch.equal(best, x.amax(-1))


# --------------------------------------------------------------------------------------------------------------- engine
def test_a_smaller_cache_gives_its_memory_back():
    """To the device, not only to the process's allocator: another process may have it."""
    model = LlamaModel(replace(PRESETS["small"], window=50, sinks=4), "cuda", seed=3)
    eng = Engine(EngineConfig(model="small", max_num_seqs=4, max_model_len=256, kv_blocks=16384), model=model)
    reqs = [eng.submit(list(range(1, 30 + i)), 30, TokenRules(repetition=1.5) if i else None) for i in range(3)]
    for _ in range(8):
        eng.step()
    assert eng.describe()["rule_graphs"] == sorted(eng._rule_graphs) != []
    size, before = eng.cache.nbytes, torch.cuda.memory_reserved()
    eng.resize_cache(100)
    assert size > 1 << 30 and eng.cache.nbytes < size // 100 and before - torch.cuda.memory_reserved() > size * 9 // 10
    assert eng.describe()["graphs"] == eng.describe()["rule_graphs"] == []
    while not eng.idle():
        eng.step()
    assert all(r.error is None and len(r.out) == 30 for r in reqs)
