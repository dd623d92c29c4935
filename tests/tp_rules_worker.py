"""One of two gloo ranks: a tensor-parallel engine with a window and with rules on the choice of tokens, against the engine that
holds the whole model. Prints one line ``RESULT {json}``."""
import json
import os
import sys
from dataclasses import replace

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from k8s_llm_monitor_amd.models.llama import PRESETS, LlamaModel  # noqa: E402
from k8s_llm_monitor_amd.ops import llm  # noqa: E402
from k8s_llm_monitor_amd.parallel.tp import TPGroup  # noqa: E402
from k8s_llm_monitor_amd.serving import Engine, EngineConfig, TokenRules  # noqa: E402


def main() -> int:
    rank = int(os.environ["RANK"])
    dist.init_process_group("gloo", rank=rank, world_size=2)
    dev = torch.device("cpu")
    tp = TPGroup(dev, data="gloo", slot_bytes=8 << 20, spin_limit_s=20.0)
    cfg = replace(PRESETS["tiny"], window=30, sinks=2)
    rules = [TokenRules(repetition=1.7, frequency=0.2), TokenRules(allowed=tuple(range(300, 330))), None, TokenRules(bias={5: 3.0, 500: 3.0}),
             TokenRules(allowed=(1, 2, 3), presence=0.5)]
    out = {}
    with torch.no_grad():
        full = LlamaModel(cfg, dev, seed=5, dtype=torch.float32)
        part = LlamaModel(cfg, dev, seed=0, dtype=torch.float32, tp=tp).load_shard_from(full)
        ecfg = EngineConfig(model="tiny", device="cpu", max_num_seqs=4, max_model_len=128, max_num_batched_tokens=50, kv_blocks=40, use_graphs=False)
        gen = torch.Generator().manual_seed(23)
        prompts = [torch.randint(0, cfg.vocab, (n,), generator=gen).tolist() for n in (40, 13, 7, 65, 30)]
        eng = Engine(ecfg, model=part)
        reqs = [eng.submit(p, 20, r) for p, r in zip(prompts, rules)] if rank == 0 else []
        eng.step_all()
        steps = 1
        while not eng.idle():
            eng.step_all()
            steps += 1
        out["steps"] = steps
        if rank == 0:
            one = Engine(ecfg, model=full)
            want = [one.submit(p, 20, r) for p, r in zip(prompts, rules)]
            while not one.idle():
                one.step()
            out["match"] = [r.out for r in reqs] == [r.out for r in want] and all(r.error is None for r in reqs)
        # all logits equal: the lowest allowed token; only the second rank's part allowed: its lowest, whatever the value
        V = part.lcfg.vocab
        z, one_set = torch.zeros(2, V), torch.ones(2)
        i32 = dict(dtype=torch.int32)
        mask = torch.full((2, cfg.vocab // 32), -1, **i32)
        mask[1, : V // 32 + 1] = 0
        lr = llm.LogitRules(torch.zeros(2, 1, **i32), torch.zeros(2, **i32), torch.zeros(2, **i32), one_set, one_set * 0, one_set * 0, mask=mask)
        ids = part._sample(z, False, lr).tolist()
        low = part._sample(torch.full((2, V), float("-inf")), False, lr).tolist()
        out["lowest_rank_of_a_tie"] = ids == [0, V + 32] and low == [0, V + 32]
    tp.barrier()
    tp.close()
    print("RESULT " + json.dumps(out), flush=True)
    dist.barrier()
    dist.destroy_process_group()
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
