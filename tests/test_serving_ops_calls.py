"""Calls of the serving operators that their documentation allows or refuses and that tests/test_serving_ops.py does not make, on the
CPU. The same operators on a GPU: tests/test_gpu_serving_ops.py, tests/test_gpu_serving_ops_calls.py."""
from types import SimpleNamespace

import pytest
import torch

from k8s_llm_monitor_amd.models.llama import LlamaModel
from k8s_llm_monitor_amd.ops import KlmOpsError, llm

from window_oracle import SCALE, make


def _pages(blocks=8):
    g = torch.Generator().manual_seed(0)
    return torch.randn(2, blocks, 1, 16, 128, generator=g), torch.randn(2, blocks, 1, 128, 16, generator=g)


# ------------------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("kind", ["decode", "prefill"])
def test_attention_out_may_be_q_but_not_share_part_of_it(kind):
    seqs = [20, 3, 40] if kind == "decode" else [(0, 2, 20), (2, 1, 3)]
    q, k, v, table = make(kind, seqs, 4, 2, 8, 2, torch.float32)
    q = q[:3].float()                                                     # contiguous [3, 512]
    lens = torch.tensor(seqs, dtype=torch.int32)

    def call(q, out=None):
        f = llm.paged_attn_decode_window if kind == "decode" else llm.paged_attn_prefill_window
        return f(q, k, v, table, lens, SCALE, 4, 8, 2, out=out)

    want = call(q)
    wide = torch.zeros(3, 1024)                                           # q as a part of fused rows
    wide[:, :512] = q
    for at in (0, 512, 1024, 1536):
        with pytest.raises(KlmOpsError):
            call(wide[:, :512], wide.view(-1)[at:at + 3 * 512].view(3, 512))
    long = torch.zeros(5, 512)
    long[:3] = q
    with pytest.raises(KlmOpsError):
        call(long[:3], long[1:4])
    assert torch.equal(call(long[:3], long[3:5].repeat(2, 1)[:3]), want)
    same = q.clone()
    assert call(same, same) is same and torch.equal(same, want)


def test_splits_of_a_prefill_stay_on_the_chip():
    """1024 blocks of a bf16 cache, 768 of an e4m3 one: more would run as a whole round and a rest."""
    pick = llm.pick_window_tiles
    assert pick(800, 1, 4, 8, 4100, 4816, False) == (1, 2) and pick(800, 1, 4, 8, 4100, 4816, True) == (1, 1)
    assert pick(520, 1, 4, 8, 4100, 4528, False) == (1, 3) and pick(520, 1, 4, 8, 4100, 4528, True) == (1, 2)
    assert pick(16, 1, 4, 8, 4096, 4016) == pick(16, 1, 4, 8, 4096, 4016, True) == (1, 20)
    for rows in (1, 60, 200, 390, 700, 900, 3000):
        for seqs in (1, 5, 40):
            for group, n_kv in ((1, 1), (4, 8), (16, 2), (7, 3), (8, 8)):
                for kv8, most in ((False, 1024), (True, 768)):
                    tiles, splits = pick(rows, seqs, group, n_kv, 4096, 5000, kv8)
                    assert splits == 1 or (tiles == 1 and splits * (-(-rows * group // 64) + seqs - 1) * n_kv <= most)


# ---------------------------------------------------------------------------------------------------------------- pages
@pytest.mark.parametrize("pairs", [[[0, 1], [2, 1]], [[0, 1], [1, 2]], [[-1, 1], [1, 2]], [[0, 8]], [[True, False]], [[0.0, 1.0]]])
def test_pairs_are_looked_at_as_numbers_whatever_holds_them(pairs):
    """A tensor of pairs, its rows in a list, its single numbers: a page written twice, or written and read, is refused in all forms."""
    k, v = _pages()
    k0 = k.clone()
    t = torch.tensor(pairs)
    for form in (pairs, tuple(map(tuple, pairs)), t, list(t), tuple(t), [tuple(row) for row in t], t.numpy(), list(t.numpy()), [tuple(row) for row in t.numpy()]):
        with pytest.raises(KlmOpsError):
            llm.copy_pages(k, v, form)
    assert torch.equal(k, k0)


def test_pairs_in_every_form_copy_the_same():
    t = torch.tensor([[0, 5], [0, 6], [-1, 7]])
    want = None
    for form in (t.tolist(), t, list(t), [tuple(row) for row in t], t.numpy(), [tuple(row) for row in t.numpy()]):
        k, v = _pages()
        llm.copy_pages(k, v, form)
        want = want or (k, v)
        assert torch.equal(k, want[0]) and torch.equal(v, want[1]) and torch.equal(k[:, 5], k[:, 0]) and not v[:, 7].any()


def test_a_pair_of_a_page_and_itself_does_nothing():
    """Neither counts as a write nor as a read of its page, but has to lie in the cache."""
    for pairs, at in (([(3, 3), (3, 4)], [0, 1, 2, 3, 3, 5, 6, 7]), ([(3, 3), (0, 3)], [0, 1, 2, 0, 4, 5, 6, 7]), ([(3, 3), (3, 3)], list(range(8)))):
        for form in (pairs, tuple(pairs), torch.tensor(pairs)):
            k, v = _pages()
            k0, v0 = k.clone(), v.clone()
            llm.copy_pages(k, v, form)
            assert torch.equal(k, k0[:, at]) and torch.equal(v, v0[:, at])
    k, v = _pages()
    for pairs in ([(8, 8)], [(-1, -1)], [(1, 1), (0, 1), (1, 2)], [(1, 1), (0, 1), (2, 1)]):
        with pytest.raises(KlmOpsError):
            llm.copy_pages(k, v, pairs)
    k2, v2 = _pages()
    with pytest.raises(KlmOpsError):                                     # another cache: the same number is another page
        llm.copy_pages(k2, v2, [(3, 3), (0, 3)], k_src=k, v_src=v)


# ------------------------------------------------------------------------------------------------------- rules on logits
def test_out_may_not_share_memory_with_a_row_of_logits():
    """Rows of logits far apart: `out` behind the first of them meets the last ones. Between them there is room."""
    B, V = 4, 24
    x = torch.randn(B, V, generator=torch.Generator().manual_seed(1))
    flat = torch.zeros(2 * B * V)
    for at in (0, 1, B * V - 7, B * V):
        with pytest.raises(KlmOpsError):
            llm.choose_tokens(flat.view(B, 2 * V)[:, :V], out=flat[at:at + B * V].view(B, V))
    half = torch.zeros(3 * B * V, dtype=torch.bfloat16)
    for at in (0, V, B * V // 2):
        with pytest.raises(KlmOpsError):
            llm.choose_tokens(half.view(B, 3 * V)[:, :V], out=half.view(torch.float32)[at:at + B * V].view(B, V))
    room = torch.empty(8 * B * V)
    for logits, at in ((room[:2 * B * V].view(B, 2 * V)[:, :V], 2 * B * V - V), (room[B * V:3 * B * V].view(B, 2 * V)[:, :V], 0),
                       (room.view(B, 8 * V)[:, :V], V), (room.view(B, 8 * V)[:, :V], 17 * V)):
        logits.copy_(x)
        out = room[at:at + B * V].view(B, V)
        ids, _ = llm.choose_tokens(logits, out=out)
        assert torch.equal(out, x) and torch.equal(logits, x) and torch.equal(ids, x.argmax(-1))


class _Ranks:
    """Two ranks' `all_gather`, one after the other: the first round collects, the second answers with what both gave."""

    def __init__(self):
        self.world, self.rank, self.given = 2, 0, {}

    def all_gather(self, x):
        self.given[self.rank] = x.clone()
        return torch.stack([self.given.get(r, x) for r in range(2)])


@pytest.mark.parametrize("low", [-float("inf"), torch.finfo(torch.float32).min, -3.0, float("nan"), float("inf")])
@pytest.mark.parametrize("high", [-float("inf"), torch.finfo(torch.float32).min, 5.0, float("nan")])
@pytest.mark.parametrize("allowed", [0b11, 0b10, 0b01, 0b00])
def test_two_ranks_choose_what_one_would(low, high, allowed):
    """Values at the ends of fp32 too: rank 0's tokens are all `low`, rank 1's all `high`; `allowed`: whose tokens the rules allow."""
    V, z, one = 32, torch.zeros(3, dtype=torch.int32), torch.ones(3)
    whole = torch.cat([torch.full((3, V), low), torch.full((3, V), high)], 1)
    mask = torch.tensor([[-(allowed & 1), -(allowed >> 1)]] * 3, dtype=torch.int32)
    rules = llm.LogitRules(torch.zeros(3, 1, dtype=torch.int32), z, z, one, one * 0, one * 0, mask=mask)
    want = llm.choose_tokens(whole, rules)[0]
    tp = _Ranks()
    model = SimpleNamespace(tp=tp)
    for _ in range(2):
        got = []
        for tp.rank in range(2):
            got.append(LlamaModel._sample(model, whole[:, tp.rank * V:(tp.rank + 1) * V].contiguous(), False, rules))
    assert got[0].tolist() == got[1].tolist() == want.tolist()


def test_blocks_of_a_choice_are_on_the_chip_at_once():
    """3 blocks a CU of 256 CUs, where 8 slices a block are enough for that."""
    for B in (1, 2, 7, 33, 64, 96, 128, 200, 256, 700):
        for V in (1, 4090, 32000, 50001, 64128, 128256):
            parts, slices = llm._lib().klm_logits_parts(B, V), -(-(V + 7) // 4096)
            per = -(-slices // parts)
            assert parts * B <= 768 or parts == -(-slices // 8), (B, V)
            assert per == 1 or -(-slices // (per - 1)) * B > 768, (B, V)       # and no fewer blocks than that takes
