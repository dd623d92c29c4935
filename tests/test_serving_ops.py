"""Windowed attention, page copies and logit rules on the CPU: the fp32 references of ops/ref.py against definitions written
key by key (token by token) in 64 bits, and what the entry points refuse. The GPU kernels: tests/test_gpu_serving_ops.py."""
import math

import pytest
import torch

from k8s_llm_monitor_amd.ops import KlmOpsError, llm, ref

from window_oracle import SCALE, by_definition, make

DECODE = [0, 1, 2, 15, 16, 17, 33, 64, 100]
PREFILL = [(2, 5, 5), (7, 1, 1), (8, 17, 40), (25, 33, 33), (58, 0, 9), (58, 4, 3), (62, 2, 90)]


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (16, 0), (17, 5), (40, 16), (1000, 4), (7, 1000)])
@pytest.mark.parametrize("kind", ["decode", "prefill"])
@pytest.mark.parametrize("n_q,n_kv", [(4, 2), (3, 1)])
def test_reference_is_the_definition(kind, window, sinks, n_q, n_kv):
    seqs = DECODE if kind == "decode" else PREFILL
    q, k, v, table = make(kind, seqs, n_q, n_kv, window, sinks, torch.float32)
    want, _ = by_definition(kind, q.double(), k, v, table, seqs, n_q, window, sinks)
    if kind == "decode":
        lens = torch.tensor(seqs, dtype=torch.int32)
        got = ref.window_attn_decode(q.double(), k, v, table, lens, SCALE, window, sinks, dtype=torch.float64)
        fp32 = llm.paged_attn_decode_window(q.float(), k, v, table, lens, SCALE, n_q, window, sinks)
    else:
        info = torch.tensor(seqs, dtype=torch.int32)
        got = ref.window_attn_prefill(q.double(), k, v, table, info, SCALE, window, sinks, dtype=torch.float64)
        fp32 = llm.paged_attn_prefill_window(q.float(), k, v, table, info, SCALE, n_q, window, sinks)
    assert torch.allclose(got, want, rtol=0, atol=1e-12)
    assert torch.allclose(fp32.double(), want, rtol=0, atol=1e-5)


def test_a_window_of_the_whole_context_is_causal_attention():
    q, k, v, table = make("decode", DECODE, 4, 2, 10 ** 9, 0, torch.float32)
    lens = torch.tensor(DECODE, dtype=torch.int32)
    a = llm.paged_attn_decode_window(q.float(), k, v, table, lens, SCALE, 4, 10 ** 9)
    b = llm.paged_attn_decode(q.float(), k, v, table, lens, SCALE, 4)
    keep = lens > 0
    assert torch.allclose(a[keep], b[keep], atol=1e-5) and not a[~keep].any()


def test_rows_of_no_sequence():
    q, k, v, table = make("prefill", PREFILL, 4, 2, 9, 2, torch.float32)
    info = torch.tensor(PREFILL, dtype=torch.int32)
    mine = torch.zeros(q.shape[0], dtype=torch.bool)
    for q0, ql, n in PREFILL:
        mine[q0:q0 + ql] |= n >= ql > 0
    fresh = llm.paged_attn_prefill_window(q.float(), k, v, table, info, SCALE, 4, 9, 2)
    given = torch.full_like(fresh, 7.0)
    assert llm.paged_attn_prefill_window(q.float(), k, v, table, info, SCALE, 4, 9, 2, out=given) is given
    assert torch.equal(given[mine], fresh[mine]) and (given[~mine] == 7).all() and not fresh[~mine].any() and (~mine).sum() > 3


def test_window_refusals():
    q, k, v, table = make("decode", [20, 3], 4, 2, 8, 0, torch.float32)
    q = q.float()
    lens = torch.tensor([20, 3], dtype=torch.int32)

    def call(q=q, k=k, v=v, table=table, lens=lens, scale=SCALE, n_q=4, window=8, sinks=0, **kw):
        return llm.paged_attn_decode_window(q, k, v, table, lens, scale, n_q, window, sinks, **kw)

    call()
    for kw in (dict(window=0), dict(sinks=-1), dict(n_q=3), dict(n_q=8), dict(n_q=0), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(lens=lens[:1]), dict(table=table[:1]), dict(table=table[:, :0]), dict(q=q[:1]), dict(v=k), dict(k=k[:, :, :8]), dict(k=k[:0], v=v[:0]),
               dict(v=v.double()), dict(k=k.transpose(0, 1)), dict(q=torch.randn(512, 2).t()), dict(out=torch.zeros(2, 511)),
               dict(out=torch.zeros(2, 512, dtype=torch.float64)), dict(num_splits=-1), dict(num_splits=257), dict(k=k[0], v=v[0])):
        with pytest.raises(KlmOpsError):
            call(**kw)
    info = torch.tensor([[0, 1, 20], [1, 1, 3]], dtype=torch.int32)
    llm.paged_attn_prefill_window(q, k, v, table, info, SCALE, 4, 8)
    for bad in (info[:1], info[:, :2], info.flatten()):
        with pytest.raises(KlmOpsError):
            llm.paged_attn_prefill_window(q, k, v, table, bad, SCALE, 4, 8)
    with pytest.raises(KlmOpsError):
        llm.paged_attn_prefill_window(q, k, v, table, info, SCALE, 4, 0)


def test_pairs_that_are_no_pairs_are_refused_alike():
    """The check of short lists and that of all else take and refuse the same."""
    k, v = torch.zeros(1, 8, 1, 16, 128), torch.zeros(1, 8, 1, 128, 16)
    for bad in ([(1, 2, 3)], [(1, 2), (3,)], [1, 2], [(1.5, 2)], [("a", 1)], [(None, 1)], [(0, 8)], [(-2, 0)], [(8, 0)], [(2 ** 40, 0)], [(0, 1), (2, 1)],
                [(0, 1), (1, 2)], [(0, 2 ** 70)]):
        for pairs in (bad, tuple(bad), bad + [(4, i) for i in range(3, 3)]):
            with pytest.raises(KlmOpsError):
                llm.copy_pages(k, v, pairs)
    for n in (1, 3):
        for same in ([(1, 1)] * n if n == 1 else [(1, 1), (2, 2), (0, 3)], [[0, 5]], ((0, 5),), torch.tensor([[0, 5]])):
            llm.copy_pages(k, v, same)


def test_tiles_and_splits_of_a_prefill():
    pick = llm.pick_window_tiles
    assert pick(8192, 1, 4, 8, 4100, 8192) == (2, 1) and pick(2048, 1, 4, 8, 2048, 2048) == (1, 1)
    assert pick(1200, 1, 8, 8, 4096, 5200) == (2, 1) and pick(500, 1, 4, 8, 500, 500) == (1, 1)
    assert pick(16, 1, 4, 8, 4096, 4016) == (1, 20) and pick(1, 1, 1, 1, 3, 16) == (1, 1)
    for rows in (1, 7, 100, 3000):
        for seqs in (1, 5, 200):
            for group, n_kv in ((1, 1), (4, 8), (16, 2), (7, 3)):
                tiles, splits = pick(rows, seqs, group, n_kv, 4096, 5000)
                assert tiles in (1, 2) and 1 <= splits <= 24 and (splits == 1 or tiles == 1)


# ---------------------------------------------------------------------------------------------------------------- pages
def _cache(layers, nb, n_kv, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(layers, nb, n_kv, 16, 128, generator=g).to(dtype), torch.randn(layers, nb, n_kv, 128, 16, generator=g).to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_copy_pages(dtype):
    k, v = _cache(3, 9, 2, dtype)
    k0, v0 = k.clone(), v.clone()
    llm.copy_pages(k, v, [(0, 5), (0, 6), (8, 1), (3, 3), (-1, 7)])
    at = [0, 8, 2, 3, 4, 0, 0, 7, 8]
    for x, x0 in ((k, k0), (v, v0)):
        want = x0.view(torch.uint8)[:, at].clone()
        want[:, 7] = 0
        assert torch.equal(x.view(torch.uint8), want)
    one, two = k[1].clone(), v[1].clone()
    llm.copy_pages(k[1], v[1], [(2, 4)])                                # one layer alone
    one[4], two[4] = one[2].clone(), two[2].clone()
    assert torch.equal(k[1].view(torch.uint8), one.view(torch.uint8)) and torch.equal(v[1].view(torch.uint8), two.view(torch.uint8))
    k2, v2 = _cache(3, 4, 2, dtype, seed=1)
    llm.copy_pages(k2, v2, [(8, 0), (0, 1), (1, 2)], k_src=k, v_src=v)    # another cache: the same numbers on both sides are other pages
    assert torch.equal(k2[:, :3].view(torch.uint8), k[:, [8, 0, 1]].view(torch.uint8)) and torch.equal(v2[:, :3].view(torch.uint8), v[:, [8, 0, 1]].view(torch.uint8))
    llm.copy_pages(k, v, [])


def test_copy_pages_refusals():
    k, v = _cache(2, 6, 2)
    k2, v2 = _cache(2, 3, 2, seed=1)
    before = k.clone()
    for pairs in ([(0, 6)], [(6, 0)], [(0, -1)], [(-2, 0)], [(0, 1), (2, 1)], [(0, 1), (1, 2)], [(0, 1), (1, 1), (1, 2)], [(-1, 1), (1, 2)], [(0, 1, 2)]):
        with pytest.raises((KlmOpsError, ValueError)):
            llm.copy_pages(k, v, pairs)
    for kw in (dict(k_src=k2), dict(k_src=k2[:1], v_src=v2[:1]), dict(k_src=k2.float(), v_src=v2.float()), dict(k_src=k2[:, :, :1], v_src=v2[:, :, :1]),
               dict(k_src=k2[:, 1:], v_src=v2[:, 1:])):
        with pytest.raises(KlmOpsError):
            llm.copy_pages(k, v, [(0, 1)], **kw)
    with pytest.raises(KlmOpsError):
        llm.copy_pages(k[0:1], v[0:1], [(0, 1)], k_src=k[0:1, :3], v_src=v[0:1, :3])         # part of the same memory
    with pytest.raises(KlmOpsError):
        llm.copy_pages(v, k, [(0, 1)])
    assert torch.equal(k, before)


# ------------------------------------------------------------------------------------------------------- rules on logits
def _rules(R, n, V, total, seed=0, bias=6, masks=3, rows=None):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, n + 3, (R,), generator=g, dtype=torch.int32)          # some beyond the list
    mask = torch.randint(-2 ** 31, 2 ** 31 - 1, (masks, -(-total // 32)), generator=g, dtype=torch.int32)
    return llm.LogitRules(torch.randint(-2, total + 3, (R, n), generator=g, dtype=torch.int32), (lens.float() * torch.rand(R, generator=g)).int(), lens,
                          torch.rand(R, generator=g) + 0.5, torch.randn(R, generator=g), torch.randn(R, generator=g),
                          torch.randint(-1, min(total, 9), (R, bias), generator=g, dtype=torch.int32), torch.randn(R, bias, generator=g), mask,
                          torch.randint(-1, masks + 1, (R,), generator=g, dtype=torch.int32), rows)


def _by_token(x, r, first, rule):
    """One row, token by token."""
    y, ok = [], []
    n = min(max(int(rule.lens[r]), 0), rule.history.shape[1])
    h = rule.history[r, :n].tolist()
    p = int(rule.prompt_lens[r])
    m = int(rule.mask_rows[r])
    for v, a in enumerate(x.double().tolist()):
        t = v + first
        c = h[p:].count(t)
        if t in h:
            a = a / float(rule.repetition[r]) if a > 0 else a * float(rule.repetition[r])
        a -= float(rule.frequency[r]) * c
        if c:
            a -= float(rule.presence[r])
        for b, w in reversed(list(zip(rule.bias_ids[r].tolist(), rule.bias_values[r].tolist()))):
            if b == t:
                a += w
                break
        fine = not 0 <= m < rule.mask.shape[0] or (int(rule.mask[m, t // 32]) >> (t % 32)) & 1
        ok.append(bool(fine))
        y.append(a if fine else -math.inf)
    live = [i for i in range(len(y)) if ok[i]]
    return y, (max(live, key=lambda i: (y[i], -i)) + first if live else -1)


@pytest.mark.parametrize("first,V", [(0, 45), (45, 45), (64, 33)])
def test_logit_reference_is_the_definition(first, V):
    B, total = 7, 140
    rows = torch.tensor([3, -1, 0, 8, 1, 2, 2], dtype=torch.int32)          # none, one beyond, one twice
    rule = _rules(5, 30, V, total, rows=rows)
    x = torch.randn(B, V, generator=torch.Generator().manual_seed(5))
    out = torch.empty(B, V)
    ids, best = llm.choose_tokens(x, rule, first_token=first, out=out)
    for b in range(B):
        r = int(rows[b])
        y, pick = _by_token(x[b], r, first, rule) if 0 <= r < 5 else (x[b].tolist(), int(x[b].argmax()) + first)
        # four operations, each off by at most half a step of a value below 16
        assert torch.allclose(out[b].double(), torch.tensor(y, dtype=torch.float64), rtol=0, atol=4 * 16 * 2.0 ** -24)
        assert int(ids[b]) == pick and float(best[b]) == (float(out[b, pick - first]) if pick >= 0 else -math.inf)


def test_choice_ties_nan_and_nothing_allowed():
    x = torch.tensor([[1.0, 3.0, 3.0, 2.0], [0.0, -0.0, -1.0, -0.0], [float("nan"), 9.0, float("nan"), float("inf")], [float("-inf")] * 4, [5.0, 4.0, 3.0, 2.0]])
    ids, best = llm.choose_tokens(x)
    assert ids.tolist() == [1, 0, 0, 0, 0] and torch.isnan(best[2]) and float(best[3]) == -math.inf
    z = torch.zeros(5, dtype=torch.int32)
    one = torch.ones(5)
    rule = llm.LogitRules(torch.zeros(5, 1, dtype=torch.int32), z, z, one, one * 0, one * 0, mask=torch.tensor([[0], [0b1010], [0b0010], [0b1000], [0b0100]], dtype=torch.int32))
    out = torch.empty(5, 4)
    ids, best = llm.choose_tokens(x, rule, out=out)
    assert ids.tolist() == [-1, 1, 1, 3, 2] and best[0] == -math.inf and best[3] == -math.inf and out[2].tolist() == [-math.inf, 9.0, -math.inf, -math.inf]


def test_logit_refusals():
    B, V, total = 4, 40, 40
    x = torch.randn(B, V)
    good = _rules(4, 8, V, total)
    llm.choose_tokens(x, good)

    def having(**kw):
        return llm.LogitRules(**{**good.__dict__, **kw})

    for kw in (dict(lens=good.lens.long()), dict(history=good.history[:3]), dict(history=good.history[0]), dict(prompt_lens=good.prompt_lens[:2]),
               dict(repetition=good.repetition.double()), dict(frequency=good.frequency[:, None]), dict(presence=good.presence[:3]), dict(bias_ids=None),
               dict(bias_values=good.bias_values[:, :2]), dict(bias_ids=good.bias_ids.long()), dict(mask=good.mask[:, :1]), dict(mask=good.mask[0]),
               dict(mask=None), dict(mask_rows=None), dict(mask_rows=good.mask_rows[:2]), dict(rows=torch.zeros(3, dtype=torch.int32)), dict(history=good.history.t().contiguous().t())):
        with pytest.raises(KlmOpsError):
            llm.choose_tokens(x, having(**kw))
    with pytest.raises(KlmOpsError):
        llm.choose_tokens(torch.randn(5, V), good)                       # more rows than sets of rules, and no `rows`
    with pytest.raises(KlmOpsError):
        llm.choose_tokens(x, good, first_token=1 << 10)                  # the masks end before
    for bad in (x.double(), x[0], x.t(), x[:, :0]):
        with pytest.raises(KlmOpsError):
            llm.choose_tokens(bad)
    with pytest.raises(KlmOpsError):
        llm.choose_tokens(x, first_token=-1)
    with pytest.raises(KlmOpsError):
        llm.choose_tokens(x, first_token=2 ** 31 - 8)
    for out in (torch.empty(B, V + 1), torch.empty(B, V, dtype=torch.bfloat16), torch.empty(V, B).t()):
        with pytest.raises(KlmOpsError):
            llm.choose_tokens(x, out=out)
    big = torch.zeros(B * V + 1)
    with pytest.raises(KlmOpsError):
        llm.choose_tokens(big[:-1].view(B, V), out=big[1:].view(B, V))
    same = x.clone()
    ids, _ = llm.choose_tokens(same, good, out=same)                     # in place
    y = torch.empty_like(x)
    assert torch.equal(ids, llm.choose_tokens(x, good, out=y)[0]) and torch.equal(same, y)
