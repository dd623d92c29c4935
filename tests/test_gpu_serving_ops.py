"""Windowed paged attention, page copies and logit rules on the GPU (ops/csrc/llm_window.hip, llm_pages.hip, llm_logits.hip)
against definitions in 64 bits. The oracles themselves are tested in tests/test_serving_ops.py."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from k8s_llm_monitor_amd.ops import KlmOpsError, llm, ref  # noqa: E402

from window_oracle import SCALE, allowed, by_definition, make  # noqa: E402

DEV = "cuda"
DECODE = [0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 129, 300]
PREFILL = [(2, 5, 5), (7, 1, 1), (8, 17, 40), (25, 33, 33), (58, 0, 9), (58, 4, 3), (62, 2, 90), (64, 70, 131)]


def _decode(q, k, v, table, seqs, n_q, window, sinks, **kw):
    lens = torch.tensor(seqs, dtype=torch.int32, device=DEV)
    return llm.paged_attn_decode_window(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), lens, SCALE, n_q, window, sinks, **kw)


def _prefill(q, k, v, table, seqs, n_q, window, sinks, **kw):
    info = torch.tensor(seqs, dtype=torch.int32, device=DEV).reshape(-1, 3)
    return llm.paged_attn_prefill_window(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), info, SCALE, n_q, window, sinks, **kw)


def _near(got, want, size):
    got = got.cpu().double()
    assert bool(torch.isfinite(got).all()), "a value that no row sees reached the result"
    over = (got - want).abs() - allowed(want, size)
    assert float(over.max()) <= 0, f"{float((got - want).abs().max()):.3g} off, {float(over.max()):.3g} more than the roundings explain"


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (15, 0), (16, 5), (17, 16), (33, 40), (200, 3), (5000, 0), (10 ** 9, 10 ** 9)])
@pytest.mark.parametrize("n_q,n_kv,dtype", [(8, 2, torch.bfloat16), (3, 1, torch.float8_e4m3fn), (20, 1, torch.bfloat16), (8, 1, torch.float8_e4m3fn)])
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_decode(window, sinks, n_q, n_kv, dtype, splits):
    q, k, v, table = make("decode", DECODE, n_q, n_kv, window, sinks, dtype)
    want, size = by_definition("decode", q, k, v, table, DECODE, n_q, window, sinks)
    _near(_decode(q, k, v, table, DECODE, n_q, window, sinks, num_splits=splits), want, size)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (15, 0), (16, 5), (17, 16), (33, 40), (200, 3), (10 ** 9, 0)])
@pytest.mark.parametrize("n_q,n_kv,dtype", [(8, 2, torch.bfloat16), (3, 1, torch.float8_e4m3fn), (20, 1, torch.bfloat16), (8, 1, torch.float8_e4m3fn), (2, 2, torch.bfloat16)])
def test_prefill(window, sinks, n_q, n_kv, dtype):
    q, k, v, table = make("prefill", PREFILL, n_q, n_kv, window, sinks, dtype)
    want, size = by_definition("prefill", q, k, v, table, PREFILL, n_q, window, sinks)
    _near(_prefill(q, k, v, table, PREFILL, n_q, window, sinks), want, size)


def _reference(kind, q, k, v, table, seqs, window, sinks):
    """The fp64 reference on the GPU, for sizes that are too slow key by key; `size` from the same with |v|."""
    a = [x.to(DEV) for x in (q, k, v, table)]
    fn = ref.window_attn_decode if kind == "decode" else ref.window_attn_prefill
    t = torch.tensor(seqs, dtype=torch.int32)
    outs = [fn(a[0].double(), a[1], x, a[3], t, SCALE, window, sinks, dtype=torch.float64).cpu() for x in (a[2], a[2].float().abs())]
    return outs


def _random(kind, seqs, n_q, n_kv, dtype, seed=0):
    """Finite values everywhere, all pages in the tables."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    ctx = [n if kind == "decode" else n[2] for n in seqs]
    width = max(1, max(-(-n // 16) for n in ctx))
    nb = sum(-(-n // 16) for n in ctx) + 5
    order = torch.randperm(nb, generator=g, device=DEV).int()
    table, at = torch.full((len(seqs), width), -1, dtype=torch.int32, device=DEV), 0
    for s, n in enumerate(ctx):
        table[s, : -(-n // 16)] = order[at:at + -(-n // 16)]
        at += -(-n // 16)
    rows = len(seqs) if kind == "decode" else max(q0 + ql for q0, ql, _ in seqs)
    r = lambda *shape: torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    return r(rows, (n_q + 2 * n_kv) * 128)[:, : n_q * 128], r(nb, n_kv, 16, 128).to(dtype), r(nb, n_kv, 128, 16).to(dtype), table


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("window,sinks", [(1000, 4), (2048, 100), (4096, 0)])
def test_decode_of_long_contexts(dtype, window, sinks):
    seqs = [5000, 1, 4097, 3071, 999, 0, 6001]
    q, k, v, table = _random("decode", seqs, 32, 8, dtype)
    want, size = _reference("decode", q, k, v, table, seqs, window, sinks)
    for splits in (0, 1, 16):
        _near(_decode(q, k, v, table, seqs, 32, window, sinks, num_splits=splits), want, size)


@pytest.mark.parametrize("n_q,n_kv,dtype", [(32, 8, torch.bfloat16), (28, 4, torch.bfloat16), (16, 1, torch.float8_e4m3fn)])
@pytest.mark.parametrize("seqs,window,sinks", [([(0, 1500, 1500)], 700, 4), ([(0, 3, 2500), (3, 700, 2000), (703, 1, 1), (704, 130, 2900)], 1024, 33),
                                               ([(0, 16, 4000)], 4096, 0)])
def test_prefill_of_long_contexts(n_q, n_kv, dtype, seqs, window, sinks):
    q, k, v, table = _random("prefill", seqs, n_q, n_kv, dtype)
    want, size = _reference("prefill", q, k, v, table, seqs, window, sinks)
    _near(_prefill(q, k, v, table, seqs, n_q, window, sinks), want, size)


def test_many_sequences_in_one_launch():
    """More sequences than a wave has lanes: the search for a block's work goes round again; some have no rows."""
    seqs, at = [], 0
    for i in range(150):
        ql = (0, 1, 9, 40)[i % 4]
        seqs.append((at, ql, ql + i % 3 * 20))
        at += ql
    q, k, v, table = _random("prefill", seqs, 4, 2, torch.bfloat16)
    want, size = _reference("prefill", q, k, v, table, seqs, 25, 2)
    _near(_prefill(q, k, v, table, seqs, 4, 25, 2), want, size)


def test_pages_that_are_not_there():
    """-1, ids beyond the cache and tokens beyond the table are not seen; a row that sees nothing is 0."""
    n, width = 100, 5                                                   # the table ends at token 80
    for kind, seqs in (("decode", [n, n, 70]), ("prefill", [(0, 30, n), (30, 2, n), (32, 50, 70)])):
        q, k, v, table = make(kind, seqs, 8, 2, 50, 3, width=8)
        table = table[:, :width].contiguous()
        table[0, 4], table[0, 0], table[2, 2], table[2, 3] = -1, k.shape[0], 2 ** 31 - 1, -2 ** 31
        want, size = by_definition(kind, q, k, v, table, seqs, 8, 50, 3)
        got = (_decode if kind == "decode" else _prefill)(q, k, v, table, seqs, 8, 50, 3)
        _near(got, want, size)
        table[:] = -1
        got = (_decode if kind == "decode" else _prefill)(q, k, v, table, seqs, 8, 50, 3)
        assert not got.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_value_reaches_only_the_rows_that_see_it(dtype, bad):
    """One token's V is NaN or infinite: tokens before it and tokens whose window has passed it are in the same query tile."""
    if dtype == torch.float8_e4m3fn and math.isinf(bad):
        pytest.skip("e4m3 has no infinity")
    seqs, window, sinks, tok = [(0, 200, 200)], 40, 2, 77
    q, k, v, table = make("prefill", seqs, 4, 2, window, sinks, dtype, spare=0)
    want, size = by_definition("prefill", q, k, v, table, seqs, 4, window, sinks)
    vb = v.float()
    vb[int(table[0, tok // 16]), 0, :, tok % 16] = bad
    got = _prefill(q, k, vb.to(dtype), table, seqs, 4, window, sinks).cpu().double()
    hit = torch.zeros(200, 4, dtype=torch.bool)
    hit[tok:tok + window, :2] = True                                    # the two query heads of kv head 0
    got, want, size = (x.view(200, 4, 128) for x in (got, want, size))
    _near(got[~hit], want[~hit], size[~hit])
    assert not torch.isfinite(got[hit]).any()
    kb = k.float()
    kb[int(table[0, tok // 16]), 0, tok % 16] = bad                     # and its K: scores of the rows that see it
    got = _prefill(q, kb.to(dtype), v, table, seqs, 4, window, sinks).cpu().double().view(200, 4, 128)
    _near(got[~hit], want[~hit], size[~hit])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("kind,seqs,n_q,n_kv,window,sinks", [("decode", DECODE, 20, 1, 50, 4), ("prefill", PREFILL, 8, 2, 50, 4), ("prefill", [(0, 300, 900)], 16, 2, 200, 3),
                                                             ("prefill", [(0, 1300, 2000)], 64, 8, 300, 20)])
def test_what_masked_places_hold_moves_no_bit(dtype, kind, seqs, n_q, n_kv, window, sinks):
    """NaN or 0 in every place that no row sees: not a value of the result may differ, whichever way the kernel took."""
    call = _decode if kind == "decode" else _prefill
    got = [call(*make(kind, seqs, n_q, n_kv, window, sinks, dtype, poison=p), seqs, n_q, window, sinks) for p in (True, False)]
    assert bool(torch.isfinite(got[0]).all()) and torch.equal(*got)


def test_large_scores_and_a_growing_maximum():
    """Scores in the hundreds, each key's larger than the one before it: the running maximum moves at every step."""
    for kind, seqs in (("decode", [150, 40]), ("prefill", [(0, 150, 150), (150, 40, 90)])):
        q, k, v, table = make(kind, seqs, 4, 2, 100, 3)
        q = (q.float().abs() * 4).to(torch.bfloat16)
        for s, row in enumerate(table.tolist()):
            for p, b in enumerate(row):
                if b >= 0:
                    k[b] = (k[b].float().abs() * (1 + 0.2 * torch.arange(p * 16, p * 16 + 16)[None, :, None])).to(torch.bfloat16)
        want, size = by_definition(kind, q, k, v, table, seqs, 4, 100, 3)
        got = (_decode if kind == "decode" else _prefill)(q, k, v, table, seqs, 4, 100, 3).cpu().double()
        # scores reach |s| = scale * sum |q k| ~ 2000 in 32 bits: 2^-24 of that times a few roundings more in each weight
        slack = 2 * 2000 * 2.0 ** -22
        assert ((got - want).abs() <= allowed(want, size) + slack * size).all()


def test_strides_given_out_and_untouched_rows():
    seqs = [(3, 40, 60), (43, 20, 20)]
    q, k, v, table = make("prefill", seqs, 8, 2, 30, 2)
    dense = q.contiguous()
    out = torch.full((q.shape[0], 8 * 128), 3.0, dtype=torch.bfloat16, device=DEV)
    assert _prefill(q, k, v, table, seqs, 8, 30, 2, out=out) is out
    assert (out[:3] == 3).all() and (out[63:] == 3).all()
    fresh = _prefill(dense, k, v, table, seqs, 8, 30, 2)
    assert torch.equal(fresh[3:63], out[3:63]) and not fresh[:3].any() and not fresh[63:].any()
    lens = [50, 9]
    q, k, v, table = make("decode", lens, 8, 2, 30, 2)
    wide = torch.randn(2, 4096, dtype=torch.float32).to(torch.bfloat16).to(DEV)
    wide[:, 64:64 + 1024] = q.to(DEV)
    a = _decode(wide[:, 64:64 + 1024], k, v, table, lens, 8, 30, 2)
    assert torch.equal(a, _decode(q.contiguous(), k, v, table, lens, 8, 30, 2))
    with pytest.raises(KlmOpsError):
        _decode(wide[:, 63:63 + 1024], k, v, table, lens, 8, 30, 2)       # 2-byte alignment


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("seqs,rows,n_q,n_kv", [([(5, 20, 3000)], 40, 8, 2), ([(0, 3, 2000), (7, 9, 10), (30, 2, 1)], 33, 4, 4), ([(9, 2000, 2100), (2010, 1, 1)], 2020, 32, 8)])
def test_rows_of_no_sequence_whatever_the_launch(dtype, seqs, rows, n_q, n_kv):
    """Few rows (split keys and their join), many rows (one pass): rows that no sequence has are 0, or as they were in a given out."""
    q, k, v, table = _random("prefill", seqs, n_q, n_kv, dtype)
    q = torch.cat([q, torch.randn(rows - q.shape[0], q.shape[1], device=DEV).to(torch.bfloat16)])
    mine = torch.zeros(rows, dtype=torch.bool)
    for q0, ql, n in seqs:
        mine[q0:q0 + ql] |= n >= ql
    want, size = _reference("prefill", q, k, v, table, seqs, 1900, 5)
    fresh = _prefill(q, k, v, table, seqs, n_q, 1900, 5)
    _near(fresh, want, size)
    assert not fresh[~mine].any()
    given = torch.full_like(fresh, 3.0)
    _prefill(q, k, v, table, seqs, n_q, 1900, 5, out=given)
    assert torch.equal(given[mine], fresh[mine]) and (given[~mine] == 3).all()


def test_rows_of_seq_info_that_are_no_sequences():
    """Queries that do not lie in q, a context shorter than the queries, negative numbers: skipped, their rows are nobody's."""
    good = (4, 6, 30)
    for bad in ((-1, 3, 10), (20, 5, 9), (0, 40, 50), (0, 3, 2), (0, -2, 5), (0, 3, -3), (2 ** 31 - 1, 3, 9), (0, 2 ** 31 - 1, 2 ** 31 - 1)):
        q, k, v, table = make("prefill", [good, (10, 2, 5)], 4, 2, 9, 2, spare=10)
        info = torch.tensor([good, bad], dtype=torch.int32, device=DEV)
        a = [x.to(DEV) for x in (q, k, v, table)]
        got = llm.paged_attn_prefill_window(*a, info, SCALE, 4, 9, 2)
        want = llm.paged_attn_prefill_window(a[0], a[1], a[2], a[3][:1].contiguous(), info[:1].contiguous(), SCALE, 4, 9, 2)
        assert torch.equal(got, want) and got[4:10].any() and not got[:4].any() and not got[10:].any()
        cpu = llm.paged_attn_prefill_window(q.float(), k.float(), v.float(), table, info.cpu(), SCALE, 4, 9, 2)
        assert torch.equal(cpu.any(1), got.cpu().any(1))


def test_refusals_on_the_gpu():
    q, k, v, table = (x.to(DEV) for x in make("decode", [20, 3], 4, 2, 8, 0))
    lens = torch.tensor([20, 3], dtype=torch.int32, device=DEV)
    for bad in (dict(q=q.float()), dict(k=k.float(), v=v.float()), dict(lens=lens.long()), dict(lens=lens.cpu()), dict(table=table.long()), dict(k=k.cpu(), v=v.cpu()),
                dict(table=table.t().contiguous().t())):
        a = {**dict(q=q, k=k, v=v, table=table, lens=lens), **bad}
        with pytest.raises(KlmOpsError):
            llm.paged_attn_decode_window(a["q"], a["k"], a["v"], a["table"], a["lens"], SCALE, 4, 8)
    small = llm.DecodeWorkspace(1, 4, 4, DEV)
    with pytest.raises(KlmOpsError):
        llm.paged_attn_decode_window(q, k, v, table, lens, SCALE, 4, 8, num_splits=4, workspace=small)
    empty = llm.paged_attn_decode_window(q[:0], k, v, table[:0], lens[:0], SCALE, 4, 8)
    assert empty.shape == (0, 512)
    assert llm.paged_attn_prefill_window(q[:0], k, v, table[:0], torch.zeros(0, 3, dtype=torch.int32, device=DEV), SCALE, 4, 8).shape == (0, 512)


def _replays(call, inputs, changes, rounds=4):
    """Captures call(), then changes its inputs and replays, with eager work in between: every replay against the eager call."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = call()
    for i in range(rounds):
        changes(i)
        g.replay()
        got = [x.clone() for x in captured]
        want = call()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)), f"replay {i}"


def test_captured_attention():
    seqs = [700, 33, 1200]
    q, k, v, table = _random("decode", seqs, 16, 4, torch.bfloat16)
    q, lens = q.contiguous(), torch.tensor(seqs, dtype=torch.int32, device=DEV)

    def change(i):
        q.copy_(torch.randn_like(q))
        lens.copy_(torch.tensor([[700, 33, 1200], [1, 0, 64], [650, 2, 1199], [16, 17, 18]][i], dtype=torch.int32))

    _replays(lambda: [llm.paged_attn_decode_window(q, k, v, table, lens, SCALE, 16, 300, 4, num_splits=5)], None, change)
    seqs = [(0, 100, 100), (100, 60, 300)]
    q2, k2, v2, table2 = _random("prefill", seqs, 16, 4, torch.bfloat16)
    q2, info = q2.contiguous(), torch.tensor(seqs, dtype=torch.int32, device=DEV)

    def change2(i):
        q2.copy_(torch.randn_like(q2))
        info.copy_(torch.tensor([[[0, 100, 100], [100, 60, 300]], [[0, 7, 50], [7, 100, 100]], [[0, 0, 0], [0, 160, 200]], [[150, 10, 11], [0, 50, 99]]][i], dtype=torch.int32))

    table2[0] = table2[1]                                               # every length up to 300 has its pages in both rows
    _replays(lambda: [llm.paged_attn_prefill_window(q2, k2, v2, table2, info, SCALE, 16, 70, 4)], None, change2)


def test_a_workspace_of_fewer_splits():
    """The choice of splits keeps within the workspace; a number that is asked for and does not fit is refused."""
    seqs = [900, 31, 0]
    q, k, v, table = make("decode", seqs, 4, 1, 600, 4)
    want, size = by_definition("decode", q, k, v, table, seqs, 4, 600, 4)
    for most in (1, 2, 3):
        ws = llm.DecodeWorkspace(4, 4, most, DEV)
        _near(_decode(q, k, v, table, seqs, 4, 600, 4, workspace=ws), want, size)
        with pytest.raises(KlmOpsError):
            _decode(q, k, v, table, seqs, 4, 600, 4, workspace=ws, num_splits=most + 1)


def test_two_streams_at_once():
    """Two calls in flight with the scratch of their own."""
    seqs = [4000] * 3
    a, b = _random("decode", seqs, 32, 8, torch.bfloat16, 1), _random("decode", seqs, 32, 8, torch.bfloat16, 2)
    lens = torch.tensor(seqs, dtype=torch.int32, device=DEV)
    call = lambda x: llm.paged_attn_decode_window(*x, lens, SCALE, 32, 3000, 4)  # noqa: E731
    want = call(a), call(b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(s1):
            x = call(a)
        with torch.cuda.stream(s2):
            y = call(b)
        torch.cuda.synchronize()
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_an_offset_past_32_bits():
    """Pages whose elements lie beyond 2^31 from the cache's start."""
    n_kv, nb = 8, 140000                                                # 140000 * 8 * 2048 elements = 2.29e9
    k = torch.zeros(nb, n_kv, 16, 128, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros(nb, n_kv, 128, 16, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    pages = [nb - 1, 139000, 0, 70000]
    for b in pages:
        k[b].normal_(generator=g)
        v[b].normal_(generator=g)
    table = torch.tensor([pages], dtype=torch.int32, device=DEV)
    near = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    q = torch.randn(1, 32 * 128, device=DEV, generator=g).to(torch.bfloat16)
    lens = torch.tensor([60], dtype=torch.int32, device=DEV)
    a = llm.paged_attn_decode_window(q, k, v, table, lens, SCALE, 32, 50, 3)
    assert torch.equal(a, llm.paged_attn_decode_window(q, k[pages], v[pages], near, lens, SCALE, 32, 50, 3)) and a.any()
    info = torch.tensor([[0, 1, 60]], dtype=torch.int32, device=DEV)
    a = llm.paged_attn_prefill_window(q, k, v, table, info, SCALE, 32, 50, 3)
    assert torch.equal(a, llm.paged_attn_prefill_window(q, k[pages], v[pages], near, info, SCALE, 32, 50, 3)) and a.any()
    llm.copy_pages(k, v, [(139000, nb - 2), (nb - 1, 5)])
    assert torch.equal(k[[nb - 2, 5]], k[[139000, nb - 1]]) and torch.equal(v[[nb - 2, 5]], v[[139000, nb - 1]])


# ---------------------------------------------------------------------------------------------------------------- pages
@pytest.mark.parametrize("layers,nb,n_kv,n,dtype", [(1, 4, 1, 1, torch.bfloat16), (3, 700, 2, 300, torch.bfloat16), (2, 40, 8, 13, torch.float8_e4m3fn),
                                                    (5, 33, 3, 11, torch.bfloat16), (1, 1200, 1, 599, torch.float8_e4m3fn)])
def test_copy_pages(layers, nb, n_kv, n, dtype):
    g = torch.Generator(device=DEV).manual_seed(1)
    k = torch.randint(0, 256, (layers, nb, n_kv, 16, 128 * (2 if dtype == torch.bfloat16 else 1)), generator=g, device=DEV, dtype=torch.uint8).view(dtype)
    v = torch.randint(0, 256, (layers, nb, n_kv, 128, 16 * (2 if dtype == torch.bfloat16 else 1)), generator=g, device=DEV, dtype=torch.uint8).view(dtype)
    order = torch.randperm(nb, generator=g, device=DEV).tolist()
    pairs = [(order[i % max(1, nb // 2)] if i % 7 != 3 else -1, order[nb // 2 + i]) for i in range(n)]
    wk, wv = k.clone(), v.clone()
    ref.copy_pages(wk.view(torch.uint8), wv.view(torch.uint8), pairs, k.view(torch.uint8), v.view(torch.uint8))
    k2, v2 = torch.zeros_like(k[:, :n]), torch.zeros_like(v[:, :n])
    llm.copy_pages(k2, v2, [(s, i) for i, (s, _) in enumerate(pairs)], k_src=k, v_src=v)
    llm.copy_pages(k, v, pairs)
    assert torch.equal(k.view(torch.uint8), wk.view(torch.uint8)) and torch.equal(v.view(torch.uint8), wv.view(torch.uint8))
    to = [d for _, d in pairs]
    assert torch.equal(k2.view(torch.uint8), k[:, to].view(torch.uint8) if dtype == torch.bfloat16 else k.view(torch.uint8)[:, to])
    assert torch.equal(v2.view(torch.uint8), v.view(torch.uint8)[:, to])
    if layers > 1:
        want = k.view(torch.uint8).clone()
        want[1, to[0]] = want[1, order[0]]
        llm.copy_pages(k[1], v[1], [(order[0], to[0])])
        assert torch.equal(k.view(torch.uint8), want)


def test_copy_pages_refuses_on_the_gpu_too():
    k = torch.zeros(2, 4, 1, 16, 128, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros(2, 4, 1, 128, 16, dtype=torch.bfloat16, device=DEV)
    for pairs in ([(0, 4)], [(4, 0)], [(0, 1), (1, 2)], [(0, 1), (2, 1)]):
        with pytest.raises(KlmOpsError):
            llm.copy_pages(k, v, pairs)
    with pytest.raises(KlmOpsError):
        llm.copy_pages(k.float(), v.float(), [(0, 1)])
    with pytest.raises(KlmOpsError):
        llm.copy_pages(k, v, [(0, 1)], k_src=k.cpu(), v_src=v.cpu())


def test_captured_copy_of_pages():
    k = torch.randn(2, 300, 2, 16, 128, device=DEV).to(torch.bfloat16)
    v = torch.randn(2, 300, 2, 128, 16, device=DEV).to(torch.bfloat16)
    pairs = [(i, 150 + i) for i in range(150)] 
    g = torch.cuda.CUDAGraph()
    llm.copy_pages(k, v, pairs)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        llm.copy_pages(k, v, pairs)
    for _ in range(3):
        k.normal_()
        v.normal_()
        g.replay()
        assert torch.equal(k[:, 150:], k[:, :150]) and torch.equal(v[:, 150:], v[:, :150])


# ------------------------------------------------------------------------------------------------------- rules on logits
def _rules(R, n, total, seed=0, bias=6, masks=3, rows=None):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, n + 3, (R,), generator=g, dtype=torch.int32)
    r = dict(history=torch.randint(-2, total + 3, (R, n), generator=g, dtype=torch.int32), prompt_lens=(lens.float() * torch.rand(R, generator=g)).int(), lens=lens,
             repetition=torch.rand(R, generator=g) + 0.5, frequency=torch.randn(R, generator=g), presence=torch.randn(R, generator=g))
    if bias:
        r.update(bias_ids=torch.randint(-1, min(total, 2 * bias), (R, bias), generator=g, dtype=torch.int32), bias_values=torch.randn(R, bias, generator=g))
    if masks:
        r.update(mask=torch.randint(-2 ** 31, 2 ** 31 - 1, (masks, -(-total // 32)), generator=g, dtype=torch.int32),
                 mask_rows=torch.randint(-1, masks + 1, (R,), generator=g, dtype=torch.int32))
        r["mask"][0] = 0                                                # a grammar that allows nothing
    if rows is not None:
        r.update(rows=torch.tensor(rows, dtype=torch.int32))
    return llm.LogitRules(**r)


def _gpu(rules):
    return llm.LogitRules(**{k: None if x is None else x.to(DEV) for k, x in rules.__dict__.items()})


@pytest.mark.parametrize("B,V,first,total,n,bias,masks", [(1, 1, 0, 1, 3, 1, 0), (3, 37, 0, 37, 5, 2, 2), (2, 4095, 0, 4095, 50, 0, 1), (2, 4096, 4096, 8192, 600, 9, 0),
                                                          (5, 4097, 31, 4200, 64, 300, 3), (9, 32000, 32000, 64000, 2000, 20, 4), (2, 50001, 0, 50001, 9000, 6, 3),
                                                          (4, 128256, 0, 128256, 1, 0, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_choose_tokens(B, V, first, total, n, bias, masks, dtype):
    """Every step is one fp32 operation: the kernel gives the reference's bits."""
    rules = _rules(B, n, total, seed=V, bias=bias, masks=masks)
    x = (torch.randn(B, V, generator=torch.Generator().manual_seed(B)) * 3).to(dtype)
    wy, wids, wbest = ref.choose_tokens(x, rules, first)
    out = torch.full((B, V), 5.0, device=DEV)
    ids, best = llm.choose_tokens(x.to(DEV), _gpu(rules), first_token=first, out=out)
    assert torch.equal(out.cpu(), wy) and torch.equal(ids.cpu(), wids) and torch.equal(best.cpu(), wbest)
    ids2, best2 = llm.choose_tokens(x.to(DEV), _gpu(rules), first_token=first)
    assert torch.equal(ids, ids2) and torch.equal(best, best2)
    plain, value = llm.choose_tokens(x.to(DEV), first_token=first)
    assert torch.equal(plain.cpu(), x.float().argmax(1) + first) and torch.equal(value.cpu(), x.float().amax(1))


@pytest.mark.parametrize("pad", [0, 1, 8])
def test_rows_strides_and_places(pad):
    """Rules by row, a row without any, sets that are not there; rows of logits further apart; in place."""
    V, total, rows = 5000, 5000, [2, -1, 0, 3, 9, 2]
    rules = _rules(4, 40, total, rows=rows)
    wide = torch.randn(6, V + pad, generator=torch.Generator().manual_seed(1))
    for dtype in (torch.float32, torch.bfloat16):
        w = wide.to(dtype)
        wy, wids, wbest = ref.choose_tokens(w[:, :V], rules, 0)
        out = torch.empty(6, V, device=DEV)
        ids, best = llm.choose_tokens(w.to(DEV)[:, :V], _gpu(rules), out=out)
        assert torch.equal(out.cpu(), wy) and torch.equal(ids.cpu(), wids) and torch.equal(best.cpu(), wbest)
    if not pad:
        y = wide.to(DEV)
        ids2, _ = llm.choose_tokens(y, _gpu(rules), out=y)
        assert torch.equal(y.cpu(), ref.choose_tokens(wide, rules, 0)[0]) and torch.equal(ids2.cpu(), ref.choose_tokens(wide, rules, 0)[1])


def test_ties_nan_infinities_and_zeros():
    V = 9000
    x = torch.full((7, V), -1.0)
    x[0, 4095], x[0, 4096], x[0, 8999] = 2.0, 2.0, 2.0                   # equals across slices: the lowest id
    x[1, :] = -0.0
    x[1, 7000] = 0.0                                                     # zeros are equal
    x[2, 5000], x[2, 100], x[2, 8000] = float("nan"), float("inf"), float("nan")
    x[3, :] = float("-inf")
    x[4, 8500], x[4, 20] = float("inf"), 3e38
    x[5, 3] = -1e-45
    x[5, :3] = -2e-45
    x[5, 4:] = -2e-45
    ids, best = llm.choose_tokens(x.to(DEV))
    # row 5: -1e-45 and -2e-45 are the same fp32 number, the smallest subnormal (1.4e-45): equals, the lowest id
    assert ids.tolist() == [4095, 0, 5000, 0, 8500, 0, 0] and math.isnan(float(best[2]))
    assert ids.tolist() == x.argmax(1).tolist()
    rules = _rules(7, 1, V, masks=1)
    rules.lens.zero_()
    rules.bias_ids.fill_(-1)
    rules.mask.fill_(-1)
    rules.mask_rows.zero_()
    rules.mask[0, 5000 // 32] &= ~(1 << (5000 % 32))                     # the NaN that won is not allowed
    out = torch.empty(7, V, device=DEV)
    ids, best = llm.choose_tokens(x.to(DEV), _gpu(rules), out=out)
    assert ids.tolist() == [4095, 0, 8000, 0, 8500, 0, 0] and float(out[2, 5000]) == -math.inf


def test_captured_choice_and_the_same_bits_again():
    rules = _gpu(_rules(3, 200, 9000, masks=2))
    x = torch.randn(3, 9000, device=DEV).to(torch.bfloat16)
    out = torch.empty(3, 9000, device=DEV)

    def change(i):
        x.copy_(torch.randn(3, 9000, device=DEV))
        rules.history.copy_(torch.randint(0, 9000, (3, 200), device=DEV, dtype=torch.int32))
        rules.lens.fill_(50 * i)

    _replays(lambda: [*llm.choose_tokens(x, rules, out=out), out], None, change)


# ----------------------------------------------------------------------------------------------------------- all together
def test_choices_of_one_prompt():
    """A prompt, forked into three sequences that share its full pages and copy the last, partly filled one; each goes on for
    some tokens through a window, gives pages back behind it and follows rules of its own."""
    n_q, n_kv, window, sinks, prompt, steps = 8, 2, 40, 4, 75, 30
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(prompt + 3 * steps, (n_q + 2 * n_kv) * 128, generator=g).to(torch.bfloat16)
    head = torch.randn(500, n_q * 128, generator=g).to(torch.bfloat16)
    nb, D = 30, 128
    k = torch.full((1, nb, n_kv, 16, D), float("nan"), dtype=torch.bfloat16, device=DEV)
    v = torch.full((1, nb, n_kv, D, 16), float("nan"), dtype=torch.bfloat16, device=DEV)

    def put(row, page, at):
        x = qkv[row].view(-1, D).to(DEV)
        k[0, page, :, at], v[0, page, :, :, at] = x[n_q:n_q + n_kv], x[n_q + n_kv:]

    pages = [list(range(5))]
    for t in range(prompt):
        put(t, pages[0][t // 16], t % 16)
    out = llm.paged_attn_prefill_window(qkv[:prompt, : n_q * D].to(DEV), k[0], v[0], torch.tensor(pages, dtype=torch.int32, device=DEV),
                                        torch.tensor([[0, prompt, prompt]], dtype=torch.int32, device=DEV), SCALE, n_q, window, sinks)
    pages += [pages[0][:4] + [5], pages[0][:4] + [6]]                   # the fork: four shared pages, the fifth copied
    llm.copy_pages(k, v, [(4, 5), (4, 6)])
    free = list(range(7, nb))
    table = torch.full((3, 8), -1, dtype=torch.int32)
    seqs = [list(range(prompt)) for _ in range(3)]
    rules = _rules(3, 64, 500, bias=4, masks=3)
    rules.mask[:] |= 0x0f0f0f0f
    rules.lens.fill_(10)
    rules.prompt_lens.fill_(4)
    for i in range(steps):
        n = prompt + i
        for b in range(3):
            if n // 16 == len(pages[b]):
                pages[b].append(free.pop())
            put(prompt + 3 * i + b, pages[b][n // 16], n % 16)
            seqs[b].append(prompt + 3 * i + b)
            table[b] = -1
            for p, page in enumerate(pages[b]):
                if (p + 1) * 16 > n + 1 - window or p * 16 < sinks:       # the others are given back
                    table[b, p] = page
        rows = [prompt + 3 * i + b for b in range(3)]
        o = llm.paged_attn_decode_window(qkv[rows, : n_q * D].to(DEV), k[0], v[0], table.to(DEV), torch.full((3,), n + 1, dtype=torch.int32, device=DEV),
                                         SCALE, n_q, window, sinks)
        x = qkv.view(-1, n_q + 2 * n_kv, D).double()
        for b in range(3):
            keys = [j for j in range(n + 1) if j > n - window or j < sinks]
            kk, vv = (x[[seqs[b][j] for j in keys], at:at + n_kv].transpose(0, 1) for at in (n_q, n_q + n_kv))
            p = torch.softmax(torch.matmul(x[rows[b], :n_q].view(n_kv, -1, D), kk.transpose(1, 2)) * SCALE, -1)
            _near(o[b:b + 1], torch.matmul(p, vv).reshape(1, -1), torch.matmul(p, vv.abs()).reshape(1, -1))
        logits = (o.float() @ head.to(DEV).float().t())
        ids, best = llm.choose_tokens(logits, _gpu(rules))
        _, wids, wbest = ref.choose_tokens(logits.cpu(), rules, 0)
        assert torch.equal(ids.cpu(), wids) and torch.equal(best.cpu(), wbest)
        rules.history[torch.arange(3), rules.lens.long()] = ids.int().cpu()
        rules.lens += 1
    assert out.shape[0] == prompt and bool(torch.isfinite(out).all())
