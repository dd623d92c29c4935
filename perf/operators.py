"""Operators of the serving engine, as one timed pass each: attention with a sliding window and sinks over the paged KV cache
(prompt chunks and single tokens), copies of cache pages, and rules on logits with the greedy choice of a token.

``own`` False: `run` computes an operator from elementary torch operations in 32 bits. True: the package's kernels, by the calls
that the engine makes. `exact` is the definition in 64 bits, written apart from both."""
import math
import random

import torch

own = False

HD, BLK = 128, 16        # head dimension and tokens per page of the engine's cache
DEV = "cuda"


# --------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one running sequence of an 8B-class model, past its window: what a user alone on the machine waits for
        dict(name="decode_one", op="decode", B=1, n_q=32, n_kv=8, ctx=1500, window=1024, sinks=4, fp8=False, lens=1),
        # a mixed batch: new, old and finished (length 0) sequences, an odd window that ends inside pages
        dict(name="decode_ragged", op="decode", B=33, n_q=32, n_kv=8, ctx=8191, window=2001, sinks=5, fp8=False, lens=2),
        # a full serving batch of a 70B-class model on an 8-bit cache: bytes of the cache are what counts
        dict(name="decode_fp8", op="decode", B=96, n_q=64, n_kv=8, ctx=8192, window=4096, sinks=64, fp8=True, lens=3),
        # short prompts of odd lengths in one launch, padded rows behind them
        dict(name="prefill_ragged", op="prefill", S=13, q=400, past=0, pad=7, n_q=32, n_kv=8, window=129, sinks=3, fp8=False, lens=4),
        # one long prompt
        dict(name="prefill_long", op="prefill", S=1, q=8192, past=0, pad=0, n_q=32, n_kv=8, window=4096, sinks=4, fp8=False, lens=5),
        # chunks of prompts whose beginning is cached already, 8-bit cache
        dict(name="prefill_chunks_fp8", op="prefill", S=4, q=1000, past=5000, pad=0, n_q=64, n_kv=8, window=2048, sinks=64, fp8=True, lens=6),
        # four more choices of one prompt: the last, partly filled page is copied in every layer
        dict(name="pages_fork", op="pages", L=32, nb=256, n_kv=8, n=4, fp8=False, two=False),
        # a third of the pages moves to the front of the pool, so that the rest can be given back
        dict(name="pages_compact", op="pages", L=32, nb=2048, n_kv=8, n=683, fp8=False, two=False),
        # pages of an 8-bit cache move into another, smaller cache
        dict(name="pages_resize_fp8", op="pages", L=80, nb=300, n_kv=8, n=250, fp8=True, two=True),
        # one sequence with penalties: the step between two tokens
        dict(name="logits_one", op="logits", B=1, V=128256, fp32=False, hist=1000, bias=0, masks=0, whole=False, first=0, lens=7),
        # a batch, every row with rules of its own, grammars among them
        dict(name="logits_batch", op="logits", B=96, V=128256, fp32=False, hist=4096, bias=50, masks=40, whole=False, first=0, lens=8),
        # a whole batch's processed logits, for a program that goes on with them; one rank's slice of the vocabulary, 32-bit logits
        dict(name="logits_whole", op="logits", B=256, V=64128, fp32=True, hist=2000, bias=8, masks=3, whole=True, first=64128, lens=9),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("decode", "prefill", "pages", "logits"))
    lens = rng.randrange(1 << 20)
    if op == "decode":
        n_q, n_kv = rng.choice(((32, 8), (64, 8), (16, 4), (4, 2), (16, 1), (8, 8), (24, 8), (28, 4)))
        return dict(op=op, B=_log(rng, 1, 96), n_q=n_q, n_kv=n_kv, ctx=_log(rng, 1, 8192), window=_log(rng, 1, 4096), sinks=rng.choice((0, 1, 4, 16, 64, 100)),
                    fp8=rng.random() < 0.4, lens=lens)
    if op == "prefill":
        n_q, n_kv = rng.choice(((32, 8), (64, 8), (16, 4), (4, 2), (16, 1), (8, 8), (24, 8), (28, 4)))
        s = _log(rng, 1, 16)
        return dict(op=op, S=s, q=_log(rng, 1, 2048 // s), past=rng.choice((0, 0, _log(rng, 1, 4000))), pad=rng.choice((0, 0, 5)), n_q=n_q, n_kv=n_kv,
                    window=_log(rng, 1, 4096), sinks=rng.choice((0, 1, 4, 16, 64, 100)), fp8=rng.random() < 0.4, lens=lens)
    if op == "pages":
        layers, two = rng.choice((1, 4, 32, 80)), rng.random() < 0.3
        nb = _log(rng, 4, 1500 * 32 // max(32, layers))
        return dict(op=op, L=layers, nb=nb, n_kv=rng.choice((1, 2, 4, 8)), n=_log(rng, 1, max(1, nb // 3)), fp8=rng.random() < 0.4, two=two)
    vocab = rng.choice((128256, 32768, 32000, 64128, 512, 16033, 50001))
    return dict(op=op, B=_log(rng, 1, 128), V=vocab, fp32=rng.random() < 0.4, hist=_log(rng, 1, 8192), bias=rng.choice((0, 1, 20, 300)), masks=rng.choice((0, 0, 1, 9)),
                whole=rng.random() < 0.4, first=rng.choice((0, 0, vocab)), lens=lens)


# --------------------------------------------------------------------------------------------- lengths, from the case alone
def _decode_lens(c):
    r = random.Random(c["lens"])
    lens = [c["ctx"]] + [int(round(c["ctx"] ** r.uniform(0.6, 1.0))) if r.random() < 0.5 else r.randint(0, c["ctx"]) for _ in range(c["B"] - 1)]
    if c["B"] >= 8:
        lens[3], lens[5] = 0, 1
    return lens


def _prefill_lens(c):
    """[(query tokens, context length)] of the sequences."""
    r = random.Random(c["lens"])
    qs = [c["q"]] + [r.randint(1, c["q"]) for _ in range(c["S"] - 1)]
    return [(q, q + (r.randint(c["past"] // 2, c["past"]) if c["past"] else 0)) for q in qs]


def _visible(pos, window, sinks):
    """Keys that a query at position `pos` sees."""
    return min(pos + 1, window) + min(sinks, max(0, pos + 1 - window))


def _logit_lens(c):
    r = random.Random(c["lens"])
    lens = [c["hist"]] + [r.randint(0, c["hist"]) for _ in range(c["B"] - 1)]
    return lens, [r.randint(0, n) for n in lens]


def work(case):
    c = case
    if c["op"] == "decode":
        seen = sum(_visible(n - 1, c["window"], c["sinks"]) for n in _decode_lens(c) if n)
        kv = seen * c["n_kv"] * 2 * HD * (1 if c["fp8"] else 2)
        return {"bytes": kv + 2 * 2 * c["B"] * c["n_q"] * HD, "flops": 4 * HD * c["n_q"] * seen}
    if c["op"] == "prefill":
        seen = keys = rows = 0
        for q, n in _prefill_lens(c):
            seen += sum(_visible(p, c["window"], c["sinks"]) for p in range(n - q, n))
            lo = max(0, n - q - c["window"] + 1)
            keys += n - lo + min(c["sinks"], lo)
            rows += q
        return {"bytes": keys * c["n_kv"] * 2 * HD * (1 if c["fp8"] else 2) + 2 * 2 * rows * c["n_q"] * HD, "flops": 4 * HD * c["n_q"] * seen}
    if c["op"] == "pages":
        return {"bytes": 2 * c["n"] * c["L"] * 2 * c["n_kv"] * BLK * HD * (1 if c["fp8"] else 2), "flops": 0}
    lens, _ = _logit_lens(c)
    n = c["B"] * c["V"]
    read = n * (4 if c["fp32"] else 2) + 4 * sum(lens) + 8 * c["B"] * c["bias"] + min(c["masks"], c["B"]) * c["V"] // 8
    return {"bytes": read + (4 * n if c["whole"] else 0) + 12 * c["B"], "flops": 2 * n}


# ------------------------------------------------------------------------------------------------------------- the inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _cache(nb, n_kv, fp8, g, layers=None):
    lead = (nb, n_kv) if layers is None else (layers, nb, n_kv)
    k = torch.empty((*lead, BLK, HD), dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    v = torch.empty((*lead, HD, BLK), dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    return (k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn)) if fp8 else (k, v)


def _tables(spans, seed):
    """spans: (context length, first position that a window reaches, sinks) of each sequence. A page table as the engine leaves
    it: pages behind the window are given back (-1), those of the sinks stay. -> table on the GPU, pages of the pool."""
    width = max(1, max(-(-n // BLK) for n, _, _ in spans))
    live = []
    for s, (n, lo, sinks) in enumerate(spans):
        live += [(s, p) for p in range(-(-n // BLK)) if (p + 1) * BLK > lo or p * BLK < sinks]
    order = list(range(len(live) + 3))
    random.Random(seed).shuffle(order)
    t = torch.full((len(spans), width), -1, dtype=torch.int32)
    if live:
        at = torch.tensor(live)
        t[at[:, 0], at[:, 1]] = torch.tensor(order[:len(live)], dtype=torch.int32)
    return t.to(DEV), len(order)


def prepare(case, seed):
    c, g = case, _generator(seed)
    st = dict(case=c)
    if c["op"] in ("decode", "prefill"):
        if c["op"] == "decode":
            lens = _decode_lens(c)
            rows = c["B"]
            spans = [(n, max(0, n - c["window"]), c["sinks"]) for n in lens]
            st["ctx_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        else:
            lens = _prefill_lens(c)
            rows = sum(q for q, _ in lens) + c["pad"]
            spans = [(n, max(0, n - q - c["window"] + 1), c["sinks"]) for q, n in lens]
            at, info = 0, []
            for q, n in lens:
                info.append((at, q, n))
                at += q
            st["seq_info"] = torch.tensor(info, dtype=torch.int32, device=DEV)
        st["tables"], nb = _tables(spans, seed)
        st["k"], st["v"] = _cache(nb, c["n_kv"], c["fp8"], g)
        qkv = torch.empty((rows, (c["n_q"] + 2 * c["n_kv"]) * HD), dtype=torch.bfloat16, device=DEV).normal_(generator=g)
        st["q"] = qkv[:, :c["n_q"] * HD]          # the projections' fused output, as the model passes it
        return st
    if c["op"] == "pages":
        st["k"], st["v"] = _cache(c["nb"], c["n_kv"], c["fp8"], g, c["L"])
        pages = list(range(c["nb"]))
        random.Random(seed).shuffle(pages)
        if c["two"]:
            st["k2"], st["v2"] = (torch.zeros_like(x[:, :c["n"] + 1]) for x in (st["k"], st["v"]))
            to = list(range(c["n"] + 1))
            random.Random(seed + 1).shuffle(to)
            st["pairs"] = list(zip(pages[:c["n"]], to))
        else:
            half = max(1, min(c["n"], c["nb"] // 2))
            to = pages[half:half + c["n"]]
            st["pairs"] = [(pages[i % half], d) for i, d in enumerate(to)]
        return st
    lens, prompts = _logit_lens(c)
    B, V, first = c["B"], c["V"], c["first"]
    x = torch.empty((B, V), dtype=torch.float32, device=DEV).normal_(0.0, 3.0, generator=g)
    st["logits"] = x if c["fp32"] else x.to(torch.bfloat16)
    total = first + 2 * V if first else V        # a slice out of the middle of a sharded vocabulary, or all of it
    r = torch.rand((B, c["hist"]), device=DEV, generator=g)
    st["history"] = (r ** 3 * total).to(torch.int32).clamp_(max=total - 1)       # low ids come again and again
    i32 = dict(dtype=torch.int32, device=DEV)
    st["lens"], st["prompt_lens"] = torch.tensor(lens, **i32), torch.tensor(prompts, **i32)
    for name, lo, hi in (("repetition", 0.8, 1.6), ("frequency", -0.3, 0.6), ("presence", -0.2, 0.9)):
        st[name] = torch.rand(B, device=DEV, generator=g) * (hi - lo) + lo
    st["bias_ids"] = st["bias_values"] = st["mask"] = st["mask_rows"] = None
    if c["bias"]:
        st["bias_ids"] = torch.randint(-1, total, (B, c["bias"]), generator=g, **i32)
        st["bias_values"] = torch.randn((B, c["bias"]), device=DEV, generator=g) * 2
    if c["masks"]:
        words = -(-total // 32)
        st["mask"] = torch.randint(-2 ** 31, 2 ** 31 - 1, (c["masks"], words), generator=g, **i32)
        st["mask"][c["masks"] - 1] = 0           # a grammar that allows nothing
        at = torch.randint(-1, c["masks"], (B,), generator=g, **i32)
        st["mask_rows"] = torch.where(at == c["masks"] - 1, at - (torch.arange(B, device=DEV, dtype=torch.int32) % 4 != 0).int(), at)
    return st


# --------------------------------------------------------------------------------------------------------- the plain forms
def _softmax_times(s, see, v):
    """softmax of the visible scores, times v; a row that sees nothing gives 0."""
    s = s.masked_fill(~see, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    z = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(z == 0, 1.0, z)


def _plain_decode(st):
    c, tab = st["case"], st["tables"]
    B, W, S, n_kv = c["B"], c["window"], c["sinks"], c["n_kv"]
    n = st["ctx_lens"].long()[:, None]
    reach = min(W, tab.shape[1] * BLK)
    pos = torch.cat([torch.arange(S, device=DEV).expand(B, S), n - reach + torch.arange(reach, device=DEV)], 1)      # sinks, then the window
    in_window = torch.arange(S + reach, device=DEV) >= S
    see = (pos >= 0) & (pos < n) & torch.where(in_window, pos >= n - W, pos < n - W)
    page = torch.gather(tab.long(), 1, (pos // BLK).clamp(0, tab.shape[1] - 1))
    see &= (page >= 0) & (page < st["k"].shape[0])
    page, off = page.clamp(0, st["k"].shape[0] - 1), pos % BLK
    bytes_k, bytes_v = (x.view(torch.uint8) if c["fp8"] else x for x in (st["k"], st["v"]))
    k, v = bytes_k[page, :, off], bytes_v[page, :, :, off]                            # [B, keys, n_kv, 128]
    if c["fp8"]:
        k, v = k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)
    k, v = k.float().transpose(1, 2), v.float().transpose(1, 2)
    q = st["q"].float().reshape(B, n_kv, c["n_q"] // n_kv, HD)
    s = torch.matmul(q, k.transpose(2, 3)) * (1 / math.sqrt(HD))
    return _softmax_times(s, see[:, None, None], v).reshape(B, -1).to(torch.bfloat16)


def _plain_prefill(st):
    c, tab, info = st["case"], st["tables"], st["seq_info"].long()
    S, n_kv, G = c["S"], c["n_kv"], c["n_q"] // c["n_kv"]
    rows, widest, keys = st["q"].shape[0], c["q"], tab.shape[1] * BLK
    ok = (tab >= 0) & (tab < st["k"].shape[0])
    page = tab.long().clamp(0, st["k"].shape[0] - 1)
    bytes_k, bytes_v = (x.view(torch.uint8) if c["fp8"] else x for x in (st["k"], st["v"]))
    k, v = bytes_k[page], bytes_v[page]                                                # [S, pages, n_kv, 16, 128], [.., 128, 16]
    if c["fp8"]:
        k, v = k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)
    k = k.float().permute(0, 2, 1, 3, 4).reshape(S, n_kv, keys, HD)
    v = v.float().permute(0, 2, 1, 4, 3).reshape(S, n_kv, keys, HD)
    at = torch.arange(widest, device=DEV)
    row = (info[:, :1] + at).clamp(max=rows - 1)                                       # [S, widest]; rows past a sequence's own are dropped below
    pos = (info[:, 2:] - info[:, 1:2] + at)[:, :, None]
    key = torch.arange(keys, device=DEV)
    see = (key <= pos) & ((key > pos - c["window"]) | (key < c["sinks"])) & ok.repeat_interleave(BLK, 1)[:, None]
    q = st["q"].float().reshape(rows, n_kv, G, HD)[row].permute(0, 2, 3, 1, 4).reshape(S, n_kv, G * widest, HD)
    s = torch.matmul(q, k.transpose(2, 3)) * (1 / math.sqrt(HD))
    o = _softmax_times(s.view(S, n_kv, G, widest, keys), see[:, None, None], v[:, :, None])
    o = o.permute(0, 3, 1, 2, 4).reshape(S, widest, -1).to(torch.bfloat16)
    out = torch.zeros((rows, c["n_q"] * HD), dtype=torch.bfloat16, device=DEV)
    mine = at < info[:, 1:2]
    out[row[mine]] = o[mine]
    return out


def _plain_pages(st):
    pairs = torch.tensor(st["pairs"], device=DEV)
    src, dst = pairs[:, 0], pairs[:, 1]
    k, v = (st["k2"], st["v2"]) if st["case"]["two"] else (st["k"], st["v"])
    for to, of in ((k, st["k"]), (v, st["v"])):
        to.view(torch.int64)[:, dst] = of.view(torch.int64)[:, src]          # whole words: the copy does not look at values
    return k, v


def _plain_logits(st):
    c = st["case"]
    B, V, first = c["B"], c["V"], c["first"]
    x = st["logits"].float()
    h = st["history"].long() - first
    at = torch.arange(c["hist"], device=DEV)
    here = (h >= 0) & (h < V)
    h = h.clamp(0, V - 1)
    live = here & (at < st["lens"][:, None])
    seen = torch.zeros((B, V), dtype=torch.int32, device=DEV).scatter_add_(1, h, live.int()) > 0
    count = torch.zeros((B, V), dtype=torch.int32, device=DEV).scatter_add_(1, h, (live & (at >= st["prompt_lens"][:, None])).int())
    r = st["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - st["frequency"][:, None] * count.float()
    x = torch.where(count > 0, x - st["presence"][:, None], x)
    if c["bias"]:
        b = st["bias_ids"].long() - first
        inside = (b >= 0) & (b < V) & (st["bias_ids"] >= 0)
        order = torch.where(inside, torch.arange(c["bias"], device=DEV) + 1, 0).expand(B, -1)      # a token twice: the later entry counts
        last = torch.zeros((B, V), dtype=torch.int64, device=DEV).scatter_reduce_(1, b.clamp(0, V - 1), order, "amax")
        x = torch.where(last > 0, x + torch.gather(st["bias_values"], 1, (last - 1).clamp(min=0)), x)
    allowed = torch.ones((B, V), dtype=torch.bool, device=DEV)
    if c["masks"]:
        token = torch.arange(first, first + V, device=DEV)
        words = st["mask"][st["mask_rows"].long().clamp(min=0)][:, token // 32]
        allowed = ((words >> (token % 32)) & 1).bool() | (st["mask_rows"] < 0)[:, None]
    x = torch.where(allowed, x, -math.inf)
    best = x.amax(1)
    token = torch.where(x == best[:, None], torch.arange(V, device=DEV), V).amin(1) + first
    ids = torch.where(allowed.any(1), token, -1)
    return (ids, best, x) if c["whole"] else (ids, best)


def _calls(st):
    """The calls that a user's program makes."""
    from k8s_llm_monitor_amd.ops import llm
    c = st["case"]
    if c["op"] == "decode":
        return llm.paged_attn_decode_window(st["q"], st["k"], st["v"], st["tables"], st["ctx_lens"], 1 / math.sqrt(HD), c["n_q"], c["window"], c["sinks"])
    if c["op"] == "prefill":
        return llm.paged_attn_prefill_window(st["q"], st["k"], st["v"], st["tables"], st["seq_info"], 1 / math.sqrt(HD), c["n_q"], c["window"], c["sinks"])
    if c["op"] == "pages":
        if c["two"]:
            llm.copy_pages(st["k2"], st["v2"], st["pairs"], k_src=st["k"], v_src=st["v"])
            return st["k2"], st["v2"]
        llm.copy_pages(st["k"], st["v"], st["pairs"])
        return st["k"], st["v"]
    rules = llm.LogitRules(**{n: st[n] for n in ("history", "prompt_lens", "lens", "repetition", "frequency", "presence", "bias_ids", "bias_values", "mask", "mask_rows")})
    if c["whole"]:
        out = torch.empty((c["B"], c["V"]), dtype=torch.float32, device=DEV)
        return (*llm.choose_tokens(st["logits"], rules, first_token=c["first"], out=out), out)
    return llm.choose_tokens(st["logits"], rules, first_token=c["first"])


def run(state):
    if own:
        return _calls(state)
    return {"decode": _plain_decode, "prefill": _plain_prefill, "pages": _plain_pages, "logits": _plain_logits}[state["case"]["op"]](state)


# ----------------------------------------------------------------------------------------------- the definitions in 64 bits
def _sequence(st, s, n):
    """K and V of one sequence in 64 bits, [n_kv, n, 128], and which positions have a page."""
    ids = st["tables"][s, :-(-n // BLK)].tolist()
    k, v = (torch.cat([x[max(i, 0)] for i in ids], dim) for x, dim in ((st["k"].double(), 1), (st["v"].double(), 2)))
    there = torch.tensor([i >= 0 for i in ids for _ in range(BLK)], device=DEV)[:n]
    return k[:, :n], v[:, :, :n].transpose(1, 2), there


def _exact_attention(st):
    c = st["case"]
    G = c["n_q"] // c["n_kv"]
    out = torch.zeros((st["q"].shape[0], c["n_kv"], G, HD), dtype=torch.float64, device=DEV)
    if c["op"] == "decode":
        spans = [(b, 1, n) for b, n in enumerate(st["ctx_lens"].tolist())]
    else:
        spans = [tuple(x) for x in st["seq_info"].tolist()]
    q = st["q"].double().reshape(-1, c["n_kv"], G, HD)
    for s, (row, m, n) in enumerate(spans):
        if not n:
            continue
        k, v, there = _sequence(st, s, n)
        pos, key = torch.arange(n - m, n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
        hidden = (key > pos) | ((key <= pos - c["window"]) & (key >= c["sinks"])) | ~there[None]
        for h in range(c["n_kv"]):
            for e in range(G):
                w = torch.softmax((q[row:row + m, h, e] @ k[h].t() / math.sqrt(HD)).masked_fill(hidden, -math.inf), -1)
                out[row:row + m, h, e] = w @ v[h]
    return out.reshape(out.shape[0], -1)


def exact(case, seed):
    st, c = prepare(case, seed), case
    if c["op"] in ("decode", "prefill"):
        return _exact_attention(st)
    if c["op"] == "pages":
        k, v = (st["k2"], st["v2"]) if c["two"] else (st["k"], st["v"])
        for s, d in st["pairs"]:
            for to, of in ((k, st["k"]), (v, st["v"])):
                to[:, d].copy_(of[:, s])
        return k, v
    ids, best, whole = [], [], []
    B, V, first = c["B"], c["V"], c["first"]
    words = None if st["mask"] is None else st["mask"].cpu().numpy().view("uint32")
    for b in range(B):
        x = st["logits"][b].double()
        n, p = int(st["lens"][b]), int(st["prompt_lens"][b])
        tokens = [t for t in st["history"][b, :n].long().tolist()]
        seen = torch.tensor(sorted({t - first for t in tokens if first <= t < first + V}), dtype=torch.long, device=DEV)
        part = x[seen]
        r = float(st["repetition"][b])
        x[seen] = torch.where(part > 0, part / r, part * r)
        times = {}
        for t in tokens[p:]:
            if first <= t < first + V:
                times[t - first] = times.get(t - first, 0) + 1
        if times:
            at = torch.tensor(list(times), device=DEV)
            x[at] -= torch.tensor(list(times.values()), dtype=torch.float64, device=DEV) * float(st["frequency"][b]) + float(st["presence"][b])
        if c["bias"]:
            add = {t - first: w for t, w in zip(st["bias_ids"][b].tolist(), st["bias_values"][b].tolist()) if t >= 0 and first <= t < first + V}
            if add:
                x[torch.tensor(list(add), device=DEV)] += torch.tensor(list(add.values()), dtype=torch.float64, device=DEV)
        m = -1 if words is None else int(st["mask_rows"][b])
        none = False
        if m >= 0:
            bits = "".join(format(int(w), "032b")[::-1] for w in words[m])[first:first + V]
            banned = torch.tensor([ch == "0" for ch in bits], device=DEV)
            x[banned] = -math.inf
            none = bool(banned.all())
        best.append(x.max())
        ids.append(-1 if none else int(torch.argmax(x)) + first)
        whole.append(x)
    ids, best = torch.tensor(ids, device=DEV), torch.stack(best)
    return (ids, best, torch.stack(whole)) if c["whole"] else (ids, best)
