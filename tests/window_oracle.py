"""Shared by the tests of windowed attention: inputs, a definition written key by key, and what an error may be."""
import math

import torch

SCALE = 1.0 / math.sqrt(128)


def sees(pos, key, window, sinks):
    return key <= pos and (key > pos - window or key < sinks)


def spans(kind, seqs):
    """(row, position) of every query. decode: context lengths; prefill: (q_start, q_len, ctx_len)."""
    if kind == "decode":
        return [(b, b, n - 1) for b, n in enumerate(seqs) if n > 0]
    return [(s, q0 + i, n - q + i) for s, (q0, q, n) in enumerate(seqs) if q > 0 and n >= q for i in range(q)]


def visible_keys(kind, seqs, window, sinks):
    """Keys of each sequence that any of its queries sees."""
    live = {}
    for s, _, pos in spans(kind, seqs):
        live.setdefault(s, set()).update(k for k in range(pos + 1) if sees(pos, k, window, sinks))
    return live


def make(kind, seqs, n_q, n_kv, window, sinks, dtype=torch.bfloat16, seed=0, spare=3, poison=True, width=None):
    """q (a view of a fused activation), K / V caches and tables on the CPU. Every byte that no query sees is NaN, pages that
    no query sees are not in the tables."""
    g = torch.Generator().manual_seed(seed)
    ctx = [n if kind == "decode" else n[2] for n in seqs]
    live = visible_keys(kind, seqs, window, sinks)
    pages = sorted({(s, k // 16) for s, ks in live.items() for k in ks})
    nb = len(pages) + spare
    order = torch.randperm(nb, generator=g)[:len(pages)].tolist()
    width = width or max(1, max([-(-n // 16) for n in ctx] + [1])) + 1
    table = torch.full((len(seqs), width), -1, dtype=torch.int32)
    k = torch.full((nb, n_kv, 16, 128), float("nan") if poison else 0.0)
    v = torch.full((nb, n_kv, 128, 16), float("nan") if poison else 0.0)
    for (s, p), b in zip(pages, order):
        table[s, p] = b
        for t in range(16):
            if p * 16 + t in live[s]:
                k[b, :, t] = torch.randn(n_kv, 128, generator=g)
                v[b, :, :, t] = torch.randn(n_kv, 128, generator=g)
    rows = len(seqs) if kind == "decode" else max([q0 + q for q0, q, _ in seqs] + [0]) + spare
    qkv = torch.randn(rows, (n_q + 2 * n_kv) * 128, generator=g).to(torch.bfloat16)
    return qkv[:, : n_q * 128], k.to(dtype), v.to(dtype), table


def by_definition(kind, q, k, v, table, seqs, n_q, window, sinks):
    """Key by key in 64 bits -> (out [rows, n_q, 128], sum of p |v|: what the rounding of the weights is relative to)."""
    n_kv = k.shape[1]
    out = torch.zeros(q.shape[0], n_q, 128, dtype=torch.float64)
    size = torch.zeros_like(out)
    kd, vd = k.double(), v.double()
    for s, row, pos in spans(kind, seqs):
        keys = [j for j in range(min(pos + 1, table.shape[1] * 16)) if sees(pos, j, window, sinks) and 0 <= int(table[s, j // 16]) < k.shape[0]]
        if not keys:
            continue
        ids = [int(table[s, j // 16]) for j in keys]
        kk = torch.stack([kd[b, :, j % 16] for b, j in zip(ids, keys)], 1)            # [n_kv, keys, 128]
        vv = torch.stack([vd[b, :, :, j % 16] for b, j in zip(ids, keys)], 1)
        qq = q[row].double().view(n_kv, n_q // n_kv, 128)
        p = torch.softmax(torch.matmul(qq, kk.transpose(1, 2)) * SCALE, -1)
        out[row] = torch.matmul(p, vv).reshape(n_q, 128)
        size[row] = torch.matmul(p, vv.abs()).reshape(n_q, 128)
    return out.view(q.shape[0], -1), size.view(q.shape[0], -1)


def allowed(out, size):
    """What a kernel may be off. Weights p_j are rounded to bf16 before they meet V (half a step, 2^-8 of each: 2^-8 * sum p|v|),
    the result is rounded to bf16 (2^-8 of itself). Scores are sums of 128 exact products in fp32: 128 * 2^-24 * sum |q k| with
    sum |q k| * scale <= 12 for unit normals gives 9e-5 of each weight, twice (weight and sum), the exponential and the running
    rescales a few 2^-23 more: under 2^-12 of sum p|v| together."""
    return (2.0 ** -8 + 2.0 ** -12) * size + (2.0 ** -8 + 2.0 ** -12) * out.abs() + 1e-30
