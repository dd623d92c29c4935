"""Plain PyTorch fp32 references of the LLM kernels in ``csrc/llm_*.hip``.

Two users: the numerics tests (``tests/test_gpu_llm.py`` compares every HIP kernel against
these on the same inputs) and the CPU path of ``ops.llm`` (a tiny model steps through the
serving engine in the CPU test suite). On a GPU the HIP kernels run, never these.

Cache layouts (see llm_attention.hip): K ``[blocks, n_kv, 16, 128]``, V ``[blocks, n_kv, 128, 16]``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

HEAD_DIM = 128
BLOCK = 16


def rope_table(max_pos: int, theta: float = 500000.0, device="cpu") -> torch.Tensor:
    """fp32 [max_pos, 128]: 64 cosines then 64 sines of pos * theta^(-2i/128)."""
    inv = 1.0 / (theta ** (torch.arange(0, HEAD_DIM, 2, dtype=torch.float64) / HEAD_DIM))
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv[None, :]
    return torch.cat([ang.cos(), ang.sin()], dim=1).to(torch.float32).to(device)


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float,
            residual: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """-> (out, new_residual); both in x.dtype, math in fp32."""
    if residual is not None:
        h = (x.float() + residual.float()).to(x.dtype)
        new_res = h
    else:
        h, new_res = x, None
    hf = h.float()
    out = hf * torch.rsqrt(hf.pow(2).mean(-1, keepdim=True) + eps) * weight.float()
    return out.to(x.dtype), new_res


def silu_mul(gate_up: torch.Tensor) -> torch.Tensor:
    """gate/up columns interleaved by 8: [.., 16j+c] gate, [.., 16j+8+c] up -> [.., 8j+c]."""
    f = gate_up.shape[-1] // 2
    v = gate_up.float().reshape(*gate_up.shape[:-1], f // 8, 2, 8)
    return (torch.nn.functional.silu(v[..., 0, :]) * v[..., 1, :]).reshape(*gate_up.shape[:-1], f).to(gate_up.dtype)


def rope(qkv: torch.Tensor, cos_sin: torch.Tensor, positions: torch.Tensor, n_q: int, n_kv: int) -> torch.Tensor:
    """Rotate-half RoPE on the q and k heads of qkv [T, (n_q + 2 n_kv) * 128]; v untouched."""
    T = qkv.shape[0]
    x = qkv.float().view(T, n_q + 2 * n_kv, HEAD_DIM)
    cs = cos_sin[positions.long().clamp(0, cos_sin.shape[0] - 1)]
    c, s = cs[:, None, :64], cs[:, None, 64:]
    rot = x[:, : n_q + n_kv]
    x1, x2 = rot[..., :64], rot[..., 64:]
    out = x.clone()
    out[:, : n_q + n_kv, :64] = x1 * c - x2 * s
    out[:, : n_q + n_kv, 64:] = x2 * c + x1 * s
    return out.view(T, -1).to(qkv.dtype)


def cache_write(qkv_rot: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                n_q: int, n_kv: int) -> None:
    T = qkv_rot.shape[0]
    x = qkv_rot.view(T, n_q + 2 * n_kv, HEAD_DIM)
    ok = (slots >= 0) & (slots < k_cache.shape[0] * BLOCK)
    idx = torch.nonzero(ok).flatten()
    if idx.numel() == 0:
        return
    sl = slots[idx].long()
    blk, off = sl // BLOCK, sl % BLOCK
    k_cache[blk, :, off, :] = x[idx, n_q:n_q + n_kv].to(k_cache.dtype)
    v_cache[blk, :, :, off] = x[idx, n_q + n_kv:].to(v_cache.dtype)


def gather_kv(k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, ctx: int):
    """-> K, V as fp32 [n_kv, ctx, 128] for one sequence."""
    nb = (ctx + BLOCK - 1) // BLOCK
    ids = table[:nb].long()
    k = k_cache[ids].permute(1, 0, 2, 3).reshape(k_cache.shape[1], nb * BLOCK, HEAD_DIM)[:, :ctx]
    v = v_cache[ids].permute(1, 0, 3, 2).reshape(v_cache.shape[1], nb * BLOCK, HEAD_DIM)[:, :ctx]
    return k.float(), v.float()


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_pos: torch.Tensor, scale: float) -> torch.Tensor:
    """q [Tq, n_q, 128] (fp32), k/v [n_kv, ctx, 128], q_pos [Tq]: causal attention with GQA."""
    n_q, n_kv = q.shape[1], k.shape[0]
    g = n_q // n_kv
    kk = k.repeat_interleave(g, dim=0)
    vv = v.repeat_interleave(g, dim=0)
    s = torch.einsum("thd,hcd->htc", q, kk) * scale
    key_pos = torch.arange(k.shape[1], device=q.device)
    mask = key_pos[None, None, :] > q_pos.long()[None, :, None]
    s = s.masked_fill(mask, float("-inf"))
    p = torch.softmax(s, dim=-1)
    return torch.einsum("htc,hcd->thd", p, vv)


def paged_attn_decode(q, k_cache, v_cache, block_tables, ctx_lens, scale: float) -> torch.Tensor:
    """q [B, n_q*128 (+ more, strided view ok)] -> [B, n_q*128]."""
    B = block_tables.shape[0]
    n_kv = k_cache.shape[1]
    n_q = q.shape[-1] // HEAD_DIM
    out = torch.zeros((B, n_q * HEAD_DIM), dtype=q.dtype, device=q.device)
    for b in range(B):
        ctx = int(ctx_lens[b])
        if ctx <= 0:
            continue
        k, v = gather_kv(k_cache, v_cache, block_tables[b], ctx)
        qq = q[b].float().view(1, n_q, HEAD_DIM)
        o = attend(qq, k, v, torch.tensor([ctx - 1], device=q.device), scale)
        out[b] = o.reshape(-1).to(q.dtype)
    del n_kv
    return out


def paged_attn_prefill(q, k_cache, v_cache, block_tables, seq_info, scale: float) -> torch.Tensor:
    """q [T, n_q*128]; seq_info [S, 3] = (q_start, q_len, ctx_len) -> [T, n_q*128]."""
    n_q = q.shape[-1] // HEAD_DIM
    out = torch.zeros((q.shape[0], n_q * HEAD_DIM), dtype=q.dtype, device=q.device)
    for s in range(seq_info.shape[0]):
        q0, ql, ctx = (int(x) for x in seq_info[s])
        if ql <= 0 or ctx < ql:
            continue
        k, v = gather_kv(k_cache, v_cache, block_tables[s], ctx)
        qq = q[q0:q0 + ql].float().view(ql, n_q, HEAD_DIM)
        pos = torch.arange(ctx - ql, ctx, device=q.device)
        out[q0:q0 + ql] = attend(qq, k, v, pos, scale).reshape(ql, -1).to(q.dtype)
    return out


def _window_rows(q, k_cache, v_cache, table, ctx: int, pos, scale: float, window: int, sinks: int) -> torch.Tensor:
    """q [Tq, n_q, 128] at positions `pos` of one sequence, limited to a window and sinks; a page id outside the cache is no page."""
    n = min(ctx, table.shape[0] * BLOCK)
    nb, n_kv = k_cache.shape[0], k_cache.shape[1]
    g = q.shape[1] // n_kv
    if n <= 0:
        return torch.zeros_like(q)
    ids = table[: (n + BLOCK - 1) // BLOCK].long()
    there = ((ids >= 0) & (ids < nb)).repeat_interleave(BLOCK)[:n]
    k, v = gather_kv(k_cache, v_cache, ids.clamp(0, nb - 1), n)
    key = torch.arange(n, device=q.device)
    p = pos.long()[:, None]
    see = (key <= p) & ((key > p - window) | (key < sinks)) & there
    any_sees = see.any(0)
    k = torch.where(any_sees[None, :, None], k, 0.0).to(q.dtype)          # keys that no row sees: their bytes do not matter
    v = torch.where(any_sees[None, :, None], v, 0.0).to(q.dtype)
    s = torch.einsum("tkgd,kcd->kgtc", q.view(q.shape[0], n_kv, g, HEAD_DIM), k) * scale
    s = s.masked_fill(~see, float("-inf"))
    m = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    z = w.sum(-1, keepdim=True)
    w = w / torch.where(z == 0, torch.ones_like(z), z)
    if bool(torch.isfinite(v).all()):
        o = torch.einsum("kgtc,kcd->tkgd", w, v)
    else:                                                                 # 0 * NaN: only the rows that see a value take it
        o = torch.where(see[None, None, :, :, None], w[..., None] * v[:, None, None], 0.0).sum(3).permute(2, 0, 1, 3)
    return o.reshape(q.shape)


def window_attn_decode(q, k_cache, v_cache, block_tables, ctx_lens, scale: float, window: int, sinks: int, dtype=torch.float32) -> torch.Tensor:
    """q [B, n_q*128] -> [B, n_q*128]; computed in `dtype`."""
    out = torch.zeros((q.shape[0], q.shape[-1]), dtype=q.dtype, device=q.device)
    for b in range(q.shape[0]):
        ctx = int(ctx_lens[b])
        if ctx > 0:
            o = _window_rows(q[b].to(dtype).view(1, -1, HEAD_DIM), k_cache, v_cache, block_tables[b], ctx,
                             torch.tensor([ctx - 1], device=q.device), scale, window, sinks)
            out[b] = o.reshape(-1).to(q.dtype)
    return out


def window_attn_prefill(q, k_cache, v_cache, block_tables, seq_info, scale: float, window: int, sinks: int, out=None,
                        dtype=torch.float32) -> torch.Tensor:
    if out is None:
        out = torch.zeros((q.shape[0], q.shape[-1]), dtype=q.dtype, device=q.device)
    for s in range(seq_info.shape[0]):
        q0, ql, ctx = (int(x) for x in seq_info[s])
        if ql <= 0 or ctx < ql or q0 < 0 or q0 + ql > q.shape[0]:
            continue
        pos = torch.arange(ctx - ql, ctx, device=q.device)
        o = _window_rows(q[q0:q0 + ql].to(dtype).view(ql, -1, HEAD_DIM), k_cache, v_cache, block_tables[s], ctx, pos, scale, window, sinks)
        out[q0:q0 + ql] = o.reshape(ql, -1).to(out.dtype)
    return out


def copy_pages(k_cache, v_cache, pairs, k_src, v_src) -> None:
    """pairs: host integers [n, 2]; -1 as a source clears."""
    if k_cache.dim() == 4:
        k_cache, v_cache, k_src, v_src = (x[None] for x in (k_cache, v_cache, k_src, v_src))
    for src, dst in ((int(a), int(b)) for a, b in pairs):
        for to, of in ((k_cache, k_src), (v_cache, v_src)):
            if src < 0:
                to[:, dst].zero_()
            else:
                to[:, dst].copy_(of[:, src])


def choose_tokens(logits, rules, first_token: int, dtype=torch.float32):
    """-> (processed logits [B, V], ids int64 [B], best [B]), computed in `dtype`, one rounded operation after another."""
    B, V = logits.shape
    y = logits.to(dtype).clone()
    ids = torch.empty(B, dtype=torch.int64, device=logits.device)
    best = torch.empty(B, dtype=torch.float32, device=logits.device)
    for b in range(B):
        x = y[b]
        allowed = torch.ones(V, dtype=torch.bool, device=logits.device)
        r = -1
        if rules is not None:
            r = b if rules.rows is None else int(rules.rows[b])
        if rules is not None and 0 <= r < rules.lens.shape[0]:
            n = min(max(int(rules.lens[r]), 0), rules.history.shape[1])
            h = rules.history[r, :n].long() - first_token
            ok = (h >= 0) & (h < V) & (rules.history[r, :n] >= 0)
            output = torch.arange(n, device=h.device) >= int(rules.prompt_lens[r])
            seen = torch.zeros(V, dtype=torch.bool, device=h.device)
            seen[h[ok]] = True
            c = torch.bincount(h[ok & output], minlength=V).to(dtype)
            rep, freq, pres = (t[r].to(dtype) for t in (rules.repetition, rules.frequency, rules.presence))
            x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
            x = torch.where(c > 0, (x - freq * c) - pres, x)
            if rules.bias_ids is not None:
                add = {}
                for i, t in enumerate(rules.bias_ids[r].tolist()):
                    if t >= 0 and 0 <= t - first_token < V:
                        add[t - first_token] = i                          # a token twice: the later entry counts
                if add:
                    at = torch.tensor(list(add), device=h.device)
                    x[at] = x[at] + rules.bias_values[r, torch.tensor(list(add.values()), device=h.device)].to(dtype)
            m = -1
            if rules.mask is not None:
                m = r if rules.mask_rows is None else int(rules.mask_rows[r])
            if rules.mask is not None and 0 <= m < rules.mask.shape[0]:
                t = torch.arange(first_token, first_token + V, device=h.device)
                allowed = ((rules.mask[m][t // 32].long() >> (t % 32)) & 1).bool()
                x = torch.where(allowed, x, torch.full_like(x, float("-inf")))
        y[b] = x
        at = torch.nonzero(allowed).flatten()
        if not at.numel():
            ids[b], best[b] = -1, float("-inf")
            continue
        z = x[at]
        nan = torch.isnan(z)
        pick = at[nan][0] if bool(nan.any()) else at[torch.nonzero(z == z.max()).flatten()[0]]
        ids[b], best[b] = pick + first_token, x[pick]
    return y, ids, best
