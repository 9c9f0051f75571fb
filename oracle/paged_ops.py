"""The paged KV-cache operators from their formulas in 64 bits (no counterpart in the reference; used by tests only).

Every function takes plain tensors on any device and loops over sequences."""
from __future__ import annotations

import math

import torch


def quantise_rows(x: torch.Tensor):
    """codes int8 and scales fp32 of rows [..., head_size]: scale = fp32(max|x| / 127), code = nearest integer of x / scale."""
    wide = x.double()
    scale = (wide.abs().amax(-1) / 127.0).float()
    code = torch.round(wide / scale.double()[..., None])
    code = torch.where(scale[..., None] == 0, torch.zeros_like(code), code)
    bad = ~torch.isfinite(wide).all(-1)
    scale = torch.where(bad, torch.full_like(scale, math.nan), scale)
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    return code.clamp(-127, 127).to(torch.int8), scale


def store(key, value, key_cache, value_cache, k_scale, v_scale, slots):
    """In place, token by token; negative slots are not stored."""
    for x, cache, scales in ((key, key_cache, k_scale), (value, value_cache, v_scale)):
        codes, s = quantise_rows(x)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < cache.shape[0] * cache.shape[1]:
                cache[slot // cache.shape[1], slot % cache.shape[1]] = codes[t]
                scales[slot // cache.shape[1], slot % cache.shape[1]] = s[t]


def rows_of(cache, scale, table_row, n):
    """The first n cached rows of one sequence in 64 bits: [n, kv_heads, head_size]"""
    at = torch.arange(n, device=cache.device)
    page, off = table_row.long()[at // cache.shape[1]], at % cache.shape[1]
    x = cache[page, off].double()
    if scale is None:
        return x
    return x * (scale.double()[None, :, None] if scale.dim() == 1 else scale[page, off].double()[..., None])


def attention(query, key_cache, value_cache, tables, lens, cu, scale, k_scale=None, v_scale=None, causal=True, window=0):
    """(out, lse, spread, mass, reach) in 64 bits.  spread[t, h, d] = sum_j p_j |v_jd|, mass the same without the weights, reach[t, h] = scale * max_j sum_d |q_d k_jd|: what the
    rounding of the weights and of the logits is measured against.  Rows outside the sequences are NaN."""
    T, Hq, D = query.shape
    H = key_cache.shape[2]
    dev = query.device
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64, device=dev)
    spread, mass = out.clone(), out.clone()
    lse = torch.full((T, Hq), math.nan, dtype=torch.float64, device=dev)
    reach = lse.clone()
    for b, n in enumerate(lens.tolist()):
        t0, t1 = int(cu[b]), int(cu[b + 1])
        if t1 == t0:
            continue
        K = rows_of(key_cache, k_scale, tables[b], n).repeat_interleave(Hq // H, 1)
        V = rows_of(value_cache, v_scale, tables[b], n).repeat_interleave(Hq // H, 1)
        q = query[t0:t1].double()
        pos = torch.arange(n - (t1 - t0), n, device=dev)[:, None]
        j = torch.arange(n, device=dev)[None, :]
        seen = torch.ones(t1 - t0, n, dtype=torch.bool, device=dev)
        if causal:
            seen &= j <= pos
        if window:
            seen &= j > pos - window
        for h in range(Hq):
            # a position that a row does not see takes no part, whatever it holds
            x = torch.where(seen, scale * (q[:, h] @ K[:, h].T), -math.inf)
            m = torch.where(seen.any(-1), x.amax(-1) if n else 0.0, 0.0) if n else torch.zeros(t1 - t0, dtype=torch.float64, device=dev)
            p = torch.where(seen, torch.exp(x - m[:, None]), 0.0)
            total = p.sum(-1)
            p = p / torch.where(total == 0, 1.0, total)[:, None]
            v = V[:, h]
            clean = torch.where(torch.isfinite(v), v, 0.0)
            o = p @ clean
            for d0 in torch.nonzero(~torch.isfinite(v).all(-1)).flatten().tolist():  # rows that see a NaN or an infinity
                o = torch.where(seen[:, d0:d0 + 1], o + p[:, d0:d0 + 1] * (v[d0] - clean[d0] if torch.isfinite(v[d0]).all() else torch.where(torch.isfinite(v[d0]), 0.0, v[d0])), o)
            out[t0:t1, h] = o
            spread[t0:t1, h] = p @ clean.abs()
            mass[t0:t1, h] = seen.double() @ clean.abs()
            lse[t0:t1, h] = torch.where(total == 0, -math.inf, m + total.log())
            r = torch.where(seen, scale * (q[:, h].abs() @ K[:, h].abs().T), 0.0)
            reach[t0:t1, h] = r.amax(-1) if n else 0.0
    return out, lse, spread, mass, reach
