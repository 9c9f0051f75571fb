"""The paged KV-cache operators: their cases, their plain forms, and the calls a user makes.

Four operators of `mcoplib_b200.op` work on the paged cache [num_blocks, block_size, kv_heads, head_size]:

  reshape_and_cache_dynamic_int8  K and V rows to int8 codes with one scale per (token, head), made as they are written
  gather_and_dequant_cache        the rows of a batch of sequences back out of the cache, packed, in the model's type
  paged_attention_decode          one new token per sequence over its cached tokens
  paged_attention_chunk           a chunk of new tokens per sequence over its cached tokens, causal from the end

The cache holds the model's type, int8 with one scale per head (what rope_kv_store_int8 writes) or int8 with one scale
per (token, head) (what reshape_and_cache_dynamic_int8 writes).
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------ cases
def _decode(name, batch, max_len, q_heads, kv_heads, dim, block, cache, dtype="bf16", spread="ragged", window=0):
    return {"name": name, "op": "decode", "batch": batch, "max_len": max_len, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "block": block,
            "cache": cache, "type": dtype, "spread": spread, "window": window}


def _chunk(name, batch, max_new, max_past, q_heads, kv_heads, dim, block, cache, dtype="bf16", spread="ragged", window=0):
    return {"name": name, "op": "chunk", "batch": batch, "max_new": max_new, "max_past": max_past, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "block": block, "cache": cache, "type": dtype, "spread": spread, "window": window}


def _rows(name, op, batch, max_len, kv_heads, dim, block, cache, dtype="bf16", spread="ragged", pad=False):
    return {"name": name, "op": op, "batch": batch, "max_len": max_len, "kv_heads": kv_heads, "dim": dim, "block": block, "cache": cache, "type": dtype,
            "spread": spread, "pad": pad}


def listed():
    return [
        # one user, a 4K conversation, the int8 cache of rope_kv_store_int8: latency
        _decode("decode_1x4k_int8", 1, 4095, 64, 8, 128, 16, "int8_head", spread="full"),
        # an ordinary serving batch of very unequal sequences, scales per token
        _decode("decode_64_ragged_int8t", 64, 8192, 64, 8, 128, 16, "int8_token"),
        # the same kind of batch on an unquantised cache, 32 query heads
        _decode("decode_32_ragged_bf16", 32, 4096, 32, 8, 128, 16, "float"),
        # the largest decode batch: throughput serving
        _decode("decode_256_int8", 256, 4096, 64, 8, 128, 16, "int8_head"),
        # a few drafted tokens per sequence checked at once
        _chunk("chunk_8x8_past2k", 8, 8, 2000, 32, 8, 128, 16, "float"),
        # long context, one prefill chunk of two requests on the int8 cache
        _chunk("chunk_2x512_past8k_int8t", 2, 512, 7680, 64, 8, 128, 16, "int8_token", spread="full"),
        # a full prefill chunk: 4096 new tokens after 4096 cached ones
        _chunk("chunk_4096_past4096", 1, 4096, 4096, 64, 8, 128, 16, "float", spread="full"),
        # mixed batch: single tokens beside chunks, sliding window, small heads, an odd group of 3
        _chunk("chunk_mixed_window_f16", 12, 1027, 3000, 12, 4, 64, 16, "float", "f16", window=1024),
        # the step's new tokens of a decode batch: latency
        _rows("store_128x1", "store", 128, 1, 8, 128, 16, "int8_token", spread="full"),
        # a prefill chunk written and read back
        _rows("store_32768", "store", 8, 4096, 8, 128, 16, "int8_token", spread="full"),
        # a short shared prefix out of the int8 cache
        _rows("gather_4_ragged_int8", "gather", 4, 777, 8, 128, 16, "int8_head"),
        # the cached part of a long batch, for a product or a transfer in the model's type
        _rows("gather_65536_int8t", "gather", 16, 4096, 8, 128, 16, "int8_token", spread="full"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    dim = rng.choice((64, 128, 128, 96))
    kv_heads = rng.choice((1, 2, 4, 8))
    q_heads = kv_heads * rng.choice((1, 3, 4, 7, 8))
    block = rng.choice((1, 16, 16, 24, 32, 64))
    cache = rng.choice(("float", "int8_head", "int8_token"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    window = rng.choice((0, 0, 0, _log(rng, 1, 2048)))
    op = rng.choice(("decode", "chunk", "store", "gather"))
    if op == "decode":
        batch = _log(rng, 1, 200)
        c = _decode("", batch, _log(rng, 1, 4096 if batch > 64 else 16384), q_heads, kv_heads, dim, block, cache, dtype, "ragged", window)
    elif op == "chunk":
        batch = _log(rng, 1, 16)
        new = _log(rng, 1, 4096 // batch)
        c = _chunk("", batch, new, _log(rng, 1, 8192 // batch + 1), q_heads, kv_heads, dim, block, cache, dtype, "ragged", window)
    else:
        batch = _log(rng, 1, 64)
        c = _rows("", op, batch, _log(rng, 1, 32768 // batch), kv_heads, dim, block, "int8_token" if op == "store" else cache, dtype, "ragged",
                  rng.random() < 0.5)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case, key, salt):
    """Sequence lengths from the case alone: the first is the longest, the others spread below it, a single token among them."""
    n, top = case["batch"], case[key]
    if case["spread"] == "full":
        return [top] * n
    r = random.Random("%s %d %d %d" % (salt, n, top, case["kv_heads"]))
    v = [top] + [max(1, int(top * r.random())) for _ in range(n - 1)]
    if n > 2:
        v[1] = 1
    return v


def _shape(case):
    """(new tokens of each sequence, cached tokens of each sequence with the new ones)"""
    if case["op"] == "chunk":
        new, past = _lengths(case, "max_new", "new"), _lengths(case, "max_past", "past")
        return new, [a + b for a, b in zip(new, past)]
    total = _lengths(case, "max_len", "len")
    return ([1] * len(total) if case["op"] == "decode" else total), total


def _randn(shape, g, dtype, gain=1.0):
    return (torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * gain).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    new, total = _shape(case)
    dtype, block, H, D = TYPES[case["type"]], case["block"], case["kv_heads"], case["dim"]
    pages = [-(-n // block) for n in total]
    blocks = sum(pages) + 3
    order = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
    start = torch.tensor([0] + pages, device=DEV).cumsum(0)[:-1]
    column = torch.arange(max(pages), device=DEV)
    table = order[(start[:, None] + column).clamp(max=blocks - 1)].contiguous()
    shape = (blocks, block, H, D)
    s = {"case": case, "table": table, "lens": torch.tensor(total, dtype=torch.int32, device=DEV), "max_len": max(total), "max_new": max(new),
         "k_scale": None, "v_scale": None}
    s["cu_lens"] = torch.tensor([0] + total, device=DEV).cumsum(0).to(torch.int32)
    s["cu_new"] = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
    if case["cache"] == "float":
        s["k_cache"], s["v_cache"] = _randn(shape, g, dtype), _randn(shape, g, dtype)
    else:
        s["k_cache"], s["v_cache"] = (_randn(shape, g, torch.float32, 32.0).round().clamp(-127, 127).to(torch.int8) for _ in range(2))
        of = (H,) if case["cache"] == "int8_head" else (blocks, block, H)
        s["k_scale"], s["v_scale"] = ((torch.rand(of, generator=g, device=DEV) * 0.02 + 0.02).contiguous() for _ in range(2))
    T = sum(new)
    seq = torch.repeat_interleave(torch.arange(len(new), device=DEV), torch.tensor(new, device=DEV))
    at = torch.arange(T, device=DEV) - s["cu_new"][seq]
    s["seq"], s["at"] = seq, at
    if case["op"] in ("decode", "chunk"):
        s["query"] = _randn((T, case["q_heads"], D), g, dtype)
        s["out"] = torch.empty_like(s["query"])
        s["lse"] = torch.empty(T, case["q_heads"], dtype=torch.float32, device=DEV)
        s["scale"] = D ** -0.5
    else:
        s["k_out"], s["v_out"] = (torch.empty(sum(total), H, D, dtype=dtype, device=DEV) for _ in range(2))
        if case["op"] == "store":
            s["key"], s["value"] = _randn((T, H, D), g, dtype), _randn((T, H, D), g, dtype)
            s["slots"] = table[seq, at // block].long() * block + at % block
            if case["pad"]:
                s["slots"][::17] = -1  # padded tokens of the batch: not stored
            s["kept"] = torch.nonzero(s["slots"] >= 0).flatten()
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _cached(s, name, slots):
    """Rows of a cache in 32 bits: [..., kv_heads, dim]"""
    cache, scale = s[name + "_cache"], s[name + "_scale"]
    rows = cache.flatten(0, 1)[slots].float()
    if scale is None:
        return rows
    return rows * (scale[:, None] if scale.dim() == 1 else scale.flatten(0, 1)[slots][..., None])


def _plain_attention(s):
    c = s["case"]
    B, H, D, L, N = c["batch"], c["kv_heads"], c["dim"], s["max_len"], s["max_new"]
    G = c["q_heads"] // H
    pos = torch.arange(L, device=DEV)
    slots = s["table"][:, pos // c["block"]].long() * c["block"] + pos % c["block"]
    first = s["cu_new"][:-1].long()
    new = s["cu_new"][1:].long() - first
    i = torch.arange(N, device=DEV)
    row = (first[:, None] + i).clamp(max=s["query"].shape[0] - 1)
    q = s["query"][row].float().view(B, N, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, N * G, D)
    k = _cached(s, "k", slots).permute(0, 2, 3, 1)
    x = torch.matmul(q, k).mul_(s["scale"]).view(B, H, N, G, L)
    here = s["lens"].long()[:, None] - new[:, None] + i
    seen = pos <= here[..., None]
    if c["window"]:
        seen &= pos > here[..., None] - c["window"]
    x.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    v = _cached(s, "v", slots).permute(0, 2, 1, 3)
    o = torch.matmul(x.view(B, H, N * G, L), v).view(B, H, N, G, D) / torch.where(total == 0, 1.0, total)
    lse = (top + total.log()).squeeze(-1)
    o = o.permute(0, 2, 1, 3, 4)[s["seq"], s["at"]].flatten(1, 2)
    return o.to(s["query"].dtype), lse.permute(0, 2, 1, 3)[s["seq"], s["at"]].flatten(1, 2)


def _plain_store(s):
    kept = s["slots"][s["kept"]]
    key, value = s["key"][s["kept"]].float(), s["value"][s["kept"]].float()
    ks, vs = key.abs().amax(-1) / 127.0, value.abs().amax(-1) / 127.0
    # the quotient in 64 bits: the code is the nearest whole number of value / scale, and 32 bits may round it onto a tie
    for x, scale, name in ((key, ks, "k"), (value, vs, "v")):
        codes = torch.where(scale[..., None] == 0, 0.0, x.double() / scale[..., None].double()).round().clamp(-127, 127)
        s[name + "_cache"].flatten(0, 1)[kept] = codes.to(torch.int8)
        s[name + "_scale"].flatten(0, 1)[kept] = scale


def _plain_gather(s):
    c = s["case"]
    total = s["cu_lens"].long()
    n = s["k_out"].shape[0]
    at = torch.arange(n, device=DEV)
    seq = torch.searchsorted(total, at, right=True) - 1
    at = at - total[seq]
    slots = s["table"][seq, at // c["block"]].long() * c["block"] + at % c["block"]
    return _cached(s, "k", slots).to(s["k_out"].dtype), _cached(s, "v", slots).to(s["v_out"].dtype)


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        from mcoplib_b200 import op as ops

        if op == "decode":
            ops.paged_attention_decode(s["out"], s["query"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["scale"], s["k_scale"], s["v_scale"],
                                       s["case"]["window"], s["lse"])
            return s["out"], s["lse"]
        if op == "chunk":
            ops.paged_attention_chunk(s["out"], s["query"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu_new"], s["scale"], s["k_scale"],
                                      s["v_scale"], True, s["case"]["window"], s["lse"])
            return s["out"], s["lse"]
        if op == "store":
            ops.reshape_and_cache_dynamic_int8(s["key"], s["value"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["slots"])
        ops.gather_and_dequant_cache(s["k_out"], s["v_out"], s["k_cache"], s["v_cache"], s["table"], s["cu_lens"], s["k_scale"], s["v_scale"])
        k, v = s["k_out"], s["v_out"]
    elif op in ("decode", "chunk"):
        return _plain_attention(s)
    else:
        if op == "store":
            _plain_store(s)
        k, v = _plain_gather(s)
    # the codes come back as the values they stand for, the scales as they are held
    return (k, v, s["k_scale"], s["v_scale"]) if op == "store" else (k, v)


# ------------------------------------------------------------------------------------------------ work
def _spans(case):
    """For each sequence: (cached tokens that some new token sees, pairs of new and cached tokens)"""
    new, total = _shape(case)
    w = case["window"]
    out = []
    for n, t in zip(new, total):
        first, last = t - n + 1, t  # how many tokens the first and the last new token would see without a window
        if not w:
            out.append((t, (first + last) * n // 2))
        else:
            out.append((t - max(0, first - w), sum(min(w, x) for x in range(first, last + 1))))
    return out


def work(case):
    new, total = _shape(case)
    H, D = case["kv_heads"], case["dim"]
    rows, T = sum(total), sum(new)
    elem = 2 if case["cache"] == "float" else 1
    one = 2 * H * (D * elem + (4 if case["cache"] == "int8_token" else 0))  # a token of the cache
    table = 4 * sum(-(-n // case["block"]) for n in total)
    if case["op"] in ("decode", "chunk"):
        spans = _spans(case)
        q = T * case["q_heads"] * D * 2
        return {"bytes": sum(a for a, _ in spans) * one + 2 * q + T * case["q_heads"] * 4 + table,
                "flops": sum(p for _, p in spans) * case["q_heads"] * D * 4}
    values = 2 * rows * H * D
    if case["op"] == "gather":
        return {"bytes": rows * one + values * 2 + table, "flops": values}
    return {"bytes": values * 2 + rows * (8 + one) + rows * one + values * 2 + table, "flops": 4 * values}


# ------------------------------------------------------------------------------------------------ 64 bits
def _wide(s, name, b, n):
    """The first n cached rows of sequence b in 64 bits: [n, kv_heads, dim]"""
    c = s["case"]
    at = torch.arange(n, device=DEV)
    page, off = s["table"][b, torch.div(at, c["block"], rounding_mode="floor")].long(), at % c["block"]
    x = s[name + "_cache"][page, off].double()
    scale = s[name + "_scale"]
    if scale is not None:
        x = x * (scale.double().view(1, -1, 1) if scale.dim() == 1 else scale[page, off].double().unsqueeze(-1))
    return x


def exact(case, seed):
    s = prepare(case, seed)
    new, total = _shape(case)
    if case["op"] in ("decode", "chunk"):
        out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEV)
        lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device=DEV)
        G, t0 = case["q_heads"] // case["kv_heads"], 0
        for b, (n, t) in enumerate(zip(new, total)):
            K, V = _wide(s, "k", b, t), _wide(s, "v", b, t)
            for lo in range(0, n, 512):
                hi = min(n, lo + 512)
                me = torch.arange(t - n + lo, t - n + hi, device=DEV).view(1, -1, 1)
                you = torch.arange(t, device=DEV).view(1, 1, -1)
                hidden = you > me
                if case["window"]:
                    hidden = hidden | (me - you >= case["window"])
                q = s["query"][t0 + lo:t0 + hi].double().transpose(0, 1)  # [q_heads, rows, dim]
                for h in range(case["kv_heads"]):
                    z = (q[h * G:(h + 1) * G] @ K[:, h].T * s["scale"]).masked_fill(hidden, -math.inf)
                    lse[t0 + lo:t0 + hi, h * G:(h + 1) * G] = torch.logsumexp(z, -1).T
                    out[t0 + lo:t0 + hi, h * G:(h + 1) * G] = (torch.softmax(z, -1) @ V[:, h]).transpose(0, 1)
            t0 += n
        return out, lse
    if case["op"] == "store":
        for x, name in ((s["key"], "k"), (s["value"], "v")):
            wide = x.double()
            scale = (wide.abs().amax(-1) / 127).float()  # held in 32 bits
            code = torch.round(wide / scale.double().unsqueeze(-1)).nan_to_num(0.0)
            written = s["slots"] >= 0
            page, off = s["slots"][written] // case["block"], s["slots"][written] % case["block"]
            s[name + "_cache"][page, off] = code[written].to(torch.int8)
            s[name + "_scale"][page, off] = scale[written]
    rows = tuple(torch.cat([_wide(s, name, b, t) for b, t in enumerate(total)]) for name in ("k", "v"))
    return rows + (s["k_scale"].double(), s["v_scale"].double()) if case["op"] == "store" else rows
