"""Decode and chunk attention over the paged cache against the formula in 64 bits."""
import math

import pytest
import torch

from mcoplib_b200 import cabi
from oracle import paged_ops as P
from tests.gpu_util import DEV, Canary
from tests.paged_util import attention_tolerance, bounds, compare, lengths, make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op():
    from mcoplib_b200 import op as _op
    return _op


def _check(out, lse, query, c, total, cu, scale, kind, causal=True, window=0, what=""):
    ref, rlse, spread, mass, reach = P.attention(query, c["k"], c["v"], c["tables"], torch.tensor(total), cu.tolist(), scale, c["ks"], c["vs"], causal, window)
    mine = ~rlse.isnan() | (reach.isnan() & ~spread.isnan().all(-1))
    tol, ltol = attention_tolerance(ref, rlse, spread, mass, reach, query.shape[2], kind, query.dtype)
    compare(out, torch.where(mine[..., None], ref, out.double()), tol, what + " out")
    compare(lse, torch.where(mine, rlse, lse.double()), ltol, what + " lse")


def _run(op, new, total, hq, hkv, D, block, kind, dtype, window=0, causal=True, decode=False, seed=0, gain=1.0):
    c = make_cache(total, hkv, D, block, kind, dtype, seed)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    T = sum(new)
    query = (torch.randn(T, hq, D, generator=g, device=DEV) * gain).to(dtype)
    out, lse = Canary((T, hq, D), dtype, 3), Canary((T, hq), torch.float32, 3)
    scale = D ** -0.5
    if decode:
        op.paged_attention_decode(out.t, query, c["k"], c["v"], c["tables"], lengths(total), scale, c["ks"], c["vs"], window, lse.t)
    else:
        op.paged_attention_chunk(out.t, query, c["k"], c["v"], c["tables"], lengths(total), bounds(new), scale, c["ks"], c["vs"], causal, window, lse.t)
    torch.cuda.synchronize()
    assert cabi.load().mcop_device_error() == 0
    out.check("out"); lse.check("lse")
    _check(out.t, lse.t, query, c, total, bounds(new), scale, kind, causal, window, str((new, total, hq, hkv, D, block, kind, dtype, window)))


KINDS = [("float", torch.bfloat16), ("float", torch.float16), ("head", torch.bfloat16), ("token", torch.bfloat16), ("head", torch.float16), ("token", torch.float16)]

DECODE = [
    ([1], 1, 1, 64, 1, 0),
    ([0], 8, 8, 128, 16, 0),
    ([1, 16, 17, 0, 63, 64, 65, 300], 8, 1, 128, 16, 0),
    ([500, 3, 1000], 64, 8, 128, 16, 0),
    ([129, 2000, 77], 14, 2, 96, 24, 0),
    ([40, 41, 4000], 6, 2, 64, 5, 100),
    ([700, 2], 32, 1, 128, 32, 1),
    ([333, 64], 12, 1, 256, 16, 0),
    ([90], 20, 1, 80, 64, 33),
    ([257, 5], 3, 3, 16, 16, 0),
    ([9000], 16, 2, 128, 16, 0),
    ([33] * 300, 4, 1, 32, 16, 0),
]


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("total,hq,hkv,D,block,window", DECODE)
def test_decode(op, total, hq, hkv, D, block, window, kind, dtype):
    _run(op, [1] * len(total), total, hq, hkv, D, block, kind, dtype, window, decode=True)


CHUNK = [
    ([1], [1], 1, 1, 64, 1, 0, True),
    ([5], [5], 8, 8, 128, 16, 0, True),
    ([0, 3, 0], [4, 3, 0], 8, 2, 128, 16, 0, True),
    ([1, 5, 17, 33], [1, 5, 40, 33], 8, 2, 64, 5, 0, True),
    ([40, 7], [20, 0], 4, 2, 128, 16, 0, True),                # more new tokens than cached ones: rows that see nothing
    ([130, 3], [130, 515], 8, 1, 128, 16, 0, True),
    ([300, 1, 129, 64], [900, 129, 129, 2000], 16, 2, 128, 32, 0, True),
    ([200], [1000], 14, 2, 96, 24, 0, True),
    ([70, 90], [90, 400], 6, 2, 64, 16, 50, True),
    ([128], [640], 8, 1, 128, 16, 1, True),
    ([60, 3], [300, 3], 4, 1, 128, 16, 0, False),
    ([33], [65], 2, 1, 128, 16, 20, False),
    ([40, 2], [200, 2], 12, 4, 256, 16, 0, True),
    ([9, 8, 1], [1000, 8, 300], 40, 1, 128, 16, 0, True),
    ([64], [5000], 8, 8, 48, 16, 0, True),
]


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("new,total,hq,hkv,D,block,window,causal", CHUNK)
def test_chunk(op, new, total, hq, hkv, D, block, window, causal, kind, dtype):
    _run(op, new, total, hq, hkv, D, block, kind, dtype, window, causal)


@pytest.mark.parametrize("decode", [True, False])
def test_peaked_logits(op, decode):
    """Logits over hundreds: the running maximum moves far, weights underflow."""
    _run(op, [1, 1] if decode else [70, 1], [800, 90], 8, 2, 128, 16, "float", torch.bfloat16, decode=decode, gain=30.0)
    _run(op, [1, 1] if decode else [70, 1], [800, 90], 8, 2, 128, 16, "token", torch.bfloat16, decode=decode, gain=30.0)


@pytest.mark.parametrize("kind", ["float", "token"])
@pytest.mark.parametrize("window", [0, 40])
def test_nan_and_infinity_reach_only_the_rows_that_see_them(op, kind, window):
    new, total, hq, hkv, D = [90], [200], 4, 2, 128
    c = make_cache(total, hkv, D, 16, kind, torch.bfloat16)
    query = torch.randn(90, hq, D, device=DEV).bfloat16()
    for pos, name, value in ((150, "v", math.nan), (170, "v", math.inf), (185, "k", math.nan), (112, "v", -math.inf)):
        page, off = int(c["tables"][0, pos // 16]), pos % 16
        if kind == "float":
            c[name][page, off, 0, 3] = value
        else:
            c[name + "s"][page, off, 0] = value
    out, lse = torch.empty_like(query), torch.empty(90, hq, device=DEV)
    op.paged_attention_chunk(out, query, c["k"], c["v"], c["tables"], lengths(total), bounds(new), D ** -0.5, c["ks"], c["vs"], True, window, lse)
    clean = make_cache(total, hkv, D, 16, kind, torch.bfloat16)
    good = torch.empty_like(query)
    op.paged_attention_chunk(good, query, clean["k"], clean["v"], clean["tables"], lengths(total), bounds(new), D ** -0.5, clean["ks"], clean["vs"],
                             True, window)
    for i in range(90):
        sees = [p for p in (150, 170, 185, 112) if p <= 110 + i and (not window or p > 110 + i - window)]
        assert torch.equal(out[i, 2:], good[i, 2:]), f"KV head 1 holds nothing special (row {i})"
        if not sees:
            assert torch.equal(out[i], good[i]), i
        elif 185 in sees or kind == "token":
            assert not bool(out[i, :2].isfinite().any()), (i, sees)
        else:
            assert not bool(out[i, :2, 3].isfinite().any()), (i, sees)
            assert torch.equal(out[i, :2, 4:], good[i, :2, 4:]) and torch.equal(out[i, :2, :3], good[i, :2, :3]), (i, sees)
        if 185 not in sees:
            assert bool(lse[i].isfinite().all())


@pytest.mark.parametrize("decode", [True, False])
def test_strided_tensors(op, decode):
    """query inside a packed qkv, out inside a wider buffer, K and V of a block beside one another, one table row for all."""
    new = [1, 1, 1] if decode else [20, 1, 60]
    total, T, D = [150, 150, 150], sum(new), 128
    c = make_cache([150], 2, D, 16, "float", torch.bfloat16)
    both = torch.stack([c["k"], c["v"]], 1)
    c["k"], c["v"], c["tables"] = both[:, 0], both[:, 1], c["tables"].expand(3, -1)
    packed = torch.randn(T, 12, D, device=DEV).bfloat16()
    wide = torch.full((T, 20, D), 7.0, device=DEV).bfloat16()
    query, out, lse = packed[:, 2:10], wide[:, 4:20:2], torch.empty(T, 8, device=DEV)
    if decode:
        op.paged_attention_decode(out, query, c["k"], c["v"], c["tables"], lengths(total), 0.1, lse=lse)
    else:
        op.paged_attention_chunk(out, query, c["k"], c["v"], c["tables"], lengths(total), bounds(new), 0.1, lse=lse)
    _check(out, lse, query, c, total, bounds(new), 0.1, "float")
    assert bool((wide[:, :4] == 7).all()) and bool((wide[:, 5::2] == 7).all())


@pytest.mark.parametrize("decode", [True, False])
def test_bad_pages_and_lengths_are_skipped_and_reported(op, decode):
    lib = cabi.load()
    c = make_cache([100, 100, 100], 2, 128, 16, "token", torch.bfloat16)
    good = c["tables"].clone()
    c["tables"][0, 2] = c["k"].shape[0] + 5
    c["tables"][1, 3] = -2
    new = [1, 1, 1] if decode else [30, 30, 30]
    q = torch.randn(sum(new), 8, 128, device=DEV).bfloat16()
    out, lse = torch.empty_like(q), torch.empty(sum(new), 8, device=DEV)

    def call(total, cu=None):
        if decode:
            op.paged_attention_decode(out, q, c["k"], c["v"], c["tables"], lengths(total), 0.1, c["ks"], c["vs"], 0, lse)
        else:
            op.paged_attention_chunk(out, q, c["k"], c["v"], c["tables"], lengths(total), bounds(new) if cu is None else cu, 0.1, c["ks"], c["vs"], True, 0, lse)
        return lib.mcop_device_error()

    assert call([100, 100, 100]) == cabi.DEVERR_SLOT
    # the bad pages are as hidden as if they were not there: sequence 0 without positions 32 .. 47, sequence 1 without 48 .. 63
    for b, hole in ((0, 2), (1, 3)):
        t = good[b:b + 1]
        without = torch.cat([t[:, :hole], t[:, hole + 1:]], 1)
        rows = slice(b * new[0], (b + 1) * new[0])
        ref, rlse, spread, mass, reach = P.attention(q[rows], c["k"], c["v"], without, torch.tensor([84]), [0, new[0]], 0.1, c["ks"], c["vs"])
        tol, ltol = attention_tolerance(ref, rlse, spread, mass, reach, 128, "token", torch.bfloat16)
        compare(out[rows], ref, tol, "hole")
        compare(lse[rows], rlse, ltol, "hole lse")
    c["tables"] = good
    assert call([100, 1000, 100]) == cabi.DEVERR_KV_INDEX
    assert call([-3, 100, 100]) == cabi.DEVERR_KV_INDEX
    if not decode:
        for cu in ([0, 60, 30, 90], [0, 30, 60, 95], [-4, 30, 60, 90]):
            assert call([100, 100, 100], torch.tensor(cu, dtype=torch.int32, device=DEV)) == cabi.DEVERR_SEQUENCE, cu
        out.fill_(7)
        lse.fill_(7)
        assert call([100, 100, 100], torch.tensor([5, 30, 60, 80], dtype=torch.int32, device=DEV)) == 0
        assert bool((out[:5] == 7).all()) and bool((out[80:] == 7).all()) and bool((lse[80:] == 7).all()) and not bool((out[5:80] == 7).all(-1).any())
    assert call([100, 100, 100]) == 0


def test_offsets_beyond_32_bits(op):
    heads, D, block = 8, 128, 64
    nb = (1 << 31) // (block * heads * D) + 5
    c = make_cache([100], heads, D, block, "float", torch.bfloat16, poison=False)
    k, v = (torch.zeros(nb, block, heads, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    far = torch.tensor([[nb - 1, nb - 3]], dtype=torch.int32, device=DEV)
    for i in range(2):
        k[far[0, i].long()], v[far[0, i].long()] = c["k"][c["tables"][0, i].long()], c["v"][c["tables"][0, i].long()]
    c["k"], c["v"], c["tables"] = k, v, far
    q = torch.randn(30, 16, D, device=DEV).bfloat16()
    out, lse = torch.empty_like(q), torch.empty(30, 16, device=DEV)
    op.paged_attention_chunk(out, q, k, v, far, lengths([100]), bounds([30]), 0.1, lse=lse)
    _check(out, lse, q, c, [100], bounds([30]), 0.1, "float")
    op.paged_attention_decode(out[:1], q[:1], k, v, far, lengths([100]), 0.1, lse=lse[:1])
    _check(out[:1], lse[:1], q[:1], c, [100], bounds([1]), 0.1, "float")


def test_serving_steps_together_captured_and_on_another_stream(op):
    """Two sequences: a prefill chunk is stored (dynamic int8) and attended, then tokens are stored and decoded one by one by
    replays of one captured graph while the lengths grow; at the end the cache is read back.  The graph runs on a side stream."""
    hq, hkv, D, block, prefill, steps = 8, 2, 128, 16, [37, 80], 5
    g = torch.Generator(device=DEV).manual_seed(5)
    nb = 40
    kc, vc = (torch.zeros(nb, block, hkv, D, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(nb, block, hkv, device=DEV) for _ in range(2))
    tables = torch.randperm(nb, generator=g, device=DEV)[:12].view(2, 6).to(torch.int32)
    c = dict(k=kc, v=vc, ks=ks, vs=vs, tables=tables)

    def slots(b, p):
        return tables[b, p // block].long() * block + p % block

    T = sum(prefill)
    seq = torch.tensor([0] * prefill[0] + [1] * prefill[1], device=DEV)
    at = torch.cat([torch.arange(n, device=DEV) for n in prefill])
    q, k, v = (torch.randn(T, h, D, generator=g, device=DEV).bfloat16() for h in (hq, hkv, hkv))
    out, lse = torch.empty_like(q), torch.empty(T, hq, device=DEV)
    op.reshape_and_cache_dynamic_int8(k, v, kc, vc, ks, vs, slots(seq, at))
    op.paged_attention_chunk(out, q, kc, vc, tables, lengths(prefill), bounds(prefill), D ** -0.5, ks, vs, lse=lse)
    _check(out, lse, q, c, prefill, bounds(prefill), D ** -0.5, "token")

    q1, k1, v1 = (torch.zeros(2, h, D, device=DEV).bfloat16() for h in (hq, hkv, hkv))
    lens, where = lengths(prefill), torch.zeros(2, dtype=torch.int64, device=DEV)
    out1, lse1, out2 = torch.empty_like(q1), torch.empty(2, hq, device=DEV), torch.empty_like(q1)
    cu = bounds([1, 1])

    def step():
        op.reshape_and_cache_dynamic_int8(k1, v1, kc, vc, ks, vs, where)
        op.paged_attention_decode(out1, q1, kc, vc, tables, lens, D ** -0.5, ks, vs, 0, lse1)
        op.paged_attention_chunk(out2, q1, kc, vc, tables, lens, cu, D ** -0.5, ks, vs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    where.fill_(-1)
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        total = list(prefill)
        for i in range(steps):
            total = [n + 1 for n in total]
            p = torch.tensor(total, device=DEV) - 1
            where.copy_(slots(torch.arange(2, device=DEV), p))
            lens.copy_(torch.tensor(total, dtype=torch.int32, device=DEV))
            for x in (q1, k1, v1):
                x.copy_(torch.randn(x.shape, generator=g, device=DEV))
            graph.replay()
            _check(out1, lse1, q1, c, total, cu, D ** -0.5, "token", what=f"step {i}")
            _check(out2, lse1, q1, c, total, cu, D ** -0.5, "token", what=f"step {i} as a chunk")
    torch.cuda.current_stream().wait_stream(side)
    ko, vo = (torch.empty(sum(total), hkv, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    op.gather_and_dequant_cache(ko, vo, kc, vc, tables, bounds(total), ks, vs)
    assert torch.equal(ko[:prefill[0]], (P.rows_of(kc, ks, tables[0], prefill[0])).float().bfloat16())
    # what was written is within half a code of what was given (and half a step of bf16 of its rounding)
    # (the product code * scale is rounded to fp32 first: at most 127 * 2^-24 < 2^-17 scales)
    step_size = (k[:prefill[0]].float().abs().amax(-1, keepdim=True) / 127).double()
    off = (ko[:prefill[0]].double() - k[:prefill[0]].double()).abs()
    near = bool((off <= step_size * (0.5 + 2.0 ** -17) + ko[:prefill[0]].double().abs() * 2.0 ** -8 * (1 + 2.0 ** -7)).all())
    assert near
    assert cabi.load().mcop_device_error() == 0


def test_same_bits_every_time(op):
    c = make_cache([4000, 10, 2500], 8, 128, 16, "token", torch.bfloat16)
    q = torch.randn(3, 64, 128, device=DEV).bfloat16()
    first = None
    for _ in range(5):
        out = torch.empty_like(q)
        op.paged_attention_decode(out, q, c["k"], c["v"], c["tables"], lengths([4000, 10, 2500]), 0.1, c["ks"], c["vs"])
        first = out if first is None else first
        assert torch.equal(out, first)


def test_two_calls_at_once_on_two_streams(op):
    c = make_cache([3000, 2000], 8, 128, 16, "float", torch.bfloat16)
    q = torch.randn(400, 16, 128, device=DEV).bfloat16()
    lens, cu = lengths([3000, 2000]), bounds([300, 100])
    want_c, want_d = torch.empty_like(q), torch.empty_like(q[:2])
    op.paged_attention_chunk(want_c, q, c["k"], c["v"], c["tables"], lens, cu, 0.1)
    op.paged_attention_decode(want_d, q[:2], c["k"], c["v"], c["tables"], lens, 0.1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [(torch.empty_like(q), torch.empty_like(q[:2])) for _ in streams]
    for _ in range(5):
        for s, (oc, od) in zip(streams, outs):
            with torch.cuda.stream(s):
                op.paged_attention_chunk(oc, q, c["k"], c["v"], c["tables"], lens, cu, 0.1)
                op.paged_attention_decode(od, q[:2], c["k"], c["v"], c["tables"], lens, 0.1)
    torch.cuda.synchronize()
    for oc, od in outs:
        assert torch.equal(oc, want_c) and torch.equal(od, want_d)


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("rising", [True, False])
def test_token_scales_over_a_wide_range(op, decode, rising):
    """V scales over 2^13 along the positions (the reference of the weights has to follow), K scales over a factor of 16."""
    new, total, D = ([1] if decode else [150]), [700], 128
    c = make_cache(total, 2, D, 16, "token", torch.bfloat16, poison=False)
    at = torch.arange(700, device=DEV)
    page, off = c["tables"][0].long()[at // 16], at % 16
    power = torch.linspace(-6, 7, 700, device=DEV) * (1 if rising else -1)
    c["vs"][page, off] = (2.0 ** power)[:, None] * 0.03
    c["ks"][page, off] *= 2.0 ** torch.randint(-2, 3, (700, 1), device=DEV)
    q = torch.randn(sum(new), 8, D, device=DEV).bfloat16()
    out, lse = torch.empty_like(q), torch.empty(sum(new), 8, device=DEV)
    if decode:
        op.paged_attention_decode(out, q, c["k"], c["v"], c["tables"], lengths(total), 0.1, c["ks"], c["vs"], 0, lse)
    else:
        op.paged_attention_chunk(out, q, c["k"], c["v"], c["tables"], lengths(total), bounds(new), 0.1, c["ks"], c["vs"], True, 0, lse)
    ref, rlse, spread, mass, reach = P.attention(q, c["k"], c["v"], c["tables"], torch.tensor(total), bounds(new).tolist(), 0.1, c["ks"], c["vs"])
    tol, ltol = attention_tolerance(ref, rlse, spread, mass, reach, D, "token", torch.bfloat16)
    # f16 holds weight * scale relative to a power of two that is at most twice the largest scale seen: below 2^-14 of it the
    # rounding is absolute, 2^-25, times |code|
    codes = c["v"][page, off].abs().double().sum(0).repeat_interleave(4, 0)
    tol = tol + 2.0 ** -24 * float(c["vs"][page, off].max()) * codes
    compare(out, ref, tol, "out")
    compare(lse, rlse, ltol, "lse")


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("kind", ["head", "token"])
def test_negative_and_zero_scales(op, decode, kind):
    new, total, D = ([1, 1] if decode else [90, 3]), [300, 40], 128
    c = make_cache(total, 3, D, 16, kind, torch.bfloat16, poison=False)
    c["ks"][..., 0] *= -1
    c["ks"][..., 1] = 0
    c["vs"][..., 2] *= -1
    if kind == "token":
        c["vs"][:, ::3, 1] = 0
    q = torch.randn(sum(new), 6, D, device=DEV).bfloat16()
    out, lse = torch.empty_like(q), torch.empty(sum(new), 6, device=DEV)
    if decode:
        op.paged_attention_decode(out, q, c["k"], c["v"], c["tables"], lengths(total), 0.1, c["ks"], c["vs"], 0, lse)
    else:
        op.paged_attention_chunk(out, q, c["k"], c["v"], c["tables"], lengths(total), bounds(new), 0.1, c["ks"], c["vs"], True, 0, lse)
    _check(out, lse, q, c, total, bounds(new), 0.1, kind)


def test_more_sequences_and_more_tiles_than_a_pass_of_the_plan(op):
    """Over 1024 sequences, and one sequence of over 1024 query tiles."""
    total = [1 + i % 3 for i in range(2100)]
    c = make_cache(total, 1, 64, 2, "head", torch.bfloat16)
    new = [0 if i % 7 == 3 else 1 for i in range(2100)]
    q = torch.randn(sum(new), 2, 64, device=DEV).bfloat16()
    out, lse = torch.empty_like(q), torch.empty(sum(new), 2, device=DEV)
    op.paged_attention_chunk(out, q, c["k"], c["v"], c["tables"], lengths(total), bounds(new), 0.1, c["ks"], c["vs"], True, 0, lse)
    _check(out, lse, q, c, total, bounds(new), 0.1, "head")
    n = 40000
    c = make_cache([n], 1, 64, 64, "float", torch.bfloat16)
    q = torch.randn(n, 8, 64, device=DEV).bfloat16()
    out, lse = torch.empty_like(q), torch.empty(n, 8, device=DEV)
    op.paged_attention_chunk(out, q, c["k"], c["v"], c["tables"], lengths([n]), bounds([n]), 0.1, window=300, lse=lse)
    for lo, hi in ((0, 60), (20000, 20060), (n - 60, n)):
        ref, rlse, spread, mass, reach = P.attention(q[lo:hi], c["k"], c["v"], c["tables"], torch.tensor([hi]), [0, hi - lo], 0.1, window=300)
        tol, ltol = attention_tolerance(ref, rlse, spread, mass, reach, 64, "float", torch.bfloat16)
        compare(out[lo:hi], ref, tol, f"rows {lo}")
        compare(lse[lo:hi], rlse, ltol, f"rows {lo} lse")
