"""Paged-cache operators at the corners of their contract: layouts that are refused, values that a row does not see, infinities in
padded heads, sequence bounds that are wrong, scales of any size."""
import math

import pytest
import torch

from mcoplib_b200 import cabi
from oracle import paged_ops as P
from tests.gpu_util import DEV
from tests.paged_util import HALF, attention_tolerance, bounds, compare, lengths, make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op():
    from mcoplib_b200 import op as _op
    return _op


def _attend(op, q, c, total, new=None, window=0, scale=0.1, causal=True):
    """new None: decode"""
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=DEV)
    if new is None:
        op.paged_attention_decode(out, q, c["k"], c["v"], c["tables"], lengths(total), scale, c["ks"], c["vs"], window, lse)
    else:
        op.paged_attention_chunk(out, q, c["k"], c["v"], c["tables"], lengths(total), bounds(new), scale, c["ks"], c["vs"], causal, window, lse)
    assert cabi.load().mcop_device_error() == 0
    return out, lse


def _place(c, b, pos):
    block = c["k"].shape[1]
    return int(c["tables"][b, pos // block]), pos % block


@pytest.mark.parametrize("which,int8", [("store", True)] + [(w, i) for w in ("gather", "decode", "chunk") for i in (False, True)])
def test_heads_of_the_value_cache_must_be_contiguous(op, which, int8):
    """Every other stride is that of the key cache."""
    dtype = torch.int8 if int8 else torch.bfloat16
    wide = [torch.zeros(4, 16, 2, 128, dtype=dtype, device=DEV) for _ in range(2)]
    k, v = wide[0][..., :64], wide[1][..., ::2]
    assert k.stride()[:3] == v.stride()[:3] and v.stride(3) == 2
    scales = [torch.ones(4, 16, 2, device=DEV) for _ in range(2)] if int8 else [None, None]
    x = torch.zeros(3, 2, 64, device=DEV).bfloat16()
    table = torch.zeros(3, 1, dtype=torch.int32, device=DEV)
    for pair in ((k, v), (v, k)):
        with pytest.raises(RuntimeError, match="heads of the caches must be contiguous"):
            if which == "store":
                op.reshape_and_cache_dynamic_int8(x, x, *pair, *scales, torch.arange(3, device=DEV))
            elif which == "gather":
                op.gather_and_dequant_cache(x, x.clone(), *pair, table, bounds([1, 1, 1]), *scales)
            elif which == "decode":
                op.paged_attention_decode(x.clone(), x, *pair, table, lengths([1, 1, 1]), 0.1, *scales)
            else:
                op.paged_attention_chunk(x.clone(), x, *pair, table, lengths([1, 1, 1]), bounds([1, 1, 1]), 0.1, *scales)


@pytest.mark.parametrize("size", [2.0 ** 30, 2.0 ** 100, 2.0 ** -60, 0.0])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("hq,hkv,D,dtype", [(4, 2, 128, torch.bfloat16), (3, 1, 64, torch.float16), (16, 1, 96, torch.bfloat16)])
def test_a_hidden_scale_changes_no_row(op, hq, hkv, D, dtype, window, size):
    """One K and V scale per token, finite and far from the others: rows that do not see the token keep every bit."""
    new, total = [230, 3], [700, 80]
    c = make_cache(total, hkv, D, 16, "token", dtype)
    q = torch.randn(sum(new), hq, D, device=DEV).to(dtype)
    out, lse = _attend(op, q, c, total, new, window)
    group = hq // hkv
    for pos in (300, 480, 512, 600, 699):                     # in front of every window, in the middle, at a tile's first token, the last
        w = dict(c, ks=c["ks"].clone(), vs=c["vs"].clone())
        page, off = _place(c, 0, pos)
        w["vs"][page, off, 0] = size
        w["ks"][page, off, 0] = min(size, 2.0 ** 30)
        out1, lse1 = _attend(op, q, w, total, new, window)
        for i in range(new[0]):
            mine = 470 + i
            if pos > mine or (window and pos <= mine - window):
                assert torch.equal(out1[i, :group], out[i, :group]) and torch.equal(lse1[i, :group], lse[i, :group]), (pos, i)
        assert torch.equal(out1[:, group:], out[:, group:]) and torch.equal(out1[new[0]:], out[new[0]:])


def _pages(c, n):
    at = torch.arange(n, device=DEV)
    return c["tables"][0].long()[at // c["k"].shape[1]], at % c["k"].shape[1]


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("rising", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,span", [(700, 13.0), (700, 24.0), (2000, 30.0)])
def test_scales_over_a_wide_range_by_what_each_row_sees(op, decode, rising, dtype, n, span):
    """V scales over 2^13 to 2^30 along the positions, the tolerance of each row from the tokens that it sees."""
    D, hq, hkv = 128, 8, 2
    new = None if decode else [200]
    c = make_cache([n], hkv, D, 16, "token", dtype, poison=False)
    page, off = _pages(c, n)
    power = torch.linspace(-span / 2, span / 2, n, device=DEV) * (1 if rising else -1)
    c["vs"][page, off] = (2.0 ** power)[:, None] * 2.0 ** -5
    q = (torch.randn(1 if decode else 200, hq, D, device=DEV) * 0.3).to(dtype)
    out, lse = _attend(op, q, c, [n], new)
    t = q.shape[0]
    ref, rlse, spread, mass, reach = P.attention(q, c["k"], c["v"], c["tables"], torch.tensor([n]), [0, t], 0.1, c["ks"], c["vs"])
    # without the part for small weights: that one stands below, from the row's own tokens
    tol, ltol = attention_tolerance(ref, rlse, spread, torch.zeros_like(mass), reach, D, "token", dtype)
    K = P.rows_of(c["k"], c["ks"], c["tables"][0], n)
    code = c["v"][page, off].double().abs()
    vs = c["vs"][page, off].double()
    seen = torch.arange(n, device=DEV)[None, :] <= torch.arange(n - t, n, device=DEV)[:, None]
    for h in range(hq):
        g = h // (hq // hkv)
        x = torch.where(seen, 0.1 * (q[:, h].double() @ K[:, g].T), -math.inf)
        p = torch.softmax(x, -1)
        # f16 holds the products of weight and scale; below 2^-14 of what they are held relative to, the rounding is absolute, 2^-25.
        # Decode: relative to at most the row's largest product, which is 1 or more as it is formed.  Chunk: to at
        # most the largest weight times a power of two that is at most twice the largest scale that the row sees.
        unit = (p * vs[:, g]).amax(-1) if decode else 2 * torch.where(seen, vs[:, g], 0.0).amax(-1) * p.amax(-1)
        tol[:, h] += 2.0 ** -25 * unit[:, None] * (seen.double() @ code[:, g])
    compare(out, ref, tol, "out")
    compare(lse, rlse, ltol, "lse")


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [16, 48, 64, 80, 96, 128, 144, 256])
def test_an_infinity_in_k_that_makes_a_logit_minus_infinity(op, D, dtype, decode):
    """Such a token has weight 0 whatever the head size is padded to; one that a row does not see has no effect at all."""
    total, hq, hkv = [300, 50], 4, 2
    new = None if decode else [40, 5]
    c = make_cache(total, hkv, D, 16, "float", dtype)
    q = torch.randn(2 if decode else 45, hq, D, device=DEV).to(dtype)
    q[..., 0] = q[..., 0].abs() + 0.5
    q[..., -1] = -q[..., -1].abs() - 0.5
    _, _, _, _, reach = P.attention(q, c["k"], c["v"], c["tables"], torch.tensor(total), bounds(new or [1, 1]).tolist(), 0.1)
    for pos, d, value in ((7, 0, -math.inf), (100, D - 1, math.inf), (250, D - 1, math.inf)):
        page, off = _place(c, 0, pos)
        c["k"][page, off, 0, d] = value
    out, lse = _attend(op, q, c, total, new)
    ref, rlse, spread, mass, _ = P.attention(q, c["k"], c["v"], c["tables"], torch.tensor(total), bounds(new or [1, 1]).tolist(), 0.1)
    tol, ltol = attention_tolerance(ref, rlse, spread, mass, reach, D, "float", dtype)  # (the reach of the finite logits)
    assert bool(ref.isfinite().all())
    compare(out, ref, tol, "out")
    compare(lse, rlse, ltol, "lse")


@pytest.mark.parametrize("D", [64, 80, 128, 192])
def test_decode_takes_no_part_of_hidden_nan_and_infinity(op, D):
    total, window = [300], 60
    c = make_cache(total, 2, D, 16, "float", torch.bfloat16)
    q = torch.randn(1, 8, D, device=DEV).bfloat16()
    want = _attend(op, q, c, total, window=window)
    for pos, name, value in ((0, "v", math.nan), (200, "k", math.inf), (239, "v", -math.inf), (238, "k", math.nan)):
        page, off = _place(c, 0, pos)
        c[name][page, off, :, D - 3] = value
    got = _attend(op, q, c, total, window=window)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kind", ["float", "token"])
@pytest.mark.parametrize("cu,kept", [
    ([0, 30, 20, 40], [(40, 50)]),              # descends: sequence 1 has no rows, 0 and 2 overlap
    ([-4, 10, 20, 30], [(0, 10), (30, 50)]),    # begins in front of the buffer: sequence 0 is left out
    ([0, 10, 20, 60], [(20, 50)]),              # ends behind it: sequence 2 is left out
    ([0, 10, 60, 70], [(10, 50)]),
])
def test_read_back_leaves_out_and_reports_sequences_outside_the_buffer(op, kind, cu, kept):
    c = make_cache([64, 64, 64], 2, 64, 16, kind, torch.bfloat16, poison=False)
    out = [torch.full((50, 2, 64), 7.0, device=DEV).bfloat16() for _ in range(2)]
    op.gather_and_dequant_cache(*out, c["k"], c["v"], c["tables"], torch.tensor(cu, dtype=torch.int32, device=DEV), c["ks"], c["vs"])
    assert cabi.load().mcop_device_error() == cabi.DEVERR_SEQUENCE
    untouched = torch.zeros(50, dtype=torch.bool, device=DEV)
    for a, b in kept:
        untouched[a:b] = True
    for o, cache, scale in zip(out, (c["k"], c["v"]), (c["ks"], c["vs"])):
        assert bool((o[untouched] == 7).all())
        rows = [P.rows_of(cache, scale, c["tables"][b], 64).float().bfloat16() for b in range(3)]
        for t in torch.nonzero(~untouched).flatten().tolist():
            mine = [rows[b][t - cu[b]] for b in range(3) if 0 <= cu[b] <= t < cu[b + 1] <= 50]
            assert any(torch.equal(o[t], r) for r in mine), t


def test_read_back_reports_bad_bounds_that_no_row_meets(op):
    c = make_cache([5] * 700, 1, 32, 16, "float", torch.bfloat16, poison=False)
    cu = bounds([0] * 650 + [5] * 50)
    cu[300] = -1                                              # an empty sequence in front of the buffer, one that descends
    out = [torch.empty(250, 1, 32, device=DEV).bfloat16() for _ in range(2)]
    op.gather_and_dequant_cache(*out, c["k"], c["v"], c["tables"], cu)
    assert cabi.load().mcop_device_error() == cabi.DEVERR_SEQUENCE


def test_store_of_fp32_rows_from_the_smallest_to_infinity(op):
    """Subnormal scales, rows near the largest float, and rows that hold infinities or NaN: scale NaN, codes 0, which equal only themselves."""
    g = torch.Generator(device=DEV).manual_seed(3)
    size = torch.tensor([0.0, 1e-44, 1e-42, 1e-38, 1e-36, 1.0, 1e30, 1e38, 1e38, 3e38], device=DEV)
    key, value = (torch.randn(10, 3, 48, generator=g, device=DEV).clamp(-1, 1) * size[:, None, None] for _ in range(2))
    value[8, 0, 5], value[8, 2, 47], key[9, 1, 0] = math.inf, -math.inf, math.nan
    kc, vc = (torch.full((2, 5, 3, 48), 9, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.full((2, 5, 3), 9.0, device=DEV) for _ in range(2))
    ref = [x.clone() for x in (kc, vc, ks, vs)]
    slots = torch.randperm(10, generator=g, device=DEV)
    P.store(key, value, *ref, slots)
    op.reshape_and_cache_dynamic_int8(key, value, kc, vc, ks, vs, slots)
    for got, want in zip((kc, vc, ks, vs), ref):
        assert bool(((got == want) | (got.isnan() & want.isnan())).all())
    assert int(ref[2].isnan().sum()) == 1 and int(ref[3].isnan().sum()) == 2


@pytest.mark.parametrize("window", [0, 500])
def test_nan_and_infinity_in_a_long_context(op, window):
    """Non-finite elements of V in tiles that all rows of an item see, and in those that some see, thousands of tokens in."""
    new, total, hq, hkv, D = [300], [6000], 4, 2, 128
    c = make_cache(total, hkv, D, 16, "float", torch.bfloat16)
    q = torch.randn(300, hq, D, device=DEV).bfloat16()
    good, lse0 = _attend(op, q, c, total, new, window)
    special = [(64, 9, math.inf), (5400, 9, -math.inf), (5820, 40, math.inf), (5990, 77, math.nan), (5999, 127, -math.inf)]
    for pos, d, value in special:
        page, off = _place(c, 0, pos)
        c["v"][page, off, 0, d] = value
    out, lse = _attend(op, q, c, total, new, window)
    assert torch.equal(lse, lse0) and torch.equal(out[:, 2:], good[:, 2:])
    for i in range(300):
        mine = 5700 + i
        hit = {}
        for pos, d, value in special:
            if pos <= mine and (not window or pos > mine - window):
                hit[d] = hit.get(d, 0.0) + value              # inf - inf is NaN, as in the sum itself
        want = good[i, :2].float()
        for d, value in hit.items():
            want[:, d] = value
        assert torch.equal(torch.nan_to_num(out[i, :2].float(), nan=-5.0, posinf=1e30, neginf=-1e30),
                           torch.nan_to_num(want, nan=-5.0, posinf=1e30, neginf=-1e30)), i


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("power", [-85, -62, 40, 62, 90])
def test_v_scales_of_any_size(op, decode, power):
    """All V scales times a power of two: the output takes it over, the log-sum-exp knows nothing of it."""
    total, D = [900, 33], 128
    new = None if decode else [70, 33]
    c = make_cache(total, 2, D, 16, "token", torch.bfloat16, poison=False)
    q = (torch.randn(2 if decode else 103, 8, D, device=DEV) * 0.3).bfloat16()
    c["vs"] *= 2.0 ** power
    out, lse = _attend(op, q, c, total, new)
    cu = bounds(new or [1, 1]).tolist()
    ref, rlse, spread, mass, reach = P.attention(q, c["k"], c["v"], c["tables"], torch.tensor(total), cu, 0.1, c["ks"], c["vs"])
    tol, ltol = attention_tolerance(ref, rlse, spread, mass, reach, D, "token", torch.bfloat16)
    # Weights are formed as 2^(x - r) with |r| <= 128: rounding the exponent moves them by at most 2^-18 * ln 2, half a step of a number
    # below 128, and log2 of their sum, below 128 in size, is off by two such steps
    compare(out, ref, tol + 2.0 ** -18 * spread, "out")
    compare(lse, rlse, ltol + 2.0 ** -16, "lse")


@pytest.mark.parametrize("kind", ["float", "token"])
@pytest.mark.parametrize("D", [64, 192])
def test_a_table_without_columns(op, kind, D):
    """Nothing is cached yet: a table of no pages per sequence is as good as an unused one."""
    c = make_cache([0, 0, 0], 2, D, 16, kind, torch.bfloat16)
    c["tables"] = torch.empty(3, 0, dtype=torch.int32, device=DEV)
    for new in (None, [2, 0, 3]):
        q = torch.randn(3 if new is None else 5, 4, D, device=DEV).bfloat16()
        out, lse = _attend(op, q, c, [0, 0, 0], new)
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    rows = [torch.full((4, 2, D), 7.0, device=DEV).bfloat16() for _ in range(2)]
    op.gather_and_dequant_cache(*rows, c["k"], c["v"], c["tables"], bounds([0, 0, 0]), c["ks"], c["vs"])
    assert bool((rows[0] == 7).all()) and bool((rows[1] == 7).all()) and cabi.load().mcop_device_error() == 0
