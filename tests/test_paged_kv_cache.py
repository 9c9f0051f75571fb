"""The dynamic int8 store and the read-back of the paged cache against their formulas in 64 bits."""
import math

import pytest
import torch

from mcoplib_b200 import cabi
from oracle import paged_ops as P
from tests.gpu_util import DEV, Canary
from tests.paged_util import bounds, make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op():
    from mcoplib_b200 import op as _op
    return _op


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,D,block", [(1, 1, 16, 1), (7, 3, 96, 24), (64, 8, 128, 16), (33, 2, 256, 5), (130, 1, 64, 32), (5, 4, 80, 16)])
def test_store_codes_and_scales_are_exact(op, tokens, heads, D, block, dtype):
    g = torch.Generator(device=DEV).manual_seed(tokens + D)
    key, value = (torch.randn(tokens, heads, D, generator=g, device=DEV).to(dtype) for _ in range(2))
    value[0] = 0.0                                            # a row of zeros
    key[-1] *= 2.0 ** -13                                     # small values (subnormal f16 among them)
    if tokens > 4:
        value[1] = (torch.arange(D, device=DEV) % 128).to(dtype)   # whole numbers up to 127 and ...
        value[2] = (torch.arange(D, device=DEV) % 128 + 0.5).to(dtype)
        value[2, :, 0] = 254.0                                # ... midpoints: s = 2, x / s = n + 1/4, and 63.5 at x = 127
        value[2, :, 1] = 127.0
        value[3, :, 5] = math.inf
        key[3, :, 7] = math.nan
    nb = -(-tokens // block) + 2
    slots = torch.randperm(nb * block, generator=g, device=DEV)[:tokens].long()
    if tokens > 4:
        slots[4] = -1
    shape = (nb, block, heads, D)
    kc, vc = Canary(shape, torch.int8, 3), Canary(shape, torch.int8, 3)
    ks, vs = Canary(shape[:3], torch.float32, 9), Canary(shape[:3], torch.float32, 9)
    ref = [x.t.clone() for x in (kc, vc, ks, vs)]
    P.store(key, value, *ref, slots)
    op.reshape_and_cache_dynamic_int8(key, value, kc.t, vc.t, ks.t, vs.t, slots)
    for got, want, name in zip((kc, vc, ks, vs), ref, ("key codes", "value codes", "key scales", "value scales")):
        got.check(name)
        assert torch.equal(torch.nan_to_num(got.t.double(), nan=-1.0), torch.nan_to_num(want.double(), nan=-1.0)), name
    assert cabi.load().mcop_device_error() == 0


def test_store_of_tiny_and_huge_fp32_rows(op):
    """Scales in the subnormal range, where 1 / s would overflow, and rows near the largest float."""
    key = torch.randn(6, 1, 32, device=DEV) * torch.tensor([1e-44, 1e-42, 1e-38, 1e-36, 1e30, 1e38], device=DEV)[:, None, None].clamp(max=1e38)
    kc, vc = (torch.zeros(1, 6, 1, 32, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(1, 6, 1, device=DEV) for _ in range(2))
    ref = [x.clone() for x in (kc, vc, ks, vs)]
    slots = torch.arange(6, device=DEV)
    P.store(key, key, *ref, slots)
    op.reshape_and_cache_dynamic_int8(key, key, kc, vc, ks, vs, slots)
    assert torch.equal(ks, ref[2]) and torch.equal(kc, ref[0]) and torch.equal(vc, ref[1])


def test_store_takes_strided_rows_and_caches_and_skips_bad_slots(op):
    packed = torch.randn(40, 12, 64, device=DEV).bfloat16()   # q, k and v of a token beside one another
    key, value = packed[:, 8:10], packed[:, 10:12]
    both = torch.zeros(6, 2, 16, 2, 64, dtype=torch.int8, device=DEV)  # K and V of a block beside one another
    ks, vs = (torch.zeros(6, 16, 2, device=DEV) for _ in range(2))
    slots = torch.randperm(96, device=DEV)[:40].long()
    slots[7] = 96
    slots[8] = 1 << 40
    ref = [both[:, 0].clone(), both[:, 1].clone(), ks.clone(), vs.clone()]
    P.store(key, value, *ref, slots)
    op.reshape_and_cache_dynamic_int8(key, value, both[:, 0], both[:, 1], ks, vs, slots)
    for got, want in zip((both[:, 0], both[:, 1], ks, vs), ref):
        assert torch.equal(got, want)
    assert cabi.load().mcop_device_error() == cabi.DEVERR_SLOT


@pytest.mark.parametrize("kind,dtype", [("float", torch.bfloat16), ("float", torch.float16), ("head", torch.bfloat16), ("token", torch.float16),
                                        ("token", torch.float32)])
@pytest.mark.parametrize("total,heads,D,block", [([1], 1, 16, 1), ([0, 5, 17, 0, 33, 0], 3, 96, 24), ([100, 1, 64], 8, 128, 16), ([9] * 70, 2, 64, 4),
                                                 ([3, 500], 1, 256, 16), ([1] * 1500, 1, 32, 2)])
def test_read_back(op, kind, dtype, total, heads, D, block):
    c = make_cache(total, heads, D, block, kind, dtype, poison=False)
    n, extra = sum(total), 3                                   # rows behind the last sequence stay as they were
    ko, vo = (Canary((n + extra, heads, D), dtype, 5) for _ in range(2))
    op.gather_and_dequant_cache(ko.t, vo.t, c["k"], c["v"], c["tables"], bounds(total), c["ks"], c["vs"])
    for out, cache, scale in ((ko, c["k"], c["ks"]), (vo, c["v"], c["vs"])):
        out.check()
        # code * scale has 31 bits: exact in 64, and rounded to fp32 first (as the operator does), then to the output type
        want = torch.cat([P.rows_of(cache, scale, c["tables"][b], t) for b, t in enumerate(total)]).float().to(dtype)
        assert torch.equal(out.t[:n], want)
        assert bool((out.t[n:] == 5).all())
    assert cabi.load().mcop_device_error() == 0


def test_read_back_leaves_rows_of_bad_pages(op):
    c = make_cache([20, 20], 2, 64, 16, "token", torch.bfloat16, poison=False)
    c["tables"][0, 1] = c["k"].shape[0]
    c["tables"][1, 0] = -1
    out = [torch.full((50, 2, 64), 7.0, device=DEV).bfloat16() for _ in range(2)]
    op.gather_and_dequant_cache(*out, c["k"], c["v"], c["tables"], torch.tensor([3, 23, 43], dtype=torch.int32, device=DEV), c["ks"], c["vs"])
    assert cabi.load().mcop_device_error() == cabi.DEVERR_SLOT
    kept = torch.zeros(50, dtype=torch.bool)
    kept[:3] = kept[19:39] = kept[43:] = True
    for o in out:
        assert bool((o[kept.to(DEV)] == 7).all())
        assert not bool((o[~kept.to(DEV)] == 7).all())
    # longer than the table, and bounds that descend
    op.gather_and_dequant_cache(*out, c["k"], c["v"], c["tables"][:1, :1], torch.tensor([0, 40], dtype=torch.int32, device=DEV), c["ks"], c["vs"])
    assert cabi.load().mcop_device_error() == cabi.DEVERR_KV_INDEX
    op.gather_and_dequant_cache(*out, c["k"], c["v"], c["tables"], torch.tensor([0, -5, 40], dtype=torch.int32, device=DEV), c["ks"], c["vs"])
    assert cabi.load().mcop_device_error() in (0, cabi.DEVERR_SEQUENCE, cabi.DEVERR_KV_INDEX, cabi.DEVERR_SLOT)


def test_offsets_beyond_32_bits(op):
    """The last pages of a cache of more than 2^31 elements."""
    heads, D, block = 8, 256, 64
    nb = (1 << 31) // (block * heads * D) + 5
    kc, vc = (torch.zeros(nb, block, heads, D, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(nb, block, heads, device=DEV) for _ in range(2))
    x, y = (torch.randn(100, heads, D, device=DEV).bfloat16() for _ in range(2))
    table = torch.tensor([[nb - 1, nb - 3]], dtype=torch.int32, device=DEV)
    at = torch.arange(100, device=DEV)
    op.reshape_and_cache_dynamic_int8(x, y, kc, vc, ks, vs, table[0].long()[at // block] * block + at % block)
    xo, yo = (torch.empty(100, heads, D, device=DEV) for _ in range(2))
    op.gather_and_dequant_cache(xo, yo, kc, vc, table, bounds([100]), ks, vs)
    for a, b in ((x, xo), (y, yo)):
        # half a code, and half an fp32 step of the product code * scale: |code| <= 127, so at most 127 * 2^-24 < 2^-17 scales
        step = (a.float().abs().amax(-1, keepdim=True) / 127).double()
        near = bool(((a.double() - b.double()).abs() <= step * (0.5 + 2.0 ** -17)).all())
        assert near
