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
