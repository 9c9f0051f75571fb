"""Refusals of the paged-cache operators, without a GPU: bad arguments are turned away before any launch."""
import pytest
import torch

from mcoplib_b200 import cabi

STORE = dict(key=16, value=16, ks=1024, vs=1024, kc=16, vc=16, bs=16384, ps=1024, hs=128, ksc=16, vsc=16, slots=16, tokens=4, heads=8, D=128,
             block=16, blocks=8, dtype=1)
GATHER = dict(ko=16, vo=16, kc=16, vc=16, bs=16384, ps=1024, hs=128, ksc=16, vsc=16, mode=2, tab=16, tstride=4, maxb=4, cu=16, batch=2, tokens=9,
              heads=8, D=128, block=16, blocks=8, dtype=1)
ATT = dict(out=16, ot=1024, oh=128, lse=None, q=16, qt=1024, qh=128, kc=16, vc=16, bs=16384, ps=1024, hs=128, ksc=None, vsc=None, mode=0, tab=16,
           tstride=4, maxb=4, lens=16)
DECODE = dict(ATT, batch=2, hq=8, heads=8, D=128, block=16, blocks=8, scale=0.1, window=0, dtype=1, ws=None, wsb=0)
CHUNK = dict(ATT, cu=16, batch=2, tokens=9, hq=8, heads=8, D=128, block=16, blocks=8, scale=0.1, causal=1, window=0, dtype=1, ws=None, wsb=0)


def _call(name, base, **change):
    lib = cabi.load()
    rc = getattr(lib, name)(*dict(base, **change).values(), None)
    return rc, cabi.last_error(lib)


COMMON = [dict(kc=None), dict(vc=8), dict(bs=16385), dict(D=100), dict(D=272), dict(block=0), dict(blocks=0),
          dict(blocks=1 << 30), dict(dtype=7), dict(heads=0)]


@pytest.mark.parametrize("change", COMMON + [dict(key=None), dict(slots=None), dict(ksc=None), dict(tokens=-1), dict(key=18), dict(ks=1001),
                                             dict(vs=-1024), dict(ps=-16)])
def test_store_refuses(change):
    rc, text = _call("mcop_reshape_and_cache_dynamic_i8", STORE, **change)
    assert rc < 0 and "reshape_and_cache_dynamic_int8" in text


@pytest.mark.parametrize("change", COMMON + [dict(ko=None), dict(cu=None), dict(ksc=None), dict(mode=3), dict(mode=0, dtype=0), dict(vo=24),
                                             dict(tokens=-1), dict(batch=-1), dict(tstride=-1), dict(maxb=-1)])
def test_gather_refuses(change):
    rc, text = _call("mcop_gather_and_dequant_cache", GATHER, **change)
    assert rc < 0 and "gather_and_dequant_cache" in text


ATTENTION = COMMON + [dict(q=None), dict(out=None), dict(lens=None), dict(tab=None), dict(mode=1), dict(mode=4), dict(dtype=0), dict(hq=12),
                      dict(hq=0), dict(q=24), dict(qt=1001), dict(oh=100), dict(tstride=-1), dict(maxb=-1), dict(maxb=1 << 28, tstride=1 << 28),
                      dict(window=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(batch=-1), dict(bs=1 << 33),
                      dict(bs=-16384)]


@pytest.mark.parametrize("change", ATTENTION + [dict(ws=24, wsb=1 << 30), dict(ws=16, wsb=64)])
def test_decode_refuses(change):
    rc, text = _call("mcop_paged_attention_decode", DECODE, **change)
    assert rc < 0 and "paged_attention_decode" in text


@pytest.mark.parametrize("change", ATTENTION + [dict(cu=None), dict(tokens=-1), dict(tokens=1 << 31)])
def test_chunk_refuses(change):
    rc, text = _call("mcop_paged_attention_chunk", CHUNK, **change)
    assert rc < 0 and "paged_attention_chunk" in text


def test_empty_calls_launch_nothing():
    assert _call("mcop_reshape_and_cache_dynamic_i8", STORE, tokens=0)[0] == 0
    assert _call("mcop_gather_and_dequant_cache", GATHER, tokens=0)[0] == 0
    assert _call("mcop_paged_attention_decode", DECODE, batch=0)[0] == 0
    assert _call("mcop_paged_attention_chunk", CHUNK, tokens=0)[0] == 0
    assert _call("mcop_paged_attention_chunk", CHUNK, batch=0)[0] == 0


def test_operators_refuse_cpu_tensors_and_are_registered():
    from mcoplib_b200 import op
    cache, q = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        op.paged_attention_decode(q, q, cache, cache, table, lens, 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        op.paged_attention_chunk(q, q, cache, cache, table, lens, lens, 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        op.gather_and_dequant_cache(q, q, cache, cache, table, lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        op.reshape_and_cache_dynamic_int8(q, q, cache, cache, q, q, lens)
    for name in ("reshape_and_cache_dynamic_int8", "gather_and_dequant_cache", "paged_attention_decode", "paged_attention_chunk"):
        assert hasattr(torch.ops.mcop_C_cache_ops, name)
