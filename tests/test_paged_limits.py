"""Sizes at the end of the 32-bit range, without a GPU: refused before any launch."""
import pytest

from tests.test_paged_cache_refusals import CHUNK, DECODE, _call

LIMIT = (1 << 31) - 1 - 255  # positions of a table, (token, query head) rows of a call


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("block", [1, 16, 255])
@pytest.mark.parametrize("name,base", [("mcop_paged_attention_decode", DECODE), ("mcop_paged_attention_chunk", CHUNK)])
def test_tables_of_nearly_2_31_positions(name, base, block, D):
    first = LIMIT // block + 1                               # the narrowest table that is refused, and the widest there is
    for maxb in (first, ((1 << 31) - 1) // block):
        rc, text = _call(name, base, maxb=maxb, tstride=maxb, block=block, D=D)
        assert rc < 0 and "block table too wide" in text, maxb
    # one page less passes that check (and is stopped by the missing workspace)
    rc, text = _call(name, base, maxb=first - 1, tstride=first - 1, block=block)
    assert rc < 0 and "workspace" in text


@pytest.mark.parametrize("tokens,hq,refused", [((1 << 31) - 1, 8, True), (LIMIT // 8, 8, False), (LIMIT // 8 + 1, 8, True), ((1 << 28) - 1, 8, True),
                                               (LIMIT // 64 + 1, 64, True), (LIMIT // 64, 64, False)])
def test_chunks_of_nearly_2_31_rows(tokens, hq, refused):
    rc, text = _call("mcop_paged_attention_chunk", CHUNK, tokens=tokens, hq=hq)
    assert rc < 0 and ("query rows" if refused else "workspace") in text
