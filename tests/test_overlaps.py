"""Operands that share memory are refused where that would let one write over another; those cut out of one tensor side by side are not.  Through the C
ABI with addresses that nothing is read from: calls that are accepted here stop at a null pointer behind the checks."""
import pytest

from tests.test_cache8_refusals import A, cache, read
from valora_amd import _lib

B = A + (1 << 27)      # away from the cache of those tests
ROW = 2 * 2 * 128      # bytes of a token's k of its heads


def message():
    return _lib.lib().mlora_last_error()


@pytest.mark.parametrize("kw", [dict(v=B), dict(v=B + ROW), dict(v=B + 2 * ROW), dict(v=B - ROW), dict(v=B + 3 * ROW - 16),
                                dict(k_stride=512, v_stride=512, v=B + ROW - 16), dict(k_stride=512, v_stride=512, v=B + ROW + 16),
                                dict(k_stride=512, v_stride=256, v=B + ROW), dict(k_stride=512, v_stride=512, v=B - ROW + 16)])
def test_read_results_that_overlap(kw):
    assert read(cache(), **dict(dict(n=3, k=B), **kw)) == -1 and b"k and v overlap" in message(), kw


@pytest.mark.parametrize("kw", [dict(v=B + 3 * ROW), dict(v=B - 3 * ROW), dict(n=1, v=B + ROW), dict(k_stride=512, v_stride=512, v=B + ROW),
                                dict(k_stride=512, v_stride=512, v=B - ROW), dict(k_stride=768, v_stride=768, v=B + 2 * ROW)])
def test_read_results_side_by_side(kw):
    assert read(cache(), **dict(dict(n=3, k=B, loc=None), **kw)) == -1 and b"null pointer" in message(), kw


def test_read_results_over_the_cache():
    end = A + 10 * 4096
    for at in (A, A + 4096, end - 16, A - 2 * ROW, A + (1 << 24), A + (1 << 25), A + (1 << 25) - 16):
        for kw in (dict(k=at, v=B), dict(k=B, v=at)):
            assert read(cache(), **kw, loc=A - (1 << 16)) == -1 and b"overlaps the cache" in message(), kw
    for kw in (dict(k=B, loc=B + 16), dict(k=B, v=B + (1 << 16), loc=B + (1 << 16) - 8)):
        assert read(cache(), **dict(dict(v=B + (1 << 12)), **kw)) == -1 and b"overlaps loc" in message(), kw
