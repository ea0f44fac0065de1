"""Operands that share memory are refused where that would let one write over another; those cut out of one tensor side by side are not.  Through the C
ABI with addresses that nothing is read from: calls that are accepted here stop at a null pointer behind the checks."""
import random

import pytest

from tests.test_cache8_refusals import A, cache, norm, read, store
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


def part(**kw):
    p = dict(src=B, dst=B, src_token_stride=512, src_head_stride=128, dst_token_stride=512, dst_head_stride=128, heads=4, flags=1)
    p.update(kw)
    return _lib.RotaryPart(*[p[n] for n, _ in _lib.RotaryPart._fields_])


def stored(q, k, v, T, k_strides=(256, 128), v_strides=(256, 128), positions=A - (1 << 20), loc=A - (1 << 19)):
    """Whether the call gets as far as the missing frequencies, or what it says."""
    rc = _lib.lib().mlora_rotary_store_codes(None, q, k, *k_strides, v, *v_strides, cache(), positions, loc, T, 128, 0, None, 1.0, 0)
    assert rc == -1
    return b"null pointer" in message() or message()


def test_q_out_over_what_the_call_reads():
    far, wide = B + (1 << 20), dict(src_token_stride=1024, dst_token_stride=1024)
    # in place, in a tensor of q, k and v side by side or head by head, or elsewhere
    assert stored(part(), far, far + (1 << 16), 3) is True
    assert stored(part(**wide), B + 1024, B + 1536, 3, (1024, 128), (1024, 128)) is True
    by_head = dict(src_token_stride=1536, dst_token_stride=1536, src_head_stride=384, dst_head_stride=384)
    assert stored(part(**by_head, heads=2), B + 256, B + 512, 3, (1536, 384), (1536, 384)) is True
    assert stored(part(dst=far), B + (1 << 16), B + (1 << 17), 3) is True
    # a token's or a head's place off, or in other strides
    for kw in (dict(dst=B + 1024), dict(dst=B - 1024), dict(dst=B + 256), dict(dst_token_stride=520), dict(dst=B + 16)):
        assert b"other heads of q" in stored(part(**kw), far, far + (1 << 16), 3), kw
    # k or v
    for at in (B, B + 256, B + 2 * 1024, B - 512, B + 3 * 1024 - 16):
        assert b"overlaps k or v" in stored(part(), at, far, 3) and b"overlaps k or v" in stored(part(), far, at, 3), at
    assert b"overlaps k or v" in stored(part(**wide), B + 1008, B + 1536, 3, (1024, 128), (1024, 128))
    for kw in (dict(positions=B + 8), dict(loc=B - 16)):
        assert b"positions or loc" in stored(part(), far, far + (1 << 16), 3, **kw)


def test_powers_over_codes():
    for kw in (dict(powers=A), dict(powers=A + 10 * 4096 - 2), dict(powers=A + (1 << 24) + 64), dict(key_stride=4160, powers=A + 4094, powers_stride=4160)):
        assert store(cache(**kw)) == -1 and b"powers overlap codes" in message(), kw
    page = dict(key_stride=4160, powers=A + 4096, powers_stride=4160)       # behind the keys' codes of each page
    assert store(cache(**page), T=0) == 0


def test_heads_of_any_strides_against_every_element():
    """Nothing that overlaps gets through, and where the two have the same strides, and rows do not interleave, nothing else is refused."""
    rng = random.Random(3)
    seen = {True: 0, False: 0}
    for _ in range(2000):
        T, hq, extra = rng.randint(1, 4), rng.randint(1, 4), 8 * rng.randint(0, 40)
        head = 128 + 8 * rng.randint(0, 40)
        token = max(head * max(hq, 2), 128) + extra
        other = rng.random() < 0.3
        k_head, k_token = (8 * rng.randint(0, 60), 8 * rng.randint(0, 200)) if other else (head, token)
        k = B + 16 * rng.randint(-token * T // 8, token * T // 8)
        taken = lambda at, n, t, h: {(at - B) // 16 + (i * t + j * h) // 8 + e for i in range(T) for j in range(n) for e in range(16)}  # noqa: E731
        q = part(heads=hq, src_token_stride=token, dst_token_stride=token, src_head_stride=head, dst_head_stride=head)
        meets = bool(taken(B, hq, token, head) & taken(k, 2, k_token, k_head))
        said = stored(q, k, A - (1 << 24), T, (k_token, k_head))
        seen[meets] += 1
        if meets:
            assert said is not True and b"overlaps k or v" in said
        elif not other:
            assert said is True, (T, hq, token, head, (k - B) // 2)
    assert min(seen.values()) > 200


def test_norm_results_beside_operands_in_one_tensor():
    """Columns of one tensor are apart where their rows are; a shift by part of a row is not.  (x is missing: what is accepted gets as far as that.)"""
    L = _lib.lib()
    wide = dict(block_stride=256, residual_stride=256, out_stride=256)

    def call(**kw):
        assert L.mlora_block_norm(None, norm(**dict(dict(x=None, x_stride=64), **kw)), 0) == -1
        return b"null pointer" in message() or message()

    assert call(block=B, residual_out=B + 128, out=B + 256, **wide) is True
    assert call(block=B + 256, residual_out=B + 128, out=B, **wide) is True
    assert call(block=B, residual_out=B + 384, gate=B + 128, gate_row_stride=256, **wide) is True
    assert call(block=B, residual_out=B + 384, gate=B + 128, gate_row_stride=256, gate_column_stride=0, **wide) is True
    assert call(block=B, residual_out=B + 128, weight=B + 256, **wide) is True                         # between the first row and the second
    assert call(block=B, out=B + 128, bias=B + 384, f32=2, **wide) is True
    assert call(block=B, residual_out=B + 256, gate=B + 384, gate_row_stride=128, gate_column_stride=0, f32=16, **wide) is True
    for kw, said in ((dict(residual_out=B + 126), b"other rows"), (dict(residual_out=B + 512 - 126), b"other rows"), (dict(out=B + 512), b"other rows"),
                     (dict(residual_out=B + 128, out=B + 130), b"results overlap"), (dict(residual_out=B + 128, out=B + 640), b"results overlap"),
                     (dict(residual_out=B + 128, gate=B + 254, gate_row_stride=256, gate_column_stride=0), b"gate"),
                     (dict(residual_out=B + 128, weight=B + 638), b"vector"), (dict(out=B + 128, bias=B + 388, f32=2), b"vector"),
                     (dict(residual_out=B + 256, gate=B + 380, gate_row_stride=128, gate_column_stride=0, f32=16), b"gate")):
        got = call(**dict(dict(block=B), **wide), **kw)
        assert got is not True and said in got, (kw, got)
