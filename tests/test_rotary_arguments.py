"""Destinations of the rotary call whose heads would share elements, refused without a GPU; the gain of a context made shorter."""
import math

import pytest

from valora_amd import _lib
from valora_amd.rotary import frequencies


def rotary(T, rows, **kw):
    p = dict(src=4096, dst=8192, src_token_stride=256, src_head_stride=64, dst_token_stride=256, dst_head_stride=64, heads=4, flags=3 if rows else 1)
    p.update(kw)
    part = _lib.RotaryPart(*[p[n] for n, _ in _lib.RotaryPart._fields_])
    # (without positions: what passes the checks of strides is refused behind them, and nothing is launched)
    return _lib.lib().mlora_rotary(None, part, 1, None, 64, rows, T, 64, 64, 0, 64, 1.0, 0)


@pytest.mark.parametrize("T,rows", [(3, 0), (1, 7), (3, 7)])
@pytest.mark.parametrize("token,head,ok", [
    (256, 64, True), (264, 64, True), (64, 64, False), (128, 64, False), (255, 64, False), (64, 128, False), (200, 100, False),
    (64, 64 * 7, True), (64, 64 * 7 - 1, False), (64, 1 << 40, True), (1 << 62, 64, True), (1 << 62, 1 << 60, True), (1 << 62, 1 << 61, False), (1 << 61, 1 << 62, False), (1, 64, False),
    (364, 100, True), (363, 100, False)])
def test_tokens_and_heads_that_share_elements(T, rows, token, head, ok):
    if not rows and (token, head) == (64, 64 * 7 - 1):
        ok = True                                        # (three tokens, not seven rows)
    rc = rotary(T, rows, dst_token_stride=token, dst_head_stride=head)
    message = _lib.lib().mlora_last_error()
    assert rc == -1 and (b"null pointer" if ok else b"overlap") in message, (rc, message)


def test_one_head_or_one_token_alone():
    """Only the stride that counts is looked at."""
    for T, rows, kw, ok in ((1, 0, dict(dst_token_stride=0), True), (1, 0, dict(dst_token_stride=64), True), (5, 0, dict(heads=1, dst_head_stride=0), True),
                            (5, 9, dict(heads=1, dst_token_stride=64, dst_head_stride=0), True), (5, 0, dict(heads=1, dst_token_stride=63), False),
                            (1, 0, dict(dst_head_stride=63), False), (1, 1, dict(dst_token_stride=0), True)):
        assert rotary(T, rows, **kw) == -1
        assert (b"null pointer" if ok else b"overlap") in _lib.lib().mlora_last_error(), kw


def test_yarn_gain_of_a_shorter_context():
    """Only a longer context sharpens the scores."""
    for factor in (1e-6, 0.25, 0.999, 1.0):
        assert frequencies(64, scaling=dict(type="yarn", factor=factor, original_max_position=4096))[1] == 1.0
        assert frequencies(64, scaling=dict(type="yarn", factor=factor, original_max_position=4096, attention_factor=0.5))[1] == 0.5
    assert frequencies(64, scaling=dict(type="yarn", factor=4.0, original_max_position=4096))[1] == 0.1 * math.log(4.0) + 1.0
