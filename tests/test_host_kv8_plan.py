"""The plan by which the 8-bit cache attention shares out its tiles: every tile of
every batch has a CTA.  Host only."""
import ctypes
import random

import pytest

from focal_b200 import _lib

ONE_CTA = {64: 18, 128: 12}  # tiles that one CTA takes whole, whatever the lengths


def covered(segs, per_seg, D, code, sms, total, top, out):
    """Whether the plan's CTAs reach the last tile, and what it writes fits into the workspace."""
    rc = _lib.lib().focal_kv8_decode_plan(segs, 64 * per_seg, D, code, sms, total, top, out)
    ctas, ways, per, ws = out
    if rc != 0 or not 1 <= ctas <= min(sms, 256):
        return False
    if ways:  # CTA c has part c % ways of segment c / ways
        return ctas >= segs * ways and per * ways >= top
    return ctas * per >= total


@pytest.mark.parametrize("D,code,sms", [(128, 0, 148), (64, 1, 148), (128, 1, 132), (64, 0, 16), (128, 0, 1), (64, 0, 300)])
def test_equal_lengths_are_covered(D, code, sms):
    """All segments have `top` tiles, `per_seg` is what the host was told."""
    out, bad = (ctypes.c_int * 4)(), []
    for segs in range(1, 2001):
        for per_seg in range(1, 41) if (D, code, sms) == (128, 0, 148) else (1, 2, 3, 4, 7, 12, 13, 18, 19, 40):
            for top in range(1, per_seg + 1):
                if not covered(segs, per_seg, D, code, sms, segs * top, top, out):
                    bad.append((segs, per_seg, top, list(out)))
    assert not bad, (len(bad), bad[:5])


def test_any_lengths_are_covered():
    rng = random.Random(1)
    out, bad = (ctypes.c_int * 4)(), []
    for _ in range(200000):
        segs = int(2 ** rng.uniform(0, 13))
        per_seg = int(2 ** rng.uniform(0, min(24, 30 - segs.bit_length())))
        top = rng.randint(0, per_seg)
        total = rng.randint(top, segs * top) if rng.random() < 0.7 else segs * top
        D, code, sms = rng.choice((64, 128)), rng.choice((0, 1)), rng.choice((148, 148, 132, 78, 160))
        if not covered(segs, per_seg, D, code, sms, total, top, out):
            bad.append((segs, per_seg, top, total, D, code, sms, list(out)))
    assert not bad, (len(bad), bad[:5])


def test_plan_fits_its_workspace():
    L, out = _lib.lib(), (ctypes.c_int * 4)()
    for D in (64, 128):
        for B in [*range(1, 700), 1000, 5000, 60000]:
            for per_seg in (1, 2, 3, 5, 12, 13, 20, 300):
                assert L.focal_kv8_decode_plan(B, 64 * per_seg, D, 0, 148, B * per_seg, per_seg, out) == 0
                assert out[3] <= L.focal_kv8_decode_workspace_size(B, 1, 1, 1, 64 * per_seg, D)


def test_plan_uses_the_gpu():
    """Batches of short sequences with more segments than SMs: no CTA has more than one
    segment above its share."""
    out = (ctypes.c_int * 4)()
    for segs in range(149, 1500):
        assert covered(segs, 1, 128, 0, 148, segs, 1, out)
        assert out[2] <= max(4, -(-segs // 148))


def test_plan_refusals():
    L, out = _lib.lib(), (ctypes.c_int * 4)()
    for args in ((0, 64, 128, 0, 148, 1, 1), (1, 0, 128, 0, 148, 1, 1), (1, 64, 128, 0, 0, 1, 1), (1, 64, 96, 0, 148, 1, 1),
                 (1, 64, 128, 2, 148, 1, 1), (1 << 20, 1 << 20, 128, 0, 148, 1, 1), (1, 64, 128, 0, 148, 2, 2),
                 (2, 64, 128, 0, 148, 3, 1), (1, 64, 128, 0, 148, -1, 1), (1, 64, 128, 0, 148, 0, -1)):
        assert L.focal_kv8_decode_plan(*args, out) != 0 and _lib.last_error()
    assert L.focal_kv8_decode_plan(1, 64, 128, 0, 148, 1, 1, None) == _lib.FOCAL_ERR_INVALID_VALUE
