"""Limits of the 8-bit cache calls that depend on several sizes together; host only."""
import ctypes

import pytest

from focal_b200 import _lib
from test_host_kv8 import decode, refused

# B, T, Hq, Hkv, max_seq_len: one below and one above 2^30 tiles of 64 positions and 16 query rows
MANY = [(16384, 1, 1, 1, 64 * 65536), (8191, 1, 32, 8, 64 * 16385), (4095, 16, 16, 1, 64 * 16388)]


@pytest.mark.parametrize("B,T,Hq,Hkv,most", MANY)
def test_tile_count_is_refused_everywhere(B, T, Hq, Hkv, most):
    """The workspace query refuses what the call would refuse, so a composite can ask before it writes."""
    size = _lib.lib().focal_kv8_decode_workspace_size
    chunks = -(-T * (Hq // Hkv) // 16)
    tiles = lambda n: B * Hkv * chunks * (-(-n // 64))  # noqa: E731
    low = most
    while tiles(low) >= 1 << 30:
        low -= 64
    high = low
    while tiles(high) < 1 << 30:
        high += 64
    assert size(B, T, Hq, Hkv, low, 128) > 0
    assert size(B, T, Hq, Hkv, high, 128) == 0
    assert "too large" in _lib.last_error()
    c = _lib.Kv8Cache(1 << 20, 1 << 20, 1 << 20, 1 << 20, 8, Hkv, 32, 128, _lib.FOCAL_E4M3)
    refused(decode(c, B=B, T=T, Hq=Hq, max_len=high, max_pages=1 << 24), _lib.FOCAL_ERR_UNSUPPORTED, "too large")
