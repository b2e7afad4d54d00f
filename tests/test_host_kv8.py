"""Refusals of the rotary, 8-bit append and 8-bit attention entry points that
the host makes before any CUDA call, through the C ABI and the PyTorch layer;
none of them touches a GPU."""
import ctypes

import pytest
import torch

import focal_b200 as F
from focal_b200 import _lib

FAKE = 1 << 20  # never dereferenced: every call below is refused first


def refused(rc, code, text):
    assert rc == code, (rc, _lib.last_error())
    assert text in _lib.last_error()


def rope(**kw):
    a = dict(x=FAKE, y=2 * FAKE, pos=FAKE, f=FAKE, T=4, H=2, D=128, rot=128, il=0, m=1.0, dt=_lib.FOCAL_BF16, p64=1,
             xt=256, xh=128, yt=256, yh=128)
    a.update(kw)
    return _lib.lib().focal_rope(*a.values(), None)


def test_rope_refusals():
    U, V = _lib.FOCAL_ERR_UNSUPPORTED, _lib.FOCAL_ERR_INVALID_VALUE
    refused(rope(dt=7), U, "dtype")
    refused(rope(D=100), U, "multiple of 8")
    refused(rope(D=2048), U, "1024")
    refused(rope(D=8, rot=16), U, "D must be")
    refused(rope(rot=24), U, "rotated dims")
    refused(rope(rot=0), U, "rotated dims")
    refused(rope(rot=144), U, "rotated dims")
    refused(rope(T=-1), U, "negative")
    refused(rope(m=float("nan")), V, "mscale")
    refused(rope(xh=4), U, "strides")
    refused(rope(yt=257), U, "strides")
    refused(rope(dt=_lib.FOCAL_FP32, xh=6), U, "strides")
    refused(rope(x=None), V, "null")
    refused(rope(f=None), V, "null")
    refused(rope(x=FAKE + 8), V, "aligned")
    refused(rope(pos=FAKE + 4), V, "aligned")
    refused(rope(y=FAKE, yt=512), V, "in place")
    assert rope(T=0, x=None) == _lib.FOCAL_OK and rope(H=0, x=None) == _lib.FOCAL_OK


def cache(**kw):
    a = dict(k_pages=FAKE, v_pages=FAKE, k_scales=FAKE, v_scales=FAKE, num_pages=8, num_kv_heads=2, page_size=32,
             head_dim=128, code=_lib.FOCAL_E4M3)
    a.update(kw)
    return _lib.Kv8Cache(*a.values())


def append(c=None, **kw):
    a = dict(k=FAKE, v=FAKE, q=None, q_out=None, block_table=FAKE, seq_lens=FAKE, cu_new=None, inv_freq=None,
             k_token_stride=256, k_head_stride=128, v_token_stride=256, v_head_stride=128, q_token_stride=0,
             q_head_stride=0, B=3, T=3, max_new=1, Hq=0, max_pages_per_seq=4, rot=0, interleaved=0,
             dtype=_lib.FOCAL_BF16, mscale=1.0)
    a.update(kw)
    return _lib.lib().focal_kv8_append(ctypes.byref(_lib.Kv8AppendArgs(*a.values())), ctypes.byref(c or cache()), None)


CACHE_REFUSALS = [(dict(code=5), "code"), (dict(head_dim=96), "head_dim"), (dict(page_size=48), "page_size"),
                  (dict(page_size=8), "page_size"), (dict(page_size=0), "page_size"), (dict(num_pages=0), "num_pages"),
                  (dict(num_kv_heads=0), "num_kv_heads")]


def test_append_refusals():
    U, V = _lib.FOCAL_ERR_UNSUPPORTED, _lib.FOCAL_ERR_INVALID_VALUE
    for kw, text in CACHE_REFUSALS:
        refused(append(cache(**kw)), U, text)
    refused(append(dtype=_lib.FOCAL_FP32), U, "dtype")
    refused(append(T=4), U, "B * max_new")
    refused(append(B=-1), U, "negative")
    refused(append(max_pages_per_seq=0), U, "max_pages_per_seq")
    refused(append(rot=40, inv_freq=FAKE), U, "rotated dims")
    refused(append(Hq=4, q=FAKE, q_out=FAKE), U, "q is only turned")
    refused(append(k_token_stride=100), U, "strides")
    refused(append(mscale=float("inf")), V, "mscale")
    refused(append(B=1 << 20, T=1 << 30, max_new=1 << 30, cu_new=FAKE), U, "too large")
    refused(append(rot=64), V, "null")
    refused(append(k=None), V, "null")
    refused(append(k=FAKE + 2), V, "aligned")
    refused(append(cache(k_pages=None)), V, "null")
    refused(append(cache(v_scales=FAKE + 4)), V, "aligned")
    refused(append(cu_new=FAKE + 2, max_new=0), V, "aligned")
    assert append(T=0, B=0, max_new=0, k=None) == _lib.FOCAL_OK
    L = _lib.lib()
    refused(L.focal_kv8_append(None, ctypes.byref(cache()), None), V, "null")
    refused(L.focal_kv8_append(ctypes.byref(_lib.Kv8AppendArgs()), None, None), V, "null")


def decode(c=None, **kw):
    a = dict(q=FAKE, o=FAKE, cache=ctypes.byref(c or cache()), table=FAKE, lens=FAKE, B=2, T=1, Hq=8, max_pages=4,
             max_len=128, scale=0.1, dtype=_lib.FOCAL_BF16, ws=FAKE, ws_bytes=1 << 40)
    a.update(kw)
    return _lib.lib().focal_kv8_decode(*a.values(), None)


def test_decode_refusals():
    U, V = _lib.FOCAL_ERR_UNSUPPORTED, _lib.FOCAL_ERR_INVALID_VALUE
    for kw, text in CACHE_REFUSALS:
        refused(decode(cache(**kw)), U, text)
    refused(decode(Hq=7), U, "multiple of Hkv")
    refused(decode(Hq=64), U, "<= 16")
    refused(decode(T=0), U, "query tokens")
    refused(decode(T=17), U, "query tokens")
    refused(decode(B=0), U, "positive")
    refused(decode(B=40000), U, "too large")
    refused(decode(max_len=129), U, "max_seq_len exceeds")
    refused(decode(max_len=0), U, "positive")
    refused(decode(max_len=(1 << 30) + 1, max_pages=1 << 30), U, "2^30")
    refused(decode(dtype=_lib.FOCAL_FP32), U, "dtype")
    refused(decode(scale=0.0), V, "scale")
    refused(decode(scale=float("nan")), V, "scale")
    refused(decode(q=None), V, "null")
    refused(decode(o=FAKE + 8), V, "aligned")
    refused(decode(cache(k_scales=None)), V, "null")
    refused(decode(ws_bytes=0), _lib.FOCAL_ERR_WORKSPACE, "workspace")
    refused(decode(ws=None), _lib.FOCAL_ERR_WORKSPACE, "workspace")
    refused(decode(ws=FAKE + 16), V, "256-byte")
    refused(_lib.lib().focal_kv8_decode(FAKE, FAKE, None, FAKE, FAKE, 2, 1, 8, 4, 128, 0.1, 0, FAKE, 1 << 40, None),
            V, "null")


def test_decode_workspace_sizing():
    L = _lib.lib()
    ws, counters = L.focal_kv8_decode_workspace_size, L.focal_kv8_decode_counter_bytes
    assert 0 < ws(1, 1, 32, 8, 512, 128) <= ws(8, 1, 32, 8, 32768, 128)
    assert counters() % 256 == 0 and counters() < ws(1, 1, 32, 8, 1, 128)
    for bad in ((0, 1, 32, 8), (1, 0, 32, 8), (1, 17, 32, 8), (1, 1, 30, 8), (1, 1, 32, 1)):
        assert ws(*bad, 512, 128) == 0
    assert ws(1, 1, 32, 8, 512, 96) == 0 and ws(1, 1, 32, 8, 0, 128) == 0


def test_python_refusals():
    with pytest.raises(ValueError, match="dtype"):
        F.kv8_cache(4, 2, 16, dtype=torch.float16, device="cpu")
    with pytest.raises(ValueError, match="page_size"):
        F.kv8_cache(4, 2, 48, device="cpu")
    with pytest.raises(ValueError, match="D must be"):
        F.kv8_cache(4, 2, 16, D=80, device="cpu")
    c = F.kv8_cache(4, 2, 32, device="cpu")
    assert c.k_pages.dtype == torch.float8_e4m3fn and c.k_scales.shape == (4, 2, 2)
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="same number"):
        F.kv8_append(k, k, c, table, lens)
    with pytest.raises(ValueError, match="max_new"):
        F.kv8_append(k, k, c, table, lens, cu_new=lens)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        F.kv8_append(k[:2], k[:2], c, table, lens)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        F.rope(k, torch.arange(3), torch.ones(64).double())
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        F.gqa_decode_attention_kv8(k, c, table, lens, 32)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        F.decode_attention_kv8(k[:2], k[:2], k[:2], c, table, lens, 32, torch.ones(64).double())
