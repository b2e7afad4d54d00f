"""8-bit cache calls at the edges of their contract: what is refused, and what a
refused call leaves as it was."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import focal_b200 as F
from test_gpu_kv8 import clones, empty_cache, ints, same, status

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, FP16 = torch.bfloat16, torch.float16


def test_too_many_tiles_leave_the_cache(cuda):
    """2^30 tiles and more: the composite refuses before it appends."""
    B, T, S, D = 4095, 16, (1 << 20) + (1 << 12), 64
    cache = empty_cache(1, 1, S, D, E4M3, cuda)
    before = clones(cache)
    q = torch.ones(B * T, 16, D, device=cuda, dtype=BF16)
    k = torch.ones(B * T, 1, D, device=cuda, dtype=BF16)
    f, _ = F.rope_inv_freq(D, device=cuda)
    table = torch.zeros(B, 1, dtype=torch.int32, device=cuda)
    with pytest.raises(RuntimeError, match="too large"):
        F.decode_attention_kv8(q, k, k, cache, table, ints([T] * B, cuda), S, f)
    assert same(cache, before) and status() == 0


def one_bad_page():
    """A step of two sequences, the first with a page id out of range: the call itself returns with the
    second sequence's output, the next call raises and leaves the cache, the one after it is fine."""
    cuda = torch.device("cuda")
    cache = empty_cache(4, 2, 16, 64, E4M3, cuda)
    for t in cache[2:]:
        t.fill_(1.0)
    f, _ = F.rope_inv_freq(64, device=cuda)
    x = torch.ones(2, 8, 64, device=cuda, dtype=BF16)
    lens = ints([1, 1], cuda)
    step = lambda pages, n=lens: F.decode_attention_kv8(x[:, :4], x[:, 4:6], x[:, 6:], cache, ints(pages, cuda), n, 16, f)  # noqa: E731
    got = step([[9], [2]])
    torch.cuda.synchronize()
    assert torch.all(got[1] == 1.0)
    before = clones(cache)
    with pytest.raises(RuntimeError, match="bad paged-KV index"):
        step([[1], [2]])
    torch.cuda.synchronize()
    assert same(cache, before)
    assert torch.all(step([[1], [2]]) == 1.0) and status() == 0


def test_a_step_that_raises_has_not_appended(cuda):
    one_bad_page()


def test_a_step_that_raises_has_not_appended_when_launches_block(cuda):
    """With every launch waited for, the append's own failure is known before the attention is launched."""
    here = Path(__file__).resolve().parent
    env = dict(os.environ, CUDA_LAUNCH_BLOCKING="1", PYTHONPATH=f"{here}{os.pathsep}{here.parent}")
    run = subprocess.run([sys.executable, "-c", "import test_gpu_kv8_limits as t; t.one_bad_page()"], env=env,
                         capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_infinities_and_nan_beside_zeros(cuda, code, dtype):
    """A block whose finite values are all zero has scale 0; infinities still get the largest code and
    NaN e4m3's NaN (int8: 0), the attention shows that NaN, and a later token's scale keeps it."""
    H, D, S, n = 2, 64, 16, 5
    cache = empty_cache(3, H, S, D, code, cuda)
    x = torch.zeros(3 * n, H, D, device=cuda, dtype=dtype)
    x[1] = -0.0
    x[n + 1, 0, 7], x[n + 2, 0, 40], x[n + 3, 1, 63] = float("inf"), float("-inf"), float("nan")
    table = ints([[2], [0], [1]], cuda)
    F.kv8_append(x, x, cache, table, ints([n] * 3, cuda))
    inf, minus, nan = (0x7E, 0xFE, 0x7F) if code == E4M3 else (127, 0x81, 0)
    want = torch.zeros(3, H, n, D, dtype=torch.uint8, device=cuda)
    want[0, 0, 1, 7], want[0, 0, 2, 40], want[0, 1, 3, 63] = inf, minus, nan
    for pages, scales in (cache[::2], cache[1::2]):
        got = pages.view(torch.uint8)[:, :, :n].clone()
        if code == E4M3:
            got[0, 1, 3, 63] &= 0x7F  # either NaN
        assert torch.equal(got, want) and torch.all(scales[:3] == 0)
    q = torch.ones(3, 2 * H, D, device=cuda, dtype=dtype)
    o = F.gqa_decode_attention_kv8(q, cache, table, ints([n] * 3, cuda), n)
    seen = torch.zeros(3, 2 * H, D, dtype=torch.bool, device=cuda)
    seen[1, H:] = code == E4M3  # K's NaN reaches all dims of its KV head
    assert torch.equal(torch.isnan(o), seen) and torch.all(o[~seen] == 0)
    one = torch.full((3, H, D), 1.5, device=cuda, dtype=dtype)
    F.kv8_append(one, one, cache, table, ints([n + 1] * 3, cuda))
    for pages, scales in (cache[::2], cache[1::2]):
        value = pages.double() * scales.double().repeat_interleave(16, 2)[..., None]
        assert torch.equal(torch.isnan(value[:, :, :n]), torch.isnan(value[:, :, :n]) & (want == nan)) and torch.all(scales > 0)
        assert bool(torch.isnan(value[0, 1, 3, 63])) == (code == E4M3)
        assert torch.all(value[:, :, :n].nan_to_num(0.0) == 0)
        # e4m3: 384 * 2^-8; int8: 127 times 1.5 / 127 rounded to fp32
        assert torch.all((value[:, :, n] - 1.5).abs() <= (0.0 if code == E4M3 else 1.5 * 2.0 ** -24))
    assert status() == 0
