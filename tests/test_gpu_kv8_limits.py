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
