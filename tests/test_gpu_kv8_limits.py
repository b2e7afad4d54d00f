"""8-bit cache calls at the edges of their contract: what is refused, and what a
refused call leaves as it was."""
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
