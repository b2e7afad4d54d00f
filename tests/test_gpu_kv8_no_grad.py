"""rope and the 8-bit cache calls have no gradient: tensors that require one are refused,
unless the caller has switched gradients off."""
import pytest
import torch

import focal_b200 as F
from test_gpu_kv8 import clones, empty_cache, ints, same, status

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_tensors_that_require_a_gradient_are_refused(cuda):
    cache = empty_cache(2, 2, 16, 64, torch.float8_e4m3fn, cuda)
    before = clones(cache)
    f, _ = F.rope_inv_freq(64, device=cuda)
    table, lens, pos = ints([[0], [1]], cuda), ints([1, 1], cuda), torch.arange(2, device=cuda)
    q, k = (torch.randn(2, h, 64, device=cuda).to(BF16) for h in (4, 2))
    leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [lambda q, k, v: F.rope(q, pos, f), lambda q, k, v: F.rope(q.detach(), pos, f, out=q),
             lambda q, k, v: F.kv8_append(k, v.detach(), cache, table, lens),
             lambda q, k, v: F.kv8_append(k.detach(), v, cache, table, lens),
             lambda q, k, v: F.kv8_append(k.detach(), v.detach(), cache, table, lens, q=q, inv_freq=f),
             lambda q, k, v: F.gqa_decode_attention_kv8(q, cache, table, lens, 16),
             lambda q, k, v: F.decode_attention_kv8(q, k.detach(), v.detach(), cache, table, lens, 16, f),
             lambda q, k, v: F.decode_attention_kv8(q.detach(), k.detach(), v, cache, table, lens, 16, f)]
    for call in calls:
        with pytest.raises(RuntimeError, match="requires a gradient"):
            call(leaf(q), leaf(k), leaf(k))
    assert same(cache, before)
    for call in calls:
        with torch.no_grad():
            call(leaf(q), leaf(k), leaf(k))
        with torch.inference_mode():
            call(q.clone(), k, k)
        call(q.clone(), k, k)
    assert status() == 0
