"""Calls of different shapes that share a stream's workspace."""
import pytest
import torch

import focal_b200 as F

pytestmark = pytest.mark.gpu


def case(cuda, B, Hq, H, L, paged, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)
    q, k, v = (torch.randn(s, device=cuda, generator=g).to(torch.bfloat16)
               for s in ((B, Hq, 128), (B, H, L, 128), (B, H, L, 128)))
    s = torch.einsum("bhgd,bhld->bhgl", q.double().view(B, H, -1, 128), k.double()) / 128 ** 0.5
    want = torch.einsum("bhgl,bhld->bhgd", s.softmax(-1), v.double()).reshape(B, Hq, 128)
    if not paged:
        return want, lambda: F.gqa_decode_attention(q, k, v)
    pages = [t.view(B, H, L // 64, 64, 128).transpose(1, 2).reshape(-1, H, 64, 128).contiguous() for t in (k, v)]
    table = torch.arange(B * (L // 64), dtype=torch.int32, device=cuda).view(B, -1)
    lens = torch.full((B,), L, dtype=torch.int32, device=cuda)
    return want, lambda: F.gqa_decode_attention_paged(q, *pages, table, lens, L)


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("many,few", [((16, 16, 8, 2048), (1, 8, 8, 20032)), ((100, 4, 1, 2048), (4, 16, 4, 10048))])
def test_attention_of_two_shapes_in_turn(cuda, paged, many, few):
    """More (sequence, KV head) pairs than 64, fewer, more again: what a call leaves in the
    workspace means nothing to the next.  Outputs are rounded once to bf16 (2^-8 of them);
    a weight is rounded to bf16 too, and |v| < 6 with weights that sum to one."""
    cases = [case(cuda, *many, paged, 1), case(cuda, *few, paged, 2)]
    for i in (0, 1, 0, 0, 1, 0):
        want, run = cases[i]
        assert float((run().double() - want).abs().max()) < 6 * 2.0 ** -8 + 2.0 ** -8
