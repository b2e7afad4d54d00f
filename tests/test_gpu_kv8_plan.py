"""Batches of short, non-empty sequences through the 8-bit cache attention: more segments
(sequence, KV head, up to 16 query rows) than SMs, one or two tiles each.  Outputs are
written into memory full of NaN, so a row that no CTA takes shows."""
import pytest
import torch

import focal_b200 as F
from focal_b200 import _lib
from test_gpu_kv8 import attention_tolerance, doubles, gen, ints, random_cache, spoil, status, table_for

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, FP16 = torch.bfloat16, torch.float16


def dense_attention(q, cache, table, lens, scale):
    """As oracle.kv8.attention, all sequences at once: (o, a, s, w), see there."""
    B, T, Hq, D = q.shape
    H, S = cache[0].shape[1:3]
    n = -(-max(lens) // S)
    at = table[:, :n].long().clamp(min=0)

    def rows(codes, scales):  # [B, H, n * S, D], 0 behind a sequence's end
        x = codes[at] * scales[at].repeat_interleave(16, 3)[..., None]
        x = x.transpose(1, 2).flatten(2, 3)
        return torch.where((torch.arange(n * S, device=q.device) < torch.tensor(lens, device=q.device)[:, None])[:, None, :, None],
                           x, torch.zeros_like(x))

    k, v = rows(cache[0], cache[2]), rows(cache[1], cache[3])
    qg = q.double().view(B, T, H, Hq // H, D)
    see = torch.tensor(lens, device=q.device)[:, None] - T + 1 + torch.arange(T, device=q.device)  # [B, T]
    seen = (torch.arange(n * S, device=q.device) < see[..., None])[:, :, None, None]
    x = torch.where(seen, torch.einsum("bthgd,bhld->bthgl", qg, k) * scale, -torch.inf)
    p = torch.softmax(x, -1).nan_to_num(0.0)
    o, a = torch.einsum("bthgl,bhld->bthgd", p, v), torch.einsum("bthgl,bhld->bthgd", p, v.abs())
    s = torch.where(seen, torch.einsum("bthgd,bhld->bthgl", qg.abs(), k.abs()) * scale, 0.0).amax(-1, keepdim=True)
    top = cache[1].abs().nan_to_num(0.0).amax() * cache[3].nan_to_num(0.0).amax()
    w = (see.clamp(min=0) * top)[:, :, None, None, None].expand_as(s)
    return [t.reshape(B, T, Hq, -1) for t in (o, a, s, w)]


def run_into_nan(q, cache, table, lens, max_len, scale):
    """focal_kv8_decode into an o full of NaN."""
    B, T, Hq, D = q.shape
    pages, H, S, _ = cache.k_pages.shape
    o = torch.full_like(q, float("nan"))
    bytes_ = _lib.lib().focal_kv8_decode_workspace_size(B, T, Hq, H, max_len, D)
    ws = torch.zeros(bytes_, dtype=torch.uint8, device=q.device)
    c = _lib.Kv8Cache(*[t.data_ptr() for t in cache], pages, H, S, D,
                      _lib.FOCAL_E4M3 if cache.k_pages.dtype == E4M3 else _lib.FOCAL_INT8)
    _lib.call("focal_kv8_decode", q.data_ptr(), o.data_ptr(), c, table.data_ptr(), lens.data_ptr(), B, T, Hq, table.shape[1],
              max_len, scale, _lib.FOCAL_BF16 if q.dtype == BF16 else _lib.FOCAL_FP16, ws.data_ptr(), bytes_,
              torch.cuda.current_stream().cuda_stream)
    return o


# B * H * row chunks, from one segment above the 148 SMs on
SHAPES = [(149, 1, 1, 2), (160, 1, 1, 1), (32, 8, 1, 4), (37, 8, 1, 2), (4, 8, 16, 8), (297, 1, 1, 1), (53, 7, 1, 4),
          (111, 2, 3, 8), (444, 1, 1, 3), (445, 1, 1, 1), (74, 8, 1, 4)]  # B, H, T, Hq / H


@pytest.mark.parametrize("max_len", [1, 16, 63, 64, 65])
@pytest.mark.parametrize("B,H,T,grp", SHAPES)
def test_short_sequences_are_all_written(cuda, B, H, T, grp, max_len):
    for D, code, dtype, S in ((128, E4M3, BF16, 64), (128, INT8, FP16, 16), (64, E4M3, FP16, 32), (64, INT8, BF16, 64),
                              (128, E4M3, FP16, 16), (128, INT8, BF16, 32), (64, E4M3, BF16, 64), (64, INT8, FP16, 16)):
        lens = [1 + (max_len - 1 - 3 * b) % max_len for b in range(B)]
        table, pages = table_for(lens, S, cuda, seed=B + D)
        cache = random_cache(pages, H, S, D, code, cuda, seed=B)
        spoil(cache, table.cpu(), lens, S)
        q = torch.randn(B, T, grp * H, D, device=cuda, generator=gen(cuda, B + 1)).to(dtype)
        scale = D ** -0.5
        got = run_into_nan(q, cache, table, ints(lens, cuda), max_len, scale)
        bounds = dense_attention(q, doubles(cache), table, lens, scale)
        err, tol = (got.double() - bounds[0]).abs(), attention_tolerance(bounds, dtype, D)
        assert torch.all(err <= tol), (D, code, dtype, int(torch.isnan(got).any(-1).sum()), float(err.nan_to_num(0.0).max()))
    assert status() == 0


@pytest.mark.parametrize("B,H,T,grp", SHAPES)
def test_short_sequences_through_the_step(cuda, B, H, T, grp):
    """decode_attention_kv8 behind an allocator whose free memory is full of NaN."""
    S, D = 16, 128
    lens = [T + (5 * b) % (64 - T + 1) for b in range(B)]
    table, pages = table_for(lens, S, cuda, seed=B)
    cache = random_cache(pages, H, S, D, E4M3, cuda, seed=B)
    x = torch.randn(B * T, (grp + 2) * H, D, device=cuda, generator=gen(cuda, B)).to(BF16)
    q, k, v = x.split([grp * H, H, H], 1)
    f, _ = F.rope_inv_freq(D, device=cuda)
    junk = [torch.full((B * T, grp * H, D), float("nan"), dtype=BF16, device=cuda) for _ in range(4)]
    del junk
    got = F.decode_attention_kv8(q, k, v, cache, table, ints(lens, cuda), max(lens), f)
    pos = (torch.tensor(lens)[:, None] - T + torch.arange(T)).flatten().to(cuda)
    turned = F.rope(q, pos, f).view(B, T, grp * H, D)
    bounds = dense_attention(turned, doubles(cache), table, lens, D ** -0.5)
    assert torch.all((got.view_as(turned).double() - bounds[0]).abs() <= attention_tolerance(bounds, BF16, D))
    assert status() == 0
