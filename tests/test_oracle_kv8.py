"""The 64-bit definitions of oracle/kv8.py against torch's own conversions and
attention, on the CPU."""
import math

import pytest
import torch

import focal_b200 as F
from oracle import kv8 as ok


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
def test_quantise_is_nearest_even(code):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4096, generator=g, dtype=torch.float64) * torch.exp(3 * torch.randn(4096, generator=g))
    x = torch.cat([x.float().double(), torch.tensor([0.0, 448.0, 1e-3, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0]).double()])
    got = ok.quantise(x, 1.0, code)
    if code == torch.int8:
        want = x.float().round().clamp(-127, 127).double()
    else:
        want = x.float().clamp(-448, 448).to(code).double()
    assert torch.equal(got, want)


def test_needed_scale():
    e4 = torch.float8_e4m3fn
    assert ok.needed_scale(448.0, e4) == 1.0 and ok.needed_scale(448.5, e4) == 2.0 and ok.needed_scale(0.0, e4) == 0.0
    assert ok.needed_scale(1e-45, e4) == 2.0 ** -126 and ok.needed_scale(254.0, torch.int8) == 2.0


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_is_a_rotation_by_the_position(interleaved):
    """Scores of turned q and k depend on the distance alone; pairs match a complex product."""
    f, _ = F.rope_inv_freq(32, device="cpu")
    g = torch.Generator().manual_seed(2)
    q, k = (torch.randn(1, 2, 48, generator=g, dtype=torch.float64) for _ in "qk")
    at = lambda x, p: ok.rope(x, torch.tensor([p]), f, interleaved)  # noqa: E731
    a = (at(q, 70) * at(k, 61)).sum(-1)
    b = (at(q, 100009) * at(k, 100000)).sum(-1)
    assert torch.allclose(a, b, atol=1e-8)
    i, j = (4, 5) if interleaved else (2, 18)
    z = complex(q[0, 0, i], q[0, 0, j]) * complex(math.cos(70 * f[2]), math.sin(70 * f[2]))
    y = at(q, 70)
    assert abs(complex(y[0, 0, i], y[0, 0, j]) - z) < 1e-12
    assert torch.equal(y[..., 32:], q[..., 32:])


def test_inv_freq_scalings():
    plain, m = F.rope_inv_freq(64, base=10000.0, device="cpu")
    assert m == 1.0 and plain.dtype == torch.float64
    assert torch.allclose(plain, 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64), rtol=1e-14)
    lin, _ = F.rope_inv_freq(64, scaling="linear", factor=4.0, device="cpu")
    assert torch.allclose(lin, plain / 4, rtol=1e-15)
    ntk, _ = F.rope_inv_freq(64, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0] == 1.0 and torch.isclose(ntk[-1], plain[-1] / 4, rtol=1e-12)  # the last pair is stretched by factor
    for kind in ("yarn", "bands"):
        f, m = F.rope_inv_freq(64, scaling=kind, factor=8.0, original_max_position=4096, device="cpu")
        turns = 4096 * plain / (2 * math.pi)
        assert torch.allclose(f[turns > 40], plain[turns > 40], rtol=1e-14)
        assert torch.allclose(f[turns < 0.5], plain[turns < 0.5] / 8, rtol=1e-14)
        assert torch.all(f <= plain * (1 + 1e-14)) and torch.all(f >= plain / 8 * (1 - 1e-14))
        assert m == (1.0 if kind == "bands" else 0.1 * math.log(8.0) + 1.0)
    for bad in (dict(rot=7), dict(rot=0), dict(rot=64, scaling="other"), dict(rot=64, base=0.5),
                dict(rot=64, factor=0.5), dict(rot=64, scaling="yarn", low=4.0, high=2.0)):
        with pytest.raises(ValueError):
            F.rope_inv_freq(device="cpu", **bad)


def test_append_then_attention_near_unquantised():
    """int8 codes of a whole prompt and of single tokens give the attention of the
    unquantised values within the codes' steps, and a block's scale only grows."""
    g = torch.Generator().manual_seed(3)
    H, D, n = 2, 64, 40
    k, v = (torch.randn(n, H, D, generator=g, dtype=torch.float64) for _ in "kv")
    table = torch.tensor([[2, 0, 1]])
    cache = [torch.zeros(3, H, 16, D, dtype=torch.float64) for _ in "kv"] + [torch.zeros(3, H, 1).double() for _ in "kv"]
    for x, c, s in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
        ok.append(x[:21], c, s, torch.int8, table, [21], [21])
        for i in range(21, n):
            ok.append(x[i:i + 1], c, s, torch.int8, table, [i + 1], [1])
        back = ok.gather(c, s, table, 0, n).transpose(0, 1)
        step = s[table[0, torch.arange(n) // 16]][..., 0]  # [n, H]
        # one rounding, and one more for each growth of the block's scale (at most 15 here)
        assert torch.all((back - x).abs() <= step[..., None] * 8)
        assert torch.all((back[:16] - x[:16]).abs() <= step[:16, :, None] * 0.5000001)
    q = torch.randn(1, 2, 4, D, generator=g, dtype=torch.float64)
    o, _, _, _ = ok.attention(q, cache, table, [n])
    want = torch.nn.functional.scaled_dot_product_attention(
        q.transpose(1, 2), ok.gather(cache[0], cache[2], table, 0, n)[None].repeat_interleave(2, 1),
        ok.gather(cache[1], cache[3], table, 0, n)[None].repeat_interleave(2, 1),
        attn_mask=torch.arange(n) < n - 1 + torch.arange(2)[:, None])
    assert torch.allclose(o, want.transpose(1, 2), atol=1e-12)


def test_attention_rows_that_see_nothing_are_zero():
    cache = [torch.ones(1, 1, 16, 64).double() for _ in "kv"] + [torch.ones(1, 1, 1).double() for _ in "kv"]
    o, _, _, _ = ok.attention(torch.ones(2, 4, 1, 64), cache, torch.zeros(2, 1, dtype=torch.int64), [2, 0])
    assert torch.all(o[0, :2] == 0) and torch.all(o[0, 2:] == 1) and torch.all(o[1] == 0)
