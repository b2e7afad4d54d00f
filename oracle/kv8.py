"""64-bit restatement of rotary positions, the 8-bit paged KV append and the
attention over it — TEST INFRASTRUCTURE ONLY.

Parity UNPINNED: the reference project has no attention code, so these are
written from the definitions (torch in float64, any device) and cross-checked on
the CPU in tests/test_oracle_kv8.py.  A cache is a list [k_pages, v_pages,
k_scales, v_scales] of float64 tensors here, codes as the numbers they are.
"""
from __future__ import annotations

import torch

GROUP = 16
TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def rope(x, positions, inv_freq, interleaved=False, mscale=1.0):
    """x [T, H, D] with its first 2 * len(inv_freq) dims turned; float64."""
    x = x.double()
    half = inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq
    c, s = (angle.cos() * mscale)[:, None], (angle.sin() * mscale)[:, None]
    y = x.clone()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., first], x[..., second]
    y[..., first] = a * c - b * s
    y[..., second] = a * s + b * c
    return y


def needed_scale(amax: float, code: torch.dtype) -> float:
    if amax == 0.0:
        return 0.0
    r = max(amax / TOP[code], 2.0 ** -126)
    if code == torch.int8:
        return r
    p = 2.0 ** -126
    while p < r:
        p *= 2.0
    return p


def quantise(x, scale: float, code: torch.dtype):
    """The codes of x / scale (as float64 numbers), nearest even, saturating."""
    r = x / (scale or 1.0)  # scale 0: zeros, infinities and NaN
    if code == torch.int8:
        return r.round().clamp(-127, 127)
    # e4m3: three mantissa bits, smallest exponent -6
    e = torch.floor(torch.log2(r.abs().clamp(min=2.0 ** -6)))
    step = torch.ldexp(torch.ones_like(r), (e - 3).int())
    return ((r / step).round() * step).clamp(-448, 448)


def append(x, codes, scales, code, block_table, seq_lens, new):
    """Rows x [T, H, D] (float64, in sequence order, new[b] of sequence b) into
    float64 codes [P, H, S, D] and scales [P, H, S / 16], in place, block by
    block and head by head."""
    page_size, done = codes.shape[2], 0
    for b, n in enumerate(new):
        at = seq_lens[b] - n
        while at < seq_lens[b]:
            base = at // GROUP * GROUP
            end = min(seq_lens[b], base + GROUP)
            page, row = int(block_table[b, base // page_size]), base % page_size
            for h in range(codes.shape[1]):
                part = x[done:done + end - at, h]
                old = float(scales[page, h, row // GROUP]) if at > base else 0.0
                scale = max(old, needed_scale(float(part.abs().max()), code))
                older = codes[page, h, row:row + at - base]
                if at > base and scale > old:
                    older.copy_(quantise(older * old, scale, code))
                codes[page, h, row + at - base:row + end - base] = quantise(part, scale, code)
                scales[page, h, row // GROUP] = scale
            done += end - at
            at = end


def gather(codes, scales, block_table, b, n):
    """Sequence b's first n positions as float64 values [H, n, D]."""
    page_size = codes.shape[2]
    pages = [int(p) for p in block_table[b, :-(-n // page_size)]]
    c = torch.cat([codes[p] for p in pages], 1)[:, :n].double()
    s = torch.cat([scales[p] for p in pages], 1).double().repeat_interleave(GROUP, 1)[:, :n]
    return c * s[..., None]


def attention(q, cache, block_table, seq_lens, scale=None):
    """(o, a, s, w): o [B, T, Hq, D] float64, and for error bounds a = sum of p |v|,
    s = the largest scale * sum |q| |k| of each row, and w = its number of positions
    times the largest V scale times the largest V code."""
    B, T, Hq, D = q.shape
    H = cache[0].shape[1]
    grp = Hq // H
    scale = D ** -0.5 if scale is None else scale
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    a, s, w = torch.zeros_like(o), torch.zeros_like(o[..., :1]), torch.zeros_like(o[..., :1])
    for b in range(B):
        n = int(seq_lens[b])
        if n == 0:
            continue
        k = gather(cache[0], cache[2], block_table, b, n)
        v = gather(cache[1], cache[3], block_table, b, n)
        for t in range(T):
            m = n - T + 1 + t
            if m < 1:
                continue
            qg = q[b, t].double().view(H, grp, D)
            p = torch.softmax(qg @ k[:, :m].transpose(1, 2) * scale, -1)
            o[b, t] = (p @ v[:, :m]).view(Hq, D)
            a[b, t] = (p @ v[:, :m].abs()).view(Hq, D)
            used = block_table[b, :-(-m // cache[1].shape[2])].long()
            top = cache[1][used].abs().nan_to_num(0.0).amax() * cache[3][used].nan_to_num(0.0).amax()
            w[b, t] = m * top
            s[b, t] = (qg.abs() @ k[:, :m].abs().transpose(1, 2) * scale).amax(-1).view(Hq, 1)
    return o, a, s, w
