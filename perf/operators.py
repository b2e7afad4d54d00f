"""Cases of the decode path around an 8-bit key/value cache: rotary positions,
the append that rotates, quantises and writes a step's or a prompt's keys and
values into pages, and grouped-query attention over those pages.

``run`` computes each operator in elementary torch operations (``own`` false)
or through focal_b200's entry points (``own`` true), on what ``prepare`` gives.

The cache: pages [num_pages, Hkv, page_size, D] of 8-bit codes (e4m3 or int8)
for K and for V, and one fp32 scale for every 16 consecutive tokens of a page
and head, [num_pages, Hkv, page_size / 16]; a code c stands for c * scale.
"""
import math
import random

import torch

own = False

GROUP = 16  # tokens that share a scale
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of eight sequences: the q and k heads of a packed QKV row
        dict(name="rope step", op="rope", tokens=8, heads=40, extra=8, dim=128, rot=128, interleaved=False,
             scaling="none", factor=1.0, max_pos=32768, dtype="bf16"),
        # a prompt of 4096 tokens in the same packed rows, positions scaled eightfold
        dict(name="rope prompt", op="rope", tokens=4096, heads=40, extra=8, dim=128, rot=128, interleaved=False,
             scaling="yarn", factor=8.0, max_pos=262144, dtype="bf16"),
        # adjacent pairs, half of a 64-wide head, an odd number of tokens
        dict(name="rope interleaved part", op="rope", tokens=1021, heads=32, extra=0, dim=64, rot=32,
             interleaved=True, scaling="linear", factor=4.0, max_pos=131072, dtype="fp16"),
        # unrounded fp32 heads at far positions, three quarters of the head rotated
        dict(name="rope fp32 far", op="rope", tokens=333, heads=9, extra=3, dim=128, rot=96, interleaved=False,
             scaling="ntk", factor=16.0, max_pos=1048576, dtype="fp32"),
        # one decode step of eight sequences: q and k rotated, k and v quantised into their pages
        dict(name="append step", op="append", batch=8, new=1, ragged=False, longest=250, heads=32, kv_heads=8, dim=128,
             rot=128, page=64, code="e4m3", dtype="bf16"),
        # one step of a large batch on small pages, keys rotated before
        dict(name="append large batch", op="append", batch=129, new=1, ragged=False, longest=61, heads=0, kv_heads=8,
             dim=128, rot=0, page=16, code="int8", dtype="bf16"),
        # prompts of different lengths, some behind a part that is cached already
        dict(name="append prompts", op="append", batch=5, new=2500, ragged=True, longest=3000, heads=32, kv_heads=8,
             dim=128, rot=128, page=64, code="e4m3", dtype="bf16"),
        # the smallest attention: one sequence, a short context
        dict(name="attend one short", op="attend", batch=1, tokens=1, longest=512, ragged=False, heads=32, kv_heads=8,
             dim=128, page=64, code="e4m3", dtype="bf16"),
        # an ordinary batch of unequal lengths on small pages
        dict(name="attend ragged int8", op="attend", batch=16, tokens=1, longest=4096, ragged=True, heads=32,
             kv_heads=8, dim=128, page=16, code="int8", dtype="fp16"),
        # long contexts of few sequences
        dict(name="attend four long", op="attend", batch=4, tokens=1, longest=32768, ragged=False, heads=32, kv_heads=8,
             dim=128, page=128, code="e4m3", dtype="bf16"),
        # four proposed tokens of each sequence checked in one pass
        dict(name="attend four tokens", op="attend", batch=8, tokens=4, longest=8191, ragged=True, heads=32,
             kv_heads=8, dim=128, page=32, code="e4m3", dtype="bf16"),
        # the largest: eight sequences of 131072 tokens
        dict(name="attend longest", op="attend", batch=8, tokens=1, longest=131072, ragged=False, heads=32, kv_heads=8,
             dim=128, page=64, code="e4m3", dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """An integer in lo .. hi, spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    op = rng.choice(("rope", "append", "attend", "attend"))
    dim = rng.choice((128, 128, 64))
    if op == "rope":
        heads = _spread(rng, 1, 48)
        return dict(op=op, tokens=_spread(rng, 1, 200000 // heads), heads=heads, extra=rng.choice((0, 0, 1, 8)), dim=dim,
                    rot=rng.randrange(16, dim + 1, 16), interleaved=rng.random() < 0.4,
                    scaling=rng.choice(("none", "linear", "ntk", "yarn")), factor=rng.choice((2.0, 4.0, 8.0, 16.0)),
                    max_pos=_spread(rng, 2048, 1048576), dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))
    kv = rng.choice((1, 2, 4, 8, 8, 16))
    group = rng.choice((1, 2, 4, 4, 7, 8, 16))
    page = rng.choice((16, 32, 64, 64, 128, 256))
    code = rng.choice(("e4m3", "e4m3", "int8"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if op == "append":
        batch = _spread(rng, 1, 256)
        new = 1 if rng.random() < 0.4 else _spread(rng, 1, max(1, 100000 // (batch * kv)))
        rot = 0 if code == "int8" else rng.choice((0, dim, dim, dim // 2))
        return dict(op=op, batch=batch, new=new, ragged=new > 1 and rng.random() < 0.5, longest=new + rng.randrange(0, 200),
                    heads=kv * group if rot and kv * group <= 64 else 0, kv_heads=kv, dim=dim, rot=rot, page=page, code=code,
                    dtype=dtype)
    batch, tokens = _spread(rng, 1, 128), rng.choice((1, 1, 1, 2, 4, 8))
    longest = _spread(rng, 1, min(131072, 16000000 // (batch * kv * max(4, tokens * group))))
    return dict(op=op, batch=batch, tokens=tokens, longest=longest, ragged=rng.random() < 0.6,
                heads=kv * group, kv_heads=kv, dim=dim, page=page, code=code, dtype=dtype)


def _lengths(case):
    """Each sequence's cached positions after the call (some are empty where lengths differ)."""
    if not case["ragged"]:
        return [case["longest"]] * case["batch"]
    rng = random.Random(case["batch"] * 7919 + case["longest"])
    got = [rng.choice((0, 1, case["longest"])) if rng.random() < 0.1 else rng.randint(1, case["longest"])
           for _ in range(case["batch"])]
    got[0] = case["longest"]
    return got


def _added(case):
    """append: each sequence's new tokens, the last of its positions."""
    if not case["ragged"]:
        return [case["new"]] * case["batch"]
    rng = random.Random(case["batch"] * 104729 + case["new"])
    got = [min(n, rng.randint(0, case["new"])) for n in _lengths(case)]
    got[0] = case["new"]
    return got


def _appended_lengths(case):
    """append: lengths after the call; unequal starts, so that blocks begin in their middle."""
    if case["ragged"]:
        return _lengths(case)
    rng = random.Random(case["batch"] + 31 * case["longest"])
    return [rng.randint(case["new"], case["longest"]) for _ in range(case["batch"])]


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rope":
        rows = case["tokens"] * case["heads"]
        return {"bytes": rows * case["dim"] * size * 2 + case["tokens"] * 8 + case["rot"] * 4,
                "flops": rows * case["rot"] * 3}
    kv, d = case["kv_heads"], case["dim"]
    per_token = 2 * kv * (d + 4 / GROUP)  # codes and scales of K and V
    if case["op"] == "append":
        n = sum(_added(case))
        return {"bytes": n * (2 * kv * d * size + per_token + 2 * case["heads"] * d * size),
                "flops": n * d * (3 * (kv + case["heads"]) + 2 * 2 * kv)}
    n = sum(_lengths(case))
    rows = case["batch"] * case["tokens"] * case["heads"]
    return {"bytes": n * per_token + 2 * rows * d * size,
            "flops": 4 * n * case["tokens"] * case["heads"] * d}


# ------------------------------------------------------------------ inputs
def _inv_freq(rot, scaling, factor, base=10000.0, original=4096):
    """(radians per position of each pair [rot / 2], factor on cos and sin), in 64 bits."""
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        return [x / factor for x in f], 1.0
    if scaling == "ntk":
        big = base * factor ** (rot / (rot - 2.0))
        return [big ** (-2.0 * i / rot) for i in range(rot // 2)], 1.0
    if scaling == "yarn":
        def pair(turns):  # the (fractional) pair that makes so many turns over the original length
            return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot // 2 - 1)
        ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))) for i in range(rot // 2)]
        return [x * (1 - r) + x / factor * r for x, r in zip(f, ramp)], 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _codes(x, code):
    """Codes and scales of x [..., 16 * n, D], made apart from any operator: an older call's cache."""
    b = x.unflatten(-2, (-1, GROUP))
    scale = b.abs().amax((-1, -2)) / TOP[code]
    c = b / scale[..., None, None]
    c = c.round().to(torch.int8) if code == "int8" else c.clamp(-448, 448).to(torch.float8_e4m3fn)
    return c.flatten(-3, -2), scale


def _pool(case, pages, gen):
    """Pages and scales of K and V: normal values, K with a few strong channels."""
    kv, d, page = case["kv_heads"], case["dim"], case["page"]
    out = []
    for strong in (True, False):
        codes = torch.empty((pages, kv, page, d), dtype=CODES[case["code"]], device="cuda")
        scales = torch.empty((pages, kv, page // GROUP), dtype=torch.float32, device="cuda")
        gain = torch.exp(0.5 * torch.randn((kv, 1, d), device="cuda", generator=gen)) if strong else 1.0
        step = max(1, (1 << 26) // (kv * page * d))
        for p in range(0, pages, step):
            x = torch.randn((min(step, pages - p), kv, page, d), device="cuda", generator=gen) * gain
            c, s = _codes(x, case["code"])
            codes[p:p + step].copy_(c)
            scales[p:p + step] = s
        out += [codes, scales]
    return out[0], out[2], out[1], out[3]


def _table(case, lengths, gen):
    """A block table of shuffled pages; entries behind a sequence's last page are -1."""
    per = [-(-n // case["page"]) for n in lengths]
    wide = max(1, max(per))
    pages = sum(per) + 3
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    first = torch.tensor([sum(per[:b]) for b in range(len(per))], device="cuda")
    j = torch.arange(wide, device="cuda")
    at = (first[:, None] + j).clamp(max=pages - 1)
    table = torch.where(j < torch.tensor(per, device="cuda")[:, None], order[at], -1)
    return table.to(torch.int32).contiguous(), pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen).to(dt)

    s = dict(case)
    if case["op"] == "rope":
        x = normal(case["tokens"], case["heads"] + case["extra"], case["dim"])
        f, s["mscale"] = _inv_freq(case["rot"], case["scaling"], case["factor"])
        first = torch.randint(0, max(1, case["max_pos"] - case["tokens"]), (1,), device="cuda", generator=gen)
        s["positions"] = first + torch.arange(case["tokens"], device="cuda")
        if case["tokens"] <= 64:  # a decode step: unrelated sequences
            s["positions"] = torch.randint(0, case["max_pos"], (case["tokens"],), device="cuda", generator=gen)
        s["x"] = x[:, :case["heads"]]
        s["inv_freq"] = torch.tensor(f, dtype=torch.float64, device="cuda")
        return s
    if case["op"] == "append":
        lengths, added = _appended_lengths(case), _added(case)
        total = sum(added)
        hq, kv, d = case["heads"], case["kv_heads"], case["dim"]
        qkv = normal(total, hq + 2 * kv, d)
        s["q"] = qkv[:, :hq] if hq else None
        s["k"], s["v"] = qkv[:, hq:hq + kv], qkv[:, hq + kv:]
        s["total"], s["max_new"] = total, max(1, max(added))
        s["cu_new"] = torch.tensor([sum(added[:b]) for b in range(len(added) + 1)], dtype=torch.int32, device="cuda")
        f, s["mscale"] = _inv_freq(case["rot"], "none", 1.0) if case["rot"] else ([], 1.0)
        s["inv_freq"] = torch.tensor(f, dtype=torch.float64, device="cuda") if f else None
    else:
        lengths = _lengths(case)
        s["x"] = normal(case["batch"], case["tokens"], case["heads"], case["dim"])
        s["scale"] = case["dim"] ** -0.5
    s["table"], pages = _table(case, lengths, gen)
    s["lens"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["cache"] = _pool(case, pages, gen)
    return s


# ------------------------------------------------------------- plain forms
def _rotate(x, positions, inv_freq, interleaved, mscale):
    rot = 2 * inv_freq.numel()
    angle = positions.double()[:, None, None] * inv_freq
    c, s = (angle.cos() * mscale).float(), (angle.sin() * mscale).float()
    y = x.float()
    r = y[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rot // 2], r[..., rot // 2:])
    u, w = a * c - b * s, a * s + b * c
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, y[..., rot:]), -1).to(x.dtype), torch.cat((turned, y[..., rot:]), -1)


def _scale_of(amax, code):
    if code == "int8":
        return torch.where(amax > 0, (amax / 127.0).clamp(min=2.0 ** -126), amax)
    m, e = torch.frexp(amax / 448.0)  # the next power of two: codes then move to a larger scale exactly
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(m), e - (m == 0.5).int()).clamp(min=2.0 ** -126), amax)


def _quantise(x, scale, code):
    r = torch.where(scale > 0, x / scale, torch.zeros_like(x)).clamp(-TOP[code], TOP[code])
    return r.round().to(torch.int8) if code == "int8" else r.to(torch.float8_e4m3fn)


def _write(x, codes, scales, block, row, code):
    """x [T, H, D] fp32 into rows `row` (0 .. 15) of blocks `block` of the pool, in place."""
    pages, h, page, d = codes.shape
    blocks = pages * page // GROUP
    old = scales.transpose(1, 2).reshape(blocks, h)
    at = block[:, None].expand(-1, h)
    amax = torch.zeros_like(old).scatter_reduce(0, at, x.abs().amax(-1), "amax")
    first = torch.full((blocks,), GROUP, device=x.device).scatter_reduce(0, block, row, "amin")
    touched = first < GROUP
    new = torch.maximum(torch.where((first > 0)[:, None], old, torch.zeros_like(old)), _scale_of(amax, code))
    new = torch.where(touched[:, None], new, old)
    mine = codes.unflatten(2, (-1, GROUP)).transpose(1, 2).reshape(blocks, h, GROUP, d)
    moved = _quantise(mine.float() * old[..., None, None], new[..., None, None], code)
    rows = torch.arange(GROUP, device=x.device)
    grown = (rows < first[:, None])[:, None, :] & (touched[:, None] & (new > old))[..., None]
    mine = torch.where(grown[..., None], moved.view(torch.uint8), mine.view(torch.uint8))
    mine[block, :, row] = _quantise(x, new[block][..., None], code).view(torch.uint8)
    back = mine.unflatten(0, (pages, -1)).transpose(1, 2).reshape(pages, h, page, d)
    codes.view(torch.uint8).copy_(back)
    scales.copy_(new.unflatten(0, (pages, -1)).transpose(1, 2))


def _plain_append(s):
    kc, vc, ks, vs = s["cache"]
    cu = s["cu_new"].long()
    seq = torch.repeat_interleave(torch.arange(s["batch"], device="cuda"), cu[1:] - cu[:-1], output_size=s["total"])
    pos = s["lens"].long()[seq] - cu[1:][seq] + torch.arange(s["total"], device="cuda")
    block = s["table"].long()[seq, pos // s["page"]] * (s["page"] // GROUP) + pos % s["page"] // GROUP
    row = pos % GROUP
    q, k = s["q"], s["k"].float()
    if s["inv_freq"] is not None:
        k = _rotate(s["k"], pos, s["inv_freq"], False, s["mscale"])[1]
        q = None if q is None else _rotate(q, pos, s["inv_freq"], False, s["mscale"])[0]
    _write(k, kc, ks, block, row, s["code"])
    _write(s["v"].float(), vc, vs, block, row, s["code"])
    return q


def _gathered(codes, scales, table):
    """fp32 [B, H, L, D] of all pages in `table`."""
    at = table.long().clamp(min=0)
    c = codes.view(torch.uint8)[at].view(codes.dtype).float().unflatten(3, (-1, GROUP)) * scales[at][..., None, None]
    return c.flatten(3, 4).transpose(1, 2).flatten(2, 3)


def _plain_attend(s):
    kc, vc, ks, vs = s["cache"]
    k, v = _gathered(kc, ks, s["table"]), _gathered(vc, vs, s["table"])
    b, t, h, d = s["x"].shape
    kv = k.shape[1]
    at = torch.arange(k.shape[2], device="cuda")
    lens = s["lens"].long()
    v = torch.where((at < lens[:, None])[:, None, :, None], v, torch.zeros_like(v))
    q = s["x"].float().unflatten(2, (kv, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [B, kv, t * group, D]
    seen = at < (lens[:, None] - t + 1 + torch.arange(t, device="cuda"))[..., None]  # [B, t, L]
    seen = seen.repeat_interleave(h // kv, 1)[:, None]
    score = torch.where(seen, q @ k.transpose(-1, -2) * s["scale"], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total > 0, total, torch.ones_like(total))
    return o.unflatten(2, (t, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3).to(s["x"].dtype)


def _stands_for(codes, scales):
    """int8 codes as the values they stand for; e4m3 ones are values in units of their scales already."""
    if codes.dtype != torch.int8:
        return codes
    return (codes.unflatten(2, (-1, GROUP)) * scales[..., None, None]).flatten(2, 3).to(torch.bfloat16)


def run(state):
    s = state
    if own:
        import focal_b200
    if s["op"] == "rope":
        if own:
            return focal_b200.rope(s["x"], s["positions"], s["inv_freq"], interleaved=s["interleaved"],
                                   mscale=s["mscale"])
        return _rotate(s["x"], s["positions"], s["inv_freq"], s["interleaved"], s["mscale"])[0]
    if s["op"] == "attend":
        if own:
            return focal_b200.gqa_decode_attention_kv8(s["x"], s["cache"], s["table"], s["lens"], s["longest"],
                                                       scale=s["scale"])
        return _plain_attend(s)
    if own:
        q = focal_b200.kv8_append(s["k"], s["v"], s["cache"], s["table"], s["lens"], cu_new=s["cu_new"],
                                  max_new=s["max_new"], q=s["q"], inv_freq=s["inv_freq"], mscale=s["mscale"])
    else:
        q = _plain_append(s)
    kc, vc, ks, vs = s["cache"]
    out = {"k": _stands_for(kc, ks), "v": _stands_for(vc, vs), "k_scales": ks, "v_scales": vs}
    return out if q is None else {**out, "q": q}


# ------------------------------------------------------ definitions, 64 bits
def _exact_turn(x, positions, inv_freq, interleaved, mscale):
    """Each pair as a complex number, times mscale * e^(i * angle)."""
    x = x.double()
    half = inv_freq.numel()
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    z = torch.complex(x[..., a], x[..., b])
    z = z * torch.polar(torch.full_like(inv_freq, mscale), positions.double()[:, None] * inv_freq)[:, None]
    y = x.clone()
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_round(x, code):
    if code == "int8":
        return x.round().clamp(-127, 127)
    step = 2.0 ** (torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (x / step).round().mul(step).clamp(-448, 448)


def _exact_append(case, s):
    lengths, added = _appended_lengths(case), _added(case)
    f = s["inv_freq"]
    out = {}
    k, q = s["k"].double(), s["q"]
    pos = torch.cat([torch.arange(n - m, n, device="cuda") for n, m in zip(lengths, added)])
    if f is not None:
        k = _exact_turn(k, pos, f, False, s["mscale"])
        if q is not None:
            out["q"] = _exact_turn(q, pos, f, False, s["mscale"])
    for name, x, codes, scales in (("k", k, s["cache"][0], s["cache"][2]),
                                   ("v", s["v"].double(), s["cache"][1], s["cache"][3])):
        codes, scales = codes.double(), scales.double()
        table, done = s["table"].tolist(), 0
        for b, (n, m) in enumerate(zip(lengths, added)):
            at = n - m
            while at < n:  # a block at a time
                row, end = at % GROUP, min(n, at // GROUP * GROUP + GROUP)
                page, j = table[b][at // case["page"]], at % case["page"] // GROUP
                part = x[done:done + end - at].transpose(0, 1)  # [H, rows, D]
                need = part.abs().amax((1, 2)) / TOP[case["code"]]
                if case["code"] == "e4m3":
                    need = 2.0 ** torch.ceil(torch.log2(need))
                had = scales[page, :, j].clone() if row else torch.zeros_like(need)
                now = torch.maximum(had, need)
                older = codes[page, :, j * GROUP:j * GROUP + row]
                older.copy_(torch.where((now > had)[:, None, None],
                                        _exact_round(older * (had / now)[:, None, None], case["code"]), older))
                codes[page, :, j * GROUP + row:j * GROUP + row + end - at] = _exact_round(part / now[:, None, None],
                                                                                        case["code"])
                scales[page, :, j] = now
                done += end - at
                at = end
        if case["code"] == "int8":
            codes = codes * scales.repeat_interleave(GROUP, 2)[..., None]
        out[name], out[name + "_scales"] = codes, scales
    return out


def _exact_attend(case, s):
    kc, vc, ks, vs = s["cache"]
    out = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    for b, n in enumerate(_lengths(case)):
        if not n:
            continue
        at = s["table"][b, :-(-n // case["page"])].tolist()
        for g in range(case["kv_heads"]):
            k, v = _exact_rows(kc, ks, at, g, n), _exact_rows(vc, vs, at, g, n)
            for t in range(case["tokens"]):
                m = n - case["tokens"] + 1 + t
                if m < 1:
                    continue
                q = s["x"][b, t, g * group:(g + 1) * group].double()
                out[b, t, g * group:(g + 1) * group] = torch.softmax(q @ k[:m].T * s["scale"], -1) @ v[:m]
    return out


def _exact_rows(codes, scales, at, g, n):
    i = torch.tensor(at, device="cuda")
    c = codes.view(torch.uint8)[i, g].view(codes.dtype).flatten(0, 1)[:n].double()
    return c * scales[i, g].flatten()[torch.arange(n, device="cuda") // GROUP].double()[:, None]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_turn(s["x"], s["positions"], s["inv_freq"], s["interleaved"], s["mscale"])
    return _exact_append(case, s) if case["op"] == "append" else _exact_attend(case, s)
