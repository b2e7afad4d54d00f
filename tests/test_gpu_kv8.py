"""The 8-bit paged KV cache on the GPU: append, attention and a run of both,
against the 64-bit definitions in oracle/kv8.py.

Append without turning is exact: the scale's division, the codes' division and
their rounding are IEEE fp32 operations on exactly representable inputs, so codes
and scales must equal an fp32 restatement bit for bit.  With turning, the fp32
turn is off by at most 4 * 2^-24 (|a| + |b|) (tests/test_gpu_rope.py), and a code
then by that and half a step.

Attention: see `attention_tolerance`."""
import ctypes

import pytest
import torch

import focal_b200 as F
from focal_b200 import _lib
from oracle import kv8 as ok

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, FP16 = torch.bfloat16, torch.float16


def gen(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


def doubles(cache):
    return [t.double() for t in cache]


def table_for(lens, page_size, device, seed, spare=2):
    """Shuffled pages for the lengths; entries behind a sequence's last page are -7."""
    per = [-(-n // page_size) for n in lens]
    pages = sum(per) + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(max(per), 1) + 1), -7, dtype=torch.int32)
    for b, n in enumerate(per):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return table.to(device), pages


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def empty_cache(pages, H, page_size, D, code, device, seed=0):
    """A cache of recycled pages: arbitrary codes (e4m3 NaN among them) and scales."""
    c = F.kv8_cache(pages, H, page_size, D, code, device)
    g = gen(device, seed)
    for t in c[:2]:
        t.view(torch.uint8).random_(0, 256, generator=g)
    for t in c[2:]:
        t.uniform_(0.5, 2.0, generator=g)
    return c


def status():
    torch.cuda.synchronize()
    st = ctypes.c_int(-1)
    _lib.call("focal_device_status", ctypes.byref(st))
    return st.value


# ------------------------------------------------------------------ append
def fp32_append(x, codes, scales, code, table, lens, new):
    """The definition in fp32 on raw codes, one block at a time (all heads at once)."""
    top = torch.full((), ok.TOP[code], device=x.device)  # on the device: torch divides by a Python number as a product
    size, done = codes.shape[2], 0

    def quant(r):
        r = r.nan_to_num(0.0) if code == INT8 else r
        return r.round().clamp(-127, 127).to(INT8) if code == INT8 else r.clamp(-448, 448).to(E4M3)

    raw = codes.view(torch.uint8)
    for b, n in enumerate(new):
        at = lens[b] - n
        while at < lens[b]:
            base = at // 16 * 16
            end = min(lens[b], base + 16)
            page, row, o = int(table[b, base // size]), base % size, at - base
            part = x[done:done + end - at].transpose(0, 1).float()  # [H, rows, D]
            amax = part.abs().nan_to_num(0.0, posinf=0.0).amax((1, 2))
            if code == INT8:
                need = (amax / top).clamp(min=2.0 ** -126)
            else:
                m, e = torch.frexp((amax / top).clamp(min=2.0 ** -126))
                need = torch.ldexp(torch.ones_like(m), e - (m == 0.5).int())
            need = torch.where(amax > 0, need, amax)
            old = scales[page, :, row // 16].clone() if o else torch.zeros_like(need)
            scale = torch.maximum(old, need)
            if o:
                moved = quant(codes[page, :, row:row + o].float() * old[:, None, None] / scale[:, None, None])
                grown = (scale > old)[:, None, None]
                raw[page, :, row:row + o] = torch.where(grown, moved.view(torch.uint8), raw[page, :, row:row + o])
            q = torch.where(scale[:, None, None] > 0, part / scale[:, None, None], torch.zeros_like(part))
            raw[page, :, row + o:row + end - base] = quant(q).view(torch.uint8)
            scales[page, :, row // 16] = scale
            done += end - at
            at = end


def clones(cache):
    return F.Kv8Cache(*[t.view(torch.uint8).clone().view(t.dtype) if t.element_size() == 1 else t.clone() for t in cache])


def same(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("H,D,page_size", [(1, 64, 16), (8, 128, 64), (3, 128, 32), (2, 64, 192)])
def test_append_is_exact(cuda, code, dtype, H, D, page_size):
    """Ragged prompts, then steps of one, then of two tokens, then nothing for some; values
    that grow from token to token, so that scales do."""
    lens0 = [1, 17, 16, 100, 63, 0, 33]
    final = [n + 40 for n in lens0]
    table, pages = table_for(final, page_size, cuda, seed=D + H)
    cache = empty_cache(pages, H, page_size, D, code, cuda, seed=3)
    mine = clones(cache)
    lens, step = [0] * len(lens0), 0
    g = gen(cuda, 5)
    for new in [lens0, [1] * 7, [1] * 7, [1] * 7, [2] * 7, [0, 3, 0, 17, 1, 16, 15], [0, 0, 0, 1, 0, 0, 0]]:
        lens = [n + m for n, m in zip(lens, new)]
        T = sum(new)
        k, v = (((torch.randn(T, H + 1, D, device=cuda, generator=g) *
                  torch.exp(torch.randn(T, 1, 1, device=cuda, generator=g) + 0.5 * step))).to(dtype)[:, 1:] for _ in "kv")
        cu = ints([sum(new[:b]) for b in range(len(new) + 1)], cuda)
        assert F.kv8_append(k, v, cache, table, ints(lens, cuda), cu_new=cu, max_new=max(new) + step % 2) is None
        fp32_append(k, mine.k_pages, mine.k_scales, code, table, lens, new)
        fp32_append(v, mine.v_pages, mine.v_scales, code, table, lens, new)
        assert same(cache, mine), step
        step += 1
    assert status() == 0


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_append_behind_rows_with_any_scale(cuda, code):
    """Blocks that something else filled, with scales that are no powers of two: some
    grow, some keep their scale and are divided by it."""
    H, D, S = 4, 64, 32
    lens0, new = [5, 20, 31, 47, 10], [3, 1, 1, 1, 6]
    table, pages = table_for([n + m for n, m in zip(lens0, new)], S, cuda, seed=6)
    cache = random_cache(pages, H, S, D, code, cuda, seed=6)
    mine = clones(cache)
    lens = [n + m for n, m in zip(lens0, new)]
    T = sum(new)
    x = (torch.randn(T, H, D, device=cuda, generator=gen(cuda, 7)) *
         torch.exp(2 * torch.randn(T, H, 1, device=cuda, generator=gen(cuda, 8)))).to(BF16)
    cu = ints([sum(new[:b]) for b in range(6)], cuda)
    F.kv8_append(x, -x, cache, table, ints(lens, cuda), cu_new=cu, max_new=6)
    fp32_append(x, mine.k_pages, mine.k_scales, code, table, lens, new)
    fp32_append(-x, mine.v_pages, mine.v_scales, code, table, lens, new)
    assert same(cache, mine) and status() == 0


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_append_extremes(cuda, code):
    """Zero blocks, the smallest and largest values, infinities and NaN, and a zero
    block that grows later."""
    H, D, S = 1, 128, 16
    table, pages = table_for([16, 16, 16, 16, 16], S, cuda, seed=1)
    cache = empty_cache(pages, H, S, D, code, cuda)
    mine = clones(cache)
    for lens in ([1] * 5, [2] * 5, [3] * 5):
        x = torch.zeros(5, H, D, device=cuda, dtype=BF16)
        if lens[0] == 2:
            x[1, 0, 5] = 2.0 ** -133  # bf16's smallest
            x[2] = torch.finfo(BF16).max
            x[3, 0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), 2.0])
        if lens[0] == 3:
            x += 1.5
        F.kv8_append(x, -x, cache, table, ints(lens, cuda))
        fp32_append(x, mine.k_pages, mine.k_scales, code, table, lens, [1] * 5)
        fp32_append(-x, mine.v_pages, mine.v_scales, code, table, lens, [1] * 5)
        for a, b in zip(cache, mine):
            assert torch.equal(a.float().nan_to_num(1e9), b.float().nan_to_num(1e9))
    assert status() == 0


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot,Hq,H", [(128, 128, 32, 8), (128, 48, 5, 1), (64, 64, 4, 4), (64, 16, 0, 2)])
def test_append_turned(cuda, code, interleaved, D, rot, Hq, H):
    lens0, new = [2000, 5, 0, 64], [33, 5, 0, 1]
    S = 32
    table, pages = table_for(lens0, S, cuda, seed=7)
    cache = empty_cache(pages, H, S, D, code, cuda)
    for t in cache[2:]:
        t.fill_(2.0 ** -20)  # the blocks' older rows: nothing that would set the scale
    T = sum(new)
    g = gen(cuda, 11)
    qkv = torch.randn(T, Hq + 2 * H, D, device=cuda, generator=g).to(BF16)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
    f, m = F.rope_inv_freq(rot, scaling="yarn", factor=2.0, device=cuda)
    cu = ints([sum(new[:b]) for b in range(5)], cuda)
    got = F.kv8_append(k, v, cache, table, ints(lens0, cuda), cu_new=cu, max_new=33, q=q if Hq else None, inv_freq=f,
                       interleaved=interleaved, mscale=m)
    pos = torch.cat([torch.arange(n - d, n) for n, d in zip(lens0, new)]).to(cuda)
    if Hq:  # the same arithmetic as rope's
        assert torch.equal(got, F.rope(q, pos, f, interleaved, m))
    else:
        assert got is None
    turned = ok.rope(k, pos, f, interleaved, m)
    noise = 8 * 2.0 ** -24 * m * k.double().abs().amax(-1, keepdim=True) * 2
    done = 0
    for b, (n, d) in enumerate(zip(lens0, new)):
        if not d:
            continue
        back = ok.gather(cache.k_pages.double(), cache.k_scales, table, b, n).transpose(0, 1)[n - d:]
        scale = cache.k_scales.double()[table[b, :-(-n // S)].long()].transpose(1, 2).flatten(0, 1)  # [blocks, H]
        want, eps = turned[done:done + d], noise[done:done + d]
        step = scale[torch.arange(n - d, n, device=cuda) // 16][..., None]
        # e4m3: half a step is 2^-4 of the value (scales are powers of two), or 2^-10 of the scale below 2^-6
        half = step * 0.5 if code == INT8 else torch.maximum(want.abs() * 2.0 ** -4, step * 2.0 ** -10)
        assert torch.all((back - want).abs() <= half * (1 + 2.0 ** -20) + 2 * eps)
        for blk in range((n - d) // 16, -(-n // 16)):  # the scale is what its rows need, and no more than that
            rows = [i for i in range(done, done + d) if (n - d + i - done) // 16 == blk]
            amax = want[[i - done for i in rows]].abs().amax((0, 2))
            top = ok.TOP[code]
            assert torch.all(scale[blk] * top >= amax * (1 - 2.0 ** -20))
            assert torch.all(scale[blk] * top <= amax * (1 + 2.0 ** -20) * (2.0 if code == E4M3 else 1.0))
        done += d
    assert status() == 0


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("new", [[700] + [1] * 40, [1] * 33 + [0, 900, 0, 17] + [2] * 30, [0] * 70 + [333]])
def test_append_one_long_among_many(cuda, code, new):
    """Thread blocks shared out by cu_new: the same bits as each sequence appended by itself,
    and a bad entry among them is reported."""
    H, D, S, Hq = 2, 128, 32, 4
    lens = [n + (b * 7) % 45 for b, n in enumerate(new)]
    table, pages = table_for(lens, S, cuda, seed=9)
    x = torch.randn(sum(new), Hq + 2 * H, D, device=cuda, generator=gen(cuda, 5)).to(BF16)
    q, k, v = x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:]
    f, m = F.rope_inv_freq(D, device=cuda)
    got, one = random_cache(pages, H, S, D, code, cuda, 9), random_cache(pages, H, S, D, code, cuda, 9)
    cu = [sum(new[:b]) for b in range(len(new) + 1)]
    turned = F.kv8_append(k, v, got, table, ints(lens, cuda), cu_new=ints(cu, cuda), max_new=max(new), q=q, inv_freq=f)
    for b, n in enumerate(new):
        if n:
            rows = slice(cu[b], cu[b + 1])
            alone = F.kv8_append(k[rows], v[rows], one, table[b:b + 1], ints([lens[b]], cuda), q=q[rows], inv_freq=f)
            assert torch.equal(alone, turned[rows])
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, one))
    assert status() == 0
    at = len(new) // 2
    for bad in (-1, sum(new) + 1):
        before = clones(got)
        F.kv8_append(k, v, got, table, ints(lens, cuda), cu_new=ints(cu[:at] + [bad] + cu[at + 1:], cuda), max_new=max(new),
                     inv_freq=f)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="bad paged-KV index"):
            F.kv8_append(k, v, got, table, ints(lens, cuda), cu_new=ints(cu, cuda), max_new=max(new), inv_freq=f)
        for t, u in zip(got, before):  # nothing of the sequences on both sides of it
            for b in (at - 1, at):
                own = table[b, :-(-lens[b] // S)].long()
                assert torch.equal(t[own].view(torch.uint8), u[own].view(torch.uint8))


def test_append_steps_equal_a_prompt(cuda):
    """e4m3: one token at a time gives the prompt's scales, and its codes wherever no
    older code sank below the smallest subnormal when it moved."""
    H, D, S, n = 2, 128, 16, 48
    table, pages = table_for([n], S, cuda, seed=2)
    a, b = (empty_cache(pages, H, S, D, E4M3, cuda, seed=s) for s in (1, 2))
    x = torch.randn(n, H, D, device=cuda, generator=gen(cuda, 4)).to(BF16)
    F.kv8_append(x, x, a, table, ints([n], cuda))
    for i in range(n):
        F.kv8_append(x[i:i + 1], x[i:i + 1], b, table, ints([i + 1], cuda))
    u, w = (ok.gather(c.k_pages.double(), c.k_scales, table, 0, n) for c in (a, b))
    used = table[0, :3].long()
    assert torch.equal(a.k_scales[used], b.k_scales[used])
    big = u.abs() >= a.k_scales[used].double().transpose(0, 1).flatten(1).repeat_interleave(16, 1)[..., None] * 2.0 ** -5
    assert torch.equal(u[big], w[big]) and torch.all((u - w).abs() <= 2.0 ** -8)


def test_append_refusals_on_the_device(cuda):
    """Bad lengths, cu_new entries and page ids set status 3 and write nothing there;
    the next call raises once."""
    H, D, S = 2, 128, 32
    f, _ = F.rope_inv_freq(128, device=cuda)
    x = torch.ones(4, H, D, device=cuda, dtype=BF16)
    good = dict(table=[[0, 1], [2, 3]], lens=[2, 34], cu=[0, 2, 4], max_new=2)
    bad = [dict(table=[[8, 1], [2, 3]]), dict(table=[[-1, 1], [2, 3]]), dict(lens=[1, 34]), dict(lens=[2, 65]),
           dict(lens=[-5, 34]), dict(cu=[0, 3, 4], max_new=2), dict(cu=[-1, 1, 4]), dict(cu=[2, 0, 4], lens=[2, 34]),
           dict(cu=[0, 2, 5], max_new=8)]
    for kw in bad:
        a = dict(good, **kw)
        cache = empty_cache(8, H, S, D, E4M3, cuda)
        before = clones(cache)
        F.kv8_append(x, x, cache, ints(a["table"], cuda), ints(a["lens"], cuda), cu_new=ints(a["cu"], cuda),
                     max_new=a["max_new"], inv_freq=f)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="bad paged-KV index"):
            F.kv8_append(x, x, cache, ints(good["table"], cuda), ints(good["lens"], cuda), inv_freq=f)
        touched = {p for row in good["table"] for p in row}
        for p in range(8):
            if p not in touched:
                assert torch.equal(cache.k_pages[p].view(torch.uint8), before.k_pages[p].view(torch.uint8))
    assert status() == 0


# --------------------------------------------------------------- attention
def attention_tolerance(bounds, dtype, D):
    """`bounds` as ok.attention gives them.  Scores: D products and sums and a handful of
    scalings in fp32, (D + 16) 2^-24 of scale * sum |q| |k| at most; a weight is off by
    twice that (numerator and sum), by half a step of the 16-bit weight (2^-11; 2^-22 for fp16,
    whose weights are two 16-bit numbers, the second the rounding of the first) and by
    the fp32 exponentials and sums, 2^-18; what a weight's error moves is at most its
    share of sum p |v|.  A weight enters as f16(2^15 p vs / R) with R at most twice the
    largest V scale: below f16's normal numbers that is off by up to 2^-25, which is
    2^-40 R / vs of the weight of the maximum, so 2^-39 times the largest V scale and
    code for each position.  Then the output's rounding (and fp16's smallest subnormal's half)."""
    o, a, s, w = bounds
    weight = 2.0 ** -22 if dtype == FP16 else 2.0 ** -11
    noise = (2 * (D + 16) * 2.0 ** -24 * s + weight + 2.0 ** -18) * a + 2.0 ** -39 * w
    return noise + (o.abs() + noise) * (torch.finfo(dtype).eps / 2) + 2.0 ** -25 * (dtype == FP16)


def random_cache(pages, H, page_size, D, code, device, seed, wild=True):
    """Codes of all magnitudes and scales that differ from block to block."""
    c = F.kv8_cache(pages, H, page_size, D, code, device)
    g = gen(device, seed)
    for t in c[:2]:
        x = torch.randn(t.shape, device=device, generator=g) * (60.0 if code == INT8 else 100.0)
        t.copy_(x.round().clamp(-127, 127).to(INT8) if code == INT8 else x.clamp(-448, 448).to(E4M3))
    for t in c[2:]:
        t.copy_(torch.exp((1.0 if wild else 0.0) * torch.randn(t.shape, device=device, generator=g)) / 100)
    return c


def spoil(cache, table, lens, page_size):
    """NaN (e4m3) or extreme codes, and NaN scales, wherever no sequence's positions are."""
    live = torch.zeros(cache.k_pages.shape[0], page_size, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(-(-n // page_size)):
            live[int(table[b, j]), :max(0, min(page_size, n - j * page_size))] = True
    dead = ~live.to(cache.k_pages.device)
    for t in cache[:2]:
        t.view(torch.uint8).masked_fill_(dead[:, None, :, None], 0x7F)
    blocks = dead.view(-1, page_size // 16, 16).all(-1)
    for t in cache[2:]:
        t.masked_fill_(blocks[:, None], float("nan"))


def check_attention(cuda, B, T, Hq, H, D, page_size, lens, max_len, code, dtype, seed, scale=None, wild=True, q_gain=1.0):
    table, pages = table_for(lens, page_size, cuda, seed=seed)
    table = torch.nn.functional.pad(table, (0, max(0, -(-max_len // page_size) - table.shape[1])), value=-7).contiguous()
    cache = random_cache(pages, H, page_size, D, code, cuda, seed, wild)
    spoil(cache, table.cpu(), lens, page_size)
    q = (torch.randn(B, T, Hq, D, device=cuda, generator=gen(cuda, seed + 1)) * q_gain).to(dtype)
    got = F.gqa_decode_attention_kv8(q[:, 0] if T == 1 else q, cache, table, ints(lens, cuda), max_len, scale)
    bounds = ok.attention(q, doubles(cache), table.cpu(), lens, scale)
    err = (got.view(q.shape).double() - bounds[0]).abs()
    tol = attention_tolerance(bounds, dtype, D)
    assert torch.all(torch.isfinite(got))
    assert torch.all(err <= tol), float((err / tol.clamp(min=1e-300)).max())
    assert status() == 0
    return got


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("D,page_size,dtype", [(128, 64, BF16), (128, 16, FP16), (64, 32, BF16), (64, 128, FP16),
                                               (128, 32, BF16), (128, 192, BF16), (64, 16, BF16)])
@pytest.mark.parametrize("T", [1, 3])
def test_attention_ragged(cuda, code, D, page_size, dtype, T):
    lens = [1, 0, 2, 15, 16, 17, 63, 64, 65, 130, 1000, 777, 511]
    check_attention(cuda, len(lens), T, 8, 2, D, page_size, lens, 1000, code, dtype, seed=D + page_size + T)


@pytest.mark.parametrize("Hq,H,T", [(1, 1, 1), (7, 1, 1), (16, 1, 1), (32, 2, 1), (9, 3, 1), (8, 8, 16), (14, 2, 4),
                                    (16, 1, 16), (32, 8, 4), (32, 8, 2), (12, 4, 7), (8, 1, 2)])
def test_attention_groups_and_tokens(cuda, Hq, H, T):
    """Every split of query rows over the heads that share a KV head, one token and more."""
    lens = [300, 5, 0, T, 129]
    check_attention(cuda, 5, T, Hq, H, 128, 64, lens, 448, E4M3, BF16, seed=Hq + T)


@pytest.mark.parametrize("B,L,H,code", [(1, 1, 8, E4M3), (1, 512, 8, E4M3), (1, 4096, 8, INT8), (1, 20011, 1, E4M3),
                                        (3, 8192, 8, E4M3), (64, 700, 4, INT8), (2, 33000, 2, E4M3)])
def test_attention_lengths(cuda, B, L, H, code):
    lens = [max(1, L - 37 * b) for b in range(B)]
    check_attention(cuda, B, 1, 4 * H, H, 128, 64, lens, L + 100, code, BF16, seed=L)


@pytest.mark.parametrize("B,H,top", [(33, 8, 200), (290, 1, 150), (700, 1, 70), (1500, 2, 20)])
def test_attention_many_sequences(cuda, B, H, top):
    """More sequences than a warp has lanes, or looks up at once; many of them empty."""
    g = torch.Generator().manual_seed(B)
    lens = (torch.randint(-top // 4, top + 1, (B,), generator=g)).clamp(min=0).tolist()
    got = check_attention(cuda, B, 1, 4 * H, H, 64, 16, lens, top, E4M3, BF16, seed=B)
    assert got[[n == 0 for n in lens]].count_nonzero() == 0
    for at in (B - 1, B // 2, 32):
        bad = list(lens)
        bad[at] = top + 1
        table, pages = table_for(lens, 16, cuda, seed=B)
        table = torch.nn.functional.pad(table, (0, 8), value=0).clamp(min=0).contiguous()
        cache = random_cache(pages, H, 16, 64, E4M3, cuda, B)
        q = torch.zeros(B, 4 * H, 64, device=cuda, dtype=BF16)
        F.gqa_decode_attention_kv8(q, cache, table, ints(bad, cuda), top)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="bad paged-KV index"):
            F.gqa_decode_attention_kv8(q, cache, table, ints(lens, cuda), top)
    assert status() == 0


def test_attention_peaked_and_flat(cuda):
    """Scores far apart (large q) and all equal (q = 0), large and tiny scales of q."""
    for gain, dtype in ((40.0, BF16), (0.0, BF16), (1e30, BF16), (1e-30, BF16), (2000.0, FP16)):
        scale = None if gain in (40.0, 0.0) else 0.05 / gain
        check_attention(cuda, 2, 1, 8, 2, 128, 64, [1000, 64], 1000, E4M3, dtype, seed=3, scale=scale, q_gain=gain)


def test_attention_scales_of_all_sizes(cuda):
    """V scales from 0 over 2^-100 to 2^20 between a sequence's blocks, K scales with zeros."""
    H, D, S, n = 1, 128, 16, 320
    table, pages = table_for([n], S, cuda, seed=1)
    cache = random_cache(pages, H, S, D, E4M3, cuda, seed=1)
    powers = [2.0 ** e for e in (-100, -60, -20, -10, 0, 20, 3, -3, 10, -126)] + [0.0] * 10
    for i, p in enumerate(powers):
        cache.v_scales[table[0, i]] = p
        if i % 3 == 0:
            cache.k_scales[table[0, i]] = 0.0
    q = torch.randn(1, 1, 4, D, device=cuda, generator=gen(cuda, 2)).to(BF16)
    for m in (n, 16, 32, 96, 160, 176, 48):
        got = F.gqa_decode_attention_kv8(q, cache, table, ints([m], cuda), n)
        bounds = ok.attention(q, doubles(cache), table.cpu(), [m])
        assert torch.all((got.double() - bounds[0]).abs() <= attention_tolerance(bounds, BF16, D)), m
    zero = torch.zeros_like(cache.v_scales)
    got = F.gqa_decode_attention_kv8(q, F.Kv8Cache(*cache[:3], zero), table, ints([n], cuda), n)
    assert torch.all(got == 0)


def test_attention_nan_where_it_is_seen(cuda):
    """A NaN code inside a sequence shows in that KV head's outputs and no others."""
    table, pages = table_for([200, 200], 64, cuda, seed=5)
    cache = random_cache(pages, 2, 64, 128, E4M3, cuda, seed=5)
    q = torch.randn(2, 8, 128, device=cuda, generator=gen(cuda, 6)).to(BF16)
    cache.k_pages.view(torch.uint8)[table[0, 1], 1, 3, 7] = 0x7F
    got = F.gqa_decode_attention_kv8(q, cache, table, ints([200, 200], cuda), 200)
    bad = torch.isnan(got)
    assert torch.all(bad[0, 4:]) and not torch.any(bad[0, :4]) and not torch.any(bad[1])


@pytest.mark.parametrize("D,Hq,H", [(128, 8, 2), (64, 16, 1)])
def test_attention_nan_that_some_queries_see(cuda, D, Hq, H):
    """NaN values among the newest positions: the queries before them do not see them, the
    others do in those dims only."""
    T, n = 5, 200
    table, pages = table_for([n, 64], 32, cuda, seed=5)
    cache = random_cache(pages, H, 32, D, E4M3, cuda, seed=5)
    q = torch.randn(2, T, Hq, D, device=cuda, generator=gen(cuda, 6)).to(BF16)
    lens = ints([n, 64], cuda)
    clean = ok.attention(q, doubles(cache), table.cpu(), [n, 64])
    raw = cache.v_pages.view(torch.uint8)
    for pos, d in ((n - 2, 7), (n - 2, 8), (n - 1, 40)):  # seen by t >= 3, t >= 3 and t = 4
        raw[table[0, pos // 32], 0, pos % 32, d] = 0xFF if d == 8 else 0x7F
    got = F.gqa_decode_attention_kv8(q, cache, table, lens, n)
    want = torch.zeros(2, T, Hq, D, dtype=torch.bool, device=cuda)
    want[0, 3:, :Hq // H, 7:9] = True
    want[0, 4:, :Hq // H, 40] = True
    assert torch.equal(torch.isnan(got), want)
    free = torch.ones_like(want)
    free[0, 3:, :Hq // H] = False  # (the others also miss nothing but the NaN codes)
    tol = attention_tolerance(clean, BF16, D)
    assert torch.all(((got.double() - clean[0]).abs() <= tol)[free])


def test_attention_is_deterministic_and_shares_pages(cuda):
    """Two sequences over the same pages agree within the bounds (where their tiles are split
    between the SMs depends on their place in the batch), and every repetition gives the same bits."""
    table, pages = table_for([5000], 64, cuda, seed=8)
    cache = random_cache(pages, 8, 64, 128, E4M3, cuda, seed=8)
    q = torch.randn(1, 1, 32, 128, device=cuda, generator=gen(cuda, 9)).to(BF16).expand(2, 1, 32, 128).contiguous()
    table = table.expand(2, -1).contiguous()
    args = (cache, table, ints([5000, 5000], cuda), 5000)
    first = F.gqa_decode_attention_kv8(q, *args)
    bounds = ok.attention(q, doubles(cache), table.cpu(), [5000, 5000])
    assert torch.all((first.double() - bounds[0]).abs() <= attention_tolerance(bounds, BF16, 128))
    for _ in range(20):
        assert torch.equal(F.gqa_decode_attention_kv8(q, *args), first)


def test_attention_bad_pages_and_lengths_set_status(cuda):
    table, pages = table_for([256, 100], 64, cuda, seed=1)
    cache = random_cache(pages, 2, 64, 128, E4M3, cuda, seed=1)
    q = torch.randn(2, 8, 128, device=cuda).to(BF16)
    good = F.gqa_decode_attention_kv8(q, cache, table, ints([256, 100], cuda), 256)
    for lens, entry in (([257, 100], None), ([256, -1], None), ([256, 100], pages), ([256, 100], -1)):
        t = table.clone()
        if entry is not None:
            t[0, 1] = entry
        got = F.gqa_decode_attention_kv8(q, cache, t, ints(lens, cuda), 256)
        assert status() == 3
        if lens[1] == 100:
            assert torch.equal(got[1], good[1])
        with pytest.raises(RuntimeError, match="bad paged-KV index"):
            F.gqa_decode_attention_kv8(q, cache, table, ints([256, 100], cuda), 256)
        assert status() == 0
    assert torch.equal(F.gqa_decode_attention_kv8(q, cache, table, ints([256, 100], cuda), 256), good)


def test_refusals(cuda):
    table, pages = table_for([64, 64], 64, cuda, seed=1)
    cache = random_cache(pages, 2, 64, 128, E4M3, cuda, seed=1)
    q = torch.zeros(2, 8, 128, device=cuda, dtype=BF16)
    lens = ints([64, 64], cuda)
    k_pages, v_pages, k_scales, v_scales = cache
    A = F.gqa_decode_attention_kv8
    for args, text in (((q.float(), cache, table, lens, 64), "dtype"), ((q[..., :64], cache, table, lens, 64), "contiguous"),
                       ((q[..., :64].contiguous(), cache, table, lens, 64), "shape"),
                       ((q[:, :7].contiguous(), cache, table, lens, 64), "multiple of Hkv"),
                       ((q, cache, table, lens, 1000), "max_seq_len"), ((q, cache, table.long(), lens, 64), "dtype"),
                       ((q, cache, table[:1], lens, 64), "shape"), ((q, cache, table, lens[:1], 64), "shape"),
                       ((q, (k_pages.view(INT8), v_pages, k_scales, v_scales), table, lens, 64), "dtype"),
                       ((q, (k_pages, v_pages, k_scales[..., :2], v_scales), table, lens, 64), "contiguous|shape"),
                       ((q, (k_pages.to(torch.bfloat16), v_pages, k_scales, v_scales), table, lens, 64), "dtype"),
                       ((q, (k_pages, v_pages[:1], k_scales, v_scales), table, lens, 64), "shape"),
                       ((q, (k_pages, v_pages.cpu(), k_scales, v_scales), table, lens, 64), "CUDA"),
                       ((q[None].expand(17, 2, 8, 128).transpose(0, 1).contiguous(), cache, table, lens, 64), "query tokens")):
        with pytest.raises(RuntimeError, match=text):
            A(*args)
    k = torch.zeros(2, 2, 128, device=cuda, dtype=BF16)
    f, _ = F.rope_inv_freq(128, device=cuda)
    for args, kw, text in (((k.float(), k, cache, table, lens), {}, "dtype"), ((k, k.half(), cache, table, lens), {}, "dtype"),
                           ((k[:, :1], k[:, :1], cache, table, lens), {}, "shape"), ((k, k[:1], cache, table, lens), {}, "shape"),
                           ((k, k, cache, table, lens), dict(q=q), "inv_freq"),
                           ((k, k, cache, table, lens), dict(cu_new=lens, max_new=1), "cu_new"),
                           ((k, k, cache, table, lens), dict(max_new=3), "B \\* max_new"),
                           ((k, k, cache, table, lens), dict(inv_freq=f.float()), "dtype"),
                           ((k, k, cache, table, lens), dict(q=q[:1], inv_freq=f), "shape"),
                           ((k, k, cache, table, lens), dict(inv_freq=F.rope_inv_freq(256, device=cuda)[0]), "rotated dims")):
        with pytest.raises(RuntimeError, match=text):
            F.kv8_append(*args, **kw)
    assert status() == 0


def test_refused_steps_leave_the_cache(cuda):
    """Whatever the composite refuses, it refuses before the append."""
    table, pages = table_for([64, 64], 64, cuda, seed=1)
    cache = random_cache(pages, 2, 64, 128, E4M3, cuda, seed=1)
    before = clones(cache)
    f, _ = F.rope_inv_freq(128, device=cuda)
    rows = lambda n, h: torch.ones(n, h, 128, device=cuda, dtype=BF16)  # noqa: E731
    lens = ints([40, 41], cuda)
    for n, h, kw, text in ((2, 7, {}, "multiple of Hkv"), (2, 64, {}, "<= 16"), (34, 8, {}, "query tokens"),
                           (0, 8, {}, "query tokens"), (3, 8, {}, "same number"), (2, 8, dict(max_len=1000), "max_seq_len"),
                           (2, 8, dict(max_len=0), "size"), (2, 8, dict(scale=0.0), "scale"),
                           (2, 8, dict(scale=1e-60), "scale"), (2, 8, dict(scale=float("inf")), "scale"),
                           (2, 8, dict(mscale=float("nan")), "mscale"), (2, 8, dict(f=f.float()), "dtype"),
                           (2, 8, dict(q=rows(1, 8)), "shape"), (2, 8, dict(q=rows(2, 8).half()), "dtype")):
        a = dict(dict(q=rows(n, h), max_len=64, f=f, mscale=1.0, scale=None), **kw)
        with pytest.raises(RuntimeError, match=text):
            F.decode_attention_kv8(a["q"], rows(n, 2), rows(n, 2), cache, table, lens, a["max_len"], a["f"],
                                   mscale=a["mscale"], scale=a["scale"])
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(cache, before))
    assert status() == 0


def test_append_of_more_than_max_new_is_reported(cuda):
    """cu_new that brings rows where max_new says none: nothing written, and status set."""
    cache = empty_cache(4, 1, 16, 64, E4M3, cuda)
    before = clones(cache)
    x = torch.ones(3, 1, 64, device=cuda, dtype=BF16)
    args = cache, ints([[0], [1]], cuda), ints([2, 1], cuda)
    F.kv8_append(x, x, *args, cu_new=ints([0, 0, 0], cuda), max_new=0)
    torch.cuda.synchronize()
    assert status() == 0
    F.kv8_append(x, x, *args, cu_new=ints([0, 2, 3], cuda), max_new=0)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="bad paged-KV index"):
        F.kv8_append(x, x, *args, cu_new=ints([0, 2, 3], cuda), max_new=2)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, before))


# ---------------------------------------------------------- used together
def decode_run(cuda, code, interleaved, steps, T, prompt, capture=False):
    """A prompt and decode steps of T tokens through the composite, as a server would
    run them; returns the last outputs and what the oracle makes of the same cache."""
    B, Hq, H, D, S = len(prompt), 8, 2, 128, 32
    final = [n + steps * T for n in prompt]
    table, pages = table_for(final, S, cuda, seed=1)
    cache = empty_cache(pages, H, S, D, code, cuda)
    f, m = F.rope_inv_freq(D, device=cuda)
    g = gen(cuda, 21)
    rows = lambda n: torch.randn(n, Hq + 2 * H, D, device=cuda, generator=g).to(BF16)  # noqa: E731
    split = lambda x: (x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:])  # noqa: E731
    q, k, v = split(rows(sum(prompt)))
    cu = ints([sum(prompt[:b]) for b in range(B + 1)], cuda)
    lens = ints(prompt, cuda)
    F.kv8_append(k, v, cache, table, lens, cu_new=cu, max_new=max(prompt), inv_freq=f, interleaved=interleaved)
    x = rows(B * T)
    graph, out = None, None
    if capture:  # one graph, replayed for every step; the warm-up runs on a copy of the cache
        call = lambda c, n: F.decode_attention_kv8(*split(x), c, table, n, max(final), f, interleaved)  # noqa: E731
        call(clones(cache), lens + T)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(cache, lens)
    for _ in range(steps):
        lens += T
        x.copy_(rows(B * T))
        if capture:
            graph.replay()
        else:
            out = F.decode_attention_kv8(*split(x), cache, table, lens, max(final), f, interleaved)
    pos = (lens[:, None].long() - T + torch.arange(T, device=cuda)).flatten()
    turned = F.rope(split(x)[0], pos, f, interleaved).view(B, T, Hq, D)
    bounds = ok.attention(turned, doubles(cache), table.cpu(), final)
    return out.view(B, T, Hq, D), bounds[0], attention_tolerance(bounds, BF16, D)


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("T,interleaved,capture", [(1, False, False), (1, True, True), (3, False, True)])
def test_decode_run(cuda, code, T, interleaved, capture):
    out, o, tol = decode_run(cuda, code, interleaved, steps=20, T=T, prompt=[100, 1, 37], capture=capture)
    assert torch.all((out.double() - o).abs() <= tol)
    assert status() == 0


def test_graphs_of_one_stream_replay_at_once(cuda):
    """Two graphs captured on one stream, replayed on two: their workspaces are their own."""
    table, pages = table_for([6000, 6000], 64, cuda, seed=3)
    cache = random_cache(pages, 4, 64, 128, E4M3, cuda, seed=3)
    lens = ints([6000, 5990], cuda)
    qs = [torch.randn(2, 16, 128, device=cuda, generator=gen(cuda, s)).to(BF16) for s in (1, 2)]
    want = [F.gqa_decode_attention_kv8(q, cache, table, lens, 6000) for q in qs]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = [F.gqa_decode_attention_kv8(q, cache, table, lens, 6000) for _ in range(8)]
        graphs.append(g)
        outs.append(got)
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for w, got in zip(want, outs):
        assert all(torch.equal(o, w) for o in got)
    assert status() == 0


def test_streams_have_their_own_workspaces(cuda):
    table, pages = table_for([9000], 64, cuda, seed=4)
    cache = random_cache(pages, 2, 64, 128, INT8, cuda, seed=4)
    q = torch.randn(1, 8, 128, device=cuda, generator=gen(cuda, 1)).to(BF16)
    lens = ints([9000], cuda)
    want = F.gqa_decode_attention_kv8(q, cache, table, lens, 9000)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(F.gqa_decode_attention_kv8(q, cache, table, lens, 9000))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("capture", [False, True])
def test_shapes_share_a_workspace(cuda, capture):
    """Many segments cut between CTAs, one long sequence, and the many again: what one call
    leaves behind in the workspace means nothing to the next."""
    big, small = [300 - b % 7 * 40 for b in range(64)], [40000]
    calls, want = [], []
    for lens, H, seed in ((big, 32, 5), (small, 2, 6)):
        table, pages = table_for(lens, 64, cuda, seed=seed)
        cache = random_cache(pages, H, 64, 64, E4M3, cuda, seed=seed)
        q = torch.randn(len(lens), 8 * H, 64, device=cuda, generator=gen(cuda, seed)).to(BF16)
        calls.append((q, cache, table, ints(lens, cuda), max(lens)))
        o, a, s, w = ok.attention(q[:, None], doubles(cache), table.cpu(), lens)
        want.append((o[:, 0], attention_tolerance((o, a, s, w), BF16, 64)[:, 0]))
    order = [0, 1, 0, 0, 1, 0]
    run = lambda: [F.gqa_decode_attention_kv8(*calls[i]) for i in order]  # noqa: E731
    outs = run()
    if capture:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = run()
        for _ in range(2):
            g.replay()
    for i, got in zip(order, outs):
        assert torch.all((got.double() - want[i][0]).abs() <= want[i][1])
    assert status() == 0


def test_cache_past_32_bits(cuda):
    """Pages whose codes lie past 2^32 bytes: written, read, and nothing at the wrapped
    addresses touched."""
    H, D, S = 8, 128, 256
    per_page = H * S * D
    pages = (1 << 32) // per_page + 40
    cache = F.kv8_cache(pages, H, S, D, E4M3, cuda)
    table = ints([[pages - 1, 3, pages - 2]], cuda)
    f, _ = F.rope_inv_freq(D, device=cuda)
    g = gen(cuda, 1)
    k, v = (torch.randn(700, H, D, device=cuda, generator=g).to(BF16) for _ in "kv")
    F.kv8_append(k, v, cache, table, ints([700], cuda), inv_freq=f)
    live = [pages - 1, 3, pages - 2]
    assert all(int(cache.k_pages[p].view(torch.uint8).count_nonzero()) > 0 for p in live)
    rest = torch.ones(pages, dtype=torch.bool)
    rest[live] = False
    for lo in range(0, pages, 1024):
        sel = rest[lo:lo + 1024].nonzero().flatten() + lo
        assert int(cache.k_pages.view(torch.uint8)[sel.to(cuda)].count_nonzero()) == 0
    small = F.Kv8Cache(*[t.view(torch.uint8)[live].view(t.dtype) if t.element_size() == 1 else t[live] for t in cache])
    q = torch.randn(1, 32, D, device=cuda, generator=g).to(BF16)
    a = F.gqa_decode_attention_kv8(q, cache, table, ints([700], cuda), 700)
    b = F.gqa_decode_attention_kv8(q, small, ints([[0, 1, 2]], cuda), ints([700], cuda), 700)
    assert torch.equal(a, b) and status() == 0
