"""focal_rope on the GPU through the PyTorch layer, against 64-bit rotations.

Tolerance of an element, from the roundings that the kernel makes: cos and sin
to fp32, two products and a sum, 2^-24 each of at most mscale (|a| + |b|) (3 on
the way of either product; 4 leaves room for CUDA's own 64-bit cos and sin),
then half a step of the output type, plus its smallest subnormal's half."""
import pytest
import torch

import focal_b200 as F
from oracle import kv8 as ok

pytestmark = pytest.mark.gpu

TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def check(y, x, positions, f, interleaved, mscale=1.0):
    want = ok.rope(x, positions, f, interleaved, mscale)
    half = f.numel()
    r = x[..., :2 * half].double().abs()
    if interleaved:
        size = (r[..., 0::2] + r[..., 1::2]).repeat_interleave(2, -1)
    else:
        size = (r[..., :half] + r[..., half:]).repeat(1, 1, 2)
    noise = torch.zeros_like(want)
    noise[..., :2 * half] = size * (mscale * 4 * 2.0 ** -24)
    tol = noise + (want.abs() + noise) * (torch.finfo(x.dtype).eps / 2) + TINY[x.dtype]
    err = (y.double() - want).abs()
    assert y.dtype == x.dtype and y.shape == x.shape
    assert torch.all(err <= tol), float((err / tol).max())
    assert torch.equal(y[..., 2 * half:], x[..., 2 * half:])


def rows(T, H, D, dtype, device, seed=0, extra=0):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(T, H + extra, D, device=device, generator=g).to(dtype)[:, :H]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D,rot", [(1, 1, 16, 16), (1, 40, 128, 128), (8, 9, 128, 64), (7, 3, 64, 16),
                                       (333, 5, 96, 80), (1025, 2, 256, 208), (65, 33, 128, 128), (3, 2, 1024, 1024),
                                       (4099, 1, 24, 16)])
def test_rope_matches_64_bits(cuda, dtype, interleaved, T, H, D, rot):
    x = rows(T, H, D, dtype, cuda, seed=T + D)
    f, m = F.rope_inv_freq(rot, scaling="yarn", factor=4.0, device=cuda)
    pos = torch.arange(T, device=cuda) * 977 + 5
    check(F.rope(x, pos, f, interleaved, m), x, pos, f, interleaved, m)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_packed_rows_and_far_positions(cuda, dtype):
    """A view of packed rows (strided heads' extent), int32 and int64 positions up to
    and past 2^31, negative ones, and rows that are read with stride 0."""
    f, m = F.rope_inv_freq(128, device=cuda)
    x = rows(6, 4, 128, dtype, cuda, extra=3)
    pos = torch.tensor([0, 1, -1, 1048575, 2 ** 31 - 1, -(2 ** 31)], device=cuda)
    for p in (pos, pos.int()):
        check(F.rope(x, p, f), x, pos, f, False)
    far = torch.tensor([2 ** 33 + 1, 2 ** 40, 5, 6, 7, 8], device=cuda)
    check(F.rope(x, far, f, True), x, far, f, True)
    one = x[:1].expand(6, 4, 128)
    check(F.rope(one, pos, f), one, pos, f, False)


def test_in_place_and_out(cuda):
    f, m = F.rope_inv_freq(64, device=cuda)
    pos = torch.arange(50, device=cuda) + 1000
    base = rows(50, 12, 128, torch.bfloat16, cuda)
    want = F.rope(base[:, 2:7], pos, f)
    buf = base.clone()
    part = buf[:, 2:7]
    assert F.rope(part, pos, f, out=part).data_ptr() == part.data_ptr()
    assert torch.equal(part, want) and torch.equal(buf[:, :2], base[:, :2]) and torch.equal(buf[:, 7:], base[:, 7:])
    out = torch.full((50, 8, 136), 3.0, dtype=torch.bfloat16, device=cuda)
    F.rope(base[:, 2:7], pos, f, out=out[:, 1:6, :128])
    assert torch.equal(out[:, 1:6, :128], want)
    out[:, 1:6, :128] = 3.0
    assert torch.all(out == 3.0)  # nothing written beside the rows


def test_infinities_and_nan_stay_in_their_pairs(cuda):
    f, _ = F.rope_inv_freq(32, device=cuda)
    x = rows(2, 1, 32, torch.bfloat16, cuda)
    x[0, 0, 3] = float("inf")
    x[1, 0, 20] = float("nan")
    pos = torch.tensor([7, 9], device=cuda)
    y = F.rope(x, pos, f)
    bad = ~torch.isfinite(y)
    assert bad[0, 0].nonzero().flatten().tolist() == [3, 19] and bad[1, 0].nonzero().flatten().tolist() == [4, 20]


def test_refusals(cuda):
    f, _ = F.rope_inv_freq(64, device=cuda)
    x = rows(4, 2, 128, torch.bfloat16, cuda)
    pos = torch.arange(4, device=cuda)
    for bad, text in (((x.transpose(1, 2), pos, f), "contiguous last"), ((x[0], pos, f), "shape"),
                      ((x.double(), pos, f), "dtype"), ((x, pos.float(), f), "dtype"), ((x, pos[:3], f), "shape"),
                      ((x, pos, f.float()), "dtype"), ((x, pos.cpu(), f), "same device"), ((x, pos, f.cpu()), "CUDA"),
                      ((x[..., 4:124], pos, f), "aligned"), ((rows(4, 2, 100, x.dtype, cuda), pos, f), "strides|multiple")):
        with pytest.raises(RuntimeError, match=text):
            F.rope(*bad)
    for out, text in ((x[:, :1].expand(4, 2, 128), "overlap|more than one element"), (x.half(), "dtype"), (x[:3], "shape"),
                      (x[:, 1:], "shape")):
        with pytest.raises(RuntimeError, match=text):
            F.rope(x, pos, f, out=out)
    assert F.rope(x[:0], pos[:0], f).shape == (0, 2, 128)


def test_other_stream_and_graph(cuda):
    f, _ = F.rope_inv_freq(128, device=cuda)
    x = rows(100, 8, 128, torch.float16, cuda)
    pos = torch.arange(100, device=cuda)
    want = F.rope(x, pos, f)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = F.rope(x, pos, f)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = F.rope(x, pos, f)
    x.copy_(rows(100, 8, 128, torch.float16, cuda, seed=9))
    pos += 17
    want = F.rope(x, pos, f)
    g.replay()
    assert torch.equal(y, want)
