"""8-bit cache calls in captures that were begun on the stream itself, without torch's graph
API: what a graph writes to between its inputs and outputs stays its own for as long as the
graph lives, and is free again behind it."""
import ctypes
import gc
import time

import pytest
import torch

import focal_b200 as F
from focal_b200 import _lib
from test_gpu_kv8 import clones, gen, ints, random_cache, same, status, table_for

pytestmark = pytest.mark.gpu

E4M3, BF16 = torch.float8_e4m3fn, torch.bfloat16


class Graph:
    """A stream capture through the runtime library that torch has loaded."""

    def __init__(self, stream):
        self.rt, self.stream = ctypes.CDLL("libcudart.so.12"), ctypes.c_void_p(stream.cuda_stream)
        self.graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()

    def __enter__(self):
        self.ok(self.rt.cudaStreamBeginCapture(self.stream, 2))  # relaxed: torch may allocate meanwhile
        return self

    def __exit__(self, *err):
        self.ok(self.rt.cudaStreamEndCapture(self.stream, ctypes.byref(self.graph)))
        self.ok(self.rt.cudaGraphInstantiate(ctypes.byref(self.exec), self.graph, ctypes.c_ulonglong(0)))
        self.ok(self.rt.cudaGraphDestroy(self.graph))  # what was instantiated lives on

    def replay(self):
        self.ok(self.rt.cudaGraphLaunch(self.exec, self.stream))

    def destroy(self):
        self.ok(self.rt.cudaGraphExecDestroy(self.exec))

    @staticmethod
    def ok(rc):
        assert rc == 0, rc


def case(cuda, B, n, seed):
    Hq, H, D, S = 16, 4, 128, 64
    lens = [n - 11 * b for b in range(B)]
    table, pages = table_for(lens, S, cuda, seed=seed)
    cache = random_cache(pages, H, S, D, E4M3, cuda, seed=seed)
    x = torch.randn(B, Hq + 2 * H, D, device=cuda, generator=gen(cuda, seed)).to(BF16)
    f, _ = F.rope_inv_freq(D, device=cuda)
    return dict(q=x[:, :Hq], k=x[:, Hq:Hq + H], v=x[:, Hq + H:], cache=cache, table=table, lens=ints(lens, cuda), n=n, f=f)


def attend(c):
    return F.gqa_decode_attention_kv8(c["q"].contiguous(), c["cache"], c["table"], c["lens"], c["n"])


def step(c):
    return F.decode_attention_kv8(c["q"], c["k"], c["v"], c["cache"], c["table"], c["lens"], c["n"], c["f"])


@pytest.mark.parametrize("call", [attend, step])
def test_graphs_keep_what_they_write_to(cuda, call):
    """Graphs captured one after another on one stream, then the stream's free memory handed out to
    others: replays give the captured call's bits and leave the others' memory alone."""
    cases = [case(cuda, B, n, seed) for B, n, seed in ((2, 6000, 1), (5, 3000, 2), (1, 900, 3))]
    if call is attend:
        for c in cases:
            c["q"] = c["q"].contiguous()  # (a copy of the call's own would be the caller's to keep)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [call(c) for c in cases]  # a second append of the same rows leaves the cache as it is
        want = [call(c) for c in cases]
        after = [clones(c["cache"]) for c in cases]
        graphs, outs = [], []
        for c in cases:
            with Graph(side) as g:
                outs.append(call(c))
            graphs.append(g)
        torch.cuda.synchronize()
        others = [torch.full((n,), 0x5A, dtype=torch.uint8, device=cuda)
                  for n in (512, 4096, 65536, 262144, 1 << 20, 2 << 20, 5 << 20, 8 << 20, 13 << 20) for _ in range(24)]
        for _ in range(3):
            for g, o in zip(graphs, outs):
                o.fill_(float("nan"))
                g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, w) for o, w in zip(outs, want))
            assert all(same(c["cache"], a) for c, a in zip(cases, after))
            assert all(torch.all(t == 0x5A) for t in others)
        torch.cuda.synchronize()
        for g in graphs:
            g.destroy()
    assert status() == 0


def test_what_a_graph_kept_is_freed_behind_it(cuda):
    """Captured and destroyed many times over, with torch's graphs and without: the memory comes back."""
    c = case(cuda, 4, 5000, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(c)
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        for i in range(6):
            if i % 2:
                with Graph(side) as g:
                    out = step(c)
                g.replay()
                torch.cuda.synchronize()
                g.destroy()
            else:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=side):
                    out = step(c)
                g.replay()
                torch.cuda.synchronize()
            del g, out
            gc.collect()
        for _ in range(100):  # the last graph's reference is given back by another thread
            step(c)
            torch.cuda.synchronize()
            if torch.cuda.memory_allocated() == base:
                break
            time.sleep(0.05)
        assert torch.cuda.memory_allocated() == base
    assert status() == 0


def test_steps_of_growing_batches_hold_little_memory(cuda):
    """Eager steps of one sequence more from call to call: the workspaces that the stream outgrows (kept for
    graphs) double at least, so all of them take less than four times the largest that is needed."""
    f, _ = F.rope_inv_freq(128, device=cuda)
    most = 200
    cache = F.kv8_cache(most, 2, 16, 128, device=cuda)
    table = torch.arange(most, dtype=torch.int32, device=cuda).view(most, 1)
    lens = torch.full((most,), 7, dtype=torch.int32, device=cuda)
    x = torch.randn(most, 36, 128, device=cuda, generator=gen(cuda, 1)).to(BF16)
    run = lambda b: F.decode_attention_kv8(x[:b, :32], x[:b, 32:34], x[:b, 34:], cache, table[:b], lens[:b], 16, f)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        base = torch.cuda.memory_allocated()
        for b in range(1, most + 1):
            run(b)
        need = _lib.lib().focal_kv8_decode_workspace_size(most, 1, 32, 2, 16, 128)
        assert torch.cuda.memory_allocated() - base < 4 * need
        torch.cuda.synchronize()
    assert status() == 0


def test_a_failure_is_not_cleared_inside_a_capture(cuda):
    """A call that is being captured reports an earlier failure and leaves it to a call outside to clear:
    the stream's workspace cannot be zeroed in between."""
    cache = random_cache(4, 2, 16, 128, E4M3, cuda, seed=1)
    k = torch.ones(1, 2, 128, device=cuda, dtype=BF16)
    q = torch.ones(1, 8, 128, device=cuda, dtype=BF16)
    one, good, bad = ints([1], cuda), ints([[2]], cuda), ints([[4]], cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = F.gqa_decode_attention_kv8(q, cache, good, one, 16)
        F.kv8_append(k, k, cache, bad, one)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="bad paged-KV index.*outside the capture"):
        with torch.cuda.graph(g, stream=side):
            k.mul_(1.0)  # (a graph with a node)
            F.kv8_append(k, k, cache, good, one)
    assert status() == 3
    with torch.cuda.stream(side):
        with pytest.raises(RuntimeError, match="bad paged-KV index.*later calls are valid"):
            F.gqa_decode_attention_kv8(q, cache, good, one, 16)
        assert torch.equal(F.gqa_decode_attention_kv8(q, cache, good, one, 16), want)
    assert status() == 0
