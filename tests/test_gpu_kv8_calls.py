"""Paged 8-bit cache on the GPU: calls that the interface allows at its edges:
many requests, many heads, pages that requests share, calls side by side."""
import math

import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_kv8 import Launches, Server, bounds, dev

pytestmark = pytest.mark.gpu


def test_attention_of_the_most_requests(kq):
    """16384 decode tokens over contexts of 1 to 4 tokens."""
    import torch
    n = 16384
    s = Server(kq, 1, 64, 16, "int8", n, 1, pages=n)
    step = s.step([1] * n)
    s.attend(step, [1] * n, 2)
    new = s.rng.integers(0, 4, n).tolist()
    step = s.step(new, padding=5)
    s.attend(step, new, 2)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_prompts_among_many_requests(kq, dtype):
    """Prompts first, last and between a thousand requests of no, one and two
    tokens, in a wide table: the search for a tile's request."""
    n = 1100
    s = Server(kq, 1, 64, 16, "int8", n, 600, pages=n + 200, dtype=dtype)
    new = s.rng.integers(0, 3, n)
    new[[0, 31, 32, 33, 500, 1024, n - 1]] = [200, 70, 0, 90, 129, 66, 150]
    new = new.tolist()
    step = s.step(new)
    with Launches(kq, "kv8_prompt") as seen:
        s.attend(step, new, 2)
    assert seen.count == 1


def test_the_most_heads(kq):
    """1024 key/value heads."""
    s = Server(kq, 1024, 64, 16, "e4m3", 2, 3, pages=5)
    for new in ([19, 3], [1, 1]):
        step = s.step(new)
        s.attend(step, new, 1024)
    s.check_pages()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new", [[1, 1, 1], [90, 1, 70]])
def test_pages_that_requests_share(kq, dtype, new):
    """A common beginning: full pages of one request in the tables of others."""
    s = Server(kq, 2, 64, 16, "int8", 3, 600, pages=90, dtype=dtype)
    s.step([320, 0, 0])
    for b in (1, 2):
        s.table[b, :20] = s.table[0, :20]
    s.table_dev.copy_(dev(s.table))
    s.context = [320, 320, 320]
    step = s.step(new)
    with Launches(kq, "kv8_prompt") as seen:
        s.attend(step, new, 4)
    assert seen.count == (new[0] > 1)
    s.check_pages()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new", [[1, 1], [100, 77]])
def test_attention_without_log_sums(kq, dtype, new):
    """lse is optional: the same output without it."""
    import torch
    s = Server(kq, 1, 128, 16, "int8", 2, 700, pages=200, dtype=dtype)
    s.step([1500, 40])
    step = s.step(new)
    T = sum(new)
    q = torch.randn(T, 4, 128, device="cuda").to(getattr(torch, dtype))
    a, b, lse = torch.empty_like(q), torch.empty_like(q), torch.empty(T, 4, device="cuda")
    ws = torch.empty(s.cache.attend_workspace_bytes(step, 4), dtype=torch.uint8, device="cuda")
    s.cache.attend(step, q, a, lse, scale=0.1, workspace=ws)
    s.cache.attend(step, q, b, scale=0.1, workspace=ws)
    assert torch.equal(a, b) and torch.isfinite(lse).all()
    kq.synchronize()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_graphs_at_the_same_time(kq, dtype):
    """Two graphs over one cache, a workspace and outputs each, replayed side
    by side: decode tokens in one, prompts in the other."""
    import torch
    s = Server(kq, 2, 128, 16, "int8", 2, 700, pages=400, dtype=dtype)
    s.step([3000, 900])
    graphs = []
    for new in ([60, 110], [1, 1]):
        step = kq.Kv8Step(2, sum(new), s.table_dev, 16)
        step.use(query_offsets=dev(np.int32(np.cumsum([0] + new))), kv_lengths=dev(np.int32(s.context)))
        q = torch.randn(sum(new), 8, 128, device="cuda").to(getattr(torch, dtype))
        out, lse = torch.empty_like(q), torch.empty(sum(new), 8, device="cuda")
        ws = torch.empty(s.cache.attend_workspace_bytes(step, 8), dtype=torch.uint8, device="cuda")
        s.cache.attend(step, q, out, lse, scale=0.1, workspace=ws)
        torch.cuda.synchronize()
        want = out.clone(), lse.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.cache.attend(step, q, out, lse, scale=0.1, workspace=ws)
        graphs.append((graph, out, lse, want, torch.cuda.Stream(), (step, q, ws)))
    for _ in range(20):
        for _, out, lse, *_ in graphs:
            out.zero_(), lse.zero_()
        torch.cuda.synchronize()
        for graph, *_, stream, _ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, lse, want, *_ in graphs:
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    kq.synchronize()
    del graphs


def test_append_and_attention_of_rows_far_apart(kq):
    """Token strides beyond 2^31 elements in all: 64-bit offsets of rows."""
    import torch
    stride = (1 << 31) // 16 + 64
    big = torch.empty(stride * 20 + 64, dtype=torch.bfloat16, device="cuda")
    far = big.as_strided((20, 1, 64), (stride, 64, 1))
    near = torch.randn(3, 20, 1, 64, device="cuda").bfloat16()
    outs = []
    for strided in (False, True):
        cache = kq.Kv8Cache(1, 64, 16, 2)
        step = kq.Kv8Step(1, 20, dev(np.int32([[1, 0]])), 16)
        ints = [dev(np.int32(a)) for a in ([0], [20], [1, 0], [0], [0])]
        cache.plan(step, *ints)
        for i in range(3):   # one strided operand at a time: the buffer is used again
            x = near[i]
            if strided:
                far.copy_(x)
                x = far
            if i == 0:
                cache.append(step, x, near[1])
            elif i == 1:
                cache.append(step, near[0], x)
            else:
                out = torch.empty(20, 1, 64, dtype=torch.bfloat16, device="cuda")
                cache.attend(step, x, out, scale=0.1)
        if strided:
            cache.attend(step, near[2], far, scale=0.1)
            assert torch.equal(far, out)
        outs.append((out, cache.codes.clone(), cache.scales.clone()))
    kq.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*outs))
