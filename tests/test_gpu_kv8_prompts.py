"""Paged 8-bit cache on the GPU: the prompt kernel at the sizes and masks where
it can go wrong.  Wide tables (contexts that could be long) send small steps to
it; every test asserts that it ran.  Bounds: test_gpu_kv8.py."""
import math

import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_kv8 import Launches, Server, bounds, dev

pytestmark = pytest.mark.gpu

DTYPES = pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
DIMS = pytest.mark.parametrize("dim", [64, 128, 256])
WIDE = 2000   # table columns of 16 tokens


def prompt(kq, s, *args, **more):
    with Launches(kq, "kv8_prompt") as seen:
        got = s.attend(*args, **more)
    assert seen.count == 1
    return got


@DTYPES
@DIMS
def test_rows_that_see_nothing(kq, dtype, dim):
    """Lengths below the new tokens leave a prompt's first rows without keys
    (whole tiles, a tile's first rows); a length of zero leaves all of them."""
    s = Server(kq, 1, dim, 16, "int8", 4, WIDE, pages=60, dtype=dtype)
    s.step([30, 20, 300, 40])
    new, lengths = [40, 70, 330, 1], [2, 0, 15, 0]
    step = kq.Kv8Step(4, sum(new) + 7, s.table_dev, 16)
    step.use(query_offsets=dev(np.int32(np.cumsum([0] + new))), kv_lengths=dev(np.int32(lengths)))
    s.context = lengths
    got, lse = prompt(kq, s, step, new, 4)
    blind = np.r_[0:38, 40:110, 110:425, 440:441]
    assert np.all(got[blind] == 0) and np.all(np.isneginf(lse[blind]))
    assert np.all(np.isfinite(lse[38:40])) and np.all(np.isfinite(lse[425:440]))


@DTYPES
@DIMS
@pytest.mark.parametrize("scale", [0.0, 40.0, -3.0])
def test_scales(kq, dtype, dim, scale):
    """Equal weights, a softmax with a single winner, a negative scale (whose
    sign goes into the queries)."""
    s = Server(kq, 2, dim, 16, "e4m3", 2, WIDE, pages=60, dtype=dtype)
    s.step([200, 63])
    new = [1, 140]
    step = s.step(new)
    prompt(kq, s, step, new, 4, scale=scale)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@DIMS
def test_pages_of_different_size(kq, fmt, dim):
    """Page scales and query rows over many orders of magnitude, zero pages
    and zero and tiny queries among them."""
    s = Server(kq, 1, dim, 16, fmt, 1, WIDE, pages=60)
    n = 600
    size = 10.0 ** s.rng.uniform(-18, 8, (n // 16 + 1, 1, 1)).repeat(16, 0)[:n]
    size[64:80] = size[320:352] = 0
    v = (s.rng.standard_normal((n, 1, dim)) * size).astype(np.float32)
    k = (s.rng.standard_normal((n, 1, dim)) * np.where(size > 0, 10.0 ** s.rng.uniform(-3, 0.5, size.shape), 0))
    s.step([n], k=k.astype(np.float32), v=v)
    step = s.step([150])
    q = s.rng.standard_normal((150, 3, dim)).astype(np.float32)
    q[:, 0] *= np.float32(1e-30)
    q[::7, 1] = 0
    q[:, 2, 1::2] *= np.float32(1e-6)
    prompt(kq, s, step, [150], 3, q=q)


@DTYPES
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_zero_pages_alone(kq, fmt, dtype):
    """Keys and values that are all zero: equal weights, output zero."""
    s = Server(kq, 1, 64, 16, fmt, 1, WIDE, pages=60, dtype=dtype)
    zero = np.zeros((200, 1, 64), np.float32)
    step = s.step([200], k=zero, v=zero)
    got, lse = prompt(kq, s, step, [200], 4)
    assert not got.any()
    assert np.all(np.abs(lse - np.log(np.arange(1, 201))[:, None]) < 1e-5)


@DTYPES
@DIMS
@pytest.mark.parametrize("hint", [1100, 4000, 100000])
def test_lengths_past_the_hint(kq, dtype, dim, hint):
    """Contexts longer than the length that the caller said to expect: the
    launch's splits take more each."""
    s = Server(kq, 2, dim, 16, "int8", 2, 500, pages=500, dtype=dtype, seed=hint)
    s.step([6000, 900])
    new = [90, 60]
    step = s.step(new)
    first = prompt(kq, s, step, new, 16, hint=hint, q=s.rng.standard_normal((150, 16, dim)).astype(np.float32))
    assert np.isfinite(first[0]).all()


@DTYPES
@DIMS
def test_splits_repeat_themselves(kq, dtype, dim):
    """The same cut gives the same bits: splits joined in order."""
    s = Server(kq, 1, dim, 32, "e4m3", 3, 1000, pages=300, dtype=dtype, seed=dim)
    s.step([5000, 40, 2500])
    new = [33, 90, 50]
    step = s.step(new, padding=11)
    q = s.rng.standard_normal((step.args.token_capacity, 8, dim)).astype(np.float32)
    a = prompt(kq, s, step, new, 8, q=q.copy())
    for _ in range(5):
        b = prompt(kq, s, step, new, 8, q=q.copy(), check=False)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@DTYPES
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("rows", [65, 127, 128, 129, 255, 256, 257, 385])
def test_tiles_that_end_anywhere(kq, dtype, page, rows):
    """One head to a group: prompts of a tile and a row more or less, over
    cached tokens that end inside a page and a step."""
    s = Server(kq, 1, 64, page, "int8", 3, WIDE * 16 // page, pages=3 * -(-900 // page), dtype=dtype, seed=rows)
    s.step([rows % 100, 0, 77])
    new = [rows, 1, rows + 1]
    step = s.step(new, padding=rows % 3)
    prompt(kq, s, step, new, 1)


def test_a_prompt_of_one_token(kq):
    """Decode tokens of more than 64 query heads to a key/value head are
    prompts too."""
    s = Server(kq, 1, 64, 16, "int8", 3, WIDE, pages=60)
    s.step([200, 63, 0])
    new = [1, 1, 1]
    step = s.step(new)
    prompt(kq, s, step, new, 100)


@DTYPES
def test_prompt_step_in_a_graph(kq, dtype):
    """A captured step of capacity for prompts, replayed with prompts, with
    decode tokens alone and with nothing."""
    import torch
    s = Server(kq, 1, 128, 32, "int8", 3, 1000, pages=200, dtype=dtype)
    s.step([2500, 9, 31])
    T = 150
    step = kq.Kv8Step(3, T, s.table_dev, 32)
    ctx, cnt, head, head_out = (dev(np.int32(a)) for a in (s.context, [1, 1, 1], [s.head], [0]))
    kind = getattr(torch, dtype)
    k, v = torch.zeros(2, T, 1, 128, device="cuda", dtype=kind)
    q, out = torch.zeros(T, 4, 128, device="cuda", dtype=kind), torch.zeros(T, 4, 128, device="cuda", dtype=kind)
    lse = torch.zeros(T, 4, device="cuda")
    ws = torch.empty(s.cache.attend_workspace_bytes(step, 4), dtype=torch.uint8, device="cuda")
    s.cache.plan(step, ctx, cnt, s.free_dev, head, head_out)   # once, outside a capture
    s.cache.attend(step, q, out, lse, scale=0.125, workspace=ws)
    torch.cuda.synchronize()
    kq.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.cache.plan(step, ctx, cnt, s.free_dev, head, head_out)
        s.cache.append(step, k, v)
        s.cache.attend(step, q, out, lse, scale=0.125, workspace=ws)
    for new in ([1, 1, 1], [100, 0, 50], [0, 0, 0], [1, 140, 2], [0, 1, 0]):
        n = sum(new)
        rows = s.rng.standard_normal((3, T, 4, 128)).astype(np.float32)
        for t, a in ((k, rows[0, :, :1]), (v, rows[1, :, :1]), (q, rows[2]), (ctx, np.int32(s.context)),
                     (cnt, np.int32(new)), (head, np.int32([s.head]))):
            t.copy_(torch.as_tensor(a))
        out.fill_(7)
        graph.replay()
        kq_rows = np.stack([k.float().cpu().numpy(), v.float().cpu().numpy()])
        torch.cuda.synchronize()
        kq.synchronize()
        want = ref.plan(32, s.context, new, s.table, s.free, s.head, T, step.page_runs.numel())
        ends = [t for t in want["page_runs"] if t >= 0] + [n]
        for a, z in zip(ends, ends[1:]):
            p = want["slots"][a]
            s.ref.append_run(p // 32, p % 32, kq_rows[:, a:z].transpose(1, 2, 0, 3))
        s.table, before = want["block_table"], s.context
        s.context, s.head = want["kv_lengths"], want["free_head"][0]
        o, l, size, top = ref.attend(s.ref, s.table, before, new, q[:n].float().cpu().numpy(), 0.125)
        bo, bl = bounds(dtype, 128, max(s.context), size, top, o, l)
        got = out.float().cpu().numpy()
        assert np.all(got[n:] == 7)
        assert np.all(np.abs(got[:n] - o) <= bo) and np.all(np.abs(lse[:n].cpu().numpy() - l) <= bl)
    del graph
