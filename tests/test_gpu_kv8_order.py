"""Paged 8-bit cache on the GPU: results that hang on the order of memory
accesses, inside the kernels and between streams."""
import math

import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_kv8 import U, Launches, Server, bounds

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim,queries", [(64, 8), (128, 4), (256, 3)])
@pytest.mark.parametrize("new", [[1, 1], [150, 40]])
def test_attention_repeats_itself(kq, dtype, dim, queries, new):
    """Rings, operand slots, TMEM and output rows that a warp takes over after
    one of its lanes has waited: the same bits in forty calls, by either kernel."""
    s = Server(kq, 2, dim, 16, "int8", 2, 700, pages=300, seed=dim, dtype=dtype)
    s.step([2900, 700])
    step = s.step(new)
    q = s.rng.standard_normal((sum(new), 2 * queries, dim)).astype(np.float32)
    with Launches(kq, "kv8_prompt") as seen:
        first = s.attend(step, new, 2 * queries, q=q.copy())
        for _ in range(39):
            again = s.attend(step, new, 2 * queries, q=q.copy(), check=False)
            assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
    assert seen.count == (40 if new[0] > 1 else 0)


def _fresh(kq, pages, seed):
    """A cache whose arrays are still being filled, and a step over its last pages."""
    cache = kq.Kv8Cache(2, 128, 64, pages)
    rng = np.random.default_rng(seed)
    ids = rng.permutation(np.arange(pages - 8, pages)).astype(np.int32)
    rows = rng.standard_normal((2, 300, 2, 128)).astype(np.float32)
    return cache, ids, rows


def _check(cache, ids, rows, values):
    want = ref.Cache(2, 128, 64, 5, "int8")
    for p in range(5):
        want.append_run(p, 0, rows[:, 64 * p:64 * p + 64].transpose(1, 2, 0, 3))
    assert np.array_equal(values.cpu().numpy(), want.values(np.arange(5)))


@pytest.mark.parametrize("side", [False, True])
def test_calls_follow_torch(kq, side):
    """A cache of 2 GB that is used while torch still fills it, arguments that
    torch has not written yet, and temporaries whose memory torch hands out
    again at once: on torch's default stream and on a side stream, with no
    synchronize before the results are read."""
    import torch
    stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
    with torch.cuda.stream(stream):
        for turn in range(4):
            cache, ids, rows = _fresh(kq, 1 << 16, turn)
            host = torch.from_numpy(rows).pin_memory()
            step = kq.Kv8Step(1, 300, torch.zeros(1, 5, dtype=torch.int32, device="cuda"), 64)
            ints = [torch.tensor(a, dtype=torch.int32).pin_memory().cuda(non_blocking=True)
                    for a in ([0], [300], ids.tolist(), [0], [0])]
            torch.cuda._sleep(3_000_000)   # what follows on this stream is late
            k, v = host.cuda(non_blocking=True)
            cache.plan(step, *ints)
            cache.append(step, k, v)
            del k, v, ints
            torch.full((2, 300, 2, 128), 9.0, device="cuda")
            values = torch.zeros(5, 2, 2, 64, 128, device="cuda")
            cache.read_pages(step.block_table[0].clone(), values)
            torch.full((5,), -1, dtype=torch.int32, device="cuda")
            _check(cache, ids, rows, values)
            kq.synchronize()
            del cache, step


def test_calls_on_the_default_stream(kq):
    """torch's default stream as the library stream, and back."""
    import torch
    own = kq.lib().kq_b200_get_stream()
    kq.set_stream(torch.cuda.current_stream())
    try:
        s = Server(kq, 2, 64, 16, "int8", 3, 300, seed=5)
        for new in ([120, 7, 31], [1, 1, 1]):
            step = s.step(new)
            s.attend(step, new, 4)
        s.check_pages()
    finally:
        kq.set_stream(None)
    assert kq.lib().kq_b200_get_stream() == own


def test_capture_of_torch_and_cache_together(kq):
    """A torch graph whose stream is not the library's: the calls join it."""
    import torch
    s = Server(kq, 2, 64, 16, "int8", 1, 200, seed=6)
    s.step([900])
    q, out = torch.zeros(1, 4, 64, device="cuda"), torch.zeros(1, 4, 64, device="cuda")
    step = s.step([1])
    ws = torch.empty(s.cache.attend_workspace_bytes(step, 4), dtype=torch.uint8, device="cuda")
    s.cache.attend(step, q, out, scale=0.125, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        double = q * 2
        s.cache.attend(step, double, out, scale=0.125, workspace=ws)
        again = out + 1
    for _ in range(3):
        x = s.rng.standard_normal((1, 4, 64)).astype(np.float32)
        q.copy_(torch.as_tensor(x))
        graph.replay()
        got = again.cpu().numpy()
        kq.synchronize()
        o, l, size, top = ref.attend(s.ref, s.table, [900], [1], 2 * x, 0.125)
        bo, _ = bounds("float32", 64, 901, size, top, o, l)
        assert np.all(np.abs(got - 1 - o) <= bo + (1 + np.abs(o)) * 2 * U)
    del graph


def test_attention_after_an_error_leaves_no_cuts(kq):
    """What a kernel that ends at once leaves in the workspace for the join:
    cuts that say nothing was cut, not what the memory held (ones here)."""
    import torch
    s = Server(kq, 1, 64, 16, "int8", 2, 500)
    s.step([50, 20])
    step = s.step([1, 1])
    q = torch.zeros(2, 4, 64, device="cuda")
    out = torch.zeros_like(q)
    nbytes = s.cache.attend_workspace_bytes(step, 4)
    ws = torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda")
    # floats of a share: two partials of 8 rows of (64 + 2), then a cut of four words, the last of them `last`
    shares = nbytes // 4 // (2 * 8 * 66 + 4)
    assert shares > 100
    s.cache.append(step, torch.full((2, 1, 64), math.inf, device="cuda"), torch.zeros(2, 1, 64, device="cuda"))
    s.cache.attend(step, q, out, scale=0.125, workspace=ws)
    with pytest.raises(kq.KQError) as e:
        kq.synchronize()
    assert e.value.status == kq.abi.NUMERIC_DOMAIN
    first = 2 * shares * 8 * 66
    last = ws.view(torch.int32)[first:first + 4 * shares].view(shares, 4)[:, 3]
    assert torch.all(last == 0)
