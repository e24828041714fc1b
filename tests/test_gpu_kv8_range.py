"""Paged 8-bit cache on the GPU: attention over values of every size that its
weights can hold, against 64 bits, with the bounds of test_gpu_kv8.py and
W = sum p |v| in place of the largest value (errors are relative to each
weight)."""
import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_kv8 import Launches, Server, bounds, dev

pytestmark = pytest.mark.gpu


def check(s, n, new, G, q, scale, got):
    if s.dtype == "bfloat16":
        q = dev(q, s.dtype).float().cpu().numpy()
    o, l, size, _ = ref.attend(s.ref, s.table, [n], [new], q, scale)
    s.ref.code[:, :, 1] = np.abs(s.ref.code[:, :, 1])
    w = ref.attend(s.ref, s.table, [n], [new], q, scale)[0].max(-1)
    bo, _ = bounds(s.dtype, s.dim, n + new, size, w, o, l)
    assert np.all(np.abs(got - o) <= bo), np.max(np.abs(got - o) / bo)
    return o


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 300])
@pytest.mark.parametrize("value", [(1e-25, 1e-25), (1e-28, 1e-28), (1e-30, 1e-30), (1e-32, 1e-32), (2e-33, 2e-33),
                                   (1e-32, 1e-20), (1e-30, 1e5)])
def test_attention_over_small_values(kq, dtype, dim, new, value):
    """Page scales down to 2^-114, alone and beside larger ones."""
    s = Server(kq, 1, dim, 16, "int8", 1, 210, pages=60, dtype=dtype, seed=dim)
    n, G = 500, 3
    size = np.exp(s.rng.uniform(*np.log(value), (50, 1, 1))).repeat(16, 0)
    v = (size * s.rng.standard_normal((800, 1, dim))).astype(np.float32)
    s.step([n], v=v[:n])
    step = s.step([new], v=v[n:n + new])
    assert np.all(s.ref.scale[s.table[0, :(n + new) // 16], :, 1] >= 2.0 ** -115)
    q = s.rng.standard_normal((new, G, dim)).astype(np.float32)
    with Launches(kq, "kv8_prompt") as seen:
        got, _ = s.attend(step, [new], G, q=q, check=False)
    assert seen.count == (new > 1)
    o = check(s, n, new, G, q, float(np.float32(dim ** -0.5)), got)
    assert np.all(o.any(-1))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 300])
def test_small_values_are_ordinary_ones_scaled(kq, dtype, dim, new):
    """Values 2^-100 times others give 2^-100 times their output, to the bit:
    every factor between them is a power of two while nothing is subnormal.
    The page scales are 2^-109, and the weights, up to 2^7.8 above a reference
    point that the first 128 tokens set, add up to 2^17."""
    n, G = 500, 3
    got = []
    for size in (0.25, 0.25 * 2.0 ** -100):
        s = Server(kq, 1, dim, 16, "int8", 1, 210, pages=60, dtype=dtype, seed=dim)
        k = np.zeros((800, 1, dim), np.float32)
        k[128:, 0, 0] = 5.4
        v = (np.float32(size) * s.rng.uniform(0.5, 1, (800, 1, dim)).astype(np.float32))
        s.step([n], k=k[:n], v=v[:n])
        step = s.step([new], k=k[n:n + new], v=v[n:n + new])
        q = np.zeros((new, G, dim), np.float32)
        q[:, :, 0] = 1
        with Launches(kq, "kv8_prompt") as seen:
            got.append(s.attend(step, [new], G, q=q, scale=1.0, check=False))
        assert seen.count == (new > 1)
    assert np.array_equal(got[0][0], got[1][0] * np.float32(2.0 ** 100)) and np.all(got[0][0] > 0.1)
    assert np.array_equal(got[0][1], got[1][1])
