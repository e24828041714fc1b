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
