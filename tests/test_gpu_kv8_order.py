"""Paged 8-bit cache on the GPU: results that hang on the order of memory
accesses, inside the kernels and between streams."""
import numpy as np
import pytest

from test_gpu_kv8 import Launches, Server

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
