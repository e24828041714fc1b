"""Paged 8-bit cache on the GPU: what failed calls leave, and what they say."""
import copy
import math

import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_kv8 import Server, dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("at", [0, 5])
def test_pages_of_a_failed_append(kq, fmt, at):
    """One NaN: its head's keys of the page stay; every other head's keys, and
    values, are whole: all old or all new.  The same append with finite rows
    then gives what it would have given at once."""
    import torch
    heads, dim, page = 5, 64, 16
    s = Server(kq, heads, dim, page, fmt, 1, 1, pages=1)
    s.step([5])
    old = copy.deepcopy(s.ref)
    rows = (3 * s.rng.standard_normal((2, 4, heads, dim))).astype(np.float32)
    s.ref.append_run(0, at, rows.transpose(1, 2, 0, 3))
    step = kq.Kv8Step(1, 4, s.table_dev, page)
    step.use(slots=dev(np.arange(at, at + 4, dtype=np.int64)), page_runs=dev(np.int32([0] + [-1] * (step.page_runs.numel() - 1))))
    k, v = dev(rows[0]), dev(rows[1])
    bad = k.clone()
    bad[2, 3, 17] = math.nan
    s.cache.append(step, bad, v)
    with pytest.raises(kq.KQError) as e:
        kq.synchronize()
    assert e.value.status == kq.abi.NUMERIC_DOMAIN
    raw, scales = s.cache.codes.cpu().numpy().reshape(heads, -1), s.cache.scales.cpu().numpy().reshape(heads, 2)
    new = 0
    for h in range(heads):
        codes = ref.from_layout(raw[h], fmt, page, dim)
        for side in range(2):
            same = [np.array_equal(codes[side], r.code[0, h, side]) and scales[h, side] == r.scale[0, h, side]
                    for r in (old, s.ref)]
            assert any(same), (h, side)
            new += same[1]
            if (h, side) == (3, 0):
                assert same[0] and not same[1]
    assert new < 2 * heads
    s.cache.append(step, k, v)
    kq.synchronize()
    s.check_pages()


@pytest.mark.parametrize("what", ["length", "row"])
def test_error_text_of_cache_calls(kq, what):
    """No state is rolled back for a cache call, and the text does not say so."""
    import torch
    s = Server(kq, 1, 64, 16, "int8", 1, 2)
    step = kq.Kv8Step(1, 3, s.table_dev, 16)
    s.cache.plan(step, *(dev(np.int32(a)) for a in ([0], [-1 if what == "length" else 3], s.free, [0], [0])))
    s.cache.append(step, torch.full((3, 1, 64), math.inf, device="cuda"), torch.zeros(3, 1, 64, device="cuda"))
    with pytest.raises(kq.KQError) as e:
        kq.synchronize()
    assert e.value.status == (kq.abi.SPAN_OUT_OF_RANGE if what == "length" else kq.abi.NUMERIC_DOMAIN)
    assert "device reported" in str(e.value) and "rolled back" not in str(e.value)
