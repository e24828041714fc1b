"""Paged 8-bit cache without a GPU: what its entry points refuse before any
device work, their sizes, and the restatement that the GPU tests use."""
import ctypes as C
import math

import numpy as np
import pytest

import kv8_reference as ref

A = 0x7F0000000000   # addresses that are never read: every call here is refused on the host


def _cache(kq, **over):
    f = dict(kv_head_count=2, head_dimension=128, page_tokens=32, page_count=10, format=0, codes=A,
             codes_bytes=2 * 10 * 2 * 32 * 128, scales=A + (1 << 30), scales_count=40)
    f.update(over)
    return kq.abi.Kv8CacheArgs(**f)


def _step(kq, **over):
    f = dict(request_count=3, token_capacity=50, table_columns=4, run_capacity=7, table_stride=4)
    f.update({n: A + (i + 2 << 30) for i, n in enumerate(
        ["block_table", "query_offsets", "kv_lengths", "slots", "positions", "run_offsets", "page_runs"])})
    f.update(over)
    return kq.abi.Kv8StepArgs(**f)


CTX, NEW, FREE, HEAD, HEAD_OUT, K, V, Q, OUT, LSE, WS = (A + (20 + i << 30) for i in range(11))


def _call(kq, name, *args):
    d = kq.abi.Diagnostic()
    st = getattr(kq.lib(), name)(*args, C.byref(d))
    assert (st == 0) or d.text()
    return st


def plan(kq, cache=None, step=None, ctx=CTX, new=NEW, free=FREE, count=20, head=HEAD, head_out=HEAD_OUT):
    return _call(kq, "kq_b200_kv8_plan", cache or _cache(kq), step or _step(kq), ctx, new, free, count, head, head_out)


def append(kq, cache=None, step=None, dtype=0, key=K, ks=256, value=V, vs=256):
    return _call(kq, "kq_b200_kv8_append", cache or _cache(kq), step or _step(kq), dtype, key, ks, value, vs)


def attend(kq, cache=None, step=None, dtype=0, q=Q, qs=1024, heads=8, scale=0.1, most=0, out=OUT, os=1024, lse=LSE,
           ws=WS, nbytes=1 << 40):
    return _call(kq, "kq_b200_kv8_attend", cache or _cache(kq), step or _step(kq), dtype, q, qs, heads, scale, most, out,
                 os, lse, ws, nbytes)


def read(kq, cache=None, pages=CTX, count=3, values=OUT, capacity=1 << 30):
    return _call(kq, "kq_b200_kv8_read", cache or _cache(kq), pages, count, values, capacity)


def test_well_formed_calls_get_as_far_as_the_device(kq):
    """The base of the refusals below: nothing on the host is wrong with these
    (no GPU: UNSUPPORTED_MODEL; a GPU that does not own the addresses:
    INVALID_ARGUMENT)."""
    got = {plan(kq), append(kq), attend(kq), read(kq)}
    assert got <= {kq.abi.UNSUPPORTED_MODEL, kq.abi.INVALID_ARGUMENT}


@pytest.mark.parametrize("over", [dict(head_dimension=96), dict(head_dimension=0), dict(page_tokens=8),
                                  dict(page_tokens=48), dict(page_tokens=256), dict(kv_head_count=0),
                                  dict(kv_head_count=1025), dict(page_count=0), dict(page_count=1 << 31),
                                  dict(format=2), dict(format=-1)])
def test_refused_geometry(kq, over):
    c = _cache(kq, **over)
    assert {plan(kq, c), append(kq, c), attend(kq, c), read(kq, c)} == {kq.abi.DIMENSION_MISMATCH}
    assert kq.lib().kq_b200_kv8_codes_bytes(c) == 0 and kq.lib().kq_b200_kv8_scales_count(c) == 0


@pytest.mark.parametrize("over,want", [(dict(codes=None), "INVALID_ARGUMENT"), (dict(scales=None), "INVALID_ARGUMENT"),
                                       (dict(codes_bytes=163839), "BUFFER_TOO_SMALL"),
                                       (dict(scales_count=39), "BUFFER_TOO_SMALL"),
                                       (dict(codes=A + 8), "INVALID_ALIGNMENT"),
                                       (dict(scales=A + (1 << 30) + 4), "INVALID_ALIGNMENT")])
def test_refused_cache_arrays(kq, over, want):
    c = _cache(kq, **over)
    assert {append(kq, c), attend(kq, c), read(kq, c)} == {getattr(kq.abi, want)}


@pytest.mark.parametrize("over,want", [(dict(request_count=0), "INVALID_ARGUMENT"),
                                       (dict(token_capacity=0), "INVALID_ARGUMENT"),
                                       (dict(table_columns=0), "INVALID_ARGUMENT"),
                                       (dict(request_count=16385), "LIMIT_EXCEEDED"),
                                       (dict(token_capacity=1 << 31), "LIMIT_EXCEEDED"),
                                       (dict(table_stride=3), "DIMENSION_MISMATCH"),
                                       (dict(table_stride=1 << 62), "ARITHMETIC_OVERFLOW")])
def test_refused_steps(kq, over, want):
    s = _step(kq, **over)
    assert {plan(kq, step=s), append(kq, step=s), attend(kq, step=s)} == {getattr(kq.abi, want)}


def test_refused_plans(kq):
    a = kq.abi
    for name in ("block_table", "query_offsets", "kv_lengths", "slots", "positions", "run_offsets", "page_runs"):
        assert plan(kq, step=_step(kq, **{name: None})) == a.INVALID_ARGUMENT, name
    assert plan(kq, step=_step(kq, run_capacity=0)) == a.INVALID_ARGUMENT
    for name in ("ctx", "new", "free", "head", "head_out"):
        assert plan(kq, **{name: None}) == a.INVALID_ARGUMENT, name
    assert plan(kq, count=1 << 31) == a.LIMIT_EXCEEDED
    assert plan(kq, step=_step(kq, slots=A + (5 << 30) + 4)) == a.INVALID_ALIGNMENT
    assert plan(kq, head_out=HEAD) == a.ALIASING_VIOLATION
    assert plan(kq, step=_step(kq, kv_lengths=CTX)) == a.ALIASING_VIOLATION
    assert plan(kq, step=_step(kq, query_offsets=A + (6 << 30) + 4 * 49)) == a.ALIASING_VIOLATION   # the last position


def test_refused_appends(kq):
    a = kq.abi
    assert append(kq, dtype=2) == a.UNSUPPORTED_TENSOR_TYPE
    assert append(kq, key=None) == a.INVALID_ARGUMENT and append(kq, value=None) == a.INVALID_ARGUMENT
    assert append(kq, step=_step(kq, slots=None)) == a.INVALID_ARGUMENT
    assert append(kq, step=_step(kq, page_runs=None)) == a.INVALID_ARGUMENT
    assert append(kq, ks=255) == a.DIMENSION_MISMATCH and append(kq, vs=0) == a.DIMENSION_MISMATCH
    assert append(kq, ks=257) == a.INVALID_ALIGNMENT and append(kq, key=K + 8) == a.INVALID_ALIGNMENT
    assert append(kq, dtype=1, vs=260) == a.INVALID_ALIGNMENT   # 520 bytes
    assert append(kq, ks=1 << 62) == a.ARITHMETIC_OVERFLOW
    assert append(kq, key=A) == a.ALIASING_VIOLATION


def test_refused_reads(kq):
    a = kq.abi
    assert read(kq, pages=None) == a.INVALID_ARGUMENT and read(kq, values=None) == a.INVALID_ARGUMENT
    assert read(kq, count=0) == a.INVALID_ARGUMENT
    assert read(kq, capacity=3 * 2 * 2 * 32 * 128 - 1) == a.BUFFER_TOO_SMALL
    assert read(kq, values=OUT + 8) == a.INVALID_ALIGNMENT
    assert read(kq, values=A + 16) == a.ALIASING_VIOLATION


def test_refused_attention(kq):
    a = kq.abi
    assert attend(kq, dtype=7) == a.UNSUPPORTED_TENSOR_TYPE
    for heads in (0, 7, 3):
        assert attend(kq, heads=heads) == a.DIMENSION_MISMATCH
    for scale in (math.nan, math.inf, -math.inf, 3e38):   # the last: not finite in base 2
        assert attend(kq, scale=scale) == a.INVALID_ARGUMENT
    for name in ("q", "out"):
        assert attend(kq, **{name: None}) == a.INVALID_ARGUMENT
    for name in ("block_table", "query_offsets", "kv_lengths"):
        assert attend(kq, step=_step(kq, **{name: None})) == a.INVALID_ARGUMENT, name
    assert attend(kq, qs=1023) == a.DIMENSION_MISMATCH and attend(kq, os=1020) == a.DIMENSION_MISMATCH
    assert attend(kq, qs=1026) == a.INVALID_ALIGNMENT and attend(kq, out=OUT + 4) == a.INVALID_ALIGNMENT
    assert attend(kq, out=Q + 1024) == a.ALIASING_VIOLATION
    assert attend(kq, lse=OUT) == a.ALIASING_VIOLATION
    # a step whose 2^28 rows of 16 heads pass 2^31 - 1 rows per key/value head
    assert attend(kq, step=_step(kq, token_capacity=1 << 28), heads=16) == a.LIMIT_EXCEEDED


def test_attention_workspace(kq):
    """A split tile needs room for its partials, and a call with less is refused."""
    s = _step(kq, token_capacity=3, table_columns=4096, table_stride=4096)
    n = C.c_uint64(1)
    assert _call(kq, "kq_b200_kv8_attend_workspace_bytes", _cache(kq), s, 8, 0, C.byref(n)) == 0
    assert n.value > 0 and n.value % 16 == 0
    assert attend(kq, step=s, nbytes=n.value - 1) == kq.abi.BUFFER_TOO_SMALL
    assert attend(kq, step=s, ws=None) == kq.abi.BUFFER_TOO_SMALL
    assert attend(kq, step=s, ws=WS + 4) == kq.abi.INVALID_ALIGNMENT
    assert attend(kq, step=s, ws=OUT, nbytes=n.value) == kq.abi.ALIASING_VIOLATION
    m = C.c_uint64(1)   # contexts that a split does not pay for
    assert _call(kq, "kq_b200_kv8_attend_workspace_bytes", _cache(kq), s, 8, 16, C.byref(m)) == 0
    assert m.value == 0
    assert _call(kq, "kq_b200_kv8_attend_workspace_bytes", _cache(kq), s, 8, 16, None) == kq.abi.INVALID_ARGUMENT


def test_sizes(kq):
    assert kq.lib().kq_b200_kv8_codes_bytes(_cache(kq)) == 163840
    assert kq.lib().kq_b200_kv8_scales_count(_cache(kq)) == 40
    run = kq.lib().kq_b200_kv8_run_capacity
    rng = np.random.default_rng(0)
    for _ in range(300):
        page, B = int(rng.choice([16, 32, 64, 128])), int(rng.integers(1, 9))
        ctx, new = rng.integers(0, 300, B), rng.integers(0, 300, B)
        runs = sum(-(-(c + n) // page) - c // page for c, n in zip(ctx, new) if n)
        assert runs <= run(int(new.sum()), B, page)
    assert run(5, 3, 0) == 0


def test_reference_rounds_like_the_format():
    """Every e4m3 value and every midpoint between neighbours (ties to even),
    and int8 halves."""
    v = ref.E4M3[:0x7F].astype(np.float64)
    assert np.array_equal(ref.encode(v, "e4m3"), v.astype(np.float32))
    mid = ((v[:-1] + v[1:]) / 2).astype(np.float32)
    even = np.where(np.arange(len(mid)) % 2 == 0, v[:-1], v[1:])
    assert np.array_equal(ref.encode(mid, "e4m3"), even.astype(np.float32))
    assert np.array_equal(ref.encode(-mid, "e4m3"), -even.astype(np.float32))
    assert np.array_equal(ref.encode(np.float32([0.5, 1.5, -2.5, 126.6, 200]), "int8"), np.float32([0, 2, -2, 127, 127]))


@pytest.mark.parametrize("columns", [1 << 28, 1 << 29, 3 << 29, (1 << 32) - 1])
@pytest.mark.parametrize("tokens", [1, 100, 800, 1600, 2400, 6000])
def test_attention_workspace_of_the_widest_tables(kq, columns, tokens):
    """A request has 2^31 - 1 tokens at most, whatever its row of the table
    could hold: tables past that are cut like one that holds as many."""
    def size(columns):
        n = C.c_uint64(1)
        s = _step(kq, token_capacity=tokens, table_columns=columns, table_stride=columns)
        assert _call(kq, "kq_b200_kv8_attend_workspace_bytes", _cache(kq, page_tokens=128), s, 8, 0, C.byref(n)) == 0
        return n.value
    assert size(columns) == size((1 << 31) // 128)


def test_attention_of_the_largest_counts(kq):
    """1024 heads, 2^31 rows a head and the longest contexts: the launch rule's
    products pass 2^64, and the step is too large, not small."""
    n = C.c_uint64(1)
    c = _cache(kq, kv_head_count=1024, page_tokens=128)
    s = _step(kq, request_count=1, token_capacity=(1 << 31) - 1, table_columns=1 << 25, table_stride=1 << 25)
    assert _call(kq, "kq_b200_kv8_attend_workspace_bytes", c, s, 1024, 0, C.byref(n)) == kq.abi.LIMIT_EXCEEDED


def test_refused_alignment_of_small_arrays(kq):
    """Arrays of 4-byte values at odd addresses: a kernel that read them would fault."""
    a = kq.abi
    arrays = {n: A + (i + 2 << 30) + 2 for i, n in enumerate(
        ["block_table", "query_offsets", "kv_lengths", "slots", "positions", "run_offsets", "page_runs"])}
    for n, p in arrays.items():
        assert plan(kq, step=_step(kq, **{n: p})) == a.INVALID_ALIGNMENT, n
    for n, p in dict(ctx=CTX, new=NEW, free=FREE, head=HEAD, head_out=HEAD_OUT).items():
        assert plan(kq, **{n: p + 2}) == a.INVALID_ALIGNMENT, n
    for n in ("slots", "page_runs"):
        assert append(kq, step=_step(kq, **{n: arrays[n]})) == a.INVALID_ALIGNMENT, n
    for n in ("block_table", "query_offsets", "kv_lengths"):
        assert attend(kq, step=_step(kq, **{n: arrays[n]})) == a.INVALID_ALIGNMENT, n
    assert attend(kq, lse=LSE + 2) == a.INVALID_ALIGNMENT
    assert read(kq, pages=CTX + 1) == a.INVALID_ALIGNMENT
