"""Paged 8-bit cache on the GPU against the plain restatement
(kv8_reference.py).

Plan, codes, scales and read values are EXACT: whole numbers, and single
correctly rounded F32 operations.  Attention is held to bounds of its
arithmetic (u = 2^-24, half an F32 step; A = the row's largest
scale * sum |q_i k_i|, V = its largest |value|):

  logit    F32 query: each element kept to 2^-22, F32 additions of 2 * d / 16
           products, a truncating adder counted as a whole step (2 u) each,
           page and row factors 4 u:            dl = A * (4 + 4 d / 16 + 4) u
           bf16 query: exact parts, d / 16 additions:  no more than that
  weight   exp2 of a logit difference: dl for each of logit and reference
           point, the subtraction and the factor log2 e: 2 u * 2 A (as |l| <= A),
           exp2 itself 4 u, F32 parts 4 u:       dp = 2 dl + 4 A u + 8 u
           bf16: the weight is rounded to fp16:  + 2^-11
  sums     weights and products over n tokens: each F32 addition 2 u; a chain
           is at most n / 16 groups of 16 products and a join:  ds = (n / 8 + 64) u
  output   |error| <= 2 (dp + ds) V, then its own rounding: 2^-24 or 2^-8 relative
  lse      |error| <= dl + dp(F32) + ds + 4 u |lse|
"""
import ctypes as C
import math

import numpy as np
import pytest

import kv8_reference as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def dev(a, dtype=None):
    import torch
    t = torch.as_tensor(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(getattr(torch, dtype))).cuda()


def bounds(dtype, dim, n, size, top, out, lse):
    dl = size * (8 + dim / 4) * U
    dp = 2 * dl + 4 * size * U + 8 * U
    ds = (n / 8 + 64) * U
    w = 2.0 ** -11 if dtype == "bfloat16" else 0.0
    o = 2 * (dp + ds + w) * top
    o = o[..., None] + (np.abs(out) + o[..., None]) * (2.0 ** -8 if dtype == "bfloat16" else U)
    return o, dl + dp + ds + 4 * U * np.abs(np.where(np.isfinite(lse), lse, 0))


class Server:
    """A cache of the library and its restatement, fed the same steps."""

    def __init__(self, kq, heads, dim, page, fmt, requests, columns, pages=None, seed=0, dtype="float32"):
        import torch
        self.kq, self.rng = kq, np.random.default_rng(seed)
        self.heads, self.dim, self.page, self.fmt, self.dtype = heads, dim, page, fmt, dtype
        pages = pages or requests * columns + 3
        self.cache = kq.Kv8Cache(heads, dim, page, pages, fmt)
        self.ref = ref.Cache(heads, dim, page, pages, fmt)
        self.free = self.rng.permutation(pages).astype(np.int32)
        self.head, self.context = 0, [0] * requests
        self.table = np.full((requests, columns), -1, np.int32)
        self.table_dev, self.free_dev = dev(self.table), dev(self.free)
        torch.cuda.synchronize()

    def step(self, new, padding=0, gain=1.0, k=None, v=None):
        """Plans and appends rows for `new` tokens of each request; returns the step."""
        import torch
        tokens = max(1, sum(new) + padding)
        step = self.kq.Kv8Step(len(new), tokens, self.table_dev, self.page)
        runs = step.page_runs.numel()
        head, out = dev(np.int32([self.head])), dev(np.int32([-7]))
        ctx, cnt = dev(np.int32(self.context)), dev(np.int32(new))
        rows = self.rng.standard_normal((2, tokens, self.heads, self.dim)).astype(np.float32) * np.float32(gain)
        if k is not None:
            rows[0, :sum(new)] = k
        if v is not None:
            rows[1, :sum(new)] = v
        rows[:, sum(new):] = np.nan   # never read
        kd, vd = dev(rows[0], self.dtype), dev(rows[1], self.dtype)
        rows = np.stack([kd.float().cpu().numpy(), vd.float().cpu().numpy()])
        torch.cuda.synchronize()
        self.cache.plan(step, ctx, cnt, self.free_dev, head, out)
        self.cache.append(step, kd, vd)
        self.kq.synchronize()
        want = ref.plan(self.page, self.context, new, self.table, self.free, self.head, tokens, runs)
        self.table = want["block_table"]
        for name, w in want.items():
            got = out if name == "free_head" else self.table_dev if name == "block_table" else getattr(step, name)
            assert np.array_equal(got.cpu().numpy(), np.asarray(w)), name
        ends = [t for t in want["page_runs"] if t >= 0] + [sum(new)]
        for a, z in zip(ends, ends[1:]):
            s = want["slots"][a]
            self.ref.append_run(s // self.page, s % self.page, rows[:, a:z].transpose(1, 2, 0, 3))
        self.head = want["free_head"][0]
        self.context = want["kv_lengths"]
        return step

    def check_pages(self):
        """Codes, scales and read values of every page, exactly."""
        import torch
        pages = np.arange(self.ref.code.shape[0], dtype=np.int32)
        got = torch.full((len(pages), self.heads, 2, self.page, self.dim), math.nan, device="cuda")
        ids = dev(pages)
        torch.cuda.synchronize()
        self.cache.read_pages(ids, got)
        self.kq.synchronize()
        assert np.array_equal(self.cache.scales.cpu().numpy().reshape(self.ref.scale.shape), self.ref.scale)
        assert np.array_equal(got.cpu().numpy(), self.ref.values(pages))

    def attend(self, step, new, query_heads, scale=None, hint=0, dtype=None, q=None, check=True):
        import torch
        dtype = dtype or self.dtype
        tokens, T = step.args.token_capacity, sum(new)
        scale = 1 / math.sqrt(self.dim) if scale is None else scale
        host = self.rng.standard_normal((tokens, query_heads, self.dim)).astype(np.float32) if q is None else q
        host[T:] = np.nan
        # queries and outputs inside wider rows, of which nothing else may change
        qw = torch.full((tokens, query_heads + 2, self.dim), math.nan, dtype=getattr(torch, dtype), device="cuda")
        qd = qw[:, 1:-1]
        qd.copy_(torch.as_tensor(host))
        wide = torch.full_like(qw, 7.0)
        out = wide[:, 1:-1]
        lse = torch.full((tokens, query_heads), 7.0, device="cuda")
        ws = torch.empty(self.cache.attend_workspace_bytes(step, query_heads, hint), dtype=torch.uint8, device="cuda")
        ws.fill_(255)   # NaNs: partials must be written before they are read
        torch.cuda.synchronize()
        self.cache.attend(step, qd, out, lse, scale=scale, max_kv_length=hint, workspace=ws)
        self.kq.synchronize()
        assert torch.all(wide[T:] == 7) and torch.all(lse[T:] == 7)
        assert torch.all(wide[:, 0] == 7) and torch.all(wide[:, -1] == 7)
        got, got_lse = out[:T].float().cpu().numpy(), lse[:T].cpu().numpy()
        if check:
            before = [c - n for c, n in zip(self.context, new)]
            f32 = np.float32(scale)
            o, l, size, top = ref.attend(self.ref, self.table, before, new, qd[:T].float().cpu().numpy(), float(f32))
            bo, bl = bounds(dtype, self.dim, max([1] + self.context), size, top, o, l)
            assert np.all(np.abs(got - o) <= bo), np.max(np.abs(got - o) / np.maximum(bo, 1e-300))
            empty = np.isinf(l)
            assert np.array_equal(np.isneginf(got_lse), empty)
            assert np.all(np.abs(got_lse[~empty] - l[~empty]) <= bl[~empty])
        return got, got_lse


# ------------------------------------------------------------------- plan

@pytest.mark.parametrize("requests,page,most", [(1, 16, 1), (1, 64, 5000), (7, 16, 40), (64, 64, 1), (300, 32, 90),
                                                (1025, 128, 9), (2000, 16, 3), (16384, 32, 2)])
def test_plan(kq, requests, page, most):
    import torch
    rng = np.random.default_rng(requests)
    context = rng.integers(0, 700, requests).tolist()
    new = rng.integers(0, most + 1, requests).tolist()   # some requests bring nothing
    new[0] = most
    columns = -(-max(c + n for c, n in zip(context, new)) // page) + 2
    pages = requests * columns + 9
    free = rng.permutation(pages).astype(np.int32)
    table = rng.integers(0, pages, (requests, columns)).astype(np.int32)
    tokens = sum(new) + 13
    # a table with longer rows than the step uses
    wide = np.full((requests, columns + 3), -5, np.int32)
    wide[:, :columns] = table
    td = dev(wide)
    step = kq.Kv8Step(requests, tokens, td[:, :columns], page)
    cache = kq.Kv8Cache(1, 64, page, pages)
    args = [dev(np.int32(a)) for a in (context, new, free, [4], [0])]
    torch.cuda.synchronize()
    for _ in range(2):   # planning a step again gives it again
        cache.plan(step, *args)
        kq.synchronize()
        want = ref.plan(page, context, new, table, free, 4, tokens, step.page_runs.numel())
        for name, w in want.items():
            got = args[4] if name == "free_head" else td[:, :columns] if name == "block_table" else getattr(step, name)
            assert np.array_equal(got.cpu().numpy(), np.asarray(w)), name
    assert np.all(td[:, columns:].cpu().numpy() == -5)


@pytest.mark.parametrize("what", ["pages", "columns", "tokens", "runs", "negative", "head", "id", "table"])
def test_plan_that_cannot_be_met(kq, what):
    """Reported at the synchronize; nothing is written where the lengths
    themselves do not fit; the next step works."""
    import torch
    page, context, new = 16, [5, 0, 40], [20, 3, 30]
    free, head, columns, tokens = np.arange(40, dtype=np.int32), [0], 5, 60
    table = np.full((3, columns), 39, np.int32)
    if what == "pages":
        free = free[:3]   # four are needed: 1 + 1 + 2
    if what == "columns":
        context[2] = 51
    if what == "tokens":
        tokens = 52
    if what == "negative":
        new[1] = -3
    if what == "head":
        head = [-1]
    if what == "id":
        free[1] = 40
    if what == "table":
        table[0, 0] = 40
    td = dev(table)
    step = kq.Kv8Step(3, tokens, td, page)
    if what == "runs":
        step.args.run_capacity = 5   # six are needed: 2 + 1 + 3
    cache = kq.Kv8Cache(1, 64, page, 40)
    arrays = [getattr(step, n) for n in ("query_offsets", "kv_lengths", "slots", "positions", "run_offsets", "page_runs")]
    for a in arrays:
        a.fill_(-99)
    args = [dev(np.int32(a)) for a in (context, new, free, head, [-99])]
    torch.cuda.synchronize()
    cache.plan(step, *args)
    with pytest.raises(kq.KQError) as e:
        kq.synchronize()
    assert e.value.status == kq.abi.SPAN_OUT_OF_RANGE
    if what not in ("id", "table"):
        assert all(torch.all(a == -99) for a in arrays + [args[4]])
        assert np.array_equal(td.cpu().numpy(), table)
    s = Server(kq, 1, 64, 16, "int8", 2, 4)
    s.step([3, 9])
    s.check_pages()


# ----------------------------------------------------------------- append

@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,dim,page", [(1, 64, 16), (2, 128, 32), (3, 64, 128), (2, 256, 64)])
def test_append_and_read(kq, fmt, dtype, heads, dim, page):
    """Runs that begin and end anywhere in a page, scales that grow, pages met
    again and again by single tokens."""
    s = Server(kq, heads, dim, page, fmt, 4, 4, seed=page + dim, dtype=dtype)
    s.step([1, page, page + 1, 2 * page - 1])
    s.step([0, 3, page - 2, 1], padding=5, gain=3.0)      # louder: kept rows are rounded again
    s.step([7, 0, 1, 2], gain=0.01)                       # quieter: scales stay
    for gain in (1.0, 5.0, 0.3):
        s.step([1, 1, 1, 1], gain=gain)
    s.check_pages()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_of_special_rows(kq, fmt):
    """Zero pages (scale 0), subnormal scales that round down below the
    quotient's range, the largest values, a page that grows from zero."""
    s = Server(kq, 1, 64, 16, fmt, 4, 2)
    zero = np.zeros((12, 1, 64), np.float32)
    tiny = np.float32(2.0 ** -149) * s.rng.integers(-300, 300, (12, 1, 64)).astype(np.float32)
    k = zero.copy()
    k[3:6] = tiny[:3]
    k[6:9] = np.float32(2.9e38) * s.rng.uniform(-1, 1, (3, 1, 64)).astype(np.float32)
    s.step([3, 3, 3, 3], k=k, v=tiny)
    s.check_pages()
    s.step([1, 1, 1, 1])
    s.check_pages()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("size", [1.0, 0.3, 1 / 3, 1.1e-20, 7e8, 2e-36, 3e33])
def test_append_at_the_rounding_borders(kq, fmt, size):
    """Every border between two codes, and the F32 values up to three steps
    from it, times the page's scale: quotients that a product with a rounded
    reciprocal would put on the other side."""
    s = Server(kq, 1, 256, 16, fmt, 1, 1)
    most = ref.LARGEST[fmt]
    codes = np.arange(-127, 128) if fmt == "int8" else np.unique(ref.E4M3[np.isfinite(ref.E4M3)])
    border = ((codes[1:].astype(np.float64) + codes[:-1]) / 2)
    x = (border * size).astype(np.float32)
    near = [x]
    for to in (np.float32(-np.inf), np.float32(np.inf)):
        y = x
        for _ in range(3):
            near.append(y := np.nextafter(y, to))
    near = np.concatenate(near)
    rows = np.zeros((2, 16 * 256), np.float32)
    rows[:, 1:1 + near.size] = near
    rows[:, 0] = np.float32(most * size)     # the scale: this / most, about `size`
    rows[1] = -rows[1]
    s.step([16], k=rows[0].reshape(16, 1, 256), v=rows[1].reshape(16, 1, 256))
    s.check_pages()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_append_of_non_finite_rows(kq, value):
    """Reported, and the (page, head, side) keeps what it held."""
    import torch
    s = Server(kq, 2, 64, 16, "int8", 1, 2)
    s.step([5])
    codes, scales = s.cache.codes.clone(), s.cache.scales.clone()
    step = kq.Kv8Step(1, 3, s.table_dev, 16)
    rows = torch.ones(3, 2, 64, device="cuda")
    rows[1, 1, 63] = value
    args = [dev(np.int32(a)) for a in ([5], [3], [0], [0], [0])]
    torch.cuda.synchronize()
    s.cache.plan(step, *args)
    s.cache.append(step, rows, rows)
    with pytest.raises(kq.KQError) as e:
        kq.synchronize()
    assert e.value.status == kq.abi.NUMERIC_DOMAIN
    page = int(s.table[0, 0])
    a = s.cache.codes.view(-1, 2, 32 * 64)[page, 1]
    assert torch.equal(a, codes.view(-1, 2, 32 * 64)[page, 1])
    assert torch.equal(s.cache.scales.view(-1, 2, 2)[page, 1], scales.view(-1, 2, 2)[page, 1])


def test_append_of_strided_rows(kq):
    """Keys and values inside one fused projection row, and slots that a
    caller made itself: runs out of range are refused, -1 is padding."""
    import torch
    heads, dim, page = 2, 64, 16
    cache, want = kq.Kv8Cache(heads, dim, page, 5, "e4m3"), ref.Cache(heads, dim, page, 5, "e4m3")
    fused = torch.randn(20, 3 * heads, dim, device="cuda")
    step = kq.Kv8Step(1, 20, dev(np.int32([[0, 1]])), page)
    slots = np.r_[4 * 16 + 3 + np.arange(13), 2 * 16 + np.arange(6), [-1]].astype(np.int64)
    runs = np.full(step.page_runs.numel(), -1, np.int32)
    runs[0], runs[2] = 0, 13
    step.use(slots=dev(slots), page_runs=dev(runs))
    torch.cuda.synchronize()
    cache.append(step, fused[:, heads:2 * heads], fused[:, 2 * heads:])
    kq.synchronize()
    f = fused.cpu().numpy()
    rows = np.stack([f[:, heads:2 * heads], f[:, 2 * heads:]], 2)
    want.append_run(4, 3, rows[:13])
    want.append_run(2, 0, rows[13:19])
    raw = cache.codes.cpu().numpy().reshape(5, heads, -1)
    for p in range(5):
        for h in range(heads):
            assert np.array_equal(ref.from_layout(raw[p, h], "e4m3", page, dim), want.code[p, h])
    assert np.array_equal(cache.scales.cpu().numpy().reshape(5, heads, 2), want.scale)
    for bad_slot, bad_run in ((5 * 16, 0), (-2, 0), (0, 20)):
        slots[0], runs[0] = bad_slot, bad_run
        step.use(slots=dev(slots), page_runs=dev(runs))
        torch.cuda.synchronize()
        cache.append(step, fused[:, heads:2 * heads], fused[:, 2 * heads:])
        with pytest.raises(kq.KQError) as e:
            kq.synchronize()
        assert e.value.status == kq.abi.SPAN_OUT_OF_RANGE


def test_read_of_pages(kq):
    """Any order, repeats; an id that is not a page is refused."""
    import torch
    s = Server(kq, 2, 64, 32, "int8", 2, 3)
    s.step([70, 11])
    ids = np.int32([int(s.table[0, 2]), int(s.table[1, 0]), int(s.table[0, 2]), 0])
    out = torch.empty(4, 2, 2, 32, 64, device="cuda")
    torch.cuda.synchronize()
    s.cache.read_pages(dev(ids), out)
    kq.synchronize()
    assert np.array_equal(out.cpu().numpy(), s.ref.values(ids))
    for bad in (-1, s.cache.pages):
        s.cache.read_pages(dev(np.int32([0, bad])), out)
        with pytest.raises(kq.KQError) as e:
            kq.synchronize()
        assert e.value.status == kq.abi.SPAN_OUT_OF_RANGE


# -------------------------------------------------------------- attention

@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,queries,dim,page", [(2, 16, 256, 64), (2, 10, 64, 16), (1, 1, 128, 128), (3, 9, 128, 32),
                                                    (1, 24, 64, 32)])
def test_attention(kq, fmt, dtype, heads, queries, dim, page):
    """Prompts, decode tokens, chunks over cached tokens, requests without new
    tokens; one to some hundred tokens."""
    s = Server(kq, heads, dim, page, fmt, 5, -(-400 // page), seed=queries, dtype=dtype)
    for new, padding in (([1, 17, 0, 130, 33], 3), ([1, 1, 1, 1, 1], 0), ([70, 2, 1, 0, 15], 9), ([0, 1, 0, 0, 0], 4)):
        step = s.step(new, padding)
        s.attend(step, new, queries)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hint", [0, 1, 100000])
def test_attention_over_long_contexts(kq, dtype, hint):
    """Contexts cut into many splits beside short ones, whatever length the
    caller said to expect."""
    s = Server(kq, 1, 64, 32, "int8", 3, 200, seed=4, dtype=dtype)
    s.step([6000, 1, 900])
    for new in ([1, 1, 1], [2, 0, 3]):
        step = s.step(new)
        s.attend(step, new, 4, hint=hint)
    new = [40, 30, 0]   # 160 and 120 rows: the prompt kernel, split
    step = s.step(new)
    s.attend(step, new, 4, hint=hint)


class Launches:
    """Launches of a kernel family while it is watched."""

    def __init__(self, kq, family):
        self.kq, self.family = kq, family

    def __enter__(self):
        self.kq.lib().kq_b200_profile_kernel(self.family.encode())
        return self

    def __exit__(self, *_):
        n, ms = C.c_uint64(), C.c_double()
        self.kq.lib().kq_b200_profile_read(C.byref(n), C.byref(ms))
        self.kq.lib().kq_b200_profile_kernel(None)
        self.count = n.value


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,queries,dim,page", [(2, 16, 256, 64), (2, 6, 128, 16), (1, 24, 64, 32), (3, 3, 128, 128)])
def test_prompts(kq, fmt, dtype, heads, queries, dim, page):
    """Long prompts and chunks beside decode tokens in one step: tiles that
    end in mid-tile, both attention kernels, pages smaller and larger than a
    step of the prompt kernel."""
    s = Server(kq, heads, dim, page, fmt, 5, -(-4000 // page), pages=5 * -(-700 // page), seed=queries, dtype=dtype)
    for new, padding in (([300, 1, 0, 37, 165], 0), ([90, 1, 130, 2, 1], 21)):
        step = s.step(new, padding)
        with Launches(kq, "kv8_prompt") as seen:
            s.attend(step, new, queries)
        assert seen.count == 1


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim,queries", [(64, 3), (128, 8), (256, 5)])
def test_prompts_over_long_contexts(kq, dtype, dim, queries):
    """Key axes cut into splits, F32 sums moved out on the way, and the same
    over one split (many tiles)."""
    s = Server(kq, 1, dim, 64, "int8", 3, 110, seed=dim, dtype=dtype)
    s.step([5000, 1300, 0])
    for new in ([90, 70, 0], [1, 200, 150]):
        step = s.step(new)
        with Launches(kq, "kv8_prompt") as seen:
            s.attend(step, new, queries)
        assert seen.count == 1
    s = Server(kq, 8, dim, 64, "e4m3", 1, 110, seed=dim, dtype=dtype)
    s.step([1100])
    new = [700]
    step = s.step(new)
    with Launches(kq, "kv8_prompt") as seen:
        s.attend(step, new, 8 * 5)
    assert seen.count == 1


def test_prompts_of_bad_contents(kq):
    """What the prompt kernel refuses, and that it works after it."""
    import torch
    for what in ("query", "page", "length"):
        s = Server(kq, 1, 128, 16, "e4m3", 2, 200, pages=60)
        s.step([50, 20])
        new = [300, 1]
        step = s.step(new)
        q = torch.randn(301, 8, 128, device="cuda")
        out = torch.empty_like(q)
        ws = torch.empty(s.cache.attend_workspace_bytes(step, 8), dtype=torch.uint8, device="cuda")
        table, lengths = s.table_dev.clone(), step.kv_lengths.clone()
        if what == "query":
            q[299, 7, 127] = math.nan
        elif what == "page":
            s.table_dev[0, 17] = -1
        else:
            step.kv_lengths[0] = 200 * 16 + 1
        torch.cuda.synchronize()
        with Launches(kq, "kv8_prompt") as seen:
            s.cache.attend(step, q, out, scale=0.1, workspace=ws)
            with pytest.raises(kq.KQError) as e:
                kq.synchronize()
        assert seen.count == 1
        assert e.value.status == (kq.abi.NUMERIC_DOMAIN if what == "query" else kq.abi.SPAN_OUT_OF_RANGE)
        s.table_dev.copy_(table)
        step.kv_lengths.copy_(lengths)
        s.attend(step, new, 8)


def test_two_threads(kq):
    """Two threads with a cache each: calls are ordered by the library."""
    from concurrent.futures import ThreadPoolExecutor

    def serve(seed):
        s = Server(kq, 2, 64, 16, "int8", 2, 30, seed=seed)
        s.step([100, 37])
        for _ in range(4):
            step = s.step([1, 1])
            s.attend(step, [1, 1], 4)
        return True

    with ThreadPoolExecutor(2) as pool:
        assert all(pool.map(serve, [1, 2]))


@pytest.mark.parametrize("queries", [8, 64])
def test_attention_of_one_request_with_all_tokens(kq, queries):
    """As many tokens as requests, all of one request: more tiles than the
    launch expects of a decode step."""
    s = Server(kq, 2, 64, 16, "e4m3", 12, 12, seed=9)
    s.step([100] + [0] * 11)
    new = [0] * 5 + [12] + [0] * 6
    step = s.step(new)
    s.attend(step, new, queries)
    new = [12] + [0] * 11
    step = s.step(new)
    s.attend(step, new, queries)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_attention_rows_that_see_nothing(kq, dtype):
    """Lengths below the new tokens (a caller's own step) leave the first rows
    without keys: zeros and -inf; a length of zero leaves all of them."""
    import torch
    s = Server(kq, 1, 64, 16, "int8", 3, 8, dtype=dtype)
    s.step([30, 20, 100])
    new, lengths = [4, 3, 90], [2, 0, 80]
    step = kq.Kv8Step(3, 97, s.table_dev, 16)
    step.use(query_offsets=dev(np.int32(np.cumsum([0] + new))), kv_lengths=dev(np.int32(lengths)))
    s.context = lengths
    got, lse = s.attend(step, new, 2)
    assert np.all(got[:2] == 0) and np.all(got[4:7] == 0) and np.all(np.isneginf(lse[4:7]))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("scale", [0.0, 40.0, -3.0])
def test_attention_scales(kq, dtype, scale):
    """Equal weights, a softmax with a single winner, a negative scale."""
    s = Server(kq, 2, 64, 16, "int8", 2, 20, dtype=dtype)
    s.step([200, 63])
    new = [1, 40]
    step = s.step(new)
    s.attend(step, new, 4, scale=scale)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_attention_over_pages_of_different_size(kq, fmt):
    """Page scales and query rows over many orders of magnitude, zero pages
    and zero queries among them."""
    s = Server(kq, 1, 64, 16, fmt, 1, 42)
    n = 600
    size = 10.0 ** s.rng.uniform(-18, 8, (n // 16 + 1, 1, 1)).repeat(16, 0)[:n]
    size[64:80] = 0
    v = (s.rng.standard_normal((n, 1, 64)) * size).astype(np.float32)
    k = (s.rng.standard_normal((n, 1, 64)) * np.where(size > 0, 10.0 ** s.rng.uniform(-3, 0.5, size.shape), 0))
    s.step([n], k=k.astype(np.float32), v=v)
    for new in ([1], [50]):
        step = s.step(new)
        q = s.rng.standard_normal((new[0], 3, 64)).astype(np.float32)
        q[:, 0] *= np.float32(1e-30)
        q[0, 1] = 0
        q[:, 2, 1::2] *= np.float32(1e-6)
        s.attend(step, new, 3, q=q)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("new", [1, 300])
def test_attention_past_large_values(kq, dtype, dim, new):
    """Pages of values 1e8 times the others', whose logits are 80 below: they
    weigh nothing (1e8 e^-80), and the others keep their bits.  The bounds of
    this file with W = sum p |v| in place of the largest value: errors are
    relative to each weight.  (Weights of 22 bits below the largest value
    alone would be wrong by 2^-5 here.)"""
    s = Server(kq, 1, dim, 16, "int8", 1, 210, pages=70, dtype=dtype)
    n, G = 700, 3
    far = np.zeros(n, bool)
    far[64:96] = far[304:320] = far[656:672] = True     # whole pages
    k = (0.1 * s.rng.standard_normal((n, 1, dim))).astype(np.float32)
    k[far] = 0
    k[far, 0, 0] = -20
    v = (s.rng.standard_normal((n, 1, dim)) * np.where(far, 1e8, 1)[:, None, None]).astype(np.float32)
    s.step([n], k=k, v=v)
    step = s.step([new], k=k[:1].repeat(new, 0), v=v[:1].repeat(new, 0))
    q = s.rng.standard_normal((new, G, dim)).astype(np.float32)
    q[:, :, 0] = 4
    with Launches(kq, "kv8_prompt") as seen:
        got, _ = s.attend(step, [new], G, scale=1.0, q=q, check=False)
    assert seen.count == (new > 1)
    if dtype == "bfloat16":
        q = dev(q, dtype).float().cpu().numpy()
    o, l, size, _ = ref.attend(s.ref, s.table, [n], [new], q, 1.0)
    s.ref.code[:, :, 1] = np.abs(s.ref.code[:, :, 1])
    w = ref.attend(s.ref, s.table, [n], [new], q, 1.0)[0].max(-1)
    bo, _ = bounds(dtype, dim, n + new, size, w, o, l)
    assert np.all(w < 10)
    assert np.all(np.abs(got - o) <= bo), np.max(np.abs(got - o) / bo)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new", [1, 300])
@pytest.mark.parametrize("value,logit", [(1e9, 1e12), (1e-7, 3e10), (1e36, 5.0), (3e-24, 5.0), (1e30, 1e-20)])
def test_attention_of_large_logits_and_values(kq, dtype, new, value, logit):
    """Logits up to 1e12, where one token wins, with values of many sizes; the
    largest and the smallest values that the reference points allow."""
    s = Server(kq, 1, 64, 16, "int8", 1, 210, pages=70, dtype=dtype, seed=3)
    n, G = 500, 3
    k = s.rng.standard_normal((n + new, 1, 64)).astype(np.float32)
    v = (value * s.rng.standard_normal((n + new, 1, 64))).astype(np.float32)
    s.step([n], k=k[:n], v=v[:n])
    step = s.step([new], k=k[n:], v=v[n:])
    q = (logit * s.rng.standard_normal((new, G, 64))).astype(np.float32)
    got, _ = s.attend(step, [new], G, scale=1.0, q=q, check=False)
    q = dev(q, dtype).float().cpu().numpy()
    o, l, size, _ = ref.attend(s.ref, s.table, [n], [new], q, 1.0)
    s.ref.code[:, :, 1] = np.abs(s.ref.code[:, :, 1])
    w = ref.attend(s.ref, s.table, [n], [new], q, 1.0)[0].max(-1)
    assert np.all(np.isfinite(got))
    if logit > 1e3:
        # rows whose winner stands out by more than the logits' errors (times 2 for a pair, and 100 to be e^-100 behind)
        kv = s.ref.rows(s.table[0], n + new)[0, 0]
        x = q.astype(np.float64) @ kv.T
        x[np.arange(n + new) > n + np.arange(new)[:, None, None].repeat(G, 1)] = -np.inf
        x.sort(-1)
        clear = x[..., -1] - x[..., -2] > 100 + 4 * size * (8 + 64 / 4) * U
        assert clear.mean() > 0.8
        step = 2.0 ** -8 + 2.0 ** -11 if dtype == "bfloat16" else 2.0 ** -20
        assert np.all(np.abs(got - o)[clear] <= (step * np.abs(o) + 2.0 ** -20 * w[..., None])[clear])
    else:
        bo, _ = bounds(dtype, 64, n + new, size, w, o, l)
        assert np.all(np.abs(got - o) <= bo), np.max(np.abs(got - o) / bo)


def test_attention_twice_is_the_same(kq):
    s = Server(kq, 2, 128, 32, "int8", 2, 100)
    s.step([3000, 50])
    for new in ([1, 1], [70, 9]):
        step = s.step(new)
        q = s.rng.standard_normal((sum(new), 8, 128)).astype(np.float32)
        a = s.attend(step, new, 8, q=q.copy(), check=False)
        b = s.attend(step, new, 8, q=q.copy(), check=False)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("new", [[1, 1], [80, 1]])
@pytest.mark.parametrize("what", ["query", "page", "length", "offsets"])
def test_attention_of_bad_contents(kq, what, new):
    """A non-finite query, a page id, a length or offsets out of range: an
    error at the synchronize, and the next call works."""
    import torch
    s = Server(kq, 1, 64, 16, "int8", 2, 12)
    s.step([50, 20])
    step = s.step(new)
    T = sum(new)
    q = torch.randn(T, 2, 64, device="cuda")
    out = torch.empty_like(q)
    ws = torch.empty(s.cache.attend_workspace_bytes(step, 2), dtype=torch.uint8, device="cuda")
    keep = {n: getattr(step, n).clone() for n in ("kv_lengths", "query_offsets")}
    table = s.table_dev.clone()
    if what == "query":
        q[0, 1, 3] = math.inf
    elif what == "page":
        s.table_dev[0, 1] = s.cache.pages
    elif what == "length":
        step.kv_lengths[0] = 12 * 16 + 1
    else:
        step.query_offsets[2] = T + 1
    torch.cuda.synchronize()
    s.cache.attend(step, q, out, scale=0.1, workspace=ws)
    with pytest.raises(kq.KQError) as e:
        kq.synchronize()
    assert e.value.status == (kq.abi.NUMERIC_DOMAIN if what == "query" else kq.abi.SPAN_OUT_OF_RANGE)
    for n, a in keep.items():
        getattr(step, n).copy_(a)
    s.table_dev.copy_(table)
    s.attend(step, new, 2)


def test_cache_beyond_32_bit_offsets(kq):
    """Codes of more than 2^32 bytes: the first and the last pages."""
    import torch
    heads, dim, page = 2, 256, 64
    pages = (1 << 32) // (2 * heads * page * dim) + 40
    cache = kq.Kv8Cache(heads, dim, page, pages, codes=torch.zeros(pages * 2 * heads * page * dim, dtype=torch.uint8,
                                                                   device="cuda"))
    ids = np.int32([pages - 1, 0, pages - 2, 1, pages - 3])
    td = dev(ids[None])
    step = kq.Kv8Step(1, 300, td, page)
    args = [dev(np.int32(a)) for a in ([0], [300], ids, [0], [0])]
    k, v = torch.randn(2, 300, heads, dim, device="cuda")
    q, out = torch.randn(300, 4, dim, device="cuda"), torch.empty(300, 4, dim, device="cuda")
    small = kq.Kv8Cache(heads, dim, page, 5)
    step2 = kq.Kv8Step(1, 300, dev(np.int32([[0, 1, 2, 3, 4]])), page)
    args2 = [dev(np.int32(a)) for a in ([0], [300], range(5), [0], [0])]
    out2, far = torch.empty_like(out), torch.empty(2, heads, 2, page, dim, device="cuda")
    near = torch.empty_like(far)
    ws = torch.empty(max(16, cache.attend_workspace_bytes(step, 4)), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for c, s, a, o, f, p in ((cache, step, args, out, far, ids[[0, 1]]), (small, step2, args2, out2, near, np.int32([0, 1]))):
        c.plan(s, *a)
        c.append(s, k, v)
        c.attend(s, q, o, scale=0.06, workspace=ws)
        c.read_pages(dev(p), f)
        kq.synchronize()
    assert torch.equal(out, out2) and torch.equal(far, near)


def test_steps_of_a_server(kq):
    """Prompts, chunks and decode steps of requests that come and go, over one
    pool whose freed pages are used again, against attention in 64 bits."""
    s = Server(kq, 2, 128, 32, "int8", 4, 8, pages=40, seed=2, dtype="bfloat16")
    for new in ([100, 33, 0, 1], [1, 1, 64, 1], [1, 1, 1, 1], [40, 1, 1, 1]):
        step = s.step(new)
        s.attend(step, new, 4)
    # request 1 ends: its pages go back to the front of the free list
    back = s.table[1, :-(-s.context[1] // 32)].copy()
    s.free = np.r_[back, s.free[s.head:]].astype(np.int32)
    s.free_dev, s.head = dev(s.free), 0
    s.context[1] = 0
    for new in ([1, 65, 1, 1], [1, 1, 1, 1]):
        step = s.step(new)
        s.attend(step, new, 4)


def test_step_in_a_graph(kq):
    """Plan, append and attention captured together on a caller's stream and
    replayed with other lengths and rows; the library's own stream after it."""
    import torch
    s = Server(kq, 2, 64, 16, "int8", 3, 200, seed=5)
    s.step([2500, 9, 31])
    stream = torch.cuda.Stream()
    step = kq.Kv8Step(3, 5, s.table_dev, 16)
    ctx, cnt, head, head_out = (dev(np.int32(a)) for a in (s.context, [1, 1, 1], [s.head], [0]))
    k, v = torch.zeros(2, 5, 2, 64, device="cuda")
    q, out, lse = torch.zeros(5, 4, 64, device="cuda"), torch.zeros(5, 4, 64, device="cuda"), torch.zeros(5, 4, device="cuda")
    ws = torch.empty(s.cache.attend_workspace_bytes(step, 4), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    d = kq.abi.Diagnostic()
    kq.abi.check(kq.lib().kq_b200_set_stream(stream.cuda_stream, C.byref(d)), d)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            s.cache.plan(step, ctx, cnt, s.free_dev, head, head_out)
            s.cache.append(step, k, v)
            s.cache.attend(step, q, out, lse, scale=0.125, workspace=ws)
        for new in ([1, 1, 1], [1, 0, 2], [0, 1, 4], [1, 1, 1]):
            T = sum(new)
            rows = s.rng.standard_normal((3, 5, 2, 64)).astype(np.float32)
            qh = s.rng.standard_normal((5, 4, 64)).astype(np.float32)
            for t, a in ((k, rows[0]), (v, rows[1]), (q, qh), (ctx, np.int32(s.context)), (cnt, np.int32(new)),
                         (head, np.int32([s.head]))):
                t.copy_(torch.as_tensor(a))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            kq.synchronize()
            want = ref.plan(16, s.context, new, s.table, s.free, s.head, 5, step.page_runs.numel())
            ends = [t for t in want["page_runs"] if t >= 0] + [T]
            for a, z in zip(ends, ends[1:]):
                p = want["slots"][a]
                s.ref.append_run(p // 16, p % 16, rows[:2, a:z].transpose(1, 2, 0, 3))
            s.table, before = want["block_table"], s.context
            s.context, s.head = want["kv_lengths"], want["free_head"][0]
            assert int(head_out) == s.head
            o, l, size, top = ref.attend(s.ref, s.table, before, new, qh[:T], 0.125)
            bo, bl = bounds("float32", 64, max(s.context), size, top, o, l)
            assert np.all(np.abs(out[:T].cpu().numpy() - o) <= bo)
            assert np.all(np.abs(lse[:T].cpu().numpy() - l) <= bl)
        del graph
    finally:
        kq.abi.check(kq.lib().kq_b200_set_stream(None, C.byref(d)), d)
    s.step([1, 1, 1])
    s.check_pages()


def test_arrays_must_be_on_the_device(kq):
    """Host memory is refused, not read."""
    import torch
    s = Server(kq, 1, 64, 16, "int8", 1, 2)
    step = s.step([3])
    host = torch.zeros(3, 1, 64)
    card = host.cuda()
    for bad in ((host, card), (card, host)):
        with pytest.raises(kq.KQError) as e:
            s.cache.append(step, *bad)
        assert e.value.status == kq.abi.INVALID_ARGUMENT
    with pytest.raises(kq.KQError):
        s.cache.attend(step, host, card, scale=1.0)
    with pytest.raises(ValueError):
        s.cache.append(step, card.half(), card)
    with pytest.raises(ValueError):
        s.cache.attend(step, card, card.bfloat16(), scale=1.0)
