"""The paged 8-bit key/value cache operators, as cases that can be measured.

``run`` makes ONE pass through an operator: with ``own`` the calls a user
makes of ``kqb200`` (plan, append and read, attend), otherwise the same
result from elementary torch operations.  Both work on the state ``prepare``
makes: the cache's code and scale arrays in the library's page layout, the
block table and the step arrays of a ragged batch.
"""
import ctypes
import math
import random
import sys
from pathlib import Path

import torch

own = False

_kq = None


def _kqb200():
    """The framework's package (imported only where ``own`` is true)."""
    global _kq
    if _kq is None:
        path = str(Path(__file__).resolve().parent.parent / "kestrel-q_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import kqb200
        _kq = kqb200
    return _kq


# ------------------------------------------------------------------- cases

def _case(name, op, requests, prompts, context, new, *, heads=(16, 2), dim=256, page=64, fmt="int8", dtype="f32",
          lengths_seed=1, padding=0):
    """`prompts` of the `requests` bring new[0]..new[1] tokens, the others one;
    contexts are uniform in context[0]..context[1] (tokens cached before)."""
    return {"name": name, "op": op, "requests": requests, "prompts": prompts, "context_min": context[0],
            "context_max": context[1], "new_min": new[0], "new_max": new[1], "query_heads": heads[0],
            "kv_heads": heads[1], "head_dim": dim, "page_tokens": page, "format": fmt, "dtype": dtype,
            "lengths_seed": lengths_seed, "padding": padding}


def listed():
    return [
        # the decode step of the benchmark's batch: 64 sequences, contexts U[1k, 32k]
        _case("plan decode 64", "plan", 64, 0, (1024, 32767), (1, 1)),
        # a prompt phase: many ragged prompts, a padded token buffer
        _case("plan prompts 512", "plan", 512, 384, (0, 4000), (1, 600), page=32, padding=1000),
        # one token of each of 64 sequences into partly filled pages, the framework's F32 activations
        _case("append decode 64 f32 int8", "append", 64, 0, (1024, 32767), (1, 1)),
        # an 8k prompt in bfloat16, e4m3 pages
        _case("append prompt 8k bf16 e4m3", "append", 1, 1, (0, 0), (8192, 8192), heads=(32, 8), dim=128, page=32,
              fmt="e4m3", dtype="bf16"),
        # chunks of many prompts that begin and end inside pages
        _case("append ragged f32 int8", "append", 48, 40, (0, 3001), (3, 2001), padding=77),
        # batch-1 decode at context 4096: latency
        _case("attend one 4k f32 int8", "attend", 1, 0, (4095, 4095), (1, 1)),
        # a few short odd requests: latency again, five heads to a key/value head
        _case("attend short odd bf16 e4m3", "attend", 7, 2, (0, 333), (1, 19), heads=(10, 2), dim=64, page=16,
              fmt="e4m3", dtype="bf16", padding=5),
        # the benchmark's decode batch: 64 sequences, contexts U[1k, 32k], F32
        _case("attend decode 64 f32 int8", "attend", 64, 0, (1024, 32767), (1, 1)),
        # a larger decode batch of shorter contexts, bfloat16 queries over e4m3 pages
        _case("attend decode 96 bf16 e4m3", "attend", 96, 0, (255, 8191), (1, 1), heads=(32, 8), dim=128, page=32,
              fmt="e4m3", dtype="bf16"),
        # single-sequence decode at 131k tokens
        _case("attend one 131k bf16 int8", "attend", 1, 0, (131071, 131071), (1, 1), dtype="bf16"),
        # an 8k prompt, bfloat16
        _case("attend prompt 8k bf16 int8", "attend", 1, 1, (0, 0), (8192, 8192), heads=(32, 8), dim=128,
              dtype="bf16"),
        # prompt chunks beside decode tokens, F32
        _case("attend mixed f32 e4m3", "attend", 24, 6, (0, 6000), (64, 700), fmt="e4m3", padding=33),
    ]


def _spread(rng, lo, hi):
    """An integer of lo..hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "append", "attend", "attend", "attend"])
    heads = rng.choice([(16, 2), (32, 8), (10, 2), (8, 8), (12, 1), (24, 4)])
    dim = rng.choice([64, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    fmt, dtype = rng.choice(["int8", "e4m3"]), rng.choice(["f32", "bf16"])
    more = dict(heads=heads, dim=dim, page=page, fmt=fmt, dtype=dtype, lengths_seed=rng.randrange(1, 1 << 20),
                padding=rng.choice([0, 0, rng.randrange(1, 300)]))
    if op == "plan":
        requests = _spread(rng, 1, 512)
        longest = _spread(rng, 1, min(600, 98304 // requests))
        case = _case("", op, requests, rng.randrange(0, requests + 1), (0, _spread(rng, 1, 32000)), (1, longest), **more)
    elif op == "append":
        requests = _spread(rng, 1, 64)
        longest = _spread(rng, 1, min(8192, 40000 // requests))
        case = _case("", op, requests, rng.randrange(0, requests + 1), (0, _spread(rng, 1, 4000)), (1, longest), **more)
    elif rng.random() < 0.5:  # decode tokens alone
        requests = _spread(rng, 1, 64)
        most = min(131071, 600000 // requests, (1 << 28) // (requests * heads[1] * dim))
        top = _spread(rng, 1, most)
        case = _case("", op, requests, 0, (rng.randrange(0, top + 1), top), (1, 1), **more)
    else:  # prompts, with and without cached tokens
        requests = _spread(rng, 1, 16)
        new = _spread(rng, 1, min(4096, 8192 // requests))
        room = (1 << 31) // (requests * new * heads[0])
        top = _spread(rng, 1, max(1, min(8191, room - new)))
        case = _case("", op, requests, rng.randrange(1, requests + 1), (0, top), (rng.randrange(1, new + 1), new), **more)
    del case["name"]
    return case


def _lengths(case):
    rng = random.Random(case["lengths_seed"])
    context = [rng.randint(case["context_min"], case["context_max"]) for _ in range(case["requests"])]
    new = [rng.randint(case["new_min"], case["new_max"]) if b < case["prompts"] else 1 for b in range(case["requests"])]
    order = list(range(case["requests"]))
    rng.shuffle(order)
    return [context[b] for b in order], [new[b] for b in order]


def _ceil(a, b):
    return -(-a // b)


def _run_capacity(tokens, requests, page):
    return min(tokens, tokens // page + 2 * requests)


# ---------------------------------------------------- the pages' layout
#
# A page holds, per key/value head, page_tokens / 16 groups of 16 tokens, each
# 16 * d key codes, then 16 * d value codes:
#   key    [j d/64][h 2][g 8][t 4][e 16]         feature = 64 j + 16 t + e, token = 8 h + g
#   value  [j d/32][g 8][t 4][i 4][h 2][e 2]     feature = 32 j + 4 g + i, token = 8 h + 2 t + e
# int8 codes are stored with 128 added, e4m3 codes as they are.

def _to_layout(codes):
    """[n][H][2][P][d] bytes -> [n][H][P/16][32 d] in page order."""
    n, heads, _, page, dim = codes.shape
    k = codes[:, :, 0].reshape(n, heads, page // 16, 2, 8, dim // 64, 4, 16).permute(0, 1, 2, 5, 3, 4, 6, 7)
    v = codes[:, :, 1].reshape(n, heads, page // 16, 2, 4, 2, dim // 32, 8, 4).permute(0, 1, 2, 6, 7, 4, 8, 3, 5)
    both = [x.reshape(n, heads, page // 16, 16 * dim) for x in (k, v)]
    return torch.cat(both, dim=-1)


def _from_layout(raw, dim):
    """The inverse of _to_layout."""
    n, heads, groups, _ = raw.shape
    k = raw[..., :16 * dim].reshape(n, heads, groups, dim // 64, 2, 8, 4, 16).permute(0, 1, 2, 4, 5, 3, 6, 7)
    v = raw[..., 16 * dim:].reshape(n, heads, groups, dim // 32, 8, 4, 4, 2, 2).permute(0, 1, 2, 7, 5, 8, 3, 4, 6)
    both = [x.reshape(n, heads, groups * 16, dim) for x in (k, v)]
    return torch.stack(both, dim=2)


_MOST = {"int8": 127.0, "e4m3": 448.0}


def _code_values(byte, fmt):
    return byte.float() - 128.0 if fmt == "int8" else byte.view(torch.float8_e4m3fn).float()


def _to_codes(x, fmt):
    """F32 quotients -> stored bytes."""
    x = x.clamp(-_MOST[fmt], _MOST[fmt])
    return (x.round() + 128.0).to(torch.uint8) if fmt == "int8" else x.to(torch.float8_e4m3fn).view(torch.uint8)


def _quotient(x, scale):
    """x / scale, 0 where the scale is 0."""
    return torch.where(scale > 0, x / torch.where(scale > 0, scale, torch.ones_like(scale)), torch.zeros_like(x))


# ----------------------------------------------------------------- inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    heads, dim, page, fmt = case["kv_heads"], case["head_dim"], case["page_tokens"], case["format"]
    dtype = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    context, new = _lengths(case)
    B, total = len(new), sum(new)
    tokens = total + case["padding"]
    before = [_ceil(c, page) for c in context]
    after = [_ceil(c + n, page) for c, n in zip(context, new)]
    columns = max(after) + 3
    used = sum(after)
    pages = used + 7
    # page ids scattered over the pool, as a server's are after a while
    ids = torch.randperm(pages, generator=gen, device=dev, dtype=torch.int64).to(torch.int32)
    ctx = torch.tensor(context, dtype=torch.int32, device=dev)
    cnt = torch.tensor(new, dtype=torch.int32, device=dev)
    held = torch.tensor(before, dtype=torch.int64, device=dev)
    final = torch.tensor(after, dtype=torch.int64, device=dev)
    col = torch.arange(columns, device=dev)[None, :]
    first = (torch.cumsum(held, 0) - held)[:, None]
    table = torch.where(col < held[:, None], ids[(first + col).clamp(max=pages - 1)], -1).to(torch.int32)
    free = ids[sum(before):].contiguous()
    state = {"case": dict(case), "tokens": tokens, "total": total, "pages": pages, "columns": columns, "ctx": ctx,
             "new": cnt, "table": table.contiguous(), "free": free,
             "free_head": torch.zeros(1, dtype=torch.int32, device=dev),
             "runs": _run_capacity(tokens, B, page), "longest": max(new), "deepest": max(after)}
    if case["op"] == "plan":
        # other tables in every seed: the free list begins at an odd place
        state["free_head"] += seed % 5
        return state
    # what the plan of this step gives: every page assigned, slots, positions, page runs
    extra = (torch.cumsum(final - held, 0) - (final - held))[:, None]
    fresh = (col >= held[:, None]) & (col < final[:, None])
    table = torch.where(fresh, free[(extra + col - held[:, None]).clamp(0, len(free) - 1)], table).contiguous()
    offsets = torch.zeros(B + 1, dtype=torch.int32, device=dev)
    offsets[1:] = torch.cumsum(cnt, 0)
    state["table"] = table
    state["step"] = _step_plain(state, table, offsets)
    # keys and values with channels of different size, as projections give them
    gain = torch.exp(0.5 * torch.randn(heads, 2, 1, dim, generator=gen, device=dev))
    if case["op"] == "append":
        state["k"] = (torch.randn(tokens, heads, dim, generator=gen, device=dev) * gain[:, 0, 0]).to(dtype)
        state["v"] = (torch.randn(tokens, heads, dim, generator=gen, device=dev) * gain[:, 1, 0]).to(dtype)
    codes = torch.empty(pages, heads, page // 16, 32 * dim, dtype=torch.uint8, device=dev)
    scales = torch.empty(pages, heads, 2, dtype=torch.float32, device=dev)
    part = max(1, (1 << 27) // (heads * 2 * page * dim))
    for a in range(0, pages, part):
        n = min(part, pages - a)
        x = torch.randn(n, heads, 2, page, dim, generator=gen, device=dev) * gain
        s = x.abs().amax(dim=(3, 4)) / _MOST[fmt]
        codes[a:a + n] = _to_layout(_to_codes(x / s[..., None, None], fmt))
        scales[a:a + n] = s
    state["codes"], state["scales"] = codes, scales
    if case["op"] == "append":
        # the pages that the step writes: one for each run
        start = state["step"]["page_runs"][:state["step_runs"]].long()
        state["touched"] = (state["step"]["slots"][start] // page).to(torch.int32).contiguous()
    else:
        q = case["query_heads"]
        state["q"] = torch.randn(tokens, q, dim, generator=gen, device=dev).to(dtype)
        state["out"] = torch.zeros(tokens, q, dim, dtype=dtype, device=dev)
        state["lse"] = torch.zeros(tokens, q, dtype=torch.float32, device=dev)
    return state


def _step_plain(state, table, offsets):
    """Slots, positions and page runs from the lengths, the block table and the query offsets."""
    page = state["case"]["page_tokens"]
    B = state["ctx"].numel()
    dev = table.device
    ctx, cnt = state["ctx"].long(), state["new"].long()
    t = torch.arange(state["tokens"], device=dev)
    b = torch.searchsorted(offsets[1:].long(), t, right=True).clamp(max=B - 1)
    inside = t < offsets[B]
    pos = ctx[b] + t - offsets[b].long()
    column = torch.where(inside, pos // page, 0)
    slot = table[b, column].long() * page + pos % page
    none = torch.full_like(slot, -1)
    slots = torch.where(inside, slot, none)
    positions = torch.where(inside, pos, none).to(torch.int32)
    count = torch.where(cnt > 0, (ctx + cnt + page - 1) // page - ctx // page, 0)
    run_offsets = torch.zeros(B + 1, dtype=torch.int64, device=dev)
    run_offsets[1:] = torch.cumsum(count, 0)
    starts = inside & ((t == offsets[b]) | (pos % page == 0))
    index = torch.where(starts, run_offsets[b] + pos // page - ctx[b] // page, state["runs"])
    runs = torch.full((state["runs"] + 1,), -1, dtype=torch.int32, device=dev)
    runs.scatter_(0, index, torch.where(starts, t, -1).to(torch.int32))
    if "step_runs" not in state:  # known to the host from the lengths
        context, new = _lengths(state["case"])
        state["step_runs"] = sum(_ceil(c + n, page) - c // page for c, n in zip(context, new) if n)
    return {"query_offsets": offsets, "kv_lengths": (ctx + cnt).to(torch.int32), "slots": slots,
            "positions": positions, "run_offsets": run_offsets.to(torch.int32), "page_runs": runs[:-1].contiguous()}


# -------------------------------------------------------------- the passes

def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "attend": _own_attend}[op](state)
    return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend}[op](state)


def _handles(state):
    """What a user's program keeps from step to step: the cache over its arrays and the step's buffers."""
    if "cache" not in state:
        kq, c = _kqb200(), state["case"]
        # the calls belong between torch's operations: one stream for both (1: CUDA's name of the default stream)
        d = kq.abi.Diagnostic()
        kq.abi.check(kq.lib().kq_b200_set_stream(torch.cuda.current_stream().cuda_stream or 1, ctypes.byref(d)), d)
        state["cache"] = kq.Kv8Cache(c["kv_heads"], c["head_dim"], c["page_tokens"], state["pages"], c["format"],
                                     codes=state.get("codes"), scales=state.get("scales"))
        step = kq.Kv8Step(c["requests"], state["tokens"], state["table"], c["page_tokens"])
        if "step" in state:
            step.use(**state["step"])
        state["handle"] = step
    return state["cache"], state["handle"]


def _own_plan(state):
    cache, step = _handles(state)
    if "free_head_out" not in state:
        state["free_head_out"] = torch.empty_like(state["free_head"])
    cache.plan(step, state["ctx"], state["new"], state["free"], state["free_head"], state["free_head_out"])
    return {"block_table": step.block_table, "query_offsets": step.query_offsets, "kv_lengths": step.kv_lengths,
            "slots": step.slots, "positions": step.positions, "run_offsets": step.run_offsets,
            "page_runs": step.page_runs, "free_head": state["free_head_out"]}


def _plain_plan(state):
    page, table = state["case"]["page_tokens"], state["table"]
    ctx, cnt, free = state["ctx"].long(), state["new"].long(), state["free"]
    B = ctx.numel()
    offsets = torch.zeros(B + 1, dtype=torch.int32, device=ctx.device)
    offsets[1:] = torch.cumsum(cnt, 0)
    held, final = (ctx + page - 1) // page, (ctx + cnt + page - 1) // page
    taken = final - held
    head = state["free_head"].long()
    col = torch.arange(state["columns"], device=ctx.device)[None, :]
    rank = head + (torch.cumsum(taken, 0) - taken)[:, None] + col - held[:, None]
    fresh = (col >= held[:, None]) & (col < final[:, None])
    table.copy_(torch.where(fresh, free[rank.clamp(0, free.numel() - 1)], table))
    step = _step_plain(state, table, offsets)
    return {"block_table": table, **step, "free_head": (head + taken.sum()).to(torch.int32)}


def _own_append(state):
    cache, step = _handles(state)
    if "values" not in state:
        c = state["case"]
        state["values"] = torch.empty(state["touched"].numel(), c["kv_heads"], 2, c["page_tokens"], c["head_dim"],
                                      device=state["k"].device)
    cache.append(step, state["k"], state["v"])
    cache.read_pages(state["touched"], state["values"])
    return {"values": state["values"], "scales": state["scales"]}


def _plain_append(state):
    c = state["case"]
    page, dim, fmt, heads = c["page_tokens"], c["head_dim"], c["format"], c["kv_heads"]
    touched = state["touched"].long()
    start = state["step"]["page_runs"][:touched.numel()].long()
    slots = state["step"]["slots"]
    at = (slots[start] % page)[:, None]
    row = torch.arange(page, device=touched.device)[None, :]
    t = (start[:, None] + row - at).clamp(0, state["tokens"] - 1)
    fresh = (row >= at) & (slots[t] == slots[start][:, None] + row - at)  # rows that the run brings
    kept = row < at
    x = torch.stack([state["k"].float()[t], state["v"].float()[t]], 1).permute(0, 3, 1, 2, 4)  # [run][H][2][P][d]
    fresh, kept = fresh[:, None, None, :, None], kept[:, None, None, :, None]
    x = torch.where(fresh, x, 0.0)
    old = torch.where((at > 0)[:, :, None], state["scales"][touched], 0.0)
    # a tensor as divisor: a number would become a product with its rounded reciprocal
    scale = torch.maximum(old, x.abs().amax(dim=(3, 4)) / torch.full_like(old, _MOST[fmt]))
    raw = _from_layout(state["codes"][touched], dim)
    ratio = _quotient(old, scale)[..., None, None]
    again = _to_codes(_code_values(raw, fmt) * ratio, fmt)
    again = torch.where(ratio == 1.0, raw, again)
    # rows behind the run: cleared by a run that begins its page, else left as they were
    behind = torch.where((at > 0)[:, None, None, :, None], raw, 128 if fmt == "int8" else 0)
    written = _to_codes(_quotient(x, scale[..., None, None]), fmt)
    codes = torch.where(fresh, written, torch.where(kept, again, behind)).to(torch.uint8)
    state["codes"][touched] = _to_layout(codes)
    state["scales"][touched] = scale
    return {"values": _code_values(codes, fmt) * scale[..., None, None], "scales": state["scales"]}


def _own_attend(state):
    cache, step = _handles(state)
    c = state["case"]
    if "workspace" not in state:
        size = cache.attend_workspace_bytes(step, c["query_heads"], state["deepest"] * c["page_tokens"])
        state["workspace"] = torch.empty(size, dtype=torch.uint8, device=state["q"].device)
    cache.attend(step, state["q"], state["out"], state["lse"], scale=1.0 / math.sqrt(c["head_dim"]),
                 max_kv_length=state["deepest"] * c["page_tokens"], workspace=state["workspace"])
    return {"out": state["out"], "lse": state["lse"]}


def _plain_attend(state):
    c, step = state["case"], state["step"]
    page, dim, heads, fmt = c["page_tokens"], c["head_dim"], c["kv_heads"], c["format"]
    G, B = c["query_heads"] // heads, c["requests"]
    table = state["table"][:, :state["deepest"]].long().clamp(min=0)
    n = table.numel()
    raw = state["codes"][table.reshape(-1)]
    scale = state["scales"][table.reshape(-1)]
    value = _code_values(_from_layout(raw, dim), fmt) * scale[..., None, None]
    value = value.view(B, n // B, heads, 2, page, dim).permute(3, 0, 2, 1, 4, 5).reshape(2, B, heads, -1, dim)
    depth = value.shape[3]
    # queries of every request, padded to the longest
    offsets, length = step["query_offsets"].long(), step["kv_lengths"].long()
    i = torch.arange(state["longest"], device=table.device)
    t = (offsets[:-1, None] + i).clamp(max=state["tokens"] - 1)
    q = state["q"].float()[t].view(B, -1, heads, G, dim).permute(0, 2, 3, 1, 4).reshape(B, heads, -1, dim)
    logits = torch.matmul(q, value[0].transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    pos = state["ctx"].long()[:, None] + i
    seen = torch.arange(depth, device=table.device) <= pos[..., None]
    logits = logits.view(B, heads, G, -1, depth).masked_fill_(~seen[:, None, None], -math.inf)
    top = logits.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weight = logits.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(B, heads, -1, depth), value[1]).view(B, heads, G, -1, dim)
    out = (out / total).permute(0, 3, 1, 2, 4).reshape(B, -1, heads * G, dim)
    lse = (top + total.log())[..., 0].permute(0, 3, 1, 2).reshape(B, -1, heads * G)
    # back to ragged rows; those behind the last request stay as they were
    u = torch.arange(state["total"], device=table.device)
    b = torch.searchsorted(offsets[1:], u, right=True)
    state["out"][:state["total"]] = out[b, u - offsets[b]].to(state["out"].dtype)
    state["lse"][:state["total"]] = lse[b, u - offsets[b]]
    return {"out": state["out"], "lse": state["lse"]}


def work(case):
    """The bytes that a pass reads and writes once, and its operations."""
    context, new = _lengths(case)
    page, dim, heads, q = case["page_tokens"], case["head_dim"], case["kv_heads"], case["query_heads"]
    size = 4 if case["dtype"] == "f32" else 2
    tokens = sum(new) + case["padding"]
    runs = sum(_ceil(c + n, page) - c // page for c, n in zip(context, new) if n)
    if case["op"] == "plan":
        taken = sum(_ceil(c + n, page) - _ceil(c, page) for c, n in zip(context, new))
        return {"bytes": 8 * len(new) + 8 * taken + 12 * tokens + 12 * len(new) + 4 * runs, "flops": 0}
    if case["op"] == "append":
        kept = sum(c % page for c in context)
        rows = 2 * heads * dim
        return {"bytes": rows * (sum(new) * (size + 1) + 2 * kept + 4 * runs * page), "flops": 4 * rows * sum(new)}
    seen = sum(n * c + n * (n + 1) // 2 for c, n in zip(context, new))
    held = sum(c + n for c, n in zip(context, new))
    return {"bytes": 2 * heads * dim * held + 8 * heads * held // page + 2 * sum(new) * q * dim * size + 4 * sum(new) * q,
            "flops": 4 * seen * q * dim}


# --------------------------------------------------- the definitions in 64 bits

def _exact_e4m3(x):
    """Nearest e4m3 value (ties to even), from the format: 3 mantissa bits, smallest exponent -6."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), torch.clamp(e - 1, min=-6) - 3)
    return torch.round(x / step) * step


def _exact_round(x, fmt):
    """The stored value nearest to the F32 quotient x (held in 64 bits)."""
    x = x.float().double().clamp(-_MOST[fmt], _MOST[fmt])
    return torch.round(x) if fmt == "int8" else _exact_e4m3(x)


def _exact_pages(state, pages):
    """Codes of pages in 64 bits, [n][H][2][P][d], one byte of the layout at a time by its place."""
    c = state["case"]
    page, dim, fmt = c["page_tokens"], c["head_dim"], c["format"]
    dev = state["codes"].device
    token = torch.arange(page, device=dev)[:, None]
    f = torch.arange(dim, device=dev)[None, :]
    w = token % 16
    key = (token // 16) * 32 * dim + (f // 64) * 1024 + (w // 8) * 512 + (w % 8) * 64 + f % 64
    val = (token // 16) * 32 * dim + 16 * dim + (f // 32) * 512 + (f % 32 // 4) * 64 + (w % 8 // 2) * 16 \
        + (f % 4) * 4 + (w // 8) * 2 + w % 2
    raw = state["codes"].view(state["pages"], c["kv_heads"], -1)[pages]
    byte = raw[:, :, torch.stack([key, val])].long()
    if fmt == "int8":
        return (byte - 128).double()
    e, m = byte // 8 % 16, byte % 8
    mag = torch.where(e > 0, torch.ldexp((8 + m).double(), e - 10), torch.ldexp(m.double(), torch.full_like(e, -9)))
    return torch.where(byte >= 128, -mag, mag)


def exact(case, seed):
    if case["op"] == "plan":
        return None
    state = prepare(case, seed)
    return _exact_append(state) if case["op"] == "append" else _exact_attend(state)


def _exact_append(state):
    c = state["case"]
    page, fmt = c["page_tokens"], c["format"]
    context, new = _lengths(c)
    scales = state["scales"].double()
    touched = state["touched"].long()
    codes = _exact_pages(state, touched)
    runs, row = [], 0
    for ctx, n in zip(context, new):
        for p in range(ctx // page, _ceil(ctx + n, page)):
            a, z = max(ctx, p * page), min(ctx + n, (p + 1) * page)
            runs.append((a - p * page, z - a, row + a - ctx))
        row += n
    at = torch.tensor([r[0] for r in runs], device=touched.device)
    count = torch.tensor([r[1] for r in runs], device=touched.device)
    first = torch.tensor([r[2] for r in runs], device=touched.device)
    place = torch.arange(page, device=touched.device)[None, :]
    token = (first[:, None] + place - at[:, None]).clamp(0, state["tokens"] - 1)
    brings = ((place >= at[:, None]) & (place < (at + count)[:, None]))[:, None, :, None]
    keeps = (place < at[:, None])[:, None, :, None]
    values = torch.empty(codes.shape, dtype=torch.float64, device=codes.device)
    for side, rows in enumerate((state["k"], state["v"])):
        x = rows.double()[token].permute(0, 2, 1, 3) * brings
        old = scales[touched, :, side] * (at > 0)[:, None]
        scale = torch.maximum(old, (x.abs().amax(dim=(2, 3)) / _MOST[fmt]).float().double())
        ratio = (old / scale).float().double()[..., None, None]
        again = torch.where(ratio == 1, codes[:, :, side], _exact_round(codes[:, :, side] * ratio, fmt))
        fresh = _exact_round(x / scale[..., None, None], fmt)
        rest = codes[:, :, side] * (at > 0)[:, None, None, None]
        code = torch.where(brings, fresh, torch.where(keeps, again, rest))
        values[:, :, side] = (code * scale[..., None, None]).float().double()
        scales[touched, :, side] = scale
    return {"values": values, "scales": scales}


def _exact_attend(state):
    c = state["case"]
    page, dim, heads = c["page_tokens"], c["head_dim"], c["kv_heads"]
    G = c["query_heads"] // heads
    context, new = _lengths(c)
    if sum(n * (x + n) for x, n in zip(context, new)) * c["query_heads"] * dim > 3e12:
        return None
    out, lse = state["out"].double(), state["lse"].double()
    row = 0
    for b, (ctx, n) in enumerate(zip(context, new)):
        if n == 0:
            continue
        pages = state["table"][b, :_ceil(ctx + n, page)].long()
        value = _exact_pages(state, pages) * state["scales"][pages].double()[..., None, None]
        value = value.permute(1, 2, 0, 3, 4).reshape(heads, 2, -1, dim)[:, :, :ctx + n]
        for h in range(heads):
            x = state["q"][row:row + n, h * G:(h + 1) * G].double()
            for a in range(0, n, 512):  # rows at a time, to bound the memory
                z = min(n, a + 512)
                logit = torch.einsum("igd,jd->igj", x[a:z], value[h, 0]) / math.sqrt(dim)
                hidden = torch.arange(ctx + n, device=x.device) > ctx + torch.arange(a, z, device=x.device)[:, None]
                logit = logit.masked_fill(hidden[:, None], -math.inf)
                out[row + a:row + z, h * G:(h + 1) * G] = torch.einsum("igj,jd->igd", torch.softmax(logit, -1), value[h, 1])
                lse[row + a:row + z, h * G:(h + 1) * G] = torch.logsumexp(logit, -1)
        row += n
    return {"out": out, "lse": lse}
