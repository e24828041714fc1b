"""Plain restatement of the paged 8-bit cache for its tests: numpy, one page
or row at a time, F32 where the definition rounds to F32 and F64 elsewhere."""
import numpy as np

LARGEST = {"int8": np.float32(127), "e4m3": np.float32(448)}


def e4m3_values() -> np.ndarray:
    """The value of every byte (the NaN codes 0x7f, 0xff as NaN)."""
    b = np.arange(256)
    e, m = b >> 3 & 15, b & 7
    v = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    v = np.where((b & 0x7F) == 0x7F, np.nan, v)
    return np.where(b >= 128, -v, v).astype(np.float32)


E4M3 = e4m3_values()
_POS = np.arange(0x7F)   # non-negative finite codes, ascending


def encode(q: np.ndarray, fmt: str) -> np.ndarray:
    """Stored values (F32) nearest to F32 quotients, ties to even."""
    q = np.clip(np.asarray(q, np.float32), -LARGEST[fmt], LARGEST[fmt])
    if fmt == "int8":
        return np.rint(q).astype(np.float32)
    v, a = E4M3[_POS].astype(np.float64), np.abs(q).astype(np.float64)
    hi = np.searchsorted(v, a).clip(0, len(v) - 1)
    lo = np.maximum(hi - 1, 0)
    up, down = v[hi] - a, a - v[lo]
    pick = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return np.copysign(v[pick], q).astype(np.float32)


def values(byte: np.ndarray, fmt: str) -> np.ndarray:
    return byte.astype(np.float32) - 128 if fmt == "int8" else E4M3[byte]


def from_layout(raw: np.ndarray, fmt: str, page: int, dim: int) -> np.ndarray:
    """Codes [2][page][dim] (as values) of one (page, head), byte by byte."""
    out = np.empty((2, page, dim), np.float32)
    f = np.arange(dim)
    for t in range(page):
        w, base = t % 16, t // 16 * 32 * dim
        key = base + f // 64 * 1024 + w // 8 * 512 + w % 8 * 64 + f % 64
        val = base + 16 * dim + f // 32 * 512 + f % 32 // 4 * 64 + w % 8 // 2 * 16 + f % 4 * 4 + w // 8 * 2 + w % 2
        out[0, t], out[1, t] = values(raw[key], fmt), values(raw[val], fmt)
    return out


class Cache:
    """Codes (as values) [page][head][2][row][feature] and scales."""

    def __init__(self, heads, dim, page, pages, fmt):
        self.heads, self.dim, self.page, self.fmt = heads, dim, page, fmt
        self.code = np.zeros((pages, heads, 2, page, dim), np.float32)
        self.scale = np.zeros((pages, heads, 2), np.float32)

    def append_run(self, page, at, rows):
        """rows: [n][head][2][feature] F32 into rows at .. at + n of a page."""
        n = rows.shape[0]
        for h in range(self.heads):
            for side in range(2):
                x = rows[:, h, side]
                old = self.scale[page, h, side] if at else np.float32(0)
                new = max(old, np.abs(x).max() / LARGEST[self.fmt])
                code = self.code[page, h, side]
                if at == 0:
                    code[n:] = 0
                elif new > old:
                    code[:at] = encode(code[:at] * np.float32(old / new), self.fmt)
                with np.errstate(divide="ignore", invalid="ignore"):
                    code[at:at + n] = encode(x / new, self.fmt) if new > 0 else 0
                self.scale[page, h, side] = new

    def values(self, pages):
        return self.code[pages] * self.scale[pages][..., None, None]

    def rows(self, table, length):
        """Values [2][head][length][feature] in F64: code times scale, not rounded."""
        p = np.asarray(table[:-(-length // self.page)], np.int64)
        v = self.code[p].astype(np.float64) * self.scale[p].astype(np.float64)[..., None, None]
        return v.transpose(2, 1, 0, 3, 4).reshape(2, self.heads, -1, self.dim)[:, :, :length]


def plan(page, context, new, table, free, head, tokens, runs):
    """The step's arrays; `table` (a copy) with the new pages."""
    table = table.copy()
    offsets, run_offsets, slots, positions, starts = [0], [0], [], [], []
    for b, (c, n) in enumerate(zip(context, new)):
        for j in range(-(-c // page), -(-(c + n) // page)):
            table[b, j] = free[head]
            head += 1
        for i in range(n):
            pos = c + i
            if i == 0 or pos % page == 0:
                starts.append(len(slots))
            slots.append(int(table[b, pos // page]) * page + pos % page)
            positions.append(pos)
        offsets.append(len(slots))
        run_offsets.append(len(starts))
    pad = tokens - len(slots)
    return {"block_table": table, "query_offsets": offsets, "kv_lengths": [c + n for c, n in zip(context, new)],
            "slots": slots + [-1] * pad, "positions": positions + [-1] * pad, "run_offsets": run_offsets,
            "page_runs": starts + [-1] * (runs - len(starts)), "free_head": [head]}


def attend(cache, table, context, new, q, scale):
    """F64 output and lse of every new token (rows in request order), and per
    row the largest sum |q_i k_i| of its logits and the largest |value|: what
    rounding errors are proportional to."""
    G = q.shape[1] // cache.heads
    out, lse = np.zeros(q.shape, np.float64), np.full(q.shape[:2], -np.inf)
    size, top = np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    row = 0
    for b, (c, n) in enumerate(zip(context, new)):
        if n and c + n > 0:
            kv = cache.rows(table[b], c + n)
            hidden = np.arange(c + n) > c + np.arange(n)[:, None]
            some = ~hidden.all(1)   # rows that see something
            for h in range(q.shape[1]):
                k, v = kv[:, h // G]
                x = q[row:row + n, h].astype(np.float64)
                l = np.where(hidden, -np.inf, x @ k.T * scale)[some]
                m = l.max(1, keepdims=True)
                w = np.exp(l - m)
                at = np.arange(row, row + n)[some]
                out[at, h] = w @ v / w.sum(1, keepdims=True)
                lse[at, h] = (m + np.log(w.sum(1, keepdims=True)))[:, 0]
                size[at, h] = np.where(hidden, 0, np.abs(x) @ np.abs(k).T)[some].max(1) * abs(scale)
                top[at, h] = np.where(hidden[some], 0, np.abs(v).max(1)).max(1)
        row += n
    return out, lse, size, top
