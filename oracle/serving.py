"""Plain 64-bit implementations of the decoder-serving operators: the 4-bit cache format, attention over it and the
next-token logits, on CPU tensors, one row after the other, from the definitions in include/chessrl_b200.h."""
import math

import torch

LIMIT = 57344.0


def held_rows(x):
    """f32 rows [..., hd] -> (codes int64 [..., hd], step, centre f64 [..., hd / 32], the values that they stand for f64)."""
    x = x.float()
    nan = torch.isnan(x).unflatten(-1, (-1, 32)).any(-1)
    r = x.clamp(-LIMIT, LIMIT).unflatten(-1, (-1, 32))
    lo, hi = r.amin(-1), r.amax(-1)
    s = ((hi - lo) * torch.tensor(1.0 / 15.0, dtype=torch.float32)).bfloat16().half().float()
    c = (lo + 8.0 * s).half().float()
    inv = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    n = ((r - c[..., None]) * inv[..., None]).nan_to_num(0.0).round().add(8.0).clamp(0.0, 15.0)
    s, c, n = s.double(), c.double(), n.double()
    s[nan], c[nan] = math.nan, math.nan
    value = (n - 8.0) * s[..., None] + c[..., None]
    return n.long().flatten(-2), s, c, value.flatten(-2)


def rotated(x, position, table, interleaved):
    """Rows [n, heads, hd] at `position` [n]: the first 2 * table.shape[1] dims rotated, f64 rounded to f32."""
    y = x.double().clone()
    half = table.shape[1]
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        cos, sin = table[position, i, 0].double()[:, None], table[position, i, 1].double()[:, None]
        y[..., a], y[..., b] = (x[..., a].double() * cos - x[..., b].double() * sin,
                                x[..., b].double() * cos + x[..., a].double() * sin)
    return y.float()


def nibble_of(kind, dim, hd):
    """Position of a dim's nibble in its row."""
    if kind == "k":
        g, t, i = dim // 32, dim % 32 // 8, dim % 8
        return t * (hd // 32) * 8 + g * 8 + i
    return dim % 8 * (hd // 8) + dim // 8


def page_rows(block, hd):
    """One block [20 * hd] uint8 (CPU) -> keys, values f64 [16, hd]."""
    out = []
    for kind, start in (("k", 0), ("v", 10 * hd)):
        codes = block[start:start + 8 * hd].reshape(16, hd // 2).long()
        sc = block[start + 8 * hd:start + 10 * hd].clone().view(torch.float16).reshape(16, hd // 32, 2).double()
        place = torch.tensor([nibble_of(kind, d, hd) for d in range(hd)])
        byte = codes[:, place // 2]
        n = torch.where(place % 2 == 1, byte >> 4, byte & 15).double()
        group = torch.arange(hd) // 32
        out.append((n - 8.0) * sc[:, group, 0] + sc[:, group, 1])
    return out


def cache_rows(pages, table_row, count, head):
    """Keys and values f64 [count, hd] of one sequence and key head; `pages` as kv4_pages lays them out, on the CPU."""
    size, hd = 16 * pages.shape[2], pages.shape[3] // 20
    used = (count + size - 1) // size
    blocks = pages[table_row[:used].long(), head].flatten(0, 1)
    rows = [page_rows(block, hd) for block in blocks]
    return tuple(torch.cat([r[i] for r in rows])[:count] if rows else torch.empty(0, hd, dtype=torch.float64) for i in (0, 1))


def attention(q, k, v, first_position, scale):
    """q f64 [n, hd] at positions first_position.. over keys / values [count, hd]; rows that see nothing are zero."""
    if k.shape[0] == 0:
        return torch.zeros_like(q)
    seen = torch.arange(k.shape[0])[None] <= first_position + torch.arange(q.shape[0])[:, None]
    score = (scale * (q @ k.T)).masked_fill(~seen, -math.inf)
    p = torch.where(seen, torch.exp(score - score.amax(1, keepdim=True)), 0.0)
    out = torch.where(seen[..., None], v[None], 0.0).mul_(p[..., None]).sum(1) if bool(v.isnan().any()) else p @ v
    return torch.where(seen.any(1, keepdim=True), out / p.sum(1, keepdim=True), 0.0)


def adjust(logits, history=None, repetition=None, frequency=None, presence=None, bias_ids=None, bias_values=None, mask=None,
           mask_rows=None, masked_value=-math.inf):
    """The logits [rows, vocab] after penalties, biases and masks, f64."""
    z = logits.double().clone()
    rows, vocab = z.shape
    for r in range(rows):
        count = {}
        for t in history[r].tolist() if history is not None else ():
            if 0 <= t < vocab:
                count[t] = count.get(t, 0) + 1
        for t, n in count.items():
            x = float(z[r, t])
            rep = float(repetition[r]) if repetition is not None else 1.0
            f = float(frequency[r]) if frequency is not None else 0.0
            p = float(presence[r]) if presence is not None else 0.0
            z[r, t] = (x / rep if x > 0 else x * rep) - (f * n + p)
        if bias_ids is not None:
            last = {t: float(b) for t, b in zip(bias_ids[r].tolist(), bias_values[r].tolist()) if 0 <= t < vocab}
            for t, b in last.items():
                z[r, t] += b
        m = r if mask_rows is None else int(mask_rows[r])
        if mask is not None and 0 <= m < mask.shape[0]:
            allowed = (mask[m].long()[torch.arange(vocab) // 8] >> (torch.arange(vocab) % 8)) & 1
            z[r, allowed == 0] = masked_value
    return z
