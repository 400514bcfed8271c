"""The decoder-serving operators as a user calls them, and their plain forms, over the sizes that they serve.

A 4-bit key/value cache: `kv4_append` quantises keys and values into pages (rotating positions on the way),
`kv4_attention` attends to them, `kv4_read` gives the held values back; `adjust_logits` applies penalties, biases and bit
masks to next-token logits. `run` computes the same in elementary torch operations unless `own` is set.

Cache format. Each (token, head) row is cut into groups of 32 dims; a group holds two f16 numbers, the step s (rounded to
eight significant bits) and the centre c, and a 4-bit code n per value, which stands for (n - 8) * s + c. A page holds
[heads][page_size / 16] blocks of 16 tokens: key codes, key (s, c), value codes, value (s, c).
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LIMIT = 57344.0


# ---- cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one game continued by one move token: 12 heads of 64, the decoder's default width; latency counts
        dict(name="append_step_1", op="append", seqs=1, tokens=1, held=69, heads=12, kv_heads=12, dim=64, page=16,
             rotate="none", rot=0, dtype="f16"),
        # a pool of games advanced by one move each, ragged lengths inside a context of 1024
        dict(name="append_step_256", op="append", seqs=256, tokens=1, held=1000, heads=12, kv_heads=12, dim=64, page=64,
             rotate="half", rot=64, dtype="f16"),
        # prompts of ragged lengths, shared key heads, half of each head rotated by neighbouring pairs
        dict(name="append_prompts", op="append", seqs=13, tokens=2048, held=77, heads=32, kv_heads=8, dim=128, page=64,
             rotate="interleaved", rot=64, dtype="bf16"),
        # one game, 64 board tokens and a few moves: the smallest call
        dict(name="attend_step_1", op="attend", seqs=1, tokens=1, held=69, heads=12, kv_heads=12, dim=64, page=16, dtype="f16"),
        # a pool of games in a context of 1024, every head with its own keys
        dict(name="attend_step_256", op="attend", seqs=256, tokens=1, held=1024, heads=12, kv_heads=12, dim=64, page=64,
             dtype="f16"),
        # few very long sequences, four query heads to a key head: the axis of keys has to be split
        dict(name="attend_step_long", op="attend", seqs=4, tokens=1, held=131001, heads=32, kv_heads=8, dim=128, page=64,
             dtype="bf16"),
        # short runs (several proposed moves checked at once) with small heads and pages that end inside a tile
        dict(name="attend_runs", op="attend", seqs=33, tokens=5, held=997, heads=16, kv_heads=4, dim=32, page=48, dtype="f16"),
        # many boards of 64 tokens each: the whole prompt in one call
        dict(name="attend_boards", op="attend", seqs=256, tokens=64, held=64, heads=12, kv_heads=12, dim=64, page=64,
             dtype="f16"),
        # long prompts: bound by the matrix products
        dict(name="attend_prompts", op="attend", seqs=2, tokens=4096, held=4131, heads=32, kv_heads=8, dim=128, page=64,
             dtype="bf16"),
        # one row over the move vocabulary with its legal moves
        dict(name="logits_1", op="logits", rows=1, vocab=1929, history=40, biases=4, mask=True, dtype="f32"),
        # the decoder's default vocabulary, long histories
        dict(name="logits_64", op="logits", rows=64, vocab=50304, history=1024, biases=64, mask=True, dtype="f16"),
        # a large pool of games over the move vocabulary (rows of odd length)
        dict(name="logits_4096", op="logits", rows=4096, vocab=1929, history=60, biases=0, mask=True, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "logits"])
    dtype = rng.choice(["f16", "bf16"])
    heads, kv = rng.choice([(12, 12), (32, 8), (16, 4), (8, 8), (7, 1), (24, 2), (5, 5)])
    dim = rng.choice([32, 64, 64, 128])
    page = rng.choice([16, 32, 48, 64, 128])
    if op == "logits":
        vocab = _log(rng, 200, 50304)
        rows = _log(rng, 1, max(1, min(4096, 8_000_000 // vocab)))
        return dict(op=op, rows=rows, vocab=vocab, history=_log(rng, 1, 1024), biases=rng.choice([0, 1, 7, 64, 300]),
                    mask=rng.random() < 0.7, dtype=rng.choice(["f32", "f16", "bf16"]))
    if op == "append":
        seqs = _log(rng, 1, 512)
        tokens = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, 16000 // seqs))
        rotate = rng.choice(["none", "half", "interleaved"])
        rot = 0 if rotate == "none" else rng.choice([dim, dim // 2, dim // 4])
        return dict(op=op, seqs=seqs, tokens=tokens, held=_log(rng, 1, 4000), heads=heads, kv_heads=kv, dim=dim, page=page,
                    rotate=rotate, rot=rot, dtype=dtype)
    kind = rng.choice(["step", "run", "prompt"])
    if kind == "prompt":
        tokens = _log(rng, 33, 2048)
        seqs = _log(rng, 1, max(1, min(128, 4096 // tokens)))
        held = tokens + rng.choice([0, 0, rng.randrange(0, 700)])
    else:
        tokens = 1 if kind == "step" else rng.randrange(2, 33)
        seqs = _log(rng, 1, 256)
        held = tokens + _log(rng, 1, min(60000, 2_000_000 // (seqs * kv)))
    return dict(op=op, seqs=seqs, tokens=tokens, held=held, heads=heads, kv_heads=kv, dim=dim, page=page, dtype=dtype)


def _ragged(case):
    """(new tokens, cache indices held before them) of every sequence: they follow from the case alone. Steps have one new
    token each; the first sequence has the largest sizes."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n, total, out = case["tokens"], case["held"], []
    for b in range(case["seqs"]):
        full = b == 0 or case["op"] == "attend" and total == n
        new = n if full or n == 1 else rng.randint(max(1, n // 2), n)
        if case["op"] == "append":
            before = total if full else rng.randint(0, total)
        else:
            before = total - new if full else rng.randint((total - new) // 2, total - new)
        out.append((new, before))
    return out


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "logits":
        cells = case["rows"] * case["vocab"]
        more = case["rows"] * (4 * case["history"] + 8 * case["biases"] + (case["vocab"] / 8 if case["mask"] else 0) + 12)
        return {"bytes": 2 * size * cells + more, "flops": 4 * cells}
    runs = _ragged(case)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    new = sum(n for n, _ in runs)
    if case["op"] == "append":
        # q in and out, keys and values in, codes and scales out, the values that they stand for out
        table = 4 * case["rot"] * new
        return {"bytes": new * (2 * h * d * size + 2 * kv * d * size + 2 * kv * d * 0.625 + 2 * kv * d * size) + table,
                "flops": new * (3 * h * d + 10 * kv * d)}
    pairs = sum(n * b + n * (n + 1) // 2 for n, b in runs)
    return {"bytes": sum((n + b) * kv * d * 1.25 for n, b in runs) + 2 * new * h * d * size, "flops": 4 * d * h * pairs}


# ---- the cache's format in elementary operations -------------------------------------------------------------------
def _key_order(d, device):
    t, g, i = torch.meshgrid(torch.arange(4), torch.arange(d // 32), torch.arange(8), indexing="ij")
    return (32 * g + 8 * t + i).reshape(-1).to(device)


def _value_order(d, device):
    r, i = torch.meshgrid(torch.arange(8), torch.arange(d // 8), indexing="ij")
    return (16 * (i // 2) + 8 * (i % 2) + r).reshape(-1).to(device)


def _block_bytes(d):
    return 2 * 16 * (d // 2 + d // 8)


def _quantise(x):
    """x [..., d] f32 -> codes [..., d] uint8, (s, c) [..., d / 32, 2] f16, values [..., d] f32."""
    r = x.clamp(-LIMIT, LIMIT).unflatten(-1, (-1, 32))
    lo, hi = r.amin(-1), r.amax(-1)
    s = ((hi - lo) / 15.0).to(torch.bfloat16).to(torch.float16)
    c = (lo + 8.0 * s.float()).to(torch.float16)
    sf, cf = s.float().unsqueeze(-1), c.float().unsqueeze(-1)
    inverse = torch.where(sf > 0, 1.0 / sf, torch.zeros_like(sf))
    n = (torch.round((r - cf) * inverse) + 8.0).clamp(0.0, 15.0)
    values = (n - 8.0) * sf + cf
    return n.to(torch.uint8).flatten(-2), torch.stack([s, c], -1), values.flatten(-2)


def _packed_rows(x, order):
    """x [..., d] f32 -> code bytes [..., d / 2], scale bytes [..., d / 8], values."""
    codes, scales, values = _quantise(x)
    codes = codes[..., order]
    return codes[..., 0::2] | (codes[..., 1::2] << 4), scales.flatten(-2).view(torch.uint8), values


def _into_pages(pages, where, k, v):
    """Rows [n, kv_heads, d] f32 into the pages at `where` = (page [n], index in the page [n]); the values they are held as."""
    d = k.shape[-1]
    page, at = where
    block, row = at // 16, at % 16
    blocks = pages.view(pages.shape[0], pages.shape[1], pages.shape[2], -1)
    half, start = d // 2, 0
    held = []
    for x, order in ((k, _key_order(d, k.device)), (v, _value_order(d, k.device))):
        codes, scales, values = _packed_rows(x, order)
        for part in (codes, scales):
            width = part.shape[-1]
            rows = blocks[..., start:start + 16 * width].unflatten(-1, (16, width))
            rows[page, :, block, row] = part
            start += 16 * width
        held.append(values)
    return held


def _from_pages(blocks, d):
    """[..., block_bytes] -> keys, values [..., 16, d] f32."""
    out, start = [], 0
    for order in (_key_order(d, blocks.device), _value_order(d, blocks.device)):
        codes = blocks[..., start:start + 8 * d].unflatten(-1, (16, d // 2))
        start += 8 * d
        scales = blocks[..., start:start + 2 * d].contiguous().view(torch.float16).unflatten(-1, (16, d // 32, 2)).float()
        start += 2 * d
        n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., torch.argsort(order)].float().unflatten(-1, (-1, 32))
        out.append(((n - 8.0) * scales[..., 0:1] + scales[..., 1:2]).flatten(-2))
    return out


def _rotate(x, table, rotate, rot):
    """x [n, heads, d], table [n, rot / 2, 2] (cos, sin): the rotated rows, formed in 64 bits and rounded to 32."""
    if rotate == "none":
        return x.float()
    turned, rest = x[..., :rot].double(), x[..., rot:].float()
    c, s = table[:, None, :, 0].double(), table[:, None, :, 1].double()
    if rotate == "half":
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([y.float(), rest], -1)


# ---- inputs --------------------------------------------------------------------------------------------------------
def _rope(rot, positions):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return torch.stack([angle.cos(), angle.sin()], -1).float().cuda()


def _pool(case, runs, gen):
    """Empty pages for every sequence, in shuffled order as a pool that has been in use gives them out, and the table."""
    size = case["page"]
    longest = max(n + b for n, b in runs)
    width = (longest + size - 1) // size
    count = [(n + b + size - 1) // size for n, b in runs]
    order = torch.randperm(sum(count), generator=gen).int()
    table = torch.zeros(len(runs), width, dtype=torch.int32)
    at = 0
    for b, c in enumerate(count):
        table[b, :c] = order[at:at + c]
        at += c
    pages = torch.zeros(sum(count), case["kv_heads"], size // 16, _block_bytes(case["dim"]), dtype=torch.uint8, device="cuda")
    return pages, table.cuda()


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dtype):
        return torch.randn(*shape, generator=dev, device="cuda", dtype=torch.float32).to(dtype)

    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        state = dict(case=case, logits=(3.0 * torch.randn(rows, vocab, generator=dev, device="cuda")).to(dtype))
        # repeats are common in what has been said; short histories are padded with -1
        spoken = torch.randint(0, max(1, vocab // 3), (rows, case["history"]), generator=gen, dtype=torch.int32)
        length = torch.randint(0, case["history"] + 1, (rows, 1), generator=gen)
        state["history"] = torch.where(torch.arange(case["history"])[None] < length, spoken, -1).int().cuda()
        state["repetition"] = (1.0 + 0.5 * torch.rand(rows, generator=gen)).cuda()
        state["frequency"] = (0.3 * torch.rand(rows, generator=gen)).cuda()
        state["presence"] = (0.5 * torch.rand(rows, generator=gen)).cuda()
        state["bias_ids"] = state["bias_values"] = state["mask"] = None
        if case["biases"]:
            state["bias_ids"] = torch.randint(0, vocab, (rows, case["biases"]), generator=gen, dtype=torch.int32).cuda()
            state["bias_values"] = (4.0 * torch.randn(rows, case["biases"], generator=gen)).cuda()
        if case["mask"]:
            # a few dozen legal entries in a small vocabulary, a grammar's share in a large one
            share = min(0.5, 40.0 / vocab if vocab < 4096 else 0.25)
            bits = (torch.rand(rows, (vocab + 7) // 8, 8, generator=dev, device="cuda") < share).to(torch.uint8)
            state["mask"] = (bits << torch.arange(8, device="cuda", dtype=torch.uint8)).sum(-1).to(torch.uint8)
        return state

    runs = _ragged(case)
    new = [n for n, _ in runs]
    starts = [b for _, b in runs]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    pages, table = _pool(case, runs, gen)
    total = sum(new)
    cu = None if case["tokens"] == 1 else _ints([sum(new[:b]) for b in range(len(new) + 1)])
    state = dict(case=case, pages=pages, table=table, starts=_ints(starts), cu=cu, total=total, longest=max(new),
                 lengths=_ints([n + b for n, b in runs]), rope=None)
    state["seq"] = torch.repeat_interleave(torch.arange(len(new), device="cuda"), _ints(new).long())
    offset = torch.arange(total, device="cuda") - torch.repeat_interleave(
        _ints([sum(new[:b]) for b in range(len(new))]), _ints(new).long())
    state["offset"] = offset
    # the rows as a fused projection leaves them: queries, keys and values side by side
    fused = normal(total, (h + 2 * kv) * d).unflatten(-1, (h + 2 * kv, d))
    state["q"], state["k"], state["v"] = fused[:, :h], fused[:, h:h + kv], fused[:, h + kv:]
    # keys have channels that stand out
    fused[:, h:h + kv] += (0.8 * torch.randn(kv, d, generator=dev, device="cuda")).to(dtype)
    if case["op"] == "append":
        if case["rot"]:
            state["rope"] = _rope(case["rot"], max(n + b for n, b in runs))
        return state
    # the cache as earlier appends left it: pages are filled in pieces of a few million rows
    page_rows = kv * case["page"]
    for first in range(0, pages.shape[0], max(1, (1 << 25) // (page_rows * d))):
        part = pages[first:first + max(1, (1 << 25) // (page_rows * d))]
        n = part.shape[0] * case["page"]
        at = torch.arange(n, device="cuda")
        mean = 0.8 * torch.randn(kv, d, generator=dev, device="cuda")
        _into_pages(part, (at // case["page"], at % case["page"]), normal(n, kv, d, dtype=torch.float32) + mean,
                    normal(n, kv, d, dtype=torch.float32))
    state["q"] = state["q"].contiguous()
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------
def _plain_append(s):
    case = s["case"]
    index = s["starts"].long()[s["seq"]] + s["offset"]
    page = s["table"].long()[s["seq"], index // case["page"]]
    turn = s["rope"][index] if case["rot"] else None
    k = _rotate(s["k"], turn, case["rotate"], case["rot"])
    q = _rotate(s["q"], turn, case["rotate"], case["rot"])
    held = _into_pages(s["pages"], (page, index % case["page"]), k, s["v"].float())
    return q.to(s["q"].dtype), held[0].to(s["q"].dtype), held[1].to(s["q"].dtype)


def _plain_attend(s):
    case = s["case"]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    b, n, g = case["seqs"], s["longest"], h // kv
    blocks = s["pages"][s["table"].long()]                              # [b, pages, kv, blocks, bytes]
    keys, values = (x.permute(0, 2, 1, 3, 4, 5).flatten(2, 4) for x in _from_pages(blocks, d))     # [b, kv, held, d]
    q = torch.zeros(b, n, h, d, device="cuda")
    q[s["seq"], s["offset"]] = s["q"].float()
    q = q.unflatten(2, (kv, g)).permute(0, 2, 3, 1, 4).flatten(2, 3)     # [b, kv, g * n, d]
    scores = (q @ keys.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).unflatten(2, (g, n))
    count = s["lengths"].long()
    last = s["starts"].long()[:, None] + torch.arange(n, device="cuda")  # the last cache index that a token sees
    last = torch.minimum(last, count[:, None] - 1)
    hidden = torch.arange(keys.shape[2], device="cuda") > last[..., None]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    out = (scores.flatten(2, 3) @ values) / scores.sum(-1).flatten(2, 3)[..., None]
    out = out.unflatten(2, (g, n)).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [b, n, h, d]
    return out[s["seq"], s["offset"]].to(s["q"].dtype)


def _plain_logits(s):
    z = s["logits"].float()
    rows, vocab = z.shape
    said = s["history"].long()
    count = torch.zeros(rows, vocab + 1, device="cuda")
    count.scatter_add_(1, torch.where(said < 0, vocab, said), torch.ones_like(said, dtype=torch.float32))
    count = count[:, :vocab]
    rep = s["repetition"][:, None]
    less = torch.where(z > 0, z / rep, z * rep) - (s["frequency"][:, None] * count + s["presence"][:, None])
    z = torch.where(count > 0, less, z)
    if s["bias_ids"] is not None:
        ids = s["bias_ids"].long()
        order = torch.arange(1, ids.shape[1] + 1, device="cuda").expand_as(ids)
        latest = torch.zeros(rows, vocab, dtype=torch.int64, device="cuda").scatter_reduce_(1, ids, order, "amax")
        padded = torch.cat([torch.zeros(rows, 1, device="cuda"), s["bias_values"]], 1)
        z = z + padded.gather(1, latest)
    if s["mask"] is not None:
        bits = (s["mask"][..., None] >> torch.arange(8, device="cuda", dtype=torch.uint8)) & 1
        z = torch.where(bits.flatten(1)[:, :vocab] != 0, z, -math.inf)
    return z.to(s["logits"].dtype)


def run(s):
    case = s["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "logits": _plain_logits}[case["op"]](s)
    import chessrl_b200 as crl
    if case["op"] == "append":
        q = crl.kv4_append(s["pages"], s["k"], s["v"], s["table"], s["starts"], cu_tokens=s["cu"], q=s["q"], rope=s["rope"],
                           interleaved=case["rotate"] == "interleaved")
        k, v = crl.kv4_read(s["pages"], s["table"], s["starts"], s["total"], cu_tokens=s["cu"], dtype=s["q"].dtype)
        return q, k, v
    if case["op"] == "attend":
        return crl.kv4_attention(s["pages"], s["q"], s["table"], s["lengths"], cu_tokens=s["cu"], max_tokens=s["longest"])
    return crl.adjust_logits(s["logits"], history=s["history"], repetition=s["repetition"], frequency=s["frequency"],
                             presence=s["presence"], bias_ids=s["bias_ids"], bias_values=s["bias_values"], mask=s["mask"])


# ---- the definition in 64 bits -------------------------------------------------------------------------------------
def _held64(r):
    """What the cache stands for when it holds the f32 rows r: the format's own roundings, values in 64 bits."""
    x = r.double().clamp(-LIMIT, LIMIT).unflatten(-1, (-1, 32))
    low = x.min(-1).values
    s = ((x.max(-1).values - low).float() / 15.0).bfloat16().half().double()
    c = (low + 8.0 * s).float().half().double()
    n = ((x - c[..., None]).float() * (1.0 / s.float())[..., None]).nan_to_num(0.0).round().double().clamp(-8.0, 7.0)
    return (n * s[..., None] + c[..., None]).flatten(-2)


def _turned64(x, index, table, case):
    y = x.double().clone()
    for i in range(case["rot"] // 2):
        a, b = (i, i + case["rot"] // 2) if case["rotate"] == "half" else (2 * i, 2 * i + 1)
        cos, sin = table[index, i, 0].double()[:, None], table[index, i, 1].double()[:, None]
        y[..., a], y[..., b] = (x[..., a].double() * cos - x[..., b].double() * sin,
                                x[..., b].double() * cos + x[..., a].double() * sin)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        z = s["logits"].double()
        said = s["history"].long()
        times = torch.zeros(z.shape[0], z.shape[1] + 1, dtype=torch.float64, device="cuda")
        times = times.scatter_add(1, said % (z.shape[1] + 1), torch.ones_like(said).double())[:, :-1]   # -1 counts apart
        rep = s["repetition"].double()[:, None]
        z = torch.where(times > 0, torch.where(z > 0, z / rep, z * rep) - s["frequency"].double()[:, None] * times
                        - s["presence"].double()[:, None], z)
        if s["bias_ids"] is not None:
            add, every = torch.zeros_like(z), torch.arange(z.shape[0], device="cuda")
            for j in range(case["biases"]):
                add[every, s["bias_ids"][:, j].long()] = s["bias_values"][:, j].double()
            z = z + add
        if s["mask"] is not None:
            for bit in range(8):
                cells = z[:, bit::8]
                cells.masked_fill_((s["mask"][:, :cells.shape[1]] >> bit) % 2 == 0, -math.inf)
        return z
    if case["op"] == "append":
        index = s["starts"].long()[s["seq"]] + s["offset"]
        q, k = (_turned64(s[x], index, s["rope"], case) for x in "qk")
        return q, _held64(k.float()), _held64(s["v"].float())
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    out, at = torch.empty(s["total"], h, d, dtype=torch.float64, device="cuda"), 0
    kp, vp = torch.empty(d, dtype=torch.int64), torch.empty(d, dtype=torch.int64)
    for x in range(d):      # the nibble that holds dim x in a key's row and in a value's row
        kp[x] = (x % 32) // 8 * (d // 4) + x // 32 * 8 + x % 8
        vp[x] = x % 8 * (d // 8) + x // 16 * 2 + x // 8 % 2

    def rows(blocks, start, place):
        raw = blocks[..., start:start + 10 * d]
        place = place.cuda()
        byte = raw[..., :8 * d].reshape(*raw.shape[:-1], 16, d // 2)[..., place // 2]
        n = torch.where(place % 2 == 1, byte // 16, byte % 16).double()
        pair = raw[..., 8 * d:].contiguous().view(torch.float16).reshape(*raw.shape[:-1], 16, d // 32, 2).double()
        pair = pair.repeat_interleave(32, -2)
        return (n - 8) * pair[..., 0] + pair[..., 1]

    for b, (n, before) in enumerate(_ragged(case)):
        used = (n + before + case["page"] - 1) // case["page"]
        mine = s["pages"][s["table"][b, :used].long()].transpose(0, 1).flatten(1, 2)     # [kv, blocks, bytes]
        seen = torch.arange(n + before, device="cuda")[None] <= before + torch.arange(n, device="cuda")[:, None]
        for j in range(kv):
            keys = rows(mine[j], 0, kp).flatten(0, 1)[:n + before]
            values = rows(mine[j], 10 * d, vp).flatten(0, 1)[:n + before]
            q = s["q"][at:at + n, j * (h // kv):(j + 1) * (h // kv)].double().transpose(0, 1)
            p = torch.softmax((q @ keys.T / d ** 0.5).masked_fill(~seen, -math.inf), -1)
            out[at:at + n, j * (h // kv):(j + 1) * (h // kv)] = (p @ values).transpose(0, 1)
        at += n
    return out
