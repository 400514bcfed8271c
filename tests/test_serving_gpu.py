"""The decoder-serving operators against plain 64-bit implementations (oracle/serving.py)."""
import math
import random

import pytest
import torch

from oracle import serving as spec

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def crl(lib):
    import chessrl_b200
    return chessrl_b200


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool(crl, lengths, page, kv, hd, gen, spare=3):
    """Pages for sequences of these lengths in shuffled order with a few unused ones, filled with bytes that no row may
    see (codes 15, NaN steps and centres), and their table padded with a page number that does not exist."""
    count = [(n + page - 1) // page for n in lengths]
    pages = crl.kv4_pages(sum(count) + spare, page, kv, hd)
    pages.fill_(255)
    order = torch.randperm(sum(count) + spare, generator=gen).int()
    table = torch.full((len(lengths), max(1, max(count))), 1 << 30, dtype=torch.int32)
    at = 0
    for b, c in enumerate(count):
        table[b, :c] = order[at:at + c]
        at += c
    return pages, table.cuda()


def filled(crl, lengths, page, kv, hd, gen, key_scale=1.0, value_scale=1.0):
    """A pool whose sequences hold random rows, written by kv4_append (checked on its own)."""
    pages, table = pool(crl, lengths, page, kv, hd, gen)
    total = sum(lengths)
    if total:
        k = (key_scale * (torch.randn(total, kv, hd, generator=gen) + 0.5 * torch.randn(kv, hd, generator=gen))).half().cuda()
        v = (value_scale * torch.randn(total, kv, hd, generator=gen)).half().cuda()
        cu = ints([sum(lengths[:b]) for b in range(len(lengths) + 1)])
        crl.kv4_append(pages, k, v, table, ints([0] * len(lengths)), cu_tokens=cu)
    return pages, table


# ---- append and read ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,kv,heads,page,rot,interleaved,runs", [
    (64, 12, 12, 16, 0, False, [(1, 69)]),
    (64, 12, 12, 64, 64, False, [(1, 5), (1, 0), (1, 63), (1, 64), (1, 200)]),
    (128, 2, 8, 48, 64, True, [(37, 11), (1, 0), (16, 16), (100, 47)]),
    (32, 3, 6, 32, 8, False, [(5, 0), (33, 31)]),
    (32, 1, 7, 128, 32, True, [(130, 3)]),
    (128, 1, 2, 16, 6, False, [(3, 15), (2, 1)]),
    (64, 5, 5, 16, 10, True, [(20, 0)]),
    (64, 2, 6, 16, 32, False, [(21, 5), (1, 0)]),
    (32, 2, 4, 16, 16, True, [(9, 30), (14, 0)]),
    (128, 1, 3, 32, 64, False, [(40, 7)]),
])
def test_append_holds_the_defined_values(crl, dtype, hd, kv, heads, page, rot, interleaved, runs):
    gen = torch.Generator().manual_seed(hd + page + rot)
    new, before = [n for n, _ in runs], [b for _, b in runs]
    total = sum(new)
    pages, table = pool(crl, [n + b for n, b in runs], page, kv, hd, gen)
    fused = torch.randn(total, (heads + 2 * kv) * hd + 8, generator=gen).to(dtype)[:, :(heads + 2 * kv) * hd]
    fused = fused.cuda().unflatten(-1, (heads + 2 * kv, hd))
    q, k, v = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
    rope = crl.rope_table(rot, max(n + b for n, b in runs)) if rot else None
    cu = None if all(n == 1 for n in new) else ints([sum(new[:b]) for b in range(len(new) + 1)])
    untouched = pages.clone()
    status = ints([0])
    got = crl.kv4_append(pages, k, v, table, ints(before), cu_tokens=cu, q=q, rope=rope, interleaved=interleaved, status=status)
    kh, vh = crl.kv4_read(pages, table, ints(before), total, cu_tokens=cu, dtype=dtype, status=status)
    assert int(status[0]) == 0
    position = torch.tensor([b + j for n, b in runs for j in range(n)])
    turn = lambda x: spec.rotated(x.cpu(), position, rope.cpu(), interleaved) if rot else x.cpu().float()  # noqa: E731
    turned = turn(k)
    # values and queries are defined up to the last rounding: they are equal
    assert torch.equal(got.cpu(), turn(q).to(dtype))
    assert torch.equal(kh.cpu(), spec.held_rows(turned)[3].float().to(dtype))
    assert torch.equal(vh.cpu(), spec.held_rows(v.cpu().float())[3].float().to(dtype))
    # the bytes are those of the documented layout, and nothing else was written
    expect = untouched.cpu()
    for kind, x, start in (("k", turned, 0), ("v", v.cpu().float(), 10 * hd)):
        codes, s, c, _ = spec.held_rows(x)
        place = torch.tensor([spec.nibble_of(kind, d, hd) for d in range(hd)])
        flat = torch.empty_like(codes)
        flat[..., place] = codes
        rows = (flat[..., 0::2] | flat[..., 1::2] << 4).to(torch.uint8)
        scales = torch.stack([s, c], -1).half().flatten(-2).view(torch.uint8)
        row = 0
        for b, (n, held) in enumerate(runs):
            for i in range(held, held + n):
                block = expect[int(table[b, i // page]), :, i % page // 16]
                lo = start + (i % 16) * (hd // 2)
                block[:, lo:lo + hd // 2] = rows[row]
                lo = start + 8 * hd + (i % 16) * (hd // 8)
                block[:, lo:lo + hd // 8] = scales[row]
                row += 1
    assert torch.equal(pages.cpu(), expect)


def test_append_of_special_values(crl):
    """Constant groups, zeros, infinities, NaN, ranges that underflow the step and the largest finite ones."""
    rows = torch.randn(12, 1, 64, generator=torch.Generator().manual_seed(3))
    rows[0] = 0.0
    rows[1] = 1.5
    rows[2, 0, 5] = math.inf
    rows[3, 0, 40] = -math.inf
    rows[4, 0, 33] = math.nan
    rows[5] = 6e-8
    rows[5, 0, :3] = 0.0
    rows[6] *= 1e-6
    rows[7] = 65504.0
    rows[7, 0, ::2] = -65504.0
    rows[8] = 65504.0
    rows[9] = -0.0
    rows[10] *= 2e4
    x = rows.half()
    pages, table = pool(crl, [12], 16, 1, 64, torch.Generator().manual_seed(1))
    crl.kv4_append(pages, x.cuda(), x.cuda(), table, ints([0]), cu_tokens=ints([0, 12]))
    k, v = crl.kv4_read(pages, table, ints([0]), 12, cu_tokens=ints([0, 12]))
    want = spec.held_rows(x.float())[3].float().half()
    for got in (k.cpu(), v.cpu()):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    assert torch.isfinite(want[2]).all() and torch.isnan(want[4, 0, 32:]).all() and torch.isfinite(want[4, 0, :32]).all()


def test_rows_behind_the_last_sequence_and_lost_indices(crl):
    """A padded batch: rows behind cu_tokens' end are not appended and their queries not written; an index without a page
    and a position past the rotation table are skipped and reported."""
    gen = torch.Generator().manual_seed(5)
    pages, table = pool(crl, [20, 3], 16, 2, 32, gen)
    before = pages.clone()
    k = torch.randn(9, 2, 32, generator=gen).half().cuda()
    status = ints([0])
    crl.kv4_append(pages, k, k, table, ints([0, 0]), cu_tokens=ints([0, 4, 6]), status=status)
    held, _ = crl.kv4_read(pages, table, ints([0, 0]), 9, cu_tokens=ints([0, 4, 6]))
    assert int(status[0]) == 0 and (held[6:] == 0).all() and (held[:6] != 0).any()
    changed = (pages != before).any(-1).any(1).nonzero()
    assert {(int(p), int(b)) for p, b in changed} == {(int(table[0, 0]), 0), (int(table[1, 0]), 0)}
    for starts, code in (([40, 0], 121), ([0, 16], 121), ([-1, 0], 121)):
        status = ints([0])
        after = pages.clone()
        crl.kv4_append(pages, k[:2], k[:2], table, ints(starts), status=status)
        assert int(status[0]) == code
        lost = 0 if starts[0] else 1
        kept, _ = crl.kv4_read(pages, table, ints(starts), 2, dtype=F16)
        assert (kept[lost] == 0).all()
        pages.copy_(after)
    status = ints([0])
    crl.kv4_append(pages, k[:2], k[:2], table, ints([17, 2]), rope=crl.rope_table(32, 10), status=status)
    assert int(status[0]) == 123


def test_append_with_empty_sequences_and_shared_rows(crl):
    """Sequences without new tokens among others, one row of keys for all heads (stride 0), more sequences than tokens."""
    gen = torch.Generator().manual_seed(16)
    new, before = [0, 3, 0, 0, 2, 0], [4, 0, 0, 9, 14, 1]
    pages, table = pool(crl, [n + b for n, b in zip(new, before)], 16, 3, 32, gen)
    cu = ints([0, 0, 3, 3, 3, 5, 5])
    k = torch.randn(5, 1, 32, generator=gen).half().cuda().expand(5, 3, 32)
    crl.kv4_append(pages, k, k, table, ints(before), cu_tokens=cu)
    kh, vh = crl.kv4_read(pages, table, ints(before), 5, cu_tokens=cu)
    want = spec.held_rows(k.cpu().float())[3].float().half()
    assert torch.equal(kh.cpu(), want) and torch.equal(vh.cpu(), want)


# ---- attention ------------------------------------------------------------------------------------------------------
def attend_case(crl, dtype, hd, heads, kv, page, runs, seed=0, key_scale=1.0, value_scale=1.0, q_scale=1.0, scale=None, order=None):
    gen = torch.Generator().manual_seed(seed)
    lengths = [n for _, n in runs]
    pages, table = filled(crl, lengths, page, kv, hd, gen, key_scale, value_scale)
    total = sum(n for n, _ in runs)
    q = (q_scale * torch.randn(total, heads, hd, generator=gen)).to(dtype).cuda()
    single = all(n == 1 for n, _ in runs)
    cu = None if single else ints([sum(n for n, _ in runs[:b]) for b in range(len(runs) + 1)])
    status = ints([0])
    got = crl.kv4_attention(pages, q, table, ints(lengths), cu_tokens=cu, max_tokens=max(n for n, _ in runs), scale=scale, status=status)
    assert int(status[0]) == 0
    check_attention(got, q, pages, table, runs, scale)
    return got


def check_attention(got, q, pages, table, runs, scale=None):
    """Every row against 64 bits. A row's error, relative to the largest value that the weights reach, is the rounding of
    each weight to f16 (half a step of a weight p s that is at most 2 to the running exponent; normal numbers), of the
    result (half a step), and fp32's part: scores are sums of up to 128 products of q <= 2 (of its own row's scale) with
    codes, 2^-24 each, times up to |score| - bounded by 2^-11 |S| here with |S| the row's largest score times 2^-8."""
    hd, kv = q.shape[2], pages.shape[1]
    g = q.shape[1] // kv
    scale = hd ** -0.5 if scale is None else scale
    cpu_pages, cpu_table, at = pages.cpu(), table.cpu(), 0
    dtype = q.dtype
    for b, (n, length) in enumerate(runs):
        for h in range(kv):
            k, v = spec.cache_rows(cpu_pages, cpu_table[b], length, h)
            for j in range(g):
                rows = q[at:at + n, h * g + j].cpu().double()
                want = spec.attention(rows, k, v, length - n, scale)
                mine = got[at:at + n, h * g + j].cpu().double()
                if length == 0 or n == 0:
                    assert (mine == 0).all()
                    continue
                top = v.abs().max()
                biggest = (scale * rows @ k.T).abs().max()
                # p rounded once: each term within half an f16 step of itself, so the sum within that of the largest |v - c|
                bound = top * (half_step(F16) * 2 + 2.0 ** -16 * (1 + biggest)) + want.abs() * half_step(dtype) + 1e-7
                assert ((mine - want).abs() <= bound).all(), (b, h, j, (mine - want).abs().max(), bound.min())
        at += n


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("heads,kv", [(3, 3), (8, 2), (7, 1), (24, 2)])
def test_attention_of_single_tokens(crl, dtype, hd, heads, kv):
    runs = [(1, n) for n in (1, 2, 15, 16, 17, 63, 64, 65, 100, 0, 513)]
    attend_case(crl, dtype, hd, heads, kv, 16, runs, seed=hd + heads)


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128])
def test_attention_over_page_sizes_and_splits(crl, page):
    """Long enough for the axis of keys to be split over a cluster; pages that end inside a tile."""
    attend_case(crl, F16, 64, 4, 2, page, [(1, 5000), (1, 4097), (1, 33), (1, 0)], seed=page)


@pytest.mark.parametrize("dtype,hd,heads,kv,runs", [
    (F16, 64, 12, 12, [(5, 69), (1, 64), (3, 3), (8, 130)]),
    (BF16, 128, 8, 2, [(2, 300), (4, 4), (1, 1), (3, 1000)]),
    (F16, 32, 6, 1, [(5, 97), (2, 2), (5, 5), (4, 64)]),
    (F16, 128, 4, 4, [(17, 40), (33, 33), (1, 90)]),
    (BF16, 64, 4, 4, [(64, 64), (64, 64), (40, 77)]),
    (F16, 64, 6, 2, [(70, 210), (0, 5), (128, 128)]),
    (BF16, 32, 8, 8, [(200, 333)]),
    (F16, 128, 8, 2, [(150, 150), (65, 1100)]),
    (F16, 128, 4, 1, [(700, 1500), (1, 1), (300, 333)]),
    (BF16, 64, 3, 1, [(900, 901), (0, 70), (257, 600)]),
    (F16, 32, 4, 2, [(500, 640), (129, 129)]),
])
def test_attention_of_runs_and_prompts(crl, dtype, hd, heads, kv, runs):
    attend_case(crl, dtype, hd, heads, kv, 32, runs, seed=hd + heads + len(runs))


def test_rows_that_see_nothing_are_zero(crl):
    """A run longer than what the cache holds: its first rows stand before the first key."""
    gen = torch.Generator().manual_seed(2)
    for n, length in ((4, 2), (40, 10), (3, 0), (400, 150)):
        pages, table = filled(crl, [max(length, 1)], 16, 2, 64, gen)
        q = torch.randn(n, 4, 64, generator=gen).half().cuda()
        out = crl.kv4_attention(pages, q, table, ints([length]), cu_tokens=ints([0, n]), max_tokens=n)
        assert (out[:n - length] == 0).all()
        if length:
            check_attention(out, q, pages, table, [(n, length)])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_of_extreme_scales(crl, dtype):
    """Tiny values (steps below f16's normal range), tiny queries, scores that leave one key, a scale of its own."""
    attend_case(crl, dtype, 64, 4, 2, 16, [(1, 200), (1, 70)], seed=1, value_scale=1e-4)
    attend_case(crl, dtype, 64, 4, 2, 16, [(1, 200), (20, 70)], seed=2, q_scale=1e-3)
    attend_case(crl, dtype, 32, 4, 2, 16, [(1, 200), (1, 3)], seed=3, key_scale=30.0)
    attend_case(crl, dtype, 128, 4, 2, 16, [(1, 200), (40, 63)], seed=4, scale=0.0)
    attend_case(crl, dtype, 64, 4, 2, 16, [(2, 200), (1, 1)], seed=5, scale=-0.3)
    attend_case(crl, dtype, 64, 4, 2, 16, [(200, 400)], seed=6, value_scale=1e-4)
    attend_case(crl, dtype, 128, 4, 2, 16, [(200, 300)], seed=7, q_scale=1e-3, scale=-0.2)
    attend_case(crl, dtype, 32, 4, 2, 16, [(200, 300)], seed=8, key_scale=30.0)
    attend_case(crl, dtype, 64, 4, 2, 16, [(150, 300)], seed=9, scale=0.0)


def test_values_growing_along_the_sequence(crl):
    """The running exponent of the values' steps has to rise tile after tile."""
    gen = torch.Generator().manual_seed(9)
    for n in (1, 40, 300):
        pages, table = pool(crl, [700], 64, 1, 64, gen)
        k = torch.randn(700, 1, 64, generator=gen).half().cuda()
        v = (torch.randn(700, 1, 64, generator=gen) * torch.linspace(-7, 9, 700).exp2()[:, None, None]).half().cuda()
        crl.kv4_append(pages, k, v, table, ints([0]), cu_tokens=ints([0, 700]))
        q = torch.randn(n, 2, 64, generator=gen).half().cuda()
        out = crl.kv4_attention(pages, q, table, ints([700]), cu_tokens=ints([0, n]), max_tokens=n)
        check_attention(out, q, pages, table, [(n, 700)])


@pytest.mark.parametrize("n", [1, 4, 40, 150])
def test_hidden_rows_do_not_leak(crl, n):
    """NaN in later tokens of the run and in the rest of the page (the pool is filled with NaN steps) stays out of the rows
    that do not see it; in what a row does see it shows."""
    gen = torch.Generator().manual_seed(4)
    held = max(50, n + 9)
    pages, table = pool(crl, [held], 32, 2, 64, gen)
    k = torch.randn(held, 2, 64, generator=gen).half()
    k[held - 1, 0] = math.nan
    v = torch.randn(held, 2, 64, generator=gen).half()
    v[held - 1, 0, 40] = math.nan
    crl.kv4_append(pages, k.cuda(), v.cuda(), table, ints([0]), cu_tokens=ints([0, held]))
    q = torch.randn(n, 2, 64, generator=gen).half().cuda()
    out = crl.kv4_attention(pages, q, table, ints([held]), cu_tokens=ints([0, n]), max_tokens=n)
    assert torch.isfinite(out[:n - 1]).all() and torch.isfinite(out[:, 1]).all()
    assert torch.isnan(out[n - 1, 0]).all()
    out = crl.kv4_attention(pages, q, table, ints([held - 1]), cu_tokens=ints([0, n]), max_tokens=n)
    check_attention(out, q, pages, table, [(n, held - 1)])


@pytest.mark.parametrize("n", [2, 40, 150])
def test_a_nan_value_reaches_its_group_of_the_rows_that_see_it(crl, n):
    gen = torch.Generator().manual_seed(8)
    held, hit = n + 20, 20 + n // 2
    pages, table = pool(crl, [held], 16, 1, 64, gen)
    k, v = torch.randn(held, 1, 64, generator=gen).half(), torch.randn(held, 1, 64, generator=gen).half()
    v[hit, 0, 40] = math.nan
    crl.kv4_append(pages, k.cuda(), v.cuda(), table, ints([0]), cu_tokens=ints([0, held]))
    q = torch.randn(n, 2, 64, generator=gen).half().cuda()
    out = crl.kv4_attention(pages, q, table, ints([held]), cu_tokens=ints([0, n]), max_tokens=n)
    sees = hit - 20      # the first row that does
    assert torch.isfinite(out[:sees]).all() and torch.isfinite(out[:, :, :32]).all() and torch.isnan(out[sees:, :, 32:]).all()


def test_attention_with_strides_and_padding(crl):
    """Queries inside fused rows that are not 16-byte aligned, an output inside a larger tensor, rows behind the last
    sequence left as they were."""
    gen = torch.Generator().manual_seed(6)
    runs = [(3, 40), (2, 18), (1, 7)]
    pages, table = filled(crl, [n for _, n in runs], 16, 2, 64, gen)
    cu = ints([0, 3, 5, 6])
    wide = torch.randn(9, 4 * 64 + 3, generator=gen).half().cuda()
    q = wide[:, 3:].unflatten(-1, (4, 64))
    out = torch.full((9, 5, 72), 7.0, dtype=F16, device="cuda")
    view = out[:, 1:, 3:67]
    back = crl.kv4_attention(pages, q, table, ints([n for _, n in runs]), cu_tokens=cu, max_tokens=3, out=view)
    assert back.data_ptr() == view.data_ptr()
    check_attention(view[:6], q[:6].contiguous(), pages, table, runs)
    assert (out[6:] == 7).all() and (out[:, 0] == 7).all() and (out[:, :, :3] == 7).all() and (out[:, :, 67:] == 7).all()
    same = crl.kv4_attention(pages, q[:6].contiguous(), table, ints([n for _, n in runs]), cu_tokens=cu, max_tokens=3)
    assert torch.equal(same, view[:6])


def test_attention_reports_what_it_skips(crl):
    gen = torch.Generator().manual_seed(7)
    pages, table = filled(crl, [40, 20], 16, 1, 64, gen)
    q = torch.randn(2, 2, 64, generator=gen).half().cuda()
    good = crl.kv4_attention(pages, q, table, ints([40, 20]))
    for bad in (-1, pages.shape[0]):
        broken = table.clone()
        broken[0, 1] = bad
        status = ints([0])
        out = crl.kv4_attention(pages, q, broken, ints([40, 20]), status=status)
        assert int(status[0]) == 121 and torch.isfinite(out).all() and torch.equal(out[1], good[1])
    status = ints([0])
    crl.kv4_attention(pages, q, table, ints([1000, 20]), status=status)
    assert int(status[0]) == 121
    status = ints([0])
    out = torch.zeros_like(q)
    crl.kv4_attention(pages, q, table, ints([40, 20]), cu_tokens=ints([0, 2, 2]), max_tokens=1, out=out, status=status)
    assert int(status[0]) == 122
    status = ints([0])
    crl.kv4_attention(pages, q, table, ints([40, 20]), cu_tokens=ints([0, 1, 9]), max_tokens=8, out=out, status=status)
    assert int(status[0]) == 122


def test_a_run_cut_short_keeps_its_positions(crl):
    """max_tokens below a sequence's new tokens: the first max_tokens of them are computed at their own positions, the rest
    of out is left alone, and the call reports it."""
    gen = torch.Generator().manual_seed(12)
    for n, most in ((6, 3), (40, 25), (500, 300)):
        pages, table = filled(crl, [n + 30], 32, 2, 64, gen)
        q = torch.randn(n, 4, 64, generator=gen).half().cuda()
        whole = crl.kv4_attention(pages, q, table, ints([n + 30]), cu_tokens=ints([0, n]), max_tokens=n)
        status, out = ints([0]), torch.full_like(q, 5.0)
        crl.kv4_attention(pages, q, table, ints([n + 30]), cu_tokens=ints([0, n]), max_tokens=most, out=out, status=status)
        assert int(status[0]) == 122 and (out[most:] == 5).all()
        check_attention(out[:most], q[:most].contiguous(), pages, table, [(most, n + 30 - (n - most))])
        assert (out[:most].float() - whole[:most].float()).abs().max() < 4e-3      # another kernel or tile, same rows


@pytest.mark.parametrize("n", [1, 20, 300])
def test_many_rows_with_odd_strides(crl, n):
    """The other kernels with rows that are not 16-byte aligned, transposed heads, and a table inside a wider one."""
    gen = torch.Generator().manual_seed(13)
    lengths = [n + 40, n]
    pages, table = filled(crl, lengths, 48, 2, 64, gen)
    wide = torch.full((2, table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = table
    total = 2 * n
    q = torch.randn(total, 6 * 64 + 1, generator=gen).half().cuda()[:, 1:].unflatten(-1, (6, 64))
    cu = ints([0, n, total])
    out = torch.zeros(6, total, 64, dtype=F16, device="cuda").transpose(0, 1)
    crl.kv4_attention(pages, q, wide[:, 2:2 + table.shape[1]], ints(lengths), cu_tokens=cu, max_tokens=n, out=out)
    check_attention(out, q.contiguous(), pages, table, [(n, lengths[0]), (n, n)])
    odd = torch.zeros(total, 6 * 64 + 1, dtype=F16, device="cuda")[:, 1:].unflatten(-1, (6, 64))
    crl.kv4_attention(pages, q.contiguous(), table, ints(lengths), cu_tokens=cu, max_tokens=n, out=odd)
    assert torch.equal(odd, out)
    with pytest.raises(ValueError, match="overlap"):
        crl.kv4_attention(pages, q, table, ints(lengths), cu_tokens=cu, max_tokens=n, out=out[:, :1].expand(total, 6, 64))


def test_a_pool_beyond_four_gigabytes(crl):
    """Offsets that pass 32 bits: pages at the end of a pool of 4.6 GB, and none of those whose offsets agree in 32 bits."""
    size, kv, hd = 128, 8, 128
    per_page = kv * size // 16 * 20 * hd
    pages = crl.kv4_pages((1 << 32) // per_page + 2000, size, kv, hd)
    gen = torch.Generator().manual_seed(14)
    last = pages.shape[0] - 1
    table = ints([last, last - 1500]).view(1, 2)
    k, v = (torch.randn(200, kv, hd, generator=gen).half().cuda() for _ in range(2))
    crl.kv4_append(pages, k, v, table, ints([0]), cu_tokens=ints([0, 200]))
    kh, _ = crl.kv4_read(pages, table, ints([0]), 200, cu_tokens=ints([0, 200]))
    assert torch.equal(kh.cpu(), spec.held_rows(k.cpu().float())[3].float().half())
    assert not pages[:2000].any() and pages[last].any()
    small, its = torch.stack([pages[last], pages[last - 1500]]), ints([0, 1]).view(1, 2)
    for n in (1, 30, 200):
        q = torch.randn(n, 8, hd, generator=gen).half().cuda()
        far = crl.kv4_attention(pages, q, table, ints([200]), cu_tokens=ints([0, n]), max_tokens=n)
        assert torch.equal(far, crl.kv4_attention(small, q, its, ints([200]), cu_tokens=ints([0, n]), max_tokens=n))


def test_sequences_that_share_a_prefix(crl):
    """Pages of a common prefix stand in several tables; each sequence goes on in its own."""
    gen = torch.Generator().manual_seed(15)
    pages, table = filled(crl, [32, 20, 20], 16, 2, 32, gen)
    both = torch.stack([torch.cat([table[0], table[1]]), torch.cat([table[0], table[2]])]).contiguous()
    runs = [(1, 52), (1, 47)]
    q = torch.randn(2, 4, 32, generator=gen).half().cuda()
    out = crl.kv4_attention(pages, q, both, ints([52, 47]))
    check_attention(out, q, pages, both, runs)


def test_first_calls_of_a_process_can_be_captured(crl):
    """Nothing has to be called before a graph is captured."""
    import subprocess
    import sys
    code = """
import torch, chessrl_b200 as crl
torch.zeros(1, device="cuda")
pages = crl.kv4_pages(8, 16, 2, 64)
table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
one, k = torch.tensor([3, 20], dtype=torch.int32, device="cuda"), torch.randn(2, 2, 64, device="cuda").half()
rope, cu = crl.rope_table(64, 64), torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
big, cub = torch.randn(400, 4, 64, device="cuda").half(), torch.tensor([0, 200, 400], dtype=torch.int32, device="cuda")
g = torch.cuda.CUDAGraph()
def work():
    q = crl.kv4_append(pages, k, k, table, one, q=k, rope=rope)
    a = crl.kv4_attention(pages, q, table, one + 1)
    b = crl.kv4_attention(pages, q.repeat(1, 5, 1), table, one + 1)
    c = crl.kv4_attention(pages, big, table, one + 1, cu_tokens=cub, max_tokens=200)
    return a, b, c, crl.adjust_logits(a.flatten(1), history=table), crl.kv4_read(pages, table, one, 2)[0]
with torch.cuda.graph(g):
    captured = work()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(x, y) for x, y in zip(captured, work()))
print("captured")
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root, timeout=300)
    assert "captured" in out.stdout, out.stderr[-2000:]


@pytest.mark.parametrize("n", [1, 6, 30, 300])
def test_keys_of_a_missing_page_are_left_out(crl, n):
    """A page number outside the pool in the middle of a sequence: its tokens are as if they were not there, in every
    kernel, and the call says so."""
    gen = torch.Generator().manual_seed(18)
    held = n + 200
    for page in (16, 64):
        pages, table = filled(crl, [held], page, 2, 64, gen)
        broken = table.clone()
        broken[0, 1] = pages.shape[0] + 3
        q = torch.randn(n, 4, 64, generator=gen).half().cuda()
        status = ints([0])
        out = crl.kv4_attention(pages, q, broken, ints([held]), cu_tokens=ints([0, n]), max_tokens=n, status=status)
        assert int(status[0]) == 121
        for h in range(4):
            k, v = spec.cache_rows(pages.cpu(), table[0].cpu(), held, h // 2)
            keep = torch.ones(held, dtype=torch.bool)
            keep[page:2 * page] = False
            score = (q[:, h].cpu().double() @ k.T / 8.0)
            seen = keep[None] & (torch.arange(held)[None] <= held - n + torch.arange(n)[:, None])
            want = torch.softmax(score.masked_fill(~seen, -math.inf), 1) @ v
            # as in check_attention
            bound = v.abs().max() * (half_step(F16) * 2 + 2.0 ** -16 * (1 + score.abs().max())) + want.abs() * half_step(F16) + 1e-7
            assert ((out[:, h].cpu().double() - want).abs() <= bound).all()


# ---- logits ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, F16, BF16])
@pytest.mark.parametrize("rows,vocab,said,biases", [(1, 1929, 40, 4), (5, 1929, 0, 0), (3, 7, 20, 9), (2, 1, 3, 1), (4, 8193, 300, 70),
                                                    (3, 50304, 1000, 33), (2, 4096, 1, 0)])
def test_logits_against_64_bits(crl, dtype, rows, vocab, said, biases):
    gen = torch.Generator().manual_seed(rows * vocab + said)
    logits = (4 * torch.randn(rows, vocab, generator=gen)).to(dtype)
    history = torch.randint(-2, min(vocab + 3, 60), (rows, said), generator=gen).int() if said else None
    rep, freq, pres = 1 + torch.rand(rows, generator=gen), torch.rand(rows, generator=gen), torch.rand(rows, generator=gen)
    ids = torch.randint(-1, min(vocab + 2, 90), (rows, biases), generator=gen).int() if biases else None
    values = 5 * torch.randn(rows, biases, generator=gen) if biases else None
    mask = torch.randint(0, 256, (3, (vocab + 7) // 8 + 1), generator=gen).to(torch.uint8)
    pick = torch.randint(-1, 3, (rows,), generator=gen).int()
    kw = dict(history=history, repetition=rep, frequency=freq, presence=pres, bias_ids=ids, bias_values=values, mask=mask, mask_rows=pick)
    want = spec.adjust(logits, **kw)
    gpu = {k: v.cuda() if v is not None else None for k, v in kw.items()}
    got = crl.adjust_logits(logits.cuda(), **gpu).cpu()
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)) and (got[~fine] == -math.inf).all()
    # five fp32 operations on numbers of up to the size of the largest operand, one rounding to the type
    big = logits.double().abs() * 2 + 2 + 1000 + (20 if biases else 0)
    touched = (want - logits.double()) != 0
    bound = want.abs() * half_step(dtype) + torch.where(touched, big * 5 * half_step(torch.float32), torch.zeros_like(want))
    assert ((got.double() - want).abs()[fine] <= bound[fine]).all()
    # in place, and in rows of a wider tensor that are not 16-byte aligned
    own = logits.cuda()
    assert crl.adjust_logits(own, out=own, **gpu) is own and torch.equal(own.cpu(), got)
    wide = torch.full((rows, vocab + 5), 3.0, dtype=dtype, device="cuda")
    wide[:, 1:vocab + 1] = logits.cuda()
    crl.adjust_logits(wide[:, 1:vocab + 1], out=wide[:, 1:vocab + 1], **gpu)
    assert torch.equal(wide[:, 1:vocab + 1].cpu(), got) and (wide[:, 0] == 3).all() and (wide[:, vocab + 1:] == 3).all()
    other = torch.full((rows, vocab + 4), 3.0, dtype=dtype, device="cuda")
    crl.adjust_logits(logits.cuda(), out=other[:, 3:vocab + 3], **gpu)
    assert torch.equal(other[:, 3:vocab + 3].cpu(), got) and (other[:, :3] == 3).all() and (other[:, vocab + 3:] == 3).all()


def test_logits_masks_that_leave_nothing_and_special_values(crl):
    logits = torch.tensor([[1.0, math.nan, math.inf, -math.inf, -3.0, 0.0, 65504.0, -65504.0, 2.0]]).repeat(3, 1)
    mask = torch.tensor([[0, 0], [255, 1], [0b10101101, 0]], dtype=torch.uint8).cuda()
    for dtype in (torch.float32, F16):
        x = logits.to(dtype).cuda()
        out = crl.adjust_logits(x, mask=mask)
        assert (out[0] == -math.inf).all()
        assert torch.equal(out[1].nan_to_num(9.0), x[1].nan_to_num(9.0))
        assert torch.equal(out[2] == -math.inf, torch.tensor([0, 1, 0, 1, 1, 0, 1, 0, 1]).bool().cuda())
        low = crl.adjust_logits(x, mask=mask, masked_value=torch.finfo(dtype).min)
        assert (low[0] == torch.finfo(dtype).min).all()
        # penalties on infinities, NaN and the type's lowest value: said tokens only
        said = torch.arange(9).int().cuda()[None].repeat(3, 1)
        out = crl.adjust_logits(x, history=said, repetition=torch.full((3,), 2.0, device="cuda"))
        want = torch.where(x.float() > 0, x.float() / 2, x.float() * 2).to(dtype)
        assert torch.equal(out.nan_to_num(9.0), want.nan_to_num(9.0))
    assert torch.equal(crl.adjust_logits(x).nan_to_num(9.0), x.nan_to_num(9.0))
    status = ints([0])
    out = crl.adjust_logits(x, mask=mask, mask_rows=ints([-1, 1, 3]), status=status)
    assert int(status[0]) == 131 and torch.equal(out[2].nan_to_num(9.0), x[2].nan_to_num(9.0))


# ---- together, streams, graphs --------------------------------------------------------------------------------------
def decode_steps(crl, dtype, steps, graph):
    """A tiny decoder: prompts of several lengths, then single tokens, every layer's cache in 4 bits; returns the last
    logits. With `graph` the step is captured once and replayed."""
    gen = torch.Generator().manual_seed(11)
    d, heads, kv, hd, vocab, layers = 128, 4, 2, 32, 1929, 2
    w = lambda *s: (torch.randn(*s, generator=gen) * s[-1] ** -0.5).to(dtype).cuda()  # noqa: E731
    embed, blocks = w(vocab, d) * 4, [(w((heads + 2 * kv) * hd, d), w(d, heads * hd)) for _ in range(layers)]
    prompts = [17, 64, 5]
    b, size = len(prompts), 16
    width = (max(prompts) + steps + size - 1) // size
    pages = [crl.kv4_pages(b * width, size, kv, hd) for _ in range(layers)]
    table = torch.randperm(b * width, generator=gen).int().view(b, width).cuda()
    rope = crl.rope_table(hd, width * size)
    tokens = torch.randint(0, vocab, (b, max(prompts) + steps), generator=gen).int().cuda()
    legal = torch.randint(0, 256, (b, (vocab + 7) // 8), generator=gen).to(torch.uint8).cuda()
    penalty = torch.full((b,), 1.3, device="cuda")

    def model(ids, starts, lengths, cu, most):
        x = embed[ids.long()]
        for (qkv, proj), pool in zip(blocks, pages):
            y = (torch.nn.functional.layer_norm(x.float(), (d,)).to(dtype) @ qkv.T).unflatten(-1, (heads + 2 * kv, hd))
            q = crl.kv4_append(pool, y[:, heads:heads + kv], y[:, heads + kv:], table, starts, cu_tokens=cu, q=y[:, :heads], rope=rope)
            x = x + crl.kv4_attention(pool, q, table, lengths, cu_tokens=cu, max_tokens=most).flatten(1) @ proj.T
        return x @ embed.T

    zero, held = ints([0] * b), ints(prompts)
    cu = ints([0, prompts[0], prompts[0] + prompts[1], sum(prompts)])
    ids = torch.cat([tokens[i, :n] for i, n in enumerate(prompts)])
    logits = model(ids, zero, held, cu, max(prompts))[cu[1:].long() - 1]
    said = torch.full((b, max(prompts) + steps), -1, dtype=torch.int32, device="cuda")
    for i, n in enumerate(prompts):
        said[i, :n] = tokens[i, :n]
    state = dict(held=held.clone(), logits=crl.adjust_logits(logits, history=said, repetition=penalty, mask=legal))

    def step():
        nxt = state["logits"].float().argmax(-1).int()
        said.scatter_(1, state["held"].long()[:, None], nxt[:, None])
        out = model(nxt, state["held"], state["held"] + 1, None, 1)
        state["held"] += 1
        state["logits"].copy_(crl.adjust_logits(out, history=said, repetition=penalty, mask=legal))

    if graph:
        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        for _ in range(steps - 1):
            g.replay()
    else:
        for _ in range(steps):
            step()
    torch.cuda.synchronize()
    return state["logits"].clone(), said.clone(), [p.clone() for p in pages], (table, embed, blocks, rope, legal, penalty, prompts)


def test_a_decoder_with_the_cache_follows_one_without(crl):
    """The same decoder recomputed from scratch over whole sequences as one prompt: the same keys and values are held, and
    the logits agree to the rounding of the activations."""
    logits, said, pages, (table, embed, blocks, rope, legal, penalty, prompts) = decode_steps(crl, F16, 6, False)
    b, steps = len(prompts), 6
    full = [n + steps for n in prompts]
    assert all(int((said[i] >= 0).sum()) == full[i] for i in range(b))
    fresh = [torch.zeros_like(p) for p in pages]
    cu = ints([0, full[0], full[0] + full[1], sum(full)])
    x = embed[torch.cat([said[i, :n] for i, n in enumerate(full)]).long()]
    for (qkv, proj), pool in zip(blocks, fresh):
        y = (torch.nn.functional.layer_norm(x.float(), (x.shape[1],)).half() @ qkv.T).unflatten(-1, (8, 32))
        q = crl.kv4_append(pool, y[:, 4:6], y[:, 6:], table, ints([0] * b), cu_tokens=cu, q=y[:, :4], rope=rope)
        x = x + crl.kv4_attention(pool, q, table, ints(full), cu_tokens=cu, max_tokens=max(full)).flatten(1) @ proj.T
    again = crl.adjust_logits((x @ embed.T)[cu[1:].long() - 1], history=said, repetition=penalty, mask=legal)
    fine = torch.isfinite(again)
    assert torch.equal(fine, torch.isfinite(logits))
    # an activation's last bit can move a 4-bit code: the two agree to a few of the codes' steps, not bit for bit
    gap = (logits[fine].float() - again[fine].float()).norm() / again[fine].float().norm()
    assert gap < 0.02


def test_captured_steps_equal_eager_ones(crl):
    eager, said, pages, _ = decode_steps(crl, BF16, 5, False)
    replayed, said2, pages2, _ = decode_steps(crl, BF16, 5, True)
    assert torch.equal(said, said2) and torch.equal(eager, replayed)
    assert all(torch.equal(a, b) for a, b in zip(pages, pages2))


def test_calls_on_two_streams_at_once(crl):
    """No workspace is shared: calls in flight at the same time give what each gives alone."""
    gen = torch.Generator().manual_seed(21)
    sets = []
    for lengths, n in (([3000, 2000], 1), ([900, 40, 700], 1)):
        pages, table = filled(crl, lengths, 64, 4, 64, gen)
        q = torch.randn(len(lengths) * n, 8, 64, generator=gen).half().cuda()
        sets.append((pages, q, table, ints(lengths)))
    alone = [crl.kv4_attention(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(10):
        for i, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[i].append(crl.kv4_attention(*s))
    torch.cuda.synchronize()
    for i, a in enumerate(alone):
        assert all(torch.equal(a, x) for x in got[i])


def test_drawn_sizes(crl):
    rng = random.Random(17)
    for seed in range(12):
        heads, kv = rng.choice([(12, 12), (8, 2), (7, 1), (6, 2), (16, 4)])
        runs = []
        for _ in range(rng.randint(1, 5)):
            n = rng.choice([1, rng.randint(2, 9), rng.randint(10, 90)])
            runs.append((n, n + rng.randint(0, 300)))
        attend_case(crl, rng.choice([F16, BF16]), rng.choice([32, 64, 128]), heads, kv, rng.choice([16, 48, 64]), runs, seed=seed)
