"""Refusals of the decoder-serving operators, and the oracle's own consistency (no GPU needed)."""
import ctypes
import math
import os
import shutil
import subprocess

import pytest
import torch

from chessrl_b200 import _lib as L
from conftest import ROOT
from oracle import serving as spec


def cache(**kw):
    c = dict(pages=1 << 20, num_pages=4, page_size=16, kv_heads=2, head_dim=64, seqs=1, block_table=1 << 21, table_stride=4, table_width=4)
    c.update(kw)
    return L.Kv4Cache(**c)


BAD_CACHES = [(dict(pages=None), -1), (dict(num_pages=0), -1), (dict(block_table=None), -1), (dict(table_stride=3), -1), (dict(seqs=-1), -1),
              (dict(kv_heads=0), -1), (dict(table_width=0), -1), (dict(head_dim=80), -2), (dict(head_dim=256), -2), (dict(page_size=24), -2),
              (dict(page_size=0), -2), (dict(pages=(1 << 20) + 8), -2), (dict(table_width=1 << 30, table_stride=1 << 30), -2)]


def test_refusals_reach_no_kernel(lib):
    """Every refused argument is an error code before anything is launched (there is no GPU here to launch on)."""
    p = 1 << 22
    append = dict(dtype=L.OUT_F16, tokens=1, k=p, v=p, starts=p, heads=0)
    read = dict(dtype=L.OUT_F16, tokens=1, k=p, v=p, starts=p)
    attend = dict(dtype=L.OUT_F16, tokens=1, q=p, out=p, lengths=p, heads=4, max_tokens=1)
    calls = [(lib.crl_kv4_append, L.Kv4AppendArgs, append), (lib.crl_kv4_read, L.Kv4ReadArgs, read),
             (lib.crl_kv4_attention, L.Kv4AttentionArgs, attend)]
    for call, cls, good in calls:
        assert call(None) == -1
        for change, rc in BAD_CACHES:
            assert call(ctypes.byref(cls(cache=cache(**change), **good))) == rc, (call, change)
        assert call(ctypes.byref(cls(cache=cache(), **{**good, "dtype": L.OUT_F32}))) == -1
        assert call(ctypes.byref(cls(cache=cache(), **{**good, "tokens": -1}))) == -1
        # nothing to do is no error and touches nothing
        assert call(ctypes.byref(cls(cache=cache(), **{**good, "tokens": 0}))) == 0
        assert call(ctypes.byref(cls(cache=cache(seqs=0), **good))) == 0
    for change, rc in ((dict(k=None), -1), (dict(heads=2), -1), (dict(heads=2, q=p, q_out=p), -1), (dict(starts=None), -1),
                       (dict(rope=p, rope_dim=63, rope_positions=8), -2), (dict(rope=p, rope_dim=128, rope_positions=8), -2),
                       (dict(rope=p, rope_dim=64, rope_positions=0), -2)):
        assert lib.crl_kv4_append(ctypes.byref(L.Kv4AppendArgs(cache=cache(), **{**append, **change}))) == rc, change
    for change, rc in ((dict(q=None), -1), (dict(heads=3), -2), (dict(heads=0), -1), (dict(lengths=None), -1)):
        assert lib.crl_kv4_attention(ctypes.byref(L.Kv4AttentionArgs(cache=cache(), **{**attend, **change}))) == rc, change
    logits = {"dtype": L.OUT_F32, "vocab": 8, "rows": 2, "logits": p, "in_stride": 8, "out": p, "out_stride": 8}
    for change, rc in ((dict(vocab=0), -1), (dict(in_stride=7), -1), (dict(out_stride=7), -1), (dict(dtype=3), -1), (dict(out=None), -1),
                       (dict(history_len=3), -1), (dict(history_len=3, history=p, history_stride=2), -1),
                       (dict(history_len=1 << 20, history=p, history_stride=1 << 20), -2),
                       (dict(biases=2, bias_ids=p, bias_stride=2), -1),
                       (dict(biases=4095, bias_ids=p, bias_stride=4095, bias_values=p, value_stride=4095), -2),
                       (dict(mask=p, mask_stride=0, mask_count=2), -1), (dict(mask=p, mask_stride=1, mask_count=1), -1), (dict(rows=-1), -1)):
        assert lib.crl_adjust_logits(ctypes.byref(L.LogitsArgs(**{**logits, **change}))) == rc, change
    assert lib.crl_adjust_logits(ctypes.byref(L.LogitsArgs(**{**logits, "rows": 0}))) == 0
    assert lib.crl_adjust_logits(None) == -1


def test_page_bytes(lib):
    assert lib.crl_kv4_page_bytes(16, 1, 64) == 1280 and lib.crl_kv4_page_bytes(48, 3, 32) == 3 * 3 * 640
    assert lib.crl_kv4_page_bytes(24, 1, 64) == 0 and lib.crl_kv4_page_bytes(16, 0, 64) == 0 and lib.crl_kv4_page_bytes(16, 1, 96) == 0


def test_tensor_checks_raise_before_the_library(lib):
    import chessrl_b200 as crl
    pages = torch.zeros(2, 2, 1, 1280, dtype=torch.uint8)
    table = torch.zeros(1, 2, dtype=torch.int32)
    k = torch.zeros(1, 2, 64, dtype=torch.float16)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        crl.kv4_append(pages, k, k, table, one)
    with pytest.raises(ValueError, match="GPU"):
        crl.kv4_attention(pages, k, table, one)
    with pytest.raises(ValueError, match="GPU"):
        crl.kv4_read(pages, table, one, 1)
    with pytest.raises(ValueError, match="GPU"):
        crl.adjust_logits(torch.zeros(1, 4))
    with pytest.raises(ValueError, match="page_size"):
        crl.kv4_pages(1, 20, 1, 64)
    with pytest.raises(ValueError, match="head_dim"):
        crl.kv4_pages(1, 16, 1, 80)
    with pytest.raises(ValueError, match="rot_dim"):
        crl.rope_table(7, 16)


def test_rope_table_far_positions():
    import chessrl_b200 as crl
    t = crl.rope_table(8, 100001, base=500.0, factor=4.0, device="cpu")
    assert t.shape == (100001, 4, 2) and t.dtype == torch.float32
    for pos, i in ((0, 0), (100000, 0), (99999, 3)):
        angle = pos / 4.0 * 500.0 ** (-2 * i / 8)
        assert abs(float(t[pos, i, 0]) - math.cos(angle)) <= 2.0 ** -24 and abs(float(t[pos, i, 1]) - math.sin(angle)) <= 2.0 ** -24


def test_ctypes_mirrors_match_the_header_layout(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    mirrors = {"crl_kv4_cache": L.Kv4Cache, "crl_kv4_append_args": L.Kv4AppendArgs, "crl_kv4_read_args": L.Kv4ReadArgs,
               "crl_kv4_attention_args": L.Kv4AttentionArgs, "crl_logits_args": L.LogitsArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "chessrl_b200.h"', 'int main(void) {']
    for cname, cls in mirrors.items():
        lines.append(f'  printf("%zu\\n", sizeof({cname}));')
        lines += [f'  printf("%zu\\n", offsetof({cname}, {f[0]}));' for f in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ['  return 0;', '}']))
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for cls in mirrors.values():
        want += [ctypes.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want


def test_oracle_format_properties():
    """A held value is within half a step (plus the step's and the centre's own roundings) of the row's, codes use the range,
    and (n - 8) * s is exact in f16."""
    x = torch.randn(200, 64, generator=torch.Generator().manual_seed(0))
    n, s, c, value = spec.held_rows(x)
    assert int(n.min()) >= 0 and int(n.max()) == 15
    step = s.repeat_interleave(32, -1)
    # the extremes may miss the end codes by what s lost to its eight bits: 8 s 2^-8, and the centre by half an f16 step
    assert ((value - x.double()).abs() <= step * (0.5 + 8 * 2.0 ** -8) + 2.0 ** -11 * c.abs().repeat_interleave(32, -1) + 1e-6).all()
    product = (n.double() - 8) * step
    assert torch.equal(product.half().double(), product)
    assert sorted(spec.nibble_of("k", d, 128) for d in range(128)) == list(range(128))
    assert sorted(spec.nibble_of("v", d, 128) for d in range(128)) == list(range(128))


def test_oracle_logits_by_hand():
    z = spec.adjust(torch.tensor([[2.0, -2.0, 1.0, 0.5]]), history=torch.tensor([[0, 1, 1, 9]]), repetition=torch.tensor([2.0]),
                    frequency=torch.tensor([0.25]), presence=torch.tensor([0.5]), bias_ids=torch.tensor([[2, 3, 2, -1]]),
                    bias_values=torch.tensor([[5.0, 1.0, 7.0, 3.0]]), mask=torch.tensor([[0b0111]], dtype=torch.uint8))
    assert z.tolist() == [[0.25, -5.0, 8.0, -math.inf]]
