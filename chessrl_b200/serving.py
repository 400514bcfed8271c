"""Decoder serving: a paged key/value cache held in 4 bits, attention over it, and next-token logits.

What `GPT`-like decoders (model_bis.py:36-83) need to continue a sequence without recomputing its prefix, which the
reference's own generation does (model_bis.py:272-320). Functions over torch tensors, like the C entry points behind them
(include/chessrl_b200.h documents the arithmetic and the page format): tensors are checked (a wrong device, dtype, shape or
stride is a ValueError), the kernels run on the tensors' GPU and its current stream, nothing is allocated but the results.

    pages = kv4_pages(num_pages, page_size, kv_heads, head_dim)      # the pool of one layer
    q = kv4_append(pages, k, v, block_table, lengths, q=q, rope=rope_table(64, 4096))
    out = kv4_attention(pages, q, block_table, lengths + 1)
    logits = adjust_logits(logits, history=tokens, repetition=penalty, mask=legal_bits)

A tensor is used on the current stream only; one that another stream is still working on has to be waited for by the
caller, as with any torch operation. `status` is an optional int32 tensor (zero before the call): a kernel that has to skip
something (a cache index without a page, a position past the rotation table, ...) leaves its code there, see the header.
"""
import ctypes
import math

import torch

from . import _lib as L

_bound = None


def _native():
    """The module that takes the tensors apart (csrc/serving_torch.cpp), bound to the loaded library."""
    global _bound
    if _bound is None:
        lib = L.load()
        try:
            from . import _serving
        except ImportError as e:
            raise RuntimeError("chessrl_b200/_serving.so is missing or was built for another torch: build it with "
                               "`python -m chessrl_b200.build`") from e
        _serving.bind(*(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value
                        for n in ("crl_kv4_append", "crl_kv4_read", "crl_kv4_attention", "crl_adjust_logits")))
        _bound = _serving
    return _bound


def kv4_pages(num_pages, page_size, kv_heads, head_dim, device="cuda"):
    """A pool of cache pages: uint8 [num_pages, kv_heads, page_size / 16, 20 * head_dim]. Its shape says everything about
    the cache; page_size is a multiple of 16, head_dim 32, 64 or 128."""
    if L.load().crl_kv4_page_bytes(page_size, kv_heads, head_dim) == 0:
        raise ValueError(f"no 4-bit pages of {page_size} tokens, {kv_heads} heads of {head_dim}: page_size is a multiple of 16, "
                         "head_dim 32, 64 or 128")
    return torch.zeros(num_pages, kv_heads, page_size // 16, 20 * head_dim, dtype=torch.uint8, device=device)


def rope_table(rot_dim, positions, base=10000.0, factor=1.0, device="cuda"):
    """(cos, sin) of the angles position / factor * base^(-2 i / rot_dim): f32 [positions, rot_dim / 2, 2], formed in 64
    bits. `factor` > 1 squeezes a longer context into the trained one (linear position interpolation); a larger `base` is
    the other usual way of scaling."""
    if rot_dim <= 0 or rot_dim % 2 != 0 or positions <= 0 or factor <= 0 or base <= 0:
        raise ValueError("rope_table needs an even rot_dim and positive positions, base and factor")
    angle = torch.arange(positions, dtype=torch.float64)[:, None] / factor * base ** (
        -torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
    return torch.stack([angle.cos(), angle.sin()], -1).float().to(device)


def kv4_append(pages, k, v, block_table, starts, cu_tokens=None, q=None, rope=None, interleaved=False, status=None):
    """Append keys and values [tokens, kv_heads, head_dim] (f16 or bf16, any strides with contiguous rows) to the cache.

    block_table int32 [seqs, pages]; starts int32 [seqs]: cache indices a sequence holds already. cu_tokens int32
    [seqs + 1]: rows cu_tokens[s] .. cu_tokens[s + 1] - 1 are sequence s's new tokens (rows behind the last sequence are
    left alone); None: one new token per sequence. rope: a `rope_table`; keys and `q` [tokens, heads, head_dim] are rotated
    at their cache index, in halves or interleaved pairs, the first rot_dim dims of a head.
    Returns the rotated queries (a new tensor), q itself where there is nothing to rotate, None without q."""
    return _native().kv4_append(pages, k, v, block_table, starts, cu_tokens, q, rope, interleaved, status)


def kv4_read(pages, block_table, starts, tokens, cu_tokens=None, dtype=torch.float16, status=None):
    """The keys and values that the cache holds, [tokens, kv_heads, head_dim] each in `dtype` (f16 or bf16): row
    cu_tokens[s] + j is cache index starts[s] + j of sequence s (without cu_tokens: row s is index starts[s]). Rows behind
    the last sequence, and rows without a page, are zero."""
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise ValueError("kv4_read gives float16 or bfloat16")
    return _native().kv4_read(pages, block_table, starts, tokens, cu_tokens, dtype is torch.bfloat16, status)


def kv4_attention(pages, q, block_table, lengths, cu_tokens=None, max_tokens=1, scale=None, out=None, status=None):
    """Causal attention of the new tokens' queries [tokens, heads, head_dim] (f16 or bf16) over the cache.

    lengths int32 [seqs]: cached tokens, the new ones included (append first). cu_tokens as in `kv4_append`, with
    max_tokens the most new tokens of any sequence (it sizes the launch; a sequence with more has the rest left out and
    reported through `status`). heads is a multiple of the cache's kv_heads. scale defaults to head_dim ** -0.5. A row that
    sees nothing is zero; rows behind the last sequence are left as they were in `out` (undefined in a new tensor)."""
    return _native().kv4_attention(pages, q, block_table, lengths, cu_tokens, max_tokens, scale, out, status)


def adjust_logits(logits, history=None, repetition=None, frequency=None, presence=None, bias_ids=None, bias_values=None,
                  mask=None, mask_rows=None, masked_value=-math.inf, out=None, status=None):
    """Penalties, biases and bit masks on next-token logits [rows, vocab] (f32, f16 or bf16), before a token is drawn.

    history int32 [rows, n]: tokens already said (entries outside the vocabulary are padding). Tokens in it have positive
    logits divided and others multiplied by repetition [rows], then frequency [rows] per occurrence and presence [rows]
    once subtracted. bias_ids int32 [rows, m] with bias_values f32 [rows, m] are added (of equal ids the last counts, ids
    outside the vocabulary are padding). mask uint8 [masks, >= ceil(vocab / 8)]: bit v clear sets masked_value (legal-move
    bitsets as positions.legal_mask_1929 and Engine.legal_masks make them); mask_rows int32 [rows] says which mask a row
    takes (negative: none), without it row r takes mask r. fp32 inside, rounded once. Returns `out` (a new tensor unless
    given; it may be `logits`)."""
    return _native().adjust_logits(logits, history, repetition, frequency, presence, bias_ids, bias_values, mask, mask_rows,
                                   masked_value, out, status)
