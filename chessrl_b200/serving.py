"""Decoder serving: a paged key/value cache held in 4 bits, attention over it, and next-token logits.

What `GPT`-like decoders (model_bis.py:36-83) need to continue a sequence without recomputing its prefix, which the
reference's own generation does (model_bis.py:272-320). Functions over torch tensors, like the C entry points behind them
(include/chessrl_b200.h documents the arithmetic and the page format): tensors are checked here, the kernels run on the
tensors' GPU and its current stream, nothing is allocated but the results.

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

_DTYPE = {torch.float32: L.OUT_F32, torch.float16: L.OUT_F16, torch.bfloat16: L.OUT_BF16}
_HALF = (torch.float16, torch.bfloat16)


def _call(name, args, device):
    lib = L.load()
    if torch.cuda.current_device() == device.index:
        args.stream = torch.cuda.current_stream(device).cuda_stream
        rc = getattr(lib, name)(ctypes.byref(args))
    else:
        with torch.cuda.device(device):
            args.stream = torch.cuda.current_stream(device).cuda_stream
            rc = getattr(lib, name)(ctypes.byref(args))
    if rc != 0:
        raise L.CrlError(rc, name)


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _check(name, t, device, dtypes, dim):
    """`t` is a tensor of `dim` dimensions on `device` with one of `dtypes`: the library gets raw pointers and sees none
    of this."""
    _need(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _need(t.device == device, f"{name} must live on {device}, got {t.device}")
    _need(t.dtype in dtypes, f"{name} must have dtype {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    _need(t.dim() == dim, f"{name} must have {dim} dimensions, got shape {tuple(t.shape)}")


def _ints(name, t, device, count):
    _check(name, t, device, (torch.int32,), 1)
    _need(t.shape[0] == count and (count <= 1 or t.stride(0) == 1), f"{name} must hold {count} contiguous int32, got shape {tuple(t.shape)}")
    return t.data_ptr()


def _status(status, device):
    if status is None:
        return None
    _check("status", status, device, (torch.int32,), 1)
    _need(status.shape[0] >= 1, "status must hold an int32")
    return status.data_ptr()


def _rows(name, t, device, dtypes, heads, dim):
    _check(name, t, device, dtypes, 3)
    _need(t.shape[2] == dim and (heads is None or t.shape[1] == heads),
          f"{name} must be [tokens, {'heads' if heads is None else heads}, {dim}], got shape {tuple(t.shape)}")
    _need(t.stride(2) == 1, f"the last dimension of {name} must be contiguous")
    return t.data_ptr(), t.stride(0), t.stride(1)


def kv4_pages(num_pages, page_size, kv_heads, head_dim, device="cuda"):
    """A pool of cache pages: uint8 [num_pages, kv_heads, page_size / 16, 20 * head_dim]. Its shape says everything about
    the cache; page_size is a multiple of 16, head_dim 32, 64 or 128."""
    _need(L.load().crl_kv4_page_bytes(page_size, kv_heads, head_dim) > 0,
          f"no 4-bit pages of {page_size} tokens, {kv_heads} heads of {head_dim}: page_size is a multiple of 16, head_dim 32, 64 or 128")
    return torch.zeros(num_pages, kv_heads, page_size // 16, 20 * head_dim, dtype=torch.uint8, device=device)


def _cache(pages, block_table):
    _need(isinstance(pages, torch.Tensor) and pages.is_cuda, "pages must be a tensor on the GPU (see kv4_pages)")
    _check("pages", pages, pages.device, (torch.uint8,), 4)
    n, heads, blocks, width = pages.shape
    _need(width in (640, 1280, 2560) and pages.is_contiguous() and pages.numel() > 0,
          "pages must be contiguous [num_pages, kv_heads, page_size / 16, 20 * head_dim] with head_dim 32, 64 or 128")
    _check("block_table", block_table, pages.device, (torch.int32,), 2)
    seqs, wide = block_table.shape
    _need(wide > 0 and (wide == 1 or block_table.stride(1) == 1), "block_table must be [seqs, pages] with contiguous rows")
    stride = block_table.stride(0) if seqs > 1 else wide
    _need(stride >= wide, "block_table rows must not overlap")
    return L.Kv4Cache(pages.data_ptr(), n, 16 * blocks, heads, width // 20, seqs, block_table.data_ptr(), stride, wide)


def rope_table(rot_dim, positions, base=10000.0, factor=1.0, device="cuda"):
    """(cos, sin) of the angles position / factor * base^(-2 i / rot_dim): f32 [positions, rot_dim / 2, 2], formed in 64
    bits. `factor` > 1 squeezes a longer context into the trained one (linear position interpolation); a larger `base` is
    the other usual way of scaling."""
    _need(rot_dim > 0 and rot_dim % 2 == 0 and positions > 0 and factor > 0 and base > 0,
          "rope_table needs an even rot_dim and positive positions, base and factor")
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
    cache = _cache(pages, block_table)
    dev = pages.device
    a = L.Kv4AppendArgs()
    a.cache = cache
    a.k, a.k_token_stride, a.k_head_stride = _rows("k", k, dev, _HALF, cache.kv_heads, cache.head_dim)
    a.v, a.v_token_stride, a.v_head_stride = _rows("v", v, dev, (k.dtype,), cache.kv_heads, cache.head_dim)
    a.tokens = k.shape[0]
    _need(v.shape[0] == k.shape[0], "k and v must have the same number of tokens")
    a.dtype = _DTYPE[k.dtype]
    a.starts = _ints("starts", starts, dev, cache.seqs)
    if cu_tokens is not None:
        a.cu_tokens = _ints("cu_tokens", cu_tokens, dev, cache.seqs + 1)
    else:
        _need(k.shape[0] == cache.seqs, "without cu_tokens there is one token per sequence")
    out = q
    if q is not None:
        q_rows = _rows("q", q, dev, (k.dtype,), None, cache.head_dim)
        _need(q.shape[0] == k.shape[0], "q and k must have the same number of tokens")
    if rope is not None:
        _check("rope", rope, dev, (torch.float32,), 3)
        _need(rope.shape[2] == 2 and rope.is_contiguous() and 0 < 2 * rope.shape[1] <= cache.head_dim and rope.shape[0] > 0,
              "rope must be a contiguous [positions, rot_dim / 2, 2] table with rot_dim <= head_dim (see rope_table)")
        a.rope, a.rope_positions, a.rope_dim, a.rope_interleaved = rope.data_ptr(), rope.shape[0], 2 * rope.shape[1], int(interleaved)
        if q is not None and q.numel() > 0:
            out = torch.empty(q.shape, dtype=q.dtype, device=dev)
            a.q, a.q_token_stride, a.q_head_stride = q_rows
            a.q_out, a.out_token_stride, a.out_head_stride = out.data_ptr(), out.stride(0), out.stride(1)
            a.heads = q.shape[1]
    a.device_status = _status(status, dev)
    if a.tokens:
        _call("crl_kv4_append", a, dev)
    return out


def kv4_read(pages, block_table, starts, tokens, cu_tokens=None, dtype=torch.float16, status=None):
    """The keys and values that the cache holds, [tokens, kv_heads, head_dim] each in `dtype` (f16 or bf16): row
    cu_tokens[s] + j is cache index starts[s] + j of sequence s (without cu_tokens: row s is index starts[s]). Rows behind
    the last sequence, and rows without a page, are zero."""
    cache = _cache(pages, block_table)
    dev = pages.device
    _need(dtype in _HALF, "kv4_read gives float16 or bfloat16")
    k = torch.zeros(tokens, cache.kv_heads, cache.head_dim, dtype=dtype, device=dev)
    v = torch.zeros_like(k)
    a = L.Kv4ReadArgs()
    a.cache, a.dtype, a.tokens = cache, _DTYPE[dtype], tokens
    a.k, a.k_token_stride, a.k_head_stride = k.data_ptr(), k.stride(0), k.stride(1)
    a.v, a.v_token_stride, a.v_head_stride = v.data_ptr(), v.stride(0), v.stride(1)
    a.starts = _ints("starts", starts, dev, cache.seqs)
    if cu_tokens is not None:
        a.cu_tokens = _ints("cu_tokens", cu_tokens, dev, cache.seqs + 1)
    else:
        _need(tokens == cache.seqs, "without cu_tokens there is one token per sequence")
    a.device_status = _status(status, dev)
    if tokens:
        _call("crl_kv4_read", a, dev)
    return k, v


def kv4_attention(pages, q, block_table, lengths, cu_tokens=None, max_tokens=1, scale=None, out=None, status=None):
    """Causal attention of the new tokens' queries [tokens, heads, head_dim] (f16 or bf16) over the cache.

    lengths int32 [seqs]: cached tokens, the new ones included (append first). cu_tokens as in `kv4_append`, with
    max_tokens the most new tokens of any sequence (it sizes the launch; a sequence with more has the rest left out and
    reported through `status`). heads is a multiple of the cache's kv_heads. scale defaults to head_dim ** -0.5. A row that
    sees nothing is zero; rows behind the last sequence are left as they were in `out` (undefined in a new tensor)."""
    cache = _cache(pages, block_table)
    dev = pages.device
    a = L.Kv4AttentionArgs()
    a.cache = cache
    a.q, a.q_token_stride, a.q_head_stride = _rows("q", q, dev, _HALF, None, cache.head_dim)
    _need(q.shape[1] > 0 and q.shape[1] % cache.kv_heads == 0, f"query heads must be a multiple of the cache's {cache.kv_heads}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    else:
        _need(isinstance(out, torch.Tensor) and out.shape[0] == q.shape[0], "out must have q's shape")
    a.out, a.out_token_stride, a.out_head_stride = _rows("out", out, dev, (q.dtype,), q.shape[1], cache.head_dim)
    a.dtype, a.heads, a.tokens = _DTYPE[q.dtype], q.shape[1], q.shape[0]
    a.lengths = _ints("lengths", lengths, dev, cache.seqs)
    if cu_tokens is not None:
        a.cu_tokens = _ints("cu_tokens", cu_tokens, dev, cache.seqs + 1)
        _need(max_tokens >= 1, "max_tokens must be at least 1")
        a.max_tokens = min(max_tokens, q.shape[0])
    else:
        _need(q.shape[0] == cache.seqs, "without cu_tokens there is one token per sequence")
        a.max_tokens = 1
    a.scale = cache.head_dim ** -0.5 if scale is None else float(scale)
    a.device_status = _status(status, dev)
    if q.shape[0]:
        _call("crl_kv4_attention", a, dev)
    return out


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
    _need(isinstance(logits, torch.Tensor) and logits.is_cuda, "logits must be a tensor on the GPU")
    dev = logits.device
    _check("logits", logits, dev, tuple(_DTYPE), 2)
    rows, vocab = logits.shape
    _need(vocab > 0, "logits must have a vocabulary")
    a = L.LogitsArgs()

    def pitch(name, t):
        _need(t.shape[1] <= 1 or t.stride(1) == 1, f"the rows of {name} must be contiguous")
        stride = t.stride(0) if t.shape[0] > 1 else t.shape[1]
        _need(stride >= t.shape[1], f"the rows of {name} must not overlap")
        return t.data_ptr(), stride

    def per_row(name, t):
        _check(name, t, dev, (torch.float32,), 1)
        _need(t.shape[0] == rows and (rows <= 1 or t.stride(0) == 1), f"{name} must hold {rows} contiguous float32")
        return t.data_ptr()

    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    _check("out", out, dev, (logits.dtype,), 2)
    _need(out.shape == logits.shape, "out must have the shape of logits")
    a.dtype, a.vocab, a.rows = _DTYPE[logits.dtype], vocab, rows
    pointer, a.in_stride = pitch("logits", logits)
    setattr(a, "in", pointer)
    a.out, a.out_stride = pitch("out", out)
    if history is not None:
        _check("history", history, dev, (torch.int32,), 2)
        _need(history.shape[0] == rows, f"history must have {rows} rows")
        a.history, a.history_stride = pitch("history", history)
        a.history_len = history.shape[1]
    for name, t in (("repetition", repetition), ("frequency", frequency), ("presence", presence)):
        if t is not None:
            setattr(a, name, per_row(name, t))
    _need((bias_ids is None) == (bias_values is None), "bias_ids and bias_values go together")
    if bias_ids is not None:
        _check("bias_ids", bias_ids, dev, (torch.int32,), 2)
        _check("bias_values", bias_values, dev, (torch.float32,), 2)
        _need(bias_ids.shape[0] == rows and bias_ids.shape == bias_values.shape, f"bias_ids and bias_values must be [{rows}, m] both")
        a.bias_ids, a.bias_stride = pitch("bias_ids", bias_ids)
        a.bias_values, a.value_stride = pitch("bias_values", bias_values)
        a.biases = bias_ids.shape[1]
    _need(mask is not None or mask_rows is None, "mask_rows needs a mask")
    if mask is not None:
        _check("mask", mask, dev, (torch.uint8,), 2)
        _need(mask.shape[1] * 8 >= vocab, f"mask rows hold {mask.shape[1]} bytes, the vocabulary needs {(vocab + 7) // 8}")
        _need(mask.shape[0] > 0 or rows == 0, "mask must have a row")
        a.mask, a.mask_stride = pitch("mask", mask)
        a.mask_count = mask.shape[0]
        if mask_rows is not None:
            a.mask_rows = _ints("mask_rows", mask_rows, dev, rows)
        else:
            _need(mask.shape[0] == rows, f"mask must have {rows} rows, or mask_rows must say which one a row takes")
    a.masked_value = float(masked_value)
    a.device_status = _status(status, dev)
    if rows:
        _call("crl_adjust_logits", a, dev)
    return out
