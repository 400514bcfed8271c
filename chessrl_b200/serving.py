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

_Tensor = torch.Tensor
_DTYPE = {torch.float32: L.OUT_F32, torch.float16: L.OUT_F16, torch.bfloat16: L.OUT_BF16}
_HALF = (torch.float16, torch.bfloat16)
_ANY, _I32, _U8, _F32 = tuple(_DTYPE), (torch.int32,), (torch.uint8,), (torch.float32,)

# A call for one token takes the GPU a few microseconds, so the host side counts: checks are single expressions whose
# message is only put together where one fails, and the stream is taken by its number.


def _call(name, args, index):
    lib = L.load()
    args.stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = getattr(lib, name)(ctypes.byref(args))
    else:
        with torch.cuda.device(index):
            rc = getattr(lib, name)(ctypes.byref(args))
    if rc != 0:
        raise L.CrlError(rc, name)


def _check(name, t, index, dtypes, dim):
    """`t` is a tensor of `dim` dimensions on GPU `index` with one of `dtypes`: the library gets raw pointers and sees none
    of this."""
    if isinstance(t, _Tensor) and t.get_device() == index and t.dtype in dtypes and t.dim() == dim:
        return
    if not isinstance(t, _Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.get_device() != index:
        raise ValueError(f"{name} must live on cuda:{index}, got {t.device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must have dtype {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    raise ValueError(f"{name} must have {dim} dimensions, got shape {tuple(t.shape)}")


def _vector(name, t, index, count, dtypes=_I32):
    _check(name, t, index, dtypes, 1)
    if t.shape[0] != count or count > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must hold {count} contiguous {str(dtypes[0])[6:]}, got shape {tuple(t.shape)}")
    return t.data_ptr()


def _status(status, index):
    if status is None:
        return None
    _check("status", status, index, _I32, 1)
    if status.shape[0] < 1:
        raise ValueError("status must hold an int32")
    return status.data_ptr()


def _rows(name, t, index, dtypes, heads, dim):
    _check(name, t, index, dtypes, 3)
    shape, stride = t.shape, t.stride()
    if shape[2] != dim or heads is not None and shape[1] != heads:
        raise ValueError(f"{name} must be [tokens, {'heads' if heads is None else heads}, {dim}], got shape {tuple(shape)}")
    if stride[2] != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    return t.data_ptr(), stride[0], stride[1]


def kv4_pages(num_pages, page_size, kv_heads, head_dim, device="cuda"):
    """A pool of cache pages: uint8 [num_pages, kv_heads, page_size / 16, 20 * head_dim]. Its shape says everything about
    the cache; page_size is a multiple of 16, head_dim 32, 64 or 128."""
    if L.load().crl_kv4_page_bytes(page_size, kv_heads, head_dim) == 0:
        raise ValueError(f"no 4-bit pages of {page_size} tokens, {kv_heads} heads of {head_dim}: page_size is a multiple of 16, "
                         "head_dim 32, 64 or 128")
    return torch.zeros(num_pages, kv_heads, page_size // 16, 20 * head_dim, dtype=torch.uint8, device=device)


def _cache(pages, block_table):
    """(the cache's description, its GPU)."""
    if not isinstance(pages, _Tensor) or not pages.is_cuda:
        raise ValueError("pages must be a tensor on the GPU (see kv4_pages)")
    index = pages.get_device()
    _check("pages", pages, index, _U8, 4)
    n, heads, blocks, width = pages.shape
    if width not in (640, 1280, 2560) or not pages.is_contiguous() or n * heads * blocks == 0:
        raise ValueError("pages must be contiguous [num_pages, kv_heads, page_size / 16, 20 * head_dim] with head_dim 32, 64 or 128")
    _check("block_table", block_table, index, _I32, 2)
    seqs, wide = block_table.shape
    stride, step = block_table.stride()
    if seqs <= 1:
        stride = wide
    if wide == 0 or wide > 1 and step != 1 or stride < wide:
        raise ValueError("block_table must be [seqs, pages] with contiguous rows that do not overlap")
    return L.Kv4Cache(pages.data_ptr(), n, 16 * blocks, heads, width // 20, seqs, block_table.data_ptr(), stride, wide), index


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
    cache, dev = _cache(pages, block_table)
    hd = cache.head_dim
    a = L.Kv4AppendArgs()
    a.cache = cache
    a.k, a.k_token_stride, a.k_head_stride = _rows("k", k, dev, _HALF, cache.kv_heads, hd)
    dtype, tokens = k.dtype, k.shape[0]
    a.v, a.v_token_stride, a.v_head_stride = _rows("v", v, dev, (dtype,), cache.kv_heads, hd)
    a.tokens, a.dtype = tokens, _DTYPE[dtype]
    if v.shape[0] != tokens or q is not None and q.shape[0] != tokens:
        raise ValueError("q, k and v must have the same number of tokens")
    a.starts = _vector("starts", starts, dev, cache.seqs)
    if cu_tokens is not None:
        a.cu_tokens = _vector("cu_tokens", cu_tokens, dev, cache.seqs + 1)
    elif tokens != cache.seqs:
        raise ValueError("without cu_tokens there is one token per sequence")
    out = q
    if q is not None:
        q_rows = _rows("q", q, dev, (dtype,), None, hd)
    if rope is not None:
        _check("rope", rope, dev, _F32, 3)
        positions, pairs, two = rope.shape
        if two != 2 or not rope.is_contiguous() or not 0 < 2 * pairs <= hd or positions == 0:
            raise ValueError("rope must be a contiguous [positions, rot_dim / 2, 2] table with rot_dim <= head_dim (see rope_table)")
        a.rope, a.rope_positions, a.rope_dim, a.rope_interleaved = rope.data_ptr(), positions, 2 * pairs, int(interleaved)
        if q is not None and q.shape[1]:
            heads = q.shape[1]
            out = torch.empty((tokens, heads, hd), dtype=dtype, device=q.device)
            a.q, a.q_token_stride, a.q_head_stride = q_rows
            a.q_out, a.out_token_stride, a.out_head_stride, a.heads = out.data_ptr(), heads * hd, hd, heads
    if status is not None:
        a.device_status = _status(status, dev)
    if tokens:
        _call("crl_kv4_append", a, dev)
    return out


def kv4_read(pages, block_table, starts, tokens, cu_tokens=None, dtype=torch.float16, status=None):
    """The keys and values that the cache holds, [tokens, kv_heads, head_dim] each in `dtype` (f16 or bf16): row
    cu_tokens[s] + j is cache index starts[s] + j of sequence s (without cu_tokens: row s is index starts[s]). Rows behind
    the last sequence, and rows without a page, are zero."""
    cache, dev = _cache(pages, block_table)
    if dtype not in _HALF:
        raise ValueError("kv4_read gives float16 or bfloat16")
    heads, hd = cache.kv_heads, cache.head_dim
    k = torch.empty((tokens, heads, hd), dtype=dtype, device=pages.device)
    v = torch.empty((tokens, heads, hd), dtype=dtype, device=pages.device)
    a = L.Kv4ReadArgs()
    a.cache, a.dtype, a.tokens = cache, _DTYPE[dtype], tokens
    a.k, a.v = k.data_ptr(), v.data_ptr()
    a.k_token_stride = a.v_token_stride = heads * hd
    a.k_head_stride = a.v_head_stride = hd
    a.starts = _vector("starts", starts, dev, cache.seqs)
    if cu_tokens is not None:
        a.cu_tokens = _vector("cu_tokens", cu_tokens, dev, cache.seqs + 1)
    elif tokens != cache.seqs:
        raise ValueError("without cu_tokens there is one token per sequence")
    if status is not None:
        a.device_status = _status(status, dev)
    if tokens:
        if cache.seqs == 0:
            return k.zero_(), v.zero_()
        _call("crl_kv4_read", a, dev)
    return k, v


def kv4_attention(pages, q, block_table, lengths, cu_tokens=None, max_tokens=1, scale=None, out=None, status=None):
    """Causal attention of the new tokens' queries [tokens, heads, head_dim] (f16 or bf16) over the cache.

    lengths int32 [seqs]: cached tokens, the new ones included (append first). cu_tokens as in `kv4_append`, with
    max_tokens the most new tokens of any sequence (it sizes the launch; a sequence with more has the rest left out and
    reported through `status`). heads is a multiple of the cache's kv_heads. scale defaults to head_dim ** -0.5. A row that
    sees nothing is zero; rows behind the last sequence are left as they were in `out` (undefined in a new tensor)."""
    cache, dev = _cache(pages, block_table)
    hd = cache.head_dim
    a = L.Kv4AttentionArgs()
    a.cache = cache
    a.q, a.q_token_stride, a.q_head_stride = _rows("q", q, dev, _HALF, None, hd)
    tokens, heads, _ = q.shape
    dtype = q.dtype
    if heads == 0 or heads % cache.kv_heads != 0:
        raise ValueError(f"query heads must be a multiple of the cache's {cache.kv_heads}, got {heads}")
    if out is None:
        out = torch.empty((tokens, heads, hd), dtype=dtype, device=q.device)
        a.out, a.out_token_stride, a.out_head_stride = out.data_ptr(), heads * hd, hd
    else:
        a.out, a.out_token_stride, a.out_head_stride = _rows("out", out, dev, (dtype,), heads, hd)
        if out.shape[0] != tokens:
            raise ValueError("out must have q's shape")
    a.dtype, a.heads, a.tokens = _DTYPE[dtype], heads, tokens
    a.lengths = _vector("lengths", lengths, dev, cache.seqs)
    if cu_tokens is not None:
        a.cu_tokens = _vector("cu_tokens", cu_tokens, dev, cache.seqs + 1)
        if max_tokens < 1:
            raise ValueError("max_tokens must be at least 1")
        a.max_tokens = min(max_tokens, tokens)
    else:
        if tokens != cache.seqs:
            raise ValueError("without cu_tokens there is one token per sequence")
        a.max_tokens = 1
    a.scale = hd ** -0.5 if scale is None else scale
    if status is not None:
        a.device_status = _status(status, dev)
    if tokens:
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
    if not isinstance(logits, _Tensor) or not logits.is_cuda:
        raise ValueError("logits must be a tensor on the GPU")
    dev = logits.get_device()
    _check("logits", logits, dev, _ANY, 2)
    rows, vocab = logits.shape
    if vocab == 0:
        raise ValueError("logits must have a vocabulary")
    a = L.LogitsArgs()

    def matrix(name, t, dtypes, count):
        """(address, elements from row to row, columns) of a matrix of `count` rows."""
        _check(name, t, dev, dtypes, 2)
        (n, wide), (stride, step) = t.shape, t.stride()
        if n != count and count is not None:
            raise ValueError(f"{name} must have {count} rows, got shape {tuple(t.shape)}")
        if n <= 1:
            stride = wide
        if wide > 1 and step != 1 or stride < wide:
            raise ValueError(f"the rows of {name} must be contiguous and not overlap")
        return t.data_ptr(), stride, wide

    if out is None:
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device)
        a.out, a.out_stride = out.data_ptr(), vocab
    else:
        a.out, a.out_stride, wide = matrix("out", out, (logits.dtype,), rows)
        if wide != vocab:
            raise ValueError("out must have the shape of logits")
    a.dtype, a.vocab, a.rows = _DTYPE[logits.dtype], vocab, rows
    a.logits, a.in_stride, _ = matrix("logits", logits, _ANY, rows)
    if history is not None:
        a.history, a.history_stride, a.history_len = matrix("history", history, _I32, rows)
    if repetition is not None:
        a.repetition = _vector("repetition", repetition, dev, rows, _F32)
    if frequency is not None:
        a.frequency = _vector("frequency", frequency, dev, rows, _F32)
    if presence is not None:
        a.presence = _vector("presence", presence, dev, rows, _F32)
    if bias_ids is not None or bias_values is not None:
        if bias_ids is None or bias_values is None:
            raise ValueError("bias_ids and bias_values go together")
        a.bias_ids, a.bias_stride, a.biases = matrix("bias_ids", bias_ids, _I32, rows)
        a.bias_values, a.value_stride, wide = matrix("bias_values", bias_values, _F32, rows)
        if wide != a.biases:
            raise ValueError("bias_ids and bias_values must have the same shape")
    if mask is not None:
        a.mask, a.mask_stride, wide = matrix("mask", mask, _U8, rows if mask_rows is None else None)
        a.mask_count = mask.shape[0]
        if wide * 8 < vocab:
            raise ValueError(f"mask rows hold {wide} bytes, the vocabulary needs {(vocab + 7) // 8}")
        if a.mask_count == 0 and rows:
            raise ValueError("mask must have a row")
        if mask_rows is not None:
            a.mask_rows = _vector("mask_rows", mask_rows, dev, rows)
    elif mask_rows is not None:
        raise ValueError("mask_rows needs a mask")
    a.masked_value = masked_value
    if status is not None:
        a.device_status = _status(status, dev)
    if rows:
        _call("crl_adjust_logits", a, dev)
    return out
