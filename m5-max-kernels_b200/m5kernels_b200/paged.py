"""A paged key/value cache and attention over it: what follows the Q/K/V projection.

`paged_append` stores the new tokens' keys and values in the cache's pages and
rotates keys and queries by their positions on the way; `paged_attention` lets
the new tokens attend over the cache.  Both take ragged batches of sequences
with any number of new tokens each (one when decoding, many for a prompt or a
chunk of one), described by

    query_start  int32 [B + 1]   rows query_start[b] .. query_start[b + 1] are sequence b's
    seq_lens     int32 [B]       its length, the new tokens included
    page_table   int32 [B, W]    its pages; position p is slot p % page of page p // page

so token i of n_b stands at position seq_lens[b] - n_b + i.  Lengths and table
are read on the device: nothing here waits for the GPU, and a captured CUDA
graph may be replayed after they changed.  The caches are [pages, kv heads,
page, head dim] tensors with any strides (the channels contiguous), so
`cache.transpose(1, 2)` presents a [pages, page, kv heads, head dim]
allocation.  The reference stops at the projection
(src/m5kernels/qk_rope.py:120-182); these operators have no twin there.
"""

from __future__ import annotations

import math
import struct
from numbers import Integral, Real

import torch

from . import _lib
from ._lib import check
from .linear import _key, _workspaces, _ws_lock

_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
# m5b_paged_batch, m5b_paged_append_args and m5b_paged_attention_args (include/m5b200.h):
# every field is 8 bytes
_PACK_APPEND = struct.Struct("@38q")
_PACK_ATTEND = struct.Struct("@29q2d5q")


def _ints(t, name):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise ValueError(f"{name} must be an int32 tensor")
    return t if t.is_contiguous() else t.contiguous()


def _rows(t, name, heads=None, dim=None):
    """A [T, heads, dim] operand with contiguous channels (copied if they are not)."""
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"{name} must have shape [tokens, heads, head_dim]")
    if (heads is not None and t.shape[1] != heads) or (dim is not None and t.shape[2] != dim):
        raise ValueError(f"{name} does not match the cache's heads and head_dim")
    return t if t.stride(2) == 1 else t.contiguous()


def _batch(tokens, q_heads, k_cache, v_cache, page_table, query_start, seq_lens):
    """The fields of m5b_paged_batch and the tensors that must outlive the call."""
    if (not isinstance(k_cache, torch.Tensor) or not isinstance(v_cache, torch.Tensor)
            or k_cache.dim() != 4 or k_cache.shape != v_cache.shape
            or k_cache.dtype != v_cache.dtype):
        raise ValueError("k_cache and v_cache must share one [pages, kv_heads, page, head_dim] "
                         "shape and dtype")
    if k_cache.dtype not in _FLOATS:
        raise ValueError("cache dtype must be float16, bfloat16 or float32")
    pages, kv_heads, page, dim = k_cache.shape
    if 0 in (pages, kv_heads, page, dim):
        raise ValueError("the cache must be nonempty")
    ks, vs = k_cache.stride(), v_cache.stride()
    if (ks[3] != 1 or vs[3] != 1) and dim > 1:
        raise ValueError("the cache's channels must be contiguous")
    query_start, seq_lens = _ints(query_start, "query_start"), _ints(seq_lens, "seq_lens")
    batch = seq_lens.numel()
    if seq_lens.dim() != 1 or batch == 0 or query_start.shape != (batch + 1,):
        raise ValueError("seq_lens must be a nonempty vector [B] and query_start [B + 1]")
    page_table = _ints(page_table, "page_table")
    if page_table.dim() != 2 or page_table.shape[0] != batch:
        raise ValueError("page_table must have shape [B, pages per sequence]")
    fields = (tokens, batch, q_heads, kv_heads, dim, query_start.data_ptr(), seq_lens.data_ptr(),
              k_cache.data_ptr(), v_cache.data_ptr(), _lib.DTYPE_CODE[k_cache.dtype], pages, page,
              ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], page_table.data_ptr(),
              page_table.shape[1], page_table.shape[1])
    return fields, (query_start, seq_lens, page_table)


def _scratch(device, nbytes):
    """Cached scratch of the attention kernels, one per device and stream."""
    if nbytes <= 0:
        return None
    key = _key(device, "paged")
    with _ws_lock:
        buf = _workspaces.get(key)
        if buf is None or buf.numel() < nbytes:
            buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
            _workspaces[key] = buf
        return buf


def paged_append(k, v, k_cache, v_cache, page_table, query_start, seq_lens, *, cos=None, sin=None,
                 q=None, layout="half"):
    """Store the new tokens' keys and values in the cache; return the rotated queries (or None).

    k, v: [T, kv_heads, head_dim], q: [T, q_heads, head_dim] - views are fine,
    the slices of one fused projection's rows or the head-major outputs of
    `projection_qkv_rope` transposed - of one floating dtype; the cache's may
    differ.  cos, sin: [positions, R] tables indexed by position, 2 R <=
    head_dim; without them nothing is rotated.  layout "half" pairs channels
    (j, j + R), "interleaved" (2j, 2j + 1).  Values are rounded once, to the
    cache's dtype, in which the queries [T, q_heads, head_dim] return too.
    A token at a position without a table row is not appended, and its query
    is zero.
    """
    k = _rows(k, "k")
    tokens = k.shape[0]
    q_heads = k.shape[1]
    if q is not None:
        q = _rows(q, "q", None, k.shape[2])
        q_heads = q.shape[1]
        if q.shape[0] != tokens or q.dtype != k.dtype:
            raise ValueError("q, k and v must share tokens and dtype")
    fields, keep = _batch(tokens, q_heads, k_cache, v_cache, page_table, query_start, seq_lens)
    kv_heads, dim = k_cache.shape[1], k_cache.shape[3]
    if k.shape[1] != kv_heads or k.shape[2] != dim:
        raise ValueError("k does not match the cache's heads and head_dim")
    v = _rows(v, "v", kv_heads, dim)
    if v.shape[0] != tokens or v.dtype != k.dtype:
        raise ValueError("q, k and v must share tokens and dtype")
    if k.dtype not in _FLOATS:
        raise ValueError("input dtype must be float16, bfloat16 or float32")
    if q_heads < 1 or q_heads % kv_heads:
        raise ValueError("q_heads must be a multiple of kv_heads")
    if layout not in ("half", "interleaved"):
        raise ValueError("layout must be 'half' or 'interleaved'")
    half = rows = table_dtype = 0
    if cos is not None or sin is not None:
        if (not isinstance(cos, torch.Tensor) or not isinstance(sin, torch.Tensor)
                or cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != sin.dtype
                or cos.dtype not in _FLOATS or 0 in cos.shape):
            raise ValueError("cos and sin must be matching floating tables [positions, R]")
        rows, half = cos.shape
        if 2 * half > dim:
            raise ValueError("cos and sin rotate 2 R channels, at most head_dim")
        table_dtype = _lib.DTYPE_CODE[cos.dtype]
        cos, sin = cos.contiguous(), sin.contiguous()
    dev = _lib.require_cuda(k, v, q, k_cache, v_cache, *keep, cos, sin)
    out = None
    if q is not None:
        out = torch.empty((tokens, q_heads, dim), dtype=k_cache.dtype, device=dev)
    if tokens == 0:
        return out
    args = _PACK_APPEND.pack(
        *fields, 0 if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(),
        _lib.DTYPE_CODE[k.dtype], 0 if q is None else q.stride(0),
        0 if q is None else q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
        0 if cos is None else cos.data_ptr(), 0 if cos is None else sin.data_ptr(), table_dtype,
        rows, half, layout == "interleaved", 0 if out is None else out.data_ptr())
    check(_lib.lib().m5b_paged_append(args, _lib.stream_handle(dev)))
    return out


def _positive(value, name, allow_none=True):
    if value is None and allow_none:
        return 0.0
    if (isinstance(value, bool) or not isinstance(value, Real) or not math.isfinite(value)
            or value <= 0):
        raise ValueError(f"{name} must be a positive finite real scalar")
    return float(value)


def paged_attention(q, k_cache, v_cache, page_table, query_start, seq_lens, *, max_query_len,
                    scale=None, softcap=None, slopes=None, window=None, prefix_lens=None,
                    return_lse=False, out=None):
    """Attention of the new tokens q [T, q_heads, head_dim] over the cache -> [T, q_heads, head_dim].

    The cache holds the new tokens' keys and values already (`paged_append`).
    Query head h reads kv head h // (q_heads // kv_heads).  Key j's score is
    x = scale q.k_j (scale: 1 / sqrt(head_dim) unless given), capped to
    softcap * tanh(x / softcap), minus slopes[h] * |pos - j| (slopes: fp32
    [q_heads]).  A token at pos sees the keys j <= pos of its sequence, of
    those the last `window` only, and the first prefix_lens[b] (int32 [B]) keys
    in any case.  A token that sees no key returns zeros.  max_query_len: the
    most new tokens of any sequence; it selects the kernel, not the result.
    With return_lse also the fp32 [T, q_heads] natural logarithm of the sum of
    exp(x), -inf for a token that sees no key.  `out` may be given, any
    strides with contiguous channels.
    """
    q = _rows(q, "q")
    tokens, q_heads, dim = q.shape
    fields, keep = _batch(tokens, q_heads, k_cache, v_cache, page_table, query_start, seq_lens)
    if dim != k_cache.shape[3] or q.dtype != k_cache.dtype:
        raise ValueError("q must have the cache's head_dim and dtype")
    if q_heads < 1 or q_heads % k_cache.shape[1]:
        raise ValueError("q_heads must be a multiple of kv_heads")
    if dim > 256:
        raise NotImplementedError("head_dim above 256 is unsupported")
    if isinstance(max_query_len, bool) or not isinstance(max_query_len, Integral) or max_query_len < 0:
        raise ValueError("max_query_len must be a whole number")
    scale = dim ** -0.5 if scale is None else _positive(scale, "scale", False)
    softcap = _positive(softcap, "softcap")
    if window is None:
        window = 0
    elif isinstance(window, bool) or not isinstance(window, Integral) or window < 1:
        raise ValueError("window must be a positive whole number")
    if slopes is not None:
        if (not isinstance(slopes, torch.Tensor) or slopes.dtype != torch.float32
                or slopes.shape != (q_heads,)):
            raise ValueError("slopes must be a float32 vector of length q_heads")
        slopes = slopes.contiguous()
    if prefix_lens is not None:
        prefix_lens = _ints(prefix_lens, "prefix_lens")
        if prefix_lens.shape != seq_lens.shape:
            raise ValueError("prefix_lens must be a vector [B]")
    if out is not None and (not isinstance(out, torch.Tensor) or out.shape != q.shape
                            or out.dtype != q.dtype or out.stride(2) != 1):
        raise ValueError("out must match q, with contiguous channels")
    dev = _lib.require_cuda(q, k_cache, v_cache, *keep, slopes, prefix_lens, out)
    if out is None:
        out = torch.empty((tokens, q_heads, dim), dtype=q.dtype, device=dev)
    lse = torch.empty((tokens, q_heads), dtype=torch.float32, device=dev) if return_lse else None
    if tokens > 0:
        lib = _lib.lib()
        ws = _scratch(dev, lib.m5b_paged_attention_workspace_bytes(dim))
        args = _PACK_ATTEND.pack(
            *fields, q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0),
            out.stride(1), 0 if lse is None else lse.data_ptr(), max_query_len, scale, softcap,
            0 if slopes is None else slopes.data_ptr(), window,
            0 if prefix_lens is None else prefix_lens.data_ptr(),
            0 if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel())
        check(lib.m5b_paged_attention(args, _lib.stream_handle(dev)))
    return (out, lse) if return_lse else out
