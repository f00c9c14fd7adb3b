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
from .linear import stream_buffer

_CODE = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
# m5b_paged_batch, m5b_paged_append_args and m5b_paged_attention_args (include/m5b200.h):
# every field is 8 bytes
_PACK_APPEND = struct.Struct("@38q")
_PACK_ATTEND = struct.Struct("@29q2d5q")
_Tensor = torch.Tensor
_CONTIGUOUS = torch.contiguous_format
_FAR = 2**31 - 1  # no position is beyond


def _ints(t, name):
    if not isinstance(t, _Tensor) or t.dtype is not torch.int32:
        raise ValueError(f"{name} must be an int32 tensor")
    return t if t.is_contiguous() else t.contiguous()


def _rows(t, name):
    """(t, shape, strides) of a [T, heads, dim] operand, its channels made contiguous."""
    if not isinstance(t, _Tensor) or t.dim() != 3:
        raise ValueError(f"{name} must have shape [tokens, heads, head_dim]")
    strides = t.stride()
    if strides[2] != 1:
        t = t.contiguous()
        strides = t.stride()
    return t, t.shape, strides


def _batch(tokens, q_heads, k_cache, v_cache, page_table, query_start, seq_lens):
    """The fields of m5b_paged_batch, the cache's shape and dtype, and the index tensors."""
    if (not isinstance(k_cache, _Tensor) or not isinstance(v_cache, _Tensor)
            or k_cache.dim() != 4 or k_cache.shape != v_cache.shape
            or k_cache.dtype is not v_cache.dtype):
        raise ValueError("k_cache and v_cache must share one [pages, kv_heads, page, head_dim] "
                         "shape and dtype")
    dtype = k_cache.dtype
    code = _CODE.get(dtype)
    if code is None:
        raise ValueError("cache dtype must be float16, bfloat16 or float32")
    shape = k_cache.shape
    pages, kv_heads, page, dim = shape
    if not (pages and kv_heads and page and dim):
        raise ValueError("the cache must be nonempty")
    kp, kh, ks, k1 = k_cache.stride()
    vp, vh, vs, v1 = v_cache.stride()
    if (k1 != 1 or v1 != 1) and dim > 1:
        raise ValueError("the cache's channels must be contiguous")
    query_start, seq_lens = _ints(query_start, "query_start"), _ints(seq_lens, "seq_lens")
    page_table = _ints(page_table, "page_table")
    batch = seq_lens.numel()
    if seq_lens.dim() != 1 or batch == 0 or query_start.shape != (batch + 1,):
        raise ValueError("seq_lens must be a nonempty vector [B] and query_start [B + 1]")
    if page_table.dim() != 2 or page_table.shape[0] != batch:
        raise ValueError("page_table must have shape [B, pages per sequence]")
    width = page_table.shape[1]
    fields = (tokens, batch, q_heads, kv_heads, dim, query_start.data_ptr(), seq_lens.data_ptr(),
              k_cache.data_ptr(), v_cache.data_ptr(), code, pages, page, kp, kh, ks, vp, vh, vs,
              page_table.data_ptr(), width, width)
    return fields, kv_heads, dim, dtype, [k_cache, v_cache, query_start, seq_lens, page_table]


def _call(function, args, index):
    """Run a C-ABI call on the device `index` and torch's current stream there."""
    if index == torch._C._cuda_getDevice():
        check(function(args, torch._C._cuda_getCurrentRawStream(index)))
    else:
        with torch.cuda.device(index):
            check(function(args, torch._C._cuda_getCurrentRawStream(index)))


def _device(tensors):
    """The CUDA device index that all the tensors share."""
    index = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != index or index < 0:
            return _lib.require_cuda(*tensors).index
    return index


_scratch_bytes: dict = {}
_COUNTER_BYTES = 4096  # M5B_PAGED_COUNTER_BYTES


def _counted(nbytes, index):
    buf = torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", index))
    buf[:_COUNTER_BYTES].zero_()
    return buf


def _scratch(index, dim):
    """The attention kernels' workspace on the current device, its counters zero:
    (pointer, bytes, the current stream, tensor to hold until the launch)."""
    stream = torch._C._cuda_getCurrentRawStream(index)
    need = _scratch_bytes.get((index, dim))
    if need is None:
        need = _scratch_bytes[index, dim] = int(_lib.lib().m5b_paged_attention_workspace_bytes(dim))
    if need <= 0:
        return 0, 0, stream, None
    buf = stream_buffer("paged", index, stream, need, _counted)
    return buf.data_ptr(), need, stream, buf


def _attend(index, dim, fields):
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return _attend(index, dim, fields)
    pointer, size, stream, _held = _scratch(index, dim)
    check(_lib.lib().m5b_paged_attention(_PACK_ATTEND.pack(*fields, pointer, size), stream))


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
    k, (tokens, kv, width), (kt, kh, _) = _rows(k, "k")
    v, v_shape, (vt, vh, _) = _rows(v, "v")
    x_dtype, q_heads = k.dtype, kv
    qt = qh = q_ptr = 0
    if q is not None:
        q, q_shape, (qt, qh, _) = _rows(q, "q")
        q_heads = q_shape[1]
        q_ptr = q.data_ptr()
    fields, kv_heads, dim, dtype, used = _batch(tokens, q_heads, k_cache, v_cache, page_table,
                                                query_start, seq_lens)
    if kv != kv_heads or width != dim:
        raise ValueError("k does not match the cache's heads and head_dim")
    x_code = _CODE.get(x_dtype)
    if x_code is None:
        raise ValueError("input dtype must be float16, bfloat16 or float32")
    if v_shape != (tokens, kv, dim) or v.dtype is not x_dtype:
        raise ValueError("q, k and v must share tokens and dtype, v also k's heads and head_dim")
    used += (k, v)
    if q is not None:
        if q_heads < 1 or q_heads % kv_heads:
            raise ValueError("q_heads must be a multiple of kv_heads")
        if q_shape != (tokens, q_heads, dim) or q.dtype is not x_dtype:
            raise ValueError("q, k and v must share tokens and dtype, q also k's head_dim")
        used.append(q)
    if layout not in ("half", "interleaved"):
        raise ValueError("layout must be 'half' or 'interleaved'")
    half = rows = table_dtype = cos_ptr = sin_ptr = 0
    if cos is not None or sin is not None:
        if (not isinstance(cos, _Tensor) or not isinstance(sin, _Tensor)
                or cos.dim() != 2 or cos.shape != sin.shape or cos.dtype is not sin.dtype
                or cos.dtype not in _CODE or cos.numel() == 0):
            raise ValueError("cos and sin must be matching floating tables [positions, R]")
        rows, half = cos.shape
        if 2 * half > dim:
            raise ValueError("cos and sin rotate 2 R channels, at most head_dim")
        table_dtype = _CODE[cos.dtype]
        cos, sin = cos.contiguous(), sin.contiguous()
        cos_ptr, sin_ptr = cos.data_ptr(), sin.data_ptr()
        used += (cos, sin)
    index = _device(used)
    out, out_ptr = None, 0
    if q is not None:
        out = torch.empty_like(q, dtype=dtype, memory_format=_CONTIGUOUS)
        out_ptr = out.data_ptr()
    if tokens > 0:
        _call(_lib.lib().m5b_paged_append, _PACK_APPEND.pack(
            *fields, q_ptr, k.data_ptr(), v.data_ptr(), x_code, qt, qh, kt, kh, vt, vh, cos_ptr,
            sin_ptr, table_dtype, rows, half, layout == "interleaved", out_ptr), index)
    return out


def _positive(value, name):
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
    in any case.  A token that sees no key returns zeros.  Slots behind a
    sequence's end, and pages that neither a prefix nor a new token's window
    reaches, may hold anything.  max_query_len: the
    most new tokens of any sequence; it selects the kernel, not the result.
    With return_lse also the fp32 [T, q_heads] natural logarithm of the sum of
    exp(x), -inf for a token that sees no key.  `out` may be given, any
    strides with contiguous channels.
    """
    q, (tokens, q_heads, width), (qt, qh, _) = _rows(q, "q")
    fields, kv_heads, dim, dtype, used = _batch(tokens, q_heads, k_cache, v_cache, page_table,
                                                query_start, seq_lens)
    if width != dim or q.dtype is not dtype:
        raise ValueError("q must have the cache's head_dim and dtype")
    if q_heads < 1 or q_heads % kv_heads:
        raise ValueError("q_heads must be a multiple of kv_heads")
    if dim > 256:
        raise NotImplementedError("head_dim above 256 is unsupported")
    if type(max_query_len) is not int and (isinstance(max_query_len, bool)
                                           or not isinstance(max_query_len, Integral)):
        raise ValueError("max_query_len must be a whole number")
    if max_query_len < 0:
        raise ValueError("max_query_len must not be negative")
    if max_query_len > _FAR:
        max_query_len = _FAR
    scale = dim ** -0.5 if scale is None else _positive(scale, "scale")
    softcap = 0.0 if softcap is None else _positive(softcap, "softcap")
    if window is None:
        window = 0
    elif isinstance(window, bool) or not isinstance(window, Integral) or window < 1:
        raise ValueError("window must be a positive whole number")
    elif window > _FAR:
        window = _FAR
    used.append(q)
    slopes_ptr = prefix_ptr = lse_ptr = 0
    if slopes is not None:
        if (not isinstance(slopes, _Tensor) or slopes.dtype is not torch.float32
                or slopes.shape != (q_heads,)):
            raise ValueError("slopes must be a float32 vector of length q_heads")
        slopes = slopes.contiguous()
        slopes_ptr = slopes.data_ptr()
        used.append(slopes)
    if prefix_lens is not None:
        prefix_lens = _ints(prefix_lens, "prefix_lens")
        if prefix_lens.shape != seq_lens.shape:
            raise ValueError("prefix_lens must be a vector [B]")
        prefix_ptr = prefix_lens.data_ptr()
        used.append(prefix_lens)
    if out is not None:
        if (not isinstance(out, _Tensor) or out.shape != q.shape or out.dtype is not dtype
                or out.stride(2) != 1):
            raise ValueError("out must match q, with contiguous channels")
        used.append(out)
    index = _device(used)
    if out is None:
        out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    lse = None
    if return_lse:
        lse = torch.empty((tokens, q_heads), dtype=torch.float32, device=q.device)
        lse_ptr = lse.data_ptr()
    if tokens > 0:
        ot, oh, _ = out.stride()
        _attend(index, dim, fields + (
            q.data_ptr(), qt, qh, out.data_ptr(), ot, oh, lse_ptr, max_query_len, scale, softcap,
            slopes_ptr, window, prefix_ptr))
    return (out, lse) if return_lse else out
