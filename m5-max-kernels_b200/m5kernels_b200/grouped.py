"""Block-scaled E4M3 products, and products whose rows are grouped by expert.

`block_quantize` makes E4M3 codes (uint8, as `quantize` does) with one fp32
scale for each block of 128 channels of a row (activations) or of 128 rows
(weights); `block_gemm` multiplies such operands.  `grouped_gemm` multiplies
each group of rows by its own weight, for operands of either kind of scales and
for unquantized ones.  An expert layer is

    codes, scales = block_quantize(x, rows=order)           # rows in the order of their experts
    h = grouped_gemm(codes, w_up, group_start, "fp8", a_scales=scales, b_scales=w_up_scales,
                     output_dtype=torch.bfloat16)           # [T, up and gate]
    codes, scales = block_quantize(h[:, :d], gate=h[:, d:])
    y = grouped_gemm(codes, w_down, group_start, "fp8", ...)

The group's bounds are read on the device: nothing here waits for the GPU, and
a captured CUDA graph may be replayed after they changed.  The reference's GEMM
takes one weight and one scale a row and channel
(src/m5kernels/metal.py:158-269); these operators have no twin there.
"""

from __future__ import annotations

import struct

import torch

from . import _lib
from ._lib import check
from .paged import _call, _device, _ints

_Tensor = torch.Tensor
BLOCK = 128
_FLOAT = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_OPERAND = {mode: (dtype, _lib.MODE[mode], dtype.itemsize) for mode, dtype in (
    ("int8", torch.int8), ("fp8", torch.uint8), ("bf16", torch.bfloat16), ("fp16", torch.float16))}
_NO_SCALES = (0,) * 7
_F32 = torch.float32
_MOST_GROUPS = 1024
# m5b_block_quantize_args and m5b_grouped_gemm_args (include/m5b200.h): every field is 8 bytes
_PACK_QUANTIZE = struct.Struct("@14q")
_PACK_GEMM = struct.Struct("@23q")


def _row_index(rows):
    if not isinstance(rows, _Tensor) or rows.dtype is not torch.int32 or rows.dim() != 1:
        raise ValueError("rows must be an int32 vector")
    return rows.contiguous()


def block_quantize(x, *, gate=None, rows=None, block_rows=1):
    """E4M3 codes with a scale for each block of 128 channels -> (codes uint8, scales fp32).

    scale = max|v| / 448 over the block (1 where that is 0), codes =
    E4M3(v / scale), nearest even, saturating, the quotient in fp32; the last
    block of a row may be shorter.  Which of the two zeros a v of -0 gets is
    not specified.

    block_rows 1 (activations): x [T, K] -> codes [T, K], scales [T, ceil(K / 128)].
    v = x, or with `gate` [T, K] v = silu(gate) * x in fp32 (the step between
    the products of a gated FFN).  With `rows` int32 [R], row r is x[rows[r]]:
    codes [R, K]; indices outside x give rows of zeros.
    block_rows 128 (weights): x [N, K] or [E, N, K]; one scale for 128 rows x
    128 channels, scales [..., ceil(N / 128), ceil(K / 128)].

    x and gate: float16, bfloat16 or float32; views with contiguous channels
    are read in place.  A block that holds an infinity or NaN gets a scale that
    is not finite.
    """
    code = _FLOAT.get(x.dtype) if isinstance(x, _Tensor) else None
    if code is None:
        raise ValueError("input dtype must be float16, bfloat16 or float32")
    if type(block_rows) is not int or block_rows not in (1, BLOCK):
        raise ValueError("block_rows must be 1 or 128")
    if block_rows == 1:
        if x.dim() != 2 or x.shape[1] == 0:
            raise ValueError("input must have shape [rows, K]")
    else:
        if x.dim() not in (2, 3) or 0 in x.shape:
            raise ValueError("weights must have nonempty shape [N, K] or [E, N, K]")
        if gate is not None or rows is not None:
            raise ValueError("gate and rows need block_rows 1")
    shape, strides = x.shape, x.stride()
    k, out_rows = shape[-1], shape[-2]
    if strides[-1] != 1:
        x = x.contiguous()
        strides = x.stride()
    used = None
    gate_ptr = gate_row = index_ptr = 0
    if gate is not None:
        if not isinstance(gate, _Tensor) or gate.shape != shape or gate.dtype is not x.dtype:
            raise ValueError("gate must have x's shape and dtype")
        if gate.stride(1) != 1:
            gate = gate.contiguous()
        gate_ptr, gate_row = gate.data_ptr(), gate.stride(0)
        used = [x, gate]
    if rows is not None:
        rows = _row_index(rows)
        index_ptr, out_rows = rows.data_ptr(), rows.shape[0]
        used = [x, rows] if used is None else [*used, rows]
    index = x.get_device() if used is None else _device(used)
    if index < 0:
        _lib.require_cuda(x)
    batch, batch_stride = (shape[0], strides[0]) if len(shape) == 3 else (1, 0)
    lead, device = shape[:-2], x.device
    # (sizes as arguments of their own take torch.empty two thirds of a tuple's time)
    codes = torch.empty(*lead, out_rows, k, dtype=torch.uint8, device=device)
    scales = torch.empty(*lead, -(-out_rows // block_rows), -(-k // BLOCK), dtype=torch.float32,
                         device=device)
    if out_rows > 0:
        _call(_lib.lib().m5b_block_quantize, _PACK_QUANTIZE.pack(
            x.data_ptr(), code, shape[-2], strides[-2], batch_stride, gate_ptr, gate_row,
            index_ptr, out_rows, k, batch, block_rows, codes.data_ptr(), scales.data_ptr()), index)
    return codes, scales


def _product(a, b, rows, groups, n, k, group_start, mode, a_scales, b_scales, output_dtype, out):
    """Both products: b [groups, N, K], or with group_start None [N, K] for all rows."""
    expected, code, size = _OPERAND[mode]
    if a.dtype is not expected or b.dtype is not expected:
        raise ValueError("operand dtypes must match the declared mode")
    if k * size & 15:
        raise NotImplementedError(f"K*{size} bytes per row must be a multiple of 16 for TMA; "
                                  "padding is not implicit")
    index = a.get_device()
    same = index >= 0 and b.get_device() == index
    blocks, scale_fields = False, _NO_SCALES
    if size == 1:
        if (not isinstance(a_scales, _Tensor) or not isinstance(b_scales, _Tensor)
                or a_scales.dtype is not _F32 or b_scales.dtype is not _F32):
            raise ValueError("float32 scales required" if group_start is not None else
                             "float32 scales of blocks of 128 channels of K required")
        a_shape, b_shape = a_scales.shape, b_scales.shape
        if len(a_shape) == 2 and mode == "fp8":
            kb, nb = -(-k // BLOCK), -(-n // BLOCK)
            blocks = a_shape == (rows, kb) and b_shape == (
                (nb, kb) if group_start is None else (groups, nb, kb))
        if not blocks and (group_start is None or a_shape != (rows,) or b_shape != (groups, n)):
            raise ValueError("scales must be those of rows and channels, or (fp8) of blocks of "
                             "128 channels of K")
        # between rows and blocks of a, groups, channels (or blocks of them) and blocks of b
        if not blocks:
            strides = (*a_scales.stride(), 0, *b_scales.stride(), 0)
        elif group_start is None:
            strides = (*a_scales.stride(), 0, *b_scales.stride())
        else:
            strides = (*a_scales.stride(), *b_scales.stride())
        scale_fields = (a_scales.data_ptr(), b_scales.data_ptr(), *strides)
        same = same and a_scales.get_device() == index and b_scales.get_device() == index
    elif a_scales is not None or b_scales is not None:
        raise ValueError("scales belong to int8 and fp8 operands")
    zero_rest = out is None
    if out is None:
        out_dtype = output_dtype or _F32
    else:
        if (not isinstance(out, _Tensor) or out.shape != (rows, n)
                or (n > 1 and out.stride(1) != 1)):
            raise ValueError("out must have shape [rows, N] and contiguous channels")
        out_dtype = out.dtype
        if output_dtype is not None and output_dtype is not out_dtype:
            raise ValueError("output_dtype must be out's")
        same = same and out.get_device() == index
    out_code = _FLOAT.get(out_dtype)
    if out_code is None:
        raise NotImplementedError("output dtype must be bfloat16, float16 or float32")
    start_ptr = 0
    if group_start is not None:
        start_ptr = group_start.data_ptr()
        same = same and group_start.get_device() == index
    if not same:
        _lib.require_cuda(a, b, a_scales, b_scales, out, group_start)
    if out is None:
        out = torch.empty(rows, n, dtype=out_dtype, device=a.device)
    if rows > 0:
        # rows that TMA can read: contiguous channels, on the 16-byte grid
        off = 16 // size - 1
        a_ptr, (a_row, a_step) = a.data_ptr(), a.stride()
        if a_ptr & 15 or a_step != 1 or a_row & off or a_row <= 0:
            a = a.clone(memory_format=torch.contiguous_format)
            a_ptr, (a_row, _) = a.data_ptr(), a.stride()
        b_ptr, strides = b.data_ptr(), b.stride()
        b_group, b_row = strides[0], strides[-2]
        if (b_ptr & 15 or strides[-1] != 1 or (b_row | b_group) & off or b_row <= 0
                or b_group <= 0):
            b = b.clone(memory_format=torch.contiguous_format)
            b_ptr, strides = b.data_ptr(), b.stride()
            b_group, b_row = strides[0], strides[-2]
        _call(_lib.lib().m5b_grouped_gemm, _PACK_GEMM.pack(
            a_ptr, b_ptr, code, rows, groups, n, k, a_row, b_group, b_row, start_ptr, blocks,
            *scale_fields, out.data_ptr(), out_code, out.stride(0), zero_rest), index)
    return out


def block_gemm(a, b, a_scales, b_scales, *, output_dtype=None, out=None):
    """Block-scaled E4M3 product a[M, K] @ b[N, K].T -> [M, N].

        out[m, n] = sum over blocks g of 128 channels of K of
                    (a_scales[m, g] * b_scales[n // 128, g]) * sum_{k in g} a[m, k] b[n, k]

    a, b: E4M3 codes (uint8), a_scales fp32 [M, ceil(K / 128)], b_scales fp32
    [ceil(N / 128), ceil(K / 128)], as `block_quantize` makes them (block_rows
    1 and 128); views of any strides are fine, but operands whose rows do not
    start on 16-byte boundaries are copied for every call.  Sums and scales in
    fp32; the product of two scales has to be in fp32's range.  K a multiple
    of 16.
    output_dtype: float32 unless given; `out` may be given, with contiguous
    channels and rows that do not overlap.
    """
    if isinstance(a, _Tensor) and isinstance(b, _Tensor):
        a_shape, b_shape = a.shape, b.shape
        if len(a_shape) == 2 and len(b_shape) == 2:
            (m, k), (n, b_k) = a_shape, b_shape
            if k == b_k and n and k:
                return _product(a, b, m, 1, n, k, None, "fp8", a_scales, b_scales, output_dtype,
                                out)
    raise ValueError("A and B must be matrices [M, K] and [N, K]")


def grouped_gemm(a, b, group_start, mode="bf16", *, a_scales=None, b_scales=None,
                 output_dtype=None, out=None):
    """Rows grouped by expert: out[t] = a[t] @ b[e].T for group_start[e] <= t < group_start[e + 1].

    a [T, K], b [E, N, K] (E up to 1024), group_start int32 [E + 1], ascending,
    read on the device; groups may be empty.  mode: "bf16", "fp16", "int8" or
    "fp8" (uint8 E4M3 codes), operands as in `gemm`.  Scales of int8 and fp8:
    a_scales [T] and b_scales [E, N], v = (acc * a_scales[t]) * b_scales[e, n];
    or for fp8 those of `block_gemm`, a_scales [T, ceil(K / 128)] and b_scales
    [E, ceil(N / 128), ceil(K / 128)].  INT32 (int8) or FP32 accumulation.
    K times the element size a multiple of 16.  Operands whose rows do not
    start on 16-byte boundaries, or whose groups or rows are expanded, are
    copied whole for every call.

    Rows outside every group are zero; where `out` is given (contiguous
    channels, rows that do not overlap, output_dtype its own) they keep what it
    holds.  output_dtype: float32 unless given.
    """
    if mode not in _OPERAND:
        if mode in ("fp32", "mxint8"):
            raise NotImplementedError(f"{mode} operands are not supported by the grouped GEMM")
        raise ValueError(f"unknown GEMM mode {mode!r}")
    a_shape = a.shape if isinstance(a, _Tensor) else ()
    b_shape = b.shape if isinstance(b, _Tensor) else ()
    if (len(a_shape) != 2 or len(b_shape) != 3 or a_shape[1] != b_shape[2]
            or not (b_shape[0] and b_shape[1] and b_shape[2])):
        raise ValueError("A and B must have shapes [T, K] and [E, N, K]")
    (rows, k), (groups, n, _) = a_shape, b_shape
    group_start = _ints(group_start, "group_start")
    if group_start.shape != (groups + 1,):
        raise ValueError("group_start must be a vector [E + 1]")
    if groups > _MOST_GROUPS:
        raise NotImplementedError("more than 1024 groups are unsupported")
    if k > 133144 and mode == "int8":
        raise NotImplementedError("INT32 worst-case overflow bound exceeded")
    return _product(a, b, rows, groups, n, k, group_start, mode, a_scales, b_scales, output_dtype,
                    out)
