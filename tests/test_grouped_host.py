"""What the block-scaled and grouped products refuse, and their argument records, without a GPU."""

import re
import struct
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
BF16, U8, I8, I32 = torch.bfloat16, torch.uint8, torch.int8, torch.int32


def refused(fn, error, match, *args, **kw):
    with pytest.raises(error, match=match):
        fn(*args, **kw)


@pytest.mark.parametrize("x,kw,match", [
    (torch.ones(4, 128, dtype=torch.float64), {}, "input dtype"),
    (torch.ones(4, 128, dtype=I8), {}, "input dtype"),
    (torch.ones(128), {}, "shape"),
    (torch.ones(2, 4, 128), {}, "shape"),
    (torch.ones(4, 0), {}, "shape"),
    (torch.ones(4, 128), dict(block_rows=64), "block_rows"),
    (torch.ones(4, 128), dict(block_rows=True), "block_rows"),
    (torch.ones(4, 128), dict(block_rows=1.0), "block_rows"),
    (torch.ones(128), dict(block_rows=128), "nonempty"),
    (torch.ones(0, 128), dict(block_rows=128), "nonempty"),
    (torch.ones(1, 2, 4, 128), dict(block_rows=128), "nonempty"),
    (torch.ones(4, 128), dict(block_rows=128, gate=torch.ones(4, 128)), "block_rows 1"),
    (torch.ones(4, 128), dict(block_rows=128, rows=torch.zeros(4, dtype=I32)), "block_rows 1"),
    (torch.ones(4, 128), dict(gate=torch.ones(4, 64)), "gate"),
    (torch.ones(4, 128), dict(gate=torch.ones(4, 128, dtype=BF16)), "gate"),
    (torch.ones(4, 128), dict(rows=torch.zeros(4, dtype=torch.int64)), "rows"),
    (torch.ones(4, 128), dict(rows=torch.zeros(4, 1, dtype=I32)), "rows"),
    (torch.ones(4, 128), dict(rows=[0, 1]), "rows"),
])
def test_block_quantize_refusals(x, kw, match):
    import m5kernels_b200 as m

    refused(m.block_quantize, ValueError, match, x, **kw)


def block_args(**change):
    args = dict(a=torch.zeros(4, 256, dtype=U8), b=torch.zeros(130, 256, dtype=U8),
                a_scales=torch.ones(4, 2), b_scales=torch.ones(2, 2))
    args.update(change)
    return args


@pytest.mark.parametrize("change,error,match", [
    (dict(a=torch.zeros(256, dtype=U8)), ValueError, "matrices"),
    (dict(a=torch.zeros(4, 128, dtype=U8)), ValueError, "matrices"),
    (dict(b=torch.zeros(0, 256, dtype=U8)), ValueError, "matrices"),
    (dict(a=torch.zeros(4, 0, dtype=U8), b=torch.zeros(130, 0, dtype=U8)), ValueError, "matrices"),
    (dict(a=torch.zeros(4, 256, dtype=I8)), ValueError, "dtypes"),
    (dict(b=torch.zeros(130, 256)), ValueError, "dtypes"),
    (dict(a_scales=torch.ones(4)), ValueError, "blocks"),
    (dict(b_scales=None), ValueError, "blocks"),
    (dict(a_scales=torch.ones(4, 3)), ValueError, "scales"),
    (dict(b_scales=torch.ones(1, 2)), ValueError, "scales"),
    (dict(a_scales=torch.ones(4, 2, dtype=BF16)), ValueError, "float32"),
    (dict(a=torch.zeros(4, 250, dtype=U8), b=torch.zeros(130, 250, dtype=U8)),
     NotImplementedError, "multiple of 16"),
    (dict(output_dtype=torch.float64), NotImplementedError, "output dtype"),
    (dict(output_dtype=I32), NotImplementedError, "output dtype"),
    (dict(out=torch.ones(4, 129)), ValueError, "out"),
    (dict(out=torch.ones(130, 4).t()), ValueError, "out"),
    (dict(out=torch.ones(4, 130), output_dtype=BF16), ValueError, "output_dtype"),
    (dict(out=torch.ones(4, 130, dtype=I32)), NotImplementedError, "output dtype"),
])
def test_block_gemm_refusals(change, error, match):
    import m5kernels_b200 as m

    refused(m.block_gemm, error, match, **block_args(**change))


def grouped_args(**change):
    args = dict(a=torch.zeros(5, 64, dtype=BF16), b=torch.zeros(3, 8, 64, dtype=BF16),
                group_start=torch.tensor([0, 2, 2, 5], dtype=I32), mode="bf16")
    args.update(change)
    return args


INT8 = dict(a=torch.zeros(5, 64, dtype=I8), b=torch.zeros(3, 8, 64, dtype=I8), mode="int8")


@pytest.mark.parametrize("change,error,match", [
    (dict(mode="fp32"), NotImplementedError, "fp32"),
    (dict(mode="mxint8"), NotImplementedError, "mxint8"),
    (dict(mode="fp4"), ValueError, "unknown"),
    (dict(b=torch.zeros(8, 64, dtype=BF16)), ValueError, "shapes"),
    (dict(a=torch.zeros(5, 32, dtype=BF16)), ValueError, "shapes"),
    (dict(b=torch.zeros(0, 8, 64, dtype=BF16)), ValueError, "shapes"),
    (dict(group_start=torch.tensor([0, 2, 5], dtype=I32)), ValueError, "group_start"),
    (dict(group_start=torch.tensor([0, 2, 2, 5])), ValueError, "int32"),
    (dict(group_start=None), ValueError, "int32"),
    (dict(a=torch.zeros(5, 64, dtype=torch.float16)), ValueError, "dtypes"),
    (dict(a_scales=torch.ones(5)), ValueError, "scales belong"),
    (dict(a=torch.zeros(5, 60, dtype=BF16), b=torch.zeros(3, 8, 60, dtype=BF16)),
     NotImplementedError, "multiple of 16"),
    (dict(INT8), ValueError, "float32 scales"),
    (dict(INT8, a_scales=torch.ones(5), b_scales=torch.ones(8)), ValueError, "scales must"),
    (dict(INT8, a_scales=torch.ones(5, 1), b_scales=torch.ones(3, 1, 1)), ValueError,
     "scales must"),
    (dict(INT8, a_scales=torch.ones(5), b_scales=torch.ones(3, 1, 1)), ValueError, "scales must"),
    (dict(b=torch.zeros(1, 1, 64, dtype=BF16).expand(1025, 1, 64),
          group_start=torch.zeros(1026, dtype=I32)), NotImplementedError, "1024"),
    (dict(a=torch.zeros(5, 133152, dtype=I8), b=torch.zeros(3, 1, 133152, dtype=I8), mode="int8"),
     NotImplementedError, "overflow"),
    (dict(out=torch.zeros(5, 9)), ValueError, "out"),
])
def test_grouped_gemm_refusals(change, error, match):
    import m5kernels_b200 as m

    refused(m.grouped_gemm, error, match, **grouped_args(**change))


def test_cpu_tensors_are_refused():
    import m5kernels_b200 as m
    from m5kernels_b200._lib import ExtensionMissing

    refused(m.block_quantize, ExtensionMissing, "CUDA", torch.ones(4, 128))
    refused(m.block_quantize, ExtensionMissing, "CUDA", torch.ones(4, 128), block_rows=128)
    refused(m.block_gemm, ExtensionMissing, "CUDA", **block_args())
    refused(m.grouped_gemm, ExtensionMissing, "CUDA", **grouped_args())


def test_argument_records_match_the_header():
    """Every field of the C structs is 8 bytes, as many as the packed records hold."""
    from m5kernels_b200 import grouped

    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "m5b200.h").read_text(), flags=re.S)
    for name, packed in (("m5b_block_quantize_args", grouped._PACK_QUANTIZE),
                         ("m5b_grouped_gemm_args", grouped._PACK_GEMM)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        decls = [d.strip() for d in body.split(";") if d.strip()]
        assert all("int64_t" in d or "*" in d for d in decls)
        count = sum(d.count(",") + 1 for d in decls)
        assert packed.format == f"@{count}q" and struct.calcsize(packed.format) == 8 * count


FAKE = 1 << 20


def test_quantize_abi_refusals_without_a_gpu():
    """Checks of sizes and pointers come before any CUDA call."""
    from m5kernels_b200 import _lib, grouped

    lib = _lib.lib()
    names = ("x", "x_dtype", "x_rows", "x_row", "x_batch", "gate", "gate_row", "index", "rows",
             "k", "batch", "block_rows", "q", "scales")
    good = dict(zip(names, (FAKE, _lib.BF16, 4, 128, 0, 0, 0, 0, 4, 128, 1, 1, FAKE, FAKE)))

    def call(**change):
        return lib.m5b_block_quantize(
            grouped._PACK_QUANTIZE.pack(*dict(good, **change).values()), None)

    for change, code, text in (
            (dict(x_dtype=_lib.I8), _lib.EINVAL, b"dtype"),
            (dict(block_rows=2), _lib.EINVAL, b"block_rows"),
            (dict(rows=-1, x_rows=-1), _lib.EINVAL, b"positive"),
            (dict(k=0), _lib.EINVAL, b"positive"),
            (dict(batch=2), _lib.EINVAL, b"batch"),
            (dict(block_rows=128, gate=FAKE), _lib.EINVAL, b"block_rows 1"),
            (dict(block_rows=128, index=FAKE), _lib.EINVAL, b"block_rows 1"),
            (dict(rows=5), _lib.EINVAL, b"row_index"),
            (dict(x=0), _lib.EINVAL, b"required"),
            (dict(q=0), _lib.EINVAL, b"required"),
            (dict(scales=0), _lib.EINVAL, b"required"),
            (dict(rows=1 << 31, x_rows=1 << 31), _lib.EUNSUPPORTED, b"range"),
            (dict(rows=1 << 30, x_rows=1 << 30, k=1 << 12), _lib.EUNSUPPORTED, b"range"),
            (dict(block_rows=128, rows=1 << 20, x_rows=1 << 20, batch=1 << 20), _lib.EUNSUPPORTED,
             b"range")):
        assert call(**change) == code and text in lib.m5b_last_error(), change
    assert call(rows=0, x_rows=0) == _lib.OK and lib.m5b_last_error() == b""
    assert lib.m5b_block_quantize(None, None) == _lib.EINVAL


def test_grouped_abi_refusals_without_a_gpu():
    from m5kernels_b200 import _lib, grouped

    lib = _lib.lib()
    names = ("a", "b", "mode", "rows", "groups", "n", "k", "a_row", "b_group", "b_row", "start",
             "block", "sa", "sb", "sa_row", "sa_block", "sb_group", "sb_row", "sb_block", "out",
             "out_dtype", "out_row", "zero_rest")
    good = dict(zip(names, (FAKE, FAKE, _lib.MODE["fp8"], 5, 3, 8, 64, 64, 512, 64, FAKE, 0, FAKE,
                            FAKE, 1, 0, 8, 1, 0, FAKE, _lib.BF16, 8, 1)))

    def call(**change):
        return lib.m5b_grouped_gemm(grouped._PACK_GEMM.pack(*dict(good, **change).values()), None)

    for change, code, text in (
            (dict(mode=7), _lib.EINVAL, b"mode"),
            (dict(mode=_lib.MODE["fp32"]), _lib.EUNSUPPORTED, b"fp32"),
            (dict(rows=-1), _lib.EINVAL, b"positive"),
            (dict(groups=0), _lib.EINVAL, b"positive"),
            (dict(n=0), _lib.EINVAL, b"positive"),
            (dict(k=0), _lib.EINVAL, b"positive"),
            (dict(start=0), _lib.EINVAL, b"group_start"),
            (dict(block=1, mode=_lib.MODE["int8"]), _lib.EINVAL, b"block scales"),
            (dict(out_dtype=_lib.I32), _lib.EUNSUPPORTED, b"output dtype"),
            (dict(groups=1025), _lib.EUNSUPPORTED, b"1024"),
            (dict(mode=_lib.MODE["int8"], k=133152), _lib.EUNSUPPORTED, b"overflow"),
            (dict(rows=1 << 31), _lib.EUNSUPPORTED, b"range"),
            (dict(rows=1 << 30, n=1 << 20), _lib.EUNSUPPORTED, b"range"),
            (dict(a=0), _lib.EINVAL, b"required"),
            (dict(out=0), _lib.EINVAL, b"required"),
            (dict(sa=0), _lib.EINVAL, b"scales"),
            (dict(a=FAKE + 8), _lib.EUNSUPPORTED, b"16-byte"),
            (dict(a_row=72), _lib.EUNSUPPORTED, b"16-byte"),
            (dict(b_row=0), _lib.EUNSUPPORTED, b"16-byte"),
            (dict(b_group=1 << 40), _lib.EUNSUPPORTED, b"16-byte")):
        assert call(**change) == code and text in lib.m5b_last_error(), change
    assert call(rows=0) == _lib.OK and lib.m5b_last_error() == b""
    assert lib.m5b_grouped_gemm(None, None) == _lib.EINVAL
