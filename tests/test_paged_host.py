"""What the paged operators refuse, and their argument records, without a GPU."""

import ctypes
import re
import struct
from pathlib import Path

import pytest
import torch

from paged_cases import Batch

ROOT = Path(__file__).resolve().parents[1]
BF16 = torch.bfloat16


def call(name, **change):
    import m5kernels_b200 as m

    batch = Batch([1, 2], [3, 0], q_heads=4, kv_heads=2, dim=64, page=16, dtype=BF16)
    args = dict(k_cache=batch.k_cache, v_cache=batch.v_cache, page_table=batch.table,
                query_start=batch.query_start, seq_lens=batch.seq_lens)
    if name == "paged_append":
        args.update(k=torch.ones(3, 2, 64, dtype=BF16), v=torch.ones(3, 2, 64, dtype=BF16))
    else:
        args.update(q=batch.q, max_query_len=2)
    args.update(change)
    return getattr(m, name)(**args)


CACHE = [
    (dict(k_cache=torch.ones(2, 2, 16, dtype=BF16)), "one \\[pages"),
    (dict(k_cache=torch.ones(2, 2, 16, 64, dtype=torch.float16)), "one \\[pages"),
    (dict(k_cache=torch.ones(5, 2, 16, 64, dtype=torch.int8),
          v_cache=torch.ones(5, 2, 16, 64, dtype=torch.int8)), "cache dtype"),
    (dict(k_cache=torch.ones(0, 2, 16, 64, dtype=BF16),
          v_cache=torch.ones(0, 2, 16, 64, dtype=BF16)), "nonempty"),
    (dict(k_cache=torch.ones(5, 2, 64, 16, dtype=BF16).transpose(2, 3),
          v_cache=torch.ones(5, 2, 16, 64, dtype=BF16)), "contiguous"),
    (dict(page_table=torch.zeros(2, 1)), "int32"),
    (dict(page_table=torch.zeros(3, 1, dtype=torch.int32)), "page_table must"),
    (dict(query_start=torch.zeros(2, dtype=torch.int32)), "query_start \\[B"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), "int32"),
    (dict(seq_lens=torch.zeros(0, dtype=torch.int32)), "nonempty"),
]


@pytest.mark.parametrize("name", ["paged_append", "paged_attention"])
@pytest.mark.parametrize("change,match", CACHE)
def test_cache_refusals(name, change, match):
    with pytest.raises(ValueError, match=match):
        call(name, **change)


@pytest.mark.parametrize("change,error,match", [
    (dict(q=torch.ones(3, 4, dtype=BF16)), ValueError, "shape"),
    (dict(q=torch.ones(3, 4, 32, dtype=BF16)), ValueError, "head_dim"),
    (dict(q=torch.ones(3, 4, 64)), ValueError, "dtype"),
    (dict(q=torch.ones(3, 3, 64, dtype=BF16)), ValueError, "multiple"),
    (dict(max_query_len=-1), ValueError, "max_query_len"),
    (dict(max_query_len=2.0), ValueError, "max_query_len"),
    (dict(scale=0.0), ValueError, "scale"),
    (dict(scale=float("nan")), ValueError, "scale"),
    (dict(softcap=-3.0), ValueError, "softcap"),
    (dict(softcap=float("inf")), ValueError, "softcap"),
    (dict(window=0), ValueError, "window"),
    (dict(window=1.5), ValueError, "window"),
    (dict(slopes=torch.ones(2)), ValueError, "slopes"),
    (dict(slopes=torch.ones(4, dtype=torch.float64)), ValueError, "slopes"),
    (dict(prefix_lens=torch.ones(3, dtype=torch.int32)), ValueError, "prefix_lens"),
    (dict(prefix_lens=torch.ones(2)), ValueError, "prefix_lens"),
    (dict(out=torch.ones(3, 4, 64)), ValueError, "out"),
    (dict(out=torch.ones(3, 64, 4, dtype=BF16).transpose(1, 2)), ValueError, "out"),
    (dict(q=torch.ones(3, 4, 320, dtype=BF16), k_cache=torch.ones(5, 2, 16, 320, dtype=BF16),
          v_cache=torch.ones(5, 2, 16, 320, dtype=BF16)), NotImplementedError, "256"),
])
def test_attention_refusals(change, error, match):
    with pytest.raises(error, match=match):
        call("paged_attention", **change)


@pytest.mark.parametrize("change,match", [
    (dict(k=torch.ones(3, 2, 32, dtype=BF16)), "head_dim"),
    (dict(v=torch.ones(2, 2, 64, dtype=BF16)), "share"),
    (dict(v=torch.ones(3, 2, 64)), "share"),
    (dict(k=torch.ones(3, 2, 64, dtype=torch.int8), v=torch.ones(3, 2, 64, dtype=torch.int8)),
     "input dtype"),
    (dict(q=torch.ones(3, 3, 64, dtype=BF16)), "multiple"),
    (dict(q=torch.ones(4, 4, 64, dtype=BF16)), "share"),
    (dict(layout="split"), "layout"),
    (dict(cos=torch.ones(8, 32)), "cos and sin"),
    (dict(cos=torch.ones(8, 32), sin=torch.ones(8, 16)), "cos and sin"),
    (dict(cos=torch.ones(8, 33), sin=torch.ones(8, 33)), "2 R"),
    (dict(cos=torch.ones(8, 4, dtype=torch.int32), sin=torch.ones(8, 4, dtype=torch.int32)),
     "cos and sin"),
])
def test_append_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        call("paged_append", **change)


@pytest.mark.parametrize("name", ["paged_append", "paged_attention"])
def test_cpu_tensors_are_refused(name):
    from m5kernels_b200._lib import ExtensionMissing

    with pytest.raises(ExtensionMissing):
        call(name)


def test_argument_records_match_the_header():
    """Every field of the C structs is 8 bytes, as many as the packed records hold."""
    from m5kernels_b200 import paged

    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "m5b200.h").read_text(), flags=re.S)

    def fields(name):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        res = []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            if decl.startswith("m5b_paged_batch"):
                res += fields("m5b_paged_batch")
            else:
                kind = "d" if decl.startswith("double") else "q"
                assert kind == "d" or "int64_t" in decl or "*" in decl, decl
                res += [kind] * (decl.count(",") + 1)
        return res

    for name, packed in (("m5b_paged_append_args", paged._PACK_APPEND),
                         ("m5b_paged_attention_args", paged._PACK_ATTEND)):
        layout = "".join(fields(name))
        expanded = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([qd])", packed.format))
        assert expanded == layout and struct.calcsize(packed.format) == 8 * len(layout)


def test_abi_refusals_without_a_gpu():
    """Checks of sizes and pointers come before any CUDA call."""
    from m5kernels_b200 import _lib, paged

    lib = _lib.lib()
    fake = 1 << 20
    good = [3, 2, 4, 2, 64, fake, fake, fake, fake, _lib.BF16, 5, 16] + [1024, 512, 64] * 2 + [fake, 1, 1]

    def attend(at=None, value=None, **kw):
        fields = list(good)
        if at is not None:
            fields[at] = value
        opt = dict(q=fake, out=fake, scale=1.0, softcap=0.0, window=0, longest=2)
        opt.update(kw)
        return lib.m5b_paged_attention(paged._PACK_ATTEND.pack(
            *fields, opt["q"], 256, 64, opt["out"], 256, 64, 0, opt["longest"], opt["scale"],
            opt["softcap"], 0, opt["window"], 0, 0, 0), None)

    for at, value, code, text in ((0, -1, _lib.EINVAL, b"positive"), (1, 0, _lib.EINVAL, b"positive"),
                                  (2, 3, _lib.EINVAL, b"multiple"), (4, 300, _lib.EUNSUPPORTED, b"256"),
                                  (5, 0, _lib.EINVAL, b"required"), (9, _lib.I8, _lib.EINVAL, b"dtype"),
                                  (11, 0, _lib.EINVAL, b"pages"), (0, 1 << 40, _lib.EUNSUPPORTED, b"range"),
                                  (18, 0, _lib.EINVAL, b"required")):
        assert attend(at, value) == code and text in lib.m5b_last_error(), (at, value)
    assert attend(q=0) == _lib.EINVAL and b"q and out" in lib.m5b_last_error()
    assert attend(scale=-1.0) == _lib.EINVAL and b"scale" in lib.m5b_last_error()
    assert attend(softcap=float("nan")) == _lib.EINVAL and b"softcap" in lib.m5b_last_error()
    assert attend(window=-1) == _lib.EINVAL and b"window" in lib.m5b_last_error()
    assert lib.m5b_paged_attention(None, None) == _lib.EINVAL
    assert lib.m5b_paged_append(None, None) == _lib.EINVAL

    def append(**kw):
        opt = dict(k=fake, q=0, x=_lib.BF16, cos=fake, rows=8, half=32, q_out=0)
        opt.update(kw)
        return lib.m5b_paged_append(paged._PACK_APPEND.pack(
            *good, opt["q"], opt["k"], fake, opt["x"], 256, 64, 128, 64, 128, 64, opt["cos"], fake,
            _lib.F32, opt["rows"], opt["half"], 0, opt["q_out"]), ctypes.c_void_p(0))

    assert append(k=0) == _lib.EINVAL and b"k and v" in lib.m5b_last_error()
    assert append(half=33) == _lib.EINVAL and b"fit" in lib.m5b_last_error()
    assert append(cos=0) == _lib.EINVAL and b"tables" in lib.m5b_last_error()
    assert append(rows=0) == _lib.EINVAL and b"tables" in lib.m5b_last_error()
    assert append(x=_lib.I8) == _lib.EINVAL and b"dtype" in lib.m5b_last_error()
    assert append(q=fake) == _lib.EINVAL and b"q_out" in lib.m5b_last_error()
