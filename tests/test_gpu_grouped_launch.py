"""Block-scaled and grouped products next to other work: kernels before them, errors before them."""

import pytest
import torch

from grouped_cases import Experts

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F32, U8 = torch.bfloat16, torch.float32, torch.uint8


@pytest.fixture(scope="module")
def ops():
    import m5kernels_b200 as m
    from m5kernels_b200 import _lib

    yield m
    assert _lib.device_status() == 0  # no bounded wait gave up


def test_a_long_kernel_before_a_dense_product(ops):
    """A product starts on SMs that the kernel before leaves idle, and waits there for its end.

    That is no wait of its own pipeline, whose waits give up after 2 s.  The kernel before is a
    block-scaled product of 256 x 9472 outputs, 37 tiles on 148 SMs, over a K that takes longer
    than that: its rows lie 16 bytes apart in one buffer, and its scales are one number.
    """
    from m5kernels_b200 import _lib

    rows, n = 256, 37 * 256
    most = 2**31 - 2**20
    buf = torch.zeros(most + 16 * n, dtype=U8, device=DEV)
    one = torch.ones(1, 1, device=DEV)

    def long_product(k):
        out = torch.empty(rows, n, dtype=BF16, device=DEV)
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        ops.block_gemm(buf.as_strided((rows, k), (16, 1)), buf.as_strided((n, k), (16, 1)),
                       one.expand(rows, k // 128), one.expand(n // 128, k // 128), out=out)
        return start, end

    def timed(k):
        start, end = long_product(k)
        end.record()
        end.synchronize()
        return start.elapsed_time(end)

    timed(2**22)
    k = min(most, int(2600 / timed(2**24) * 2**24)) // 128 * 128
    case = Experts([3], n=200, k=2064, mode="fp8", scales="block", seed=21)
    args = case.on(DEV)
    want = ops.block_gemm(args["a"], args["b"][0], args["a_scales"], args["b_scales"][0])
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    start, end = long_product(k)
    out = ops.block_gemm(args["a"], args["b"][0], args["a_scales"], args["b_scales"][0])
    end.record()
    end.synchronize()
    if start.elapsed_time(end) < 2100:
        pytest.skip("the kernel before ends too soon here")
    assert _lib.device_status() == 0 and torch.equal(out, want)


def test_an_earlier_error_is_not_reported_again(ops):
    """A call that failed has said so; the next one succeeds and says that."""
    import ctypes

    from m5kernels_b200 import _lib

    lib = _lib.lib()
    buf = torch.zeros(1 << 21, dtype=U8, device=DEV)
    handle, offset = (ctypes.c_uint8 * 64)(), ctypes.c_int64(0)
    case = Experts([3, 5], n=200, k=272, mode="fp8", scales="block", seed=22)
    args = case.on(DEV)
    x = torch.randn(4, 256, device=DEV)

    def fail():  # a process cannot import what it exported itself
        mapped = ctypes.c_void_p()
        with pytest.raises(RuntimeError):
            _lib.check(lib.m5b_ipc_import(handle, offset, ctypes.byref(mapped)))

    def grouped():
        return ops.grouped_gemm(args["a"], args["b"], args["group_start"], "fp8",
                                a_scales=args["a_scales"], b_scales=args["b_scales"])

    calls = (lambda: ops.block_quantize(x)[0], lambda: ops.block_quantize(x, block_rows=128)[0],
             lambda: ops.block_gemm(args["a"], args["b"][0], args["a_scales"],
                                    args["b_scales"][0]),
             grouped, lambda: ops.quantize(x, "int8")[0],
             lambda: ops.gemm(x.to(BF16), x.to(BF16)))
    want = [call() for call in calls]
    _lib.check(lib.m5b_ipc_export(ctypes.c_void_p(buf.data_ptr()), handle, ctypes.byref(offset)))
    for call, expected in zip(calls, want):
        fail()
        assert torch.equal(call(), expected)


def test_rows_of_out_that_overlap_are_refused(ops):
    case = Experts([3, 5], n=200, k=272, mode="bf16", seed=23)
    args = case.on(DEV)
    buf = torch.zeros(9 * 200, dtype=BF16, device=DEV)
    for step in (0, 1, 199):
        with pytest.raises(ValueError, match="overlap"):
            ops.grouped_gemm(args["a"], args["b"], args["group_start"],
                             out=buf.as_strided((8, 200), (step, 1)))
    assert (buf == 0).all()
    out = buf.as_strided((8, 200), (200, 1))
    ops.grouped_gemm(args["a"], args["b"], args["group_start"], out=out)
    assert torch.equal(out, ops.grouped_gemm(args["a"], args["b"], args["group_start"],
                                             output_dtype=BF16))
