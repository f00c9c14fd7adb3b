"""A GEMM behind a kernel of this library that lets it start early and takes longer than the 2 s
after which the GEMM's own waits give up: it waits for that kernel's end for as long as that takes."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, U8 = torch.bfloat16, torch.uint8


@pytest.mark.parametrize("mode", ["bf16", "int8"])
def test_a_long_kernel_before_a_gemm(mode):
    import m5kernels_b200 as ops
    from m5kernels_b200 import _lib

    # a block-scaled product of 37 tiles on 148 SMs over a long K: its rows lie 16 bytes apart in
    # one buffer, and its scales are one number
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
    g = torch.Generator(device=DEV).manual_seed(41)
    a, b = (torch.randn(r, 512, generator=g, device=DEV) for r in (40, 256))
    if mode == "bf16":
        args = dict(a=a.to(BF16), b=b.to(BF16), mode="bf16")
    else:
        (aq, sa), (bq, sb) = ops.quantize(a, "int8"), ops.quantize(b, "int8")
        args = dict(a=aq, b=bq, mode="int8", a_scales=sa, b_scales=sb)
    want = ops.gemm(**args)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    start, end = long_product(k)
    out = ops.gemm(**args)
    end.record()
    end.synchronize()
    if start.elapsed_time(end) < 2100:
        pytest.skip("the kernel before ends too soon here")
    assert _lib.device_status() == 0 and torch.equal(out, want)
