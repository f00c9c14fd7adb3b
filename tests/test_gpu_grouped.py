"""Block-scaled and grouped products on the GPU against 64-bit oracles."""

import pytest
import torch

from grouped_cases import (BLOCK, Experts, check_product, dequantized, quantize_oracle, values)

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    import m5kernels_b200 as m
    from m5kernels_b200 import _lib

    yield m
    assert _lib.device_status() == 0  # no bounded wait gave up


def activations(rows, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g) * torch.exp(torch.randn(k, generator=g))
    return x.to(dtype)


def check_codes(codes, scales, v, block_rows=1):
    """Bit for bit, but for the sign of codes that are zero."""
    want, want_scales = quantize_oracle(v.float(), block_rows)
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(values(codes.cpu()), want)


# ---------------------------------------------------------------- quantization
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 128), (3, 127), (2, 130), (7, 16), (5, 1000),
                                    (33, 256), (64, 2064), (300, 4096), (1, 16384)])
def test_quantize(ops, rows, k, dtype):
    x = activations(rows, k, dtype)
    codes, scales = ops.block_quantize(x.to(DEV))
    assert codes.dtype == torch.uint8 and codes.shape == (rows, k)
    check_codes(codes, scales, x)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (129, 130), (100, 1000), (5, 2064),
                                   (300, 520), (3, 200, 264), (2, 128, 72), (4, 1, 8)])
def test_quantize_weights(ops, shape, dtype):
    rows = 1
    for s in shape[:-1]:
        rows *= s
    w = activations(rows, shape[-1], dtype).view(shape)
    codes, scales = ops.block_quantize(w.to(DEV), block_rows=BLOCK)
    assert codes.shape == shape
    each = w[None] if w.dim() == 2 else w
    codes, scales = (codes[None], scales[None]) if w.dim() == 2 else (codes, scales)
    for e in range(each.shape[0]):
        check_codes(codes[e], scales[e], each[e], BLOCK)


@pytest.mark.parametrize("dtype,k", [(BF16, 1000), (F16, 256), (F32, 131)])
def test_quantize_rows(ops, dtype, k):
    """Rows in another order, repeated, and from outside."""
    x = activations(50, k, dtype)
    rows = torch.randint(0, 50, (170,), generator=torch.Generator().manual_seed(1))
    rows[7] = rows[8] = 49
    picked = x[rows].clone()
    index = rows.to(torch.int32)
    for at, bad in ((3, -1), (20, 50), (21, 2**31 - 1), (169, -2**31)):
        index[at] = bad
        picked[at] = 0
    codes, scales = ops.block_quantize(x.to(DEV), rows=index.to(DEV))
    check_codes(codes, scales, picked)


def gated(x, g):
    x, g = x.double(), g.double()
    return g * torch.sigmoid(g) * x


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,k", [(1, 8), (5, 127), (40, 1000), (129, 512)])
def test_quantize_gated(ops, rows, k, dtype):
    """Codes times scales against silu(gate) x in 64 bits.

    fp32 silu: exp to 2 units, a sum, a quotient and a product, at most 2^-21
    of the value; the scale as much of the block's peak; a code half a step,
    2^-4 of its value or 2^-10 of the scale.
    """
    both = activations(rows, 2 * k, dtype)
    both[:, k:] *= 3.0
    dev = both.to(DEV)
    codes, scales = ops.block_quantize(dev[:, :k], gate=dev[:, k:])
    want = gated(both[:, :k], both[:, k:])
    peak = torch.nn.functional.pad(want.abs(), (0, -k % BLOCK)).view(rows, -1, BLOCK).amax(2)
    scales = scales.double().cpu()
    assert ((scales - peak / 448).abs() <= 2.0**-20 * peak / 448).all()
    got = dequantized(codes.cpu(), scales.float(), 1)
    step = scales.repeat_interleave(BLOCK, 1)[:, :k]
    assert ((got - want).abs() <= (2.0**-4 + 2.0**-18) * want.abs() + 2.0**-10 * step).all()


def test_quantize_gate_and_rows(ops):
    both = activations(30, 512, BF16)
    rows = torch.tensor([3, 3, 0, 29, 30, 7], dtype=torch.int32)
    dev = both.to(DEV)
    codes, scales = ops.block_quantize(dev[:, :256], gate=dev[:, 256:], rows=rows.to(DEV))
    take = dev[[3, 3, 0, 29, 0, 7]]
    take[4] = 0
    want, want_scales = ops.block_quantize(take[:, :256], gate=take[:, 256:])
    assert torch.equal(codes, want) and torch.equal(scales, want_scales)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_quantize_far_values(ops, dtype):
    """Zeros, the type's smallest and largest values, peaks whose scale is tiny or zero."""
    info = torch.finfo(dtype)
    x = torch.zeros(8, 256, dtype=dtype)
    x[1, :5] = info.smallest_normal
    x[2, 3] = info.max
    x[2, 4] = -info.max / 3
    x[3, 200] = info.max
    x[3, 201] = info.tiny
    x[4] = torch.finfo(dtype).smallest_normal / 16  # (subnormal)
    x[5] = -0.0
    x[6, ::2] = 448.0
    x[6, 1::2] = torch.linspace(-1, 1, 128).to(dtype)
    x[7, 1] = 1.0
    codes, scales = ops.block_quantize(x.to(DEV))
    check_codes(codes, scales, x)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("block_rows", [1, BLOCK])
def test_quantize_not_finite(ops, bad, block_rows):
    """Such a block's scale shows it; its neighbours are as without it."""
    x = activations(130, 384, BF16)
    want, want_scales = ops.block_quantize(x.to(DEV), block_rows=block_rows)
    x[40, 200] = bad
    codes, scales = ops.block_quantize(x.to(DEV), block_rows=block_rows)
    at = (40 // block_rows, 1)
    assert not torch.isfinite(scales[at])
    same = torch.ones_like(scales, dtype=torch.bool)
    same[at] = False
    assert torch.equal(scales[same], want_scales[same])
    wide = same.repeat_interleave(block_rows, 0)[:130].repeat_interleave(BLOCK, 1)
    assert torch.equal(codes[wide], want[wide])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantize_views(ops, dtype):
    """Rows off the 16-byte grid, channels that are not contiguous, every second row."""
    x = activations(41, 520, dtype).to(DEV)
    for v in (x[:, 1:513], x[::2, 8:264], x[:, ::2], x.t(), x[:0]):
        codes, scales = ops.block_quantize(v)
        assert codes.shape == v.shape
        if v.numel():
            check_codes(codes, scales, v.cpu())
    stack = activations(64, 260, dtype).view(4, 16, 260).to(DEV)
    for v in (stack[:, :, :256], stack.transpose(0, 1), stack[::2, 1:, 4:]):
        codes, scales = ops.block_quantize(v, block_rows=BLOCK)
        for e in range(v.shape[0]):
            check_codes(codes[e], scales[e], v[e].cpu(), BLOCK)


# ---------------------------------------------------------------- products
MODES = [("bf16", "none"), ("fp16", "none"), ("int8", "row"), ("fp8", "row"), ("fp8", "block")]
SIZES = {
    "one_row": [1],
    "one_group": [200],
    "tokens": [1, 0, 3, 2, 0, 0, 1],
    "small": [5, 64, 65, 1, 16, 17, 40],
    "mixed": [300, 1, 0, 257, 33, 512],
    "none": [0, 0, 0],
    "many": [n % 5 for n in range(77)],
}


def product(ops, case, **kw):
    args = case.on(DEV)
    return ops.grouped_gemm(args.pop("a"), args.pop("b"), args.pop("group_start"),
                            args.pop("mode"), **args, **kw)


def check(ops, case, dtype):
    got = product(ops, case, output_dtype=dtype)
    assert got.dtype == dtype and got.shape == (case.rows, case.n)
    if not case.rows:
        return got
    out, spread = case.oracle()
    check_product(got, out, spread, case.k)
    return got


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("mode,scales", MODES)
@pytest.mark.parametrize("n,k,dtype", [(256, 256, BF16), (72, 1040, F16), (331, 144, F32),
                                       (640, 528, BF16), (129, 16, BF16)])
def test_grouped(ops, sizes, mode, scales, n, k, dtype):
    check(ops, Experts(SIZES[sizes], n=n, k=k, mode=mode, scales=scales, seed=1), dtype)


@pytest.mark.parametrize("mode,scales", MODES)
@pytest.mark.parametrize("rows", [1, 8, 9, 16, 60, 64, 65, 128, 255, 256, 257, 700])
def test_rows_of_one_group(ops, rows, mode, scales):
    check(ops, Experts([rows], n=384, k=2064, mode=mode, scales=scales, seed=2), BF16)
