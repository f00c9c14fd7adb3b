"""block_quantize at every scale's rounding boundaries, over whole grids, and with far gates."""

import pytest
import torch

from grouped_cases import BLOCK, quantize_oracle, values

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    import m5kernels_b200 as m

    return m


# The quotients halfway between two codes: of normal codes (8 mantissas), of subnormal ones.
TIES = [(8 + i + 0.5) / 8 for i in range(8)] + [(i + 0.5) / 512 for i in range(8)]


@pytest.mark.parametrize("exponent", [-75, 0, 90])
def test_every_scale_at_its_ties(ops, exponent):
    """For each of the 2^23 mantissas of a block's peak, the values next to all ties.

    The kernel does not divide: its reciprocal of the scale may be off by the rarest ulp, and its
    quotient has to be RN(v / scale) where that decides on the code.  RN(peak / 448) and the
    quotients are those of 64 bits, rounded once to fp32 (a quotient of fp32 numbers that is not a
    midpoint of two of them is further from one than 64 bits err), the codes those of the
    conversion of that.
    """
    ties = torch.tensor(TIES, dtype=torch.float64, device=DEV)
    step = 1 << 18
    for first in range(0, 1 << 23, step):
        mantissa = torch.arange(first, first + step, device=DEV, dtype=torch.int32)
        peak = ((127 + exponent) << 23 | mantissa).view(F32)
        scale = (peak.double() / 448.0).float()
        x = torch.zeros(step, BLOCK, device=DEV)
        x[:, 0] = peak
        near = (ties * scale.double()[:, None]).float().view(torch.int32)
        for i, ulps in enumerate((-2, -1, 0, 1, 2)):
            x[:, 1 + 16 * i:17 + 16 * i] = (near + ulps).view(F32)
        x[:, 81:97] = -x[:, 33:49]
        x[:, 97:113] = 16.0 * x[:, 33:49]
        codes, scales = ops.block_quantize(x)
        assert torch.equal(scales[:, 0], scale)
        want = (x.double() / scale.double()[:, None]).float().to(torch.float8_e4m3fn)
        assert torch.equal(codes.view(torch.float8_e4m3fn).float(), want.float())


def many(rows, k, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, k, generator=g, device=DEV)
    return (x * torch.exp(torch.randn(k, generator=g, device=DEV))).to(dtype)


def check_exact(codes, scales, v):
    want, want_scales = quantize_oracle(v.float())
    assert torch.equal(scales, want_scales) and torch.equal(values(codes), want)


def check_gated(codes, scales, x, gate):
    """fp32 silu: exp to 2 units, a sum, a quotient and a product, at most 2^-21 of the value; the
    scale as much of the block's peak; a code half a step, 2^-4 of its value or 2^-10 of the scale."""
    k = x.shape[1]
    x, gate, scales = x.double(), gate.double(), scales.double()
    want = gate * torch.sigmoid(gate) * x
    peak = torch.nn.functional.pad(want.abs(), (0, -k % BLOCK)).view(len(x), -1, BLOCK).amax(2)
    assert ((scales - peak / 448).abs() <= 2.0**-20 * peak / 448).all()
    step = scales.repeat_interleave(BLOCK, 1)[:, :k]
    off = (values(codes) * step - want).abs()
    assert (off <= (2.0**-4 + 2.0**-18) * want.abs() + 2.0**-10 * step).all()


# More blocks than all resident lanes take at a time (148 SMs: 23680, gated ones 94720), several
# times over, so that rows and blocks are counted on; odd numbers of blocks in a row.
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,k", [(40001, 256), (30011, 400), (150000, 16), (7001, 2000),
                                    (333, 16384)])
@pytest.mark.parametrize("shift", [0, 1])
def test_whole_grids(ops, rows, k, dtype, shift):
    x = many(rows, k + 8, dtype)[:, shift:shift + k]
    codes, scales = ops.block_quantize(x)
    check_exact(codes, scales, x)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,rows,k,shift", [(5000, 40003, 400, 0), (5000, 40003, 400, 1),
                                                 (70000, 110001, 130, 0), (9, 60000, 128, 0)])
def test_whole_grids_of_rows(ops, tokens, rows, k, dtype, shift):
    x = many(tokens, k + 8, dtype)[:, shift:shift + k]
    g = torch.Generator(device=DEV).manual_seed(1)
    index = torch.randint(-3, tokens + 3, (rows,), generator=g, device=DEV, dtype=torch.int32)
    codes, scales = ops.block_quantize(x, rows=index)
    inside = (index >= 0) & (index < tokens)
    picked = torch.where(inside[:, None], x[index.clamp(0, tokens - 1).long()], 0)
    check_exact(codes, scales, picked)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,k,shift", [(60001, 256, 0), (60001, 250, 0), (200000, 16, 0),
                                          (13007, 2000, 1), (1500, 16384, 0)])
def test_whole_grids_of_gates(ops, rows, k, dtype, shift):
    both = many(rows, 2 * k + 8, dtype)
    x, gate = both[:, shift:shift + k], both[:, shift + k:shift + 2 * k]
    codes, scales = ops.block_quantize(x, gate=gate)
    check_gated(codes, scales, x, gate)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_whole_grids_of_gates_and_rows(ops, dtype):
    tokens, rows, k = 3000, 60000, 272
    both = many(tokens, 2 * k, dtype)
    g = torch.Generator(device=DEV).manual_seed(2)
    index = torch.randint(0, tokens, (rows,), generator=g, device=DEV, dtype=torch.int32)
    codes, scales = ops.block_quantize(both[:, :k], gate=both[:, k:], rows=index)
    once, once_scales = ops.block_quantize(both[:, :k], gate=both[:, k:])
    assert torch.equal(codes, once[index.long()])
    assert torch.equal(scales, once_scales[index.long()])


INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("k", [384, 383])
@pytest.mark.parametrize("gate,x,finite", [
    (NAN, 1.0, False), (INF, 1.0, False), (-INF, 1.0, False), (INF, 0.0, False),
    (1.0, NAN, False), (1.0, -INF, False), (0.0, INF, False), (-3e4, 2.0, True),
    (-100.0, 1.0, True), (100.0, 3.0, True), (-80.0, 1.0, True), (80.0, 1.0, True),
    (-0.0, 1.0, True), (6e4, 1.0, True)])
def test_far_gates(ops, gate, x, finite, dtype, k):
    """silu(gate) x that is not finite shows in its block's scale, and in no other block."""
    both = many(9, 2 * k, dtype, seed=3)
    xs, gates = both[:, :k].contiguous(), both[:, k:].contiguous()
    want, want_scales = ops.block_quantize(xs, gate=gates)
    xs[4, 200], gates[4, 200] = x, gate
    codes, scales = ops.block_quantize(xs, gate=gates)
    if finite:
        check_gated(codes, scales, xs, gates)
    else:
        assert not torch.isfinite(scales[4, 1])
    same = torch.ones_like(scales, dtype=torch.bool)
    same[4, 1] = False
    assert torch.equal(scales[same], want_scales[same])
    wide = same.repeat_interleave(BLOCK, 1)[:, :k]
    assert torch.equal(codes[wide], want[wide])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("block_rows", [1, BLOCK])
def test_zeros_of_either_sign(ops, dtype, block_rows):
    """Codes of zeros are zeros; which of the two is not specified."""
    x = torch.zeros(130, 260, dtype=dtype, device=DEV)
    x[::2] = -0.0
    x[5, 7], x[70, 133], x[100, 259] = 1.0, -3.0, 2.0**-14
    codes, scales = ops.block_quantize(x, block_rows=block_rows)
    assert (codes[x == 0] & 0x7F == 0).all()
    want, want_scales = quantize_oracle(x.float(), block_rows)
    assert torch.equal(scales, want_scales) and torch.equal(values(codes), want)
