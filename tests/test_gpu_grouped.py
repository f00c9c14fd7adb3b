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


@pytest.mark.parametrize("sizes", [[1100], [300, 1, 0, 257, 33, 512], [32] * 40, [700, 500]])
@pytest.mark.parametrize("mode,scales", MODES)
@pytest.mark.parametrize("n,k,dtype", [(2048, 528, BF16), (1801, 144, F32), (2056, 1040, F16),
                                       (2306, 16, BF16), (2240, 272, F32), (1900, 400, F16)])
def test_tiles_of_pairs(ops, sizes, mode, scales, n, k, dtype):
    """More tiles of 128 channels x 64 rows than SMs: CTA pairs take tiles of 256 x 256."""
    check(ops, Experts(sizes, n=n, k=k, mode=mode, scales=scales, lead=3, behind=30, seed=16),
          dtype)


@pytest.mark.parametrize("mode,scales", MODES)
@pytest.mark.parametrize("rows", [1, 8, 9, 16, 60, 64, 65, 128, 255, 256, 257, 700])
def test_rows_of_one_group(ops, rows, mode, scales):
    check(ops, Experts([rows], n=384, k=2064, mode=mode, scales=scales, seed=2), BF16)


@pytest.mark.parametrize("rows,n,k", [(1, 128, 4096), (3, 1000, 16384), (17, 256, 2064),
                                      (33, 130, 8192), (64, 512, 4096), (50, 64, 528)])
@pytest.mark.parametrize("mode,scales", MODES)
def test_few_rows_of_a_long_sum(ops, rows, n, k, mode, scales):
    """K shared by several CTAs: 2, 4 and 8 of them, ranges that are not equal."""
    check(ops, Experts([rows], n=n, k=k, mode=mode, scales=scales, seed=3), F32)


@pytest.mark.parametrize("mode", ["bf16", "fp16"])
@pytest.mark.parametrize("sizes,n", [([40], 300), ([300, 200], 300), ([700], 300), ([900], 1600)])
def test_fp32_results_of_long_sums(ops, mode, sizes, n):
    """Parts of four blocks (16 instructions) are added in fp32: the error does not grow with K
    but for the rounding of those additions, e = (16 + K / 256 + 3) 2^-22 of the magnitudes."""
    k = 16384
    case = Experts(sizes, n=n, k=k, mode=mode, seed=4)
    got = product(ops, case, output_dtype=F32).double().cpu()
    out, spread = case.oracle()
    e = (16 + k // 256 + 3) * 2.0**-22
    assert ((got - out).abs() <= 2.0**-24 * out.abs() + e * spread).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("sizes,n", [("small", 264), ("mixed", 264), ("many", 264),
                                     ("mixed", 2304)])
def test_int8_is_gemm_of_each_group(ops, sizes, n, dtype):
    case = Experts(SIZES[sizes], n=n, k=1040, mode="int8", scales="row", seed=5)
    args = case.on(DEV)
    got = product(ops, case, output_dtype=dtype)
    for e, rows in enumerate(case.sizes):
        if rows:
            mine = slice(case.starts[e], case.starts[e + 1])
            want = ops.gemm(args["a"][mine], args["b"][e], "int8", a_scales=args["a_scales"][mine],
                            b_scales=args["b_scales"][e], output_dtype=dtype)
            assert torch.equal(got[mine], want)


@pytest.mark.parametrize("mode,scales", MODES)
@pytest.mark.parametrize("sizes,n", [([0, 0], 136), ([3, 0, 40], 136), ([100, 200, 0, 300], 136),
                                     ([100, 200, 0, 600], 1800)])
def test_rows_outside_the_groups(ops, mode, scales, sizes, n):
    """They are zero in a fresh output, kept in a given one, and their NaNs reach nothing."""
    case = Experts(sizes, n=n, k=272, mode=mode, scales=scales, lead=7, behind=70, seed=6)
    fresh = check(ops, case, BF16)
    assert (fresh[case.outside.to(DEV)] == 0).all()
    given = torch.full((case.rows, case.n), 5.0, dtype=BF16, device=DEV)
    assert product(ops, case, out=given) is given
    assert (given[case.outside.to(DEV)] == 5.0).all()
    assert torch.equal(given[~case.outside.to(DEV)], fresh[~case.outside.to(DEV)])


@pytest.mark.parametrize("starts,means", [
    ([0, 20, 20, 90], [0, 20, 20, 64]), ([-5, 20, 30, 64], [0, 20, 30, 64]),
    ([0, 30, 10, 64], [0, 30, 30, 64]), ([50, 40, 30, 20], [50, 50, 50, 50]),
    ([2**31 - 1, 0, 64, 64], [64, 64, 64, 64]), ([-2**31, 64, -2**31, 2**31 - 1], [0, 64, 64, 64])])
@pytest.mark.parametrize("mode,scales", MODES)
def test_bounds_that_do_not_ascend(ops, starts, means, mode, scales):
    case = Experts([20, 0, 44], n=72, k=144, mode=mode, scales=scales, seed=7)
    case.group_start = torch.tensor(starts, dtype=torch.int32)
    got = product(ops, case, output_dtype=F32)
    case.group_start = torch.tensor(means, dtype=torch.int32)
    assert torch.equal(got, product(ops, case, output_dtype=F32))
    case.starts, case.sizes = means, [b - a for a, b in zip(means, means[1:])]
    out, spread = case.oracle()
    check_product(got, out, spread, case.k)


@pytest.mark.parametrize("groups", [1, 31, 32, 33, 1024])
@pytest.mark.parametrize("mode,scales", [("bf16", "none"), ("fp8", "block")])
def test_number_of_groups(ops, groups, mode, scales):
    check(ops, Experts([(7 * e) % 4 for e in range(groups)], n=24, k=48, mode=mode, scales=scales,
                       seed=8), BF16)


@pytest.mark.parametrize("mode,scales", MODES)
@pytest.mark.parametrize("sizes,n", [([30, 0, 65], 200), ([500, 0, 600], 1800)])
def test_views(ops, mode, scales, sizes, n):
    """Operands, scales and outputs of other strides and alignments."""
    case = Experts(sizes, n=n, k=272, mode=mode, scales=scales, seed=9)
    want = product(ops, case, output_dtype=BF16)
    args = case.on(DEV)
    a, b, start = args["a"], args["b"], args["group_start"]
    kw = dict(a_scales=args["a_scales"], b_scales=args["b_scales"])
    wide = torch.zeros(case.rows, 512, dtype=a.dtype, device=DEV)
    odd = torch.zeros(case.rows, 301, dtype=a.dtype, device=DEV)
    wide[:, 16:288], odd[:, 3:275] = a, a
    stack = torch.zeros(3, n + 10, 320, dtype=b.dtype, device=DEV)
    stack[:, 5:5 + n, 32:304] = b
    turned = b.transpose(1, 2).contiguous().transpose(1, 2)
    for x, w in ((wide[:, 16:288], b), (odd[:, 3:275], b), (a, stack[:, 5:5 + n, 32:304]),
                 (a, turned), (a.t().contiguous().t(), b)):
        assert torch.equal(ops.grouped_gemm(x, w, start, mode, output_dtype=BF16, **kw), want)
    if scales != "none":
        other = {k: v.transpose(0, 1).contiguous().transpose(0, 1) if v.dim() > 1
                 else torch.stack([v, v], 1)[:, 1] for k, v in kw.items()}
        assert torch.equal(ops.grouped_gemm(a, b, start, mode, output_dtype=BF16, **other), want)
    for dtype in (BF16, F16, F32):
        want = ops.grouped_gemm(a, b, start, mode, output_dtype=dtype, **kw)
        for more, at in ((56, 0), (11, 0), (11, 5), (8, 1)):
            buf = torch.full((case.rows + 2, n + more), 7.0, dtype=dtype, device=DEV)
            out = buf[1:-1, at:at + n]
            ops.grouped_gemm(a, b, start, mode, out=out, **kw)
            assert torch.equal(out, want)
            out.fill_(7.0)
            assert (buf == 7.0).all()


@pytest.mark.parametrize("mode,scales", [m for m in MODES if m[0] != "int8"])
@pytest.mark.parametrize("rows,n", [(60, 300), (300, 300), (900, 1700)])
def test_nan_stays_in_its_row_and_channel(ops, rows, n, mode, scales):
    case = Experts([rows], n=n, k=400, mode=mode, scales=scales, seed=10)
    want = product(ops, case, output_dtype=F32)
    case.a[13, 7] = 0x7F if mode == "fp8" else float("nan")
    case.b[0, 200, 390] = 0x7F if mode == "fp8" else float("nan")
    got = product(ops, case, output_dtype=F32)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[13], bad[:, 200] = True, True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 7168, 5376), (2, 129, 128), (63, 200, 144),
                                   (65, 256, 2048), (129, 1000, 1040), (256, 128, 512),
                                   (300, 384, 4096), (520, 640, 656), (1000, 2176, 912),
                                   (1285, 1793, 528)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_block_gemm(ops, m, n, k, dtype):
    case = Experts([m], n=n, k=k, mode="fp8", scales="block", seed=11)
    args = case.on(DEV)
    got = ops.block_gemm(args["a"], args["b"][0], args["a_scales"], args["b_scales"][0],
                         output_dtype=dtype)
    check_product(got, *case.oracle(), k)
    out = torch.empty(m, n + 3, dtype=dtype, device=DEV)[:, :n]
    assert ops.block_gemm(args["a"], args["b"][0], args["a_scales"], args["b_scales"][0],
                          out=out) is out and torch.equal(out, got)


def test_defaults_and_no_rows(ops):
    a, b = torch.zeros(0, 128, dtype=torch.uint8, device=DEV), torch.zeros(
        5, 128, dtype=torch.uint8, device=DEV)
    out = ops.block_gemm(a, b, torch.ones(0, 1, device=DEV), torch.ones(1, 1, device=DEV))
    assert out.shape == (0, 5) and out.dtype == F32
    codes, scales = ops.block_quantize(torch.zeros(0, 300, device=DEV))
    assert codes.shape == (0, 300) and scales.shape == (0, 3)
    codes, scales = ops.block_quantize(
        torch.ones(4, 300, device=DEV), rows=torch.zeros(0, dtype=torch.int32, device=DEV))
    assert codes.shape == (0, 300) and scales.shape == (0, 3)
    codes, scales = ops.block_quantize(
        torch.ones(0, 256, device=DEV), rows=torch.zeros(2, dtype=torch.int32, device=DEV))
    assert (values(codes.cpu()) == 0).all() and (scales == 1).all()
    x = torch.randn(6, 32, device=DEV, dtype=BF16)
    out = ops.grouped_gemm(x, torch.ones(1, 3, 32, device=DEV, dtype=BF16),
                           torch.tensor([0, 6], dtype=torch.int32, device=DEV))
    assert out.dtype == F32 and out.shape == (6, 3)


def test_quantize_and_multiply(ops):
    """The two together: what E4M3 with these scales makes of a product."""
    g = torch.Generator().manual_seed(12)
    x, w = torch.randn(150, 700, generator=g), 0.02 * torch.randn(260, 700, generator=g)
    w = torch.nn.functional.pad(w, (0, 4))
    x = torch.nn.functional.pad(x, (0, 4))  # 704: rows on the 16-byte grid
    a, sa = ops.block_quantize(x.to(DEV, BF16))
    b, sb = ops.block_quantize(w.to(DEV), block_rows=BLOCK)
    got = ops.block_gemm(a, b, sa, sb)
    x8, w8 = dequantized(a.cpu(), sa.cpu(), 1), dequantized(b.cpu(), sb.cpu(), BLOCK)
    check_product(got, x8 @ w8.T, x8.abs() @ w8.abs().T, 704)


@pytest.mark.parametrize("tokens,experts,top", [(5, 8, 2), (64, 4, 2), (300, 6, 3)])
def test_expert_layer(ops, tokens, experts, top):
    """Rows to their experts, up and gate, silu, down, as they are used together.

    Each step is checked against 64 bits of what it was given.
    """
    g = torch.Generator().manual_seed(13)
    d, inner = 512, 384
    x = torch.randn(tokens, d, generator=g).to(BF16)
    w_up = 0.05 * torch.randn(experts, 2 * inner, d, generator=g)
    w_down = 0.05 * torch.randn(experts, d, inner, generator=g)
    chosen = torch.stack([torch.randperm(experts, generator=g)[:top] for _ in range(tokens)])
    expert, order = chosen.flatten().sort(stable=True)
    rows = (order // top).to(torch.int32)
    start = torch.searchsorted(expert, torch.arange(experts + 1)).to(torch.int32)
    up, up_scales = ops.block_quantize(w_up.to(DEV), block_rows=BLOCK)
    down, down_scales = ops.block_quantize(w_down.to(DEV), block_rows=BLOCK)

    a, sa = ops.block_quantize(x.to(DEV), rows=rows.to(DEV))
    check_codes(a, sa, x[rows.long()])
    h = ops.grouped_gemm(a, up, start.to(DEV), "fp8", a_scales=sa, b_scales=up_scales,
                         output_dtype=BF16)
    b, sb = ops.block_quantize(h[:, :inner], gate=h[:, inner:])
    y = ops.grouped_gemm(b, down, start.to(DEV), "fp8", a_scales=sb, b_scales=down_scales,
                         output_dtype=F32)

    for got, codes, scales, w, w_scales, k in ((h, a, sa, up, up_scales, d),
                                               (y, b, sb, down, down_scales, inner)):
        out = torch.zeros(got.shape, dtype=torch.float64)
        spread = torch.zeros_like(out)
        for e in range(experts):
            mine = slice(int(start[e]), int(start[e + 1]))
            p = dequantized(codes[mine].cpu(), scales[mine].cpu(), 1)
            q = dequantized(w[e].cpu(), w_scales[e].cpu(), BLOCK)
            out[mine], spread[mine] = p @ q.T, p.abs() @ q.abs().T
        check_product(got, out, spread, k)
    want = gated(h[:, :inner].cpu(), h[:, inner:].cpu())
    step = sb.double().cpu().repeat_interleave(BLOCK, 1)
    off = (dequantized(b.cpu(), sb.cpu(), 1) - want).abs()
    assert (off <= (2.0**-4 + 2.0**-18) * want.abs() + 2.0**-10 * step).all()


@pytest.mark.parametrize("tokens,n", [(40, 200), (900, 200), (900, 2000)])
def test_graph_replays_with_other_bounds(ops, tokens, n):
    """Captured calls read the bounds when they are replayed; two graphs run beside each other."""
    case = Experts([tokens // 2, 0, tokens - tokens // 2], n=n, k=272, mode="fp8",
                   scales="block", seed=14)
    args = case.on(DEV)
    x = torch.randn(tokens, 272, device=DEV)
    start = args["group_start"]

    def step():
        codes, scales = ops.block_quantize(x)
        return ops.grouped_gemm(codes, args["b"], start, "fp8", a_scales=scales,
                                b_scales=args["b_scales"], output_dtype=BF16)

    step()
    graphs, outs = [], []
    for _ in range(2):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(step())
        graphs.append(graph)
    for bounds in ([0, 1, 2, tokens], [0, tokens, tokens, tokens], [0, 0, 20, 30]):
        start.copy_(torch.tensor(bounds, dtype=torch.int32))
        x.normal_()
        want = step()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out in outs)


def test_calls_on_several_streams(ops):
    """Calls side by side do not share anything, and repeat to the bit."""
    cases = [Experts(s, n=n, k=1040, mode=m, scales=sc, seed=15)
             for s, n, (m, sc) in zip(([200, 300], [7, 0, 9], [800], [64], [433, 600]),
                                      (384, 384, 1800, 384, 2048), MODES)]
    args = [c.on(DEV) for c in cases]

    def run(a):
        return ops.grouped_gemm(a["a"], a["b"], a["group_start"], a["mode"],
                                a_scales=a["a_scales"], b_scales=a["b_scales"], output_dtype=F32)

    want = [run(a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    for _ in range(4):
        got = []
        for a, stream in zip(args, streams):
            with torch.cuda.stream(stream):
                got.append(run(a))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_offsets_beyond_32_bits(ops):
    """Outputs, activations and weights of more than 2^31 elements."""
    rows, n = 70000, 32768
    a = torch.randn(rows, 16, device=DEV, dtype=BF16)
    b = torch.randn(1, n, 16, device=DEV, dtype=BF16)
    out = ops.grouped_gemm(a, b, torch.tensor([0, rows], dtype=torch.int32, device=DEV),
                           output_dtype=BF16)
    for at in (slice(0, 3), slice(rows - 3, rows)):
        want = a[at].double() @ b[0].double().T
        assert ((out[at].double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-16).all()
    del out
    experts = torch.zeros(130, 4096, 4112, dtype=torch.int8, device=DEV)
    experts[128:] = torch.randint(-9, 10, (2, 4096, 4112), device=DEV, dtype=torch.int8)
    a = torch.randint(-9, 10, (5, 4112), device=DEV, dtype=torch.int8)
    start = torch.zeros(131, dtype=torch.int32, device=DEV)
    start[129], start[130] = 2, 5
    ones = torch.ones(130, 4096, device=DEV)
    got = ops.grouped_gemm(a, experts, start, "int8", a_scales=ones[0, :5], b_scales=ones)
    for e, mine in ((128, slice(0, 2)), (129, slice(2, 5))):
        assert torch.equal(got[mine].double(), a[mine].double() @ experts[e].double().T)
    del experts
    x = torch.zeros(140000, 16384, device=DEV, dtype=BF16)
    x[-2:] = torch.randn(2, 16384, device=DEV, dtype=BF16)
    codes, scales = ops.block_quantize(x)
    check_codes(codes[-3:], scales[-3:], x[-3:].cpu())
    assert (codes[:-2].view(torch.int64) == 0).all() and (scales[:-2] == 1).all()


@pytest.mark.parametrize("sizes,n", [([40], 300), ([300, 200], 300), ([900], 1600)])
def test_fp32_results_of_long_e4m3_sums(ops, sizes, n):
    """As test_fp32_results_of_long_sums: parts of four blocks of 128 channels (16 instructions),
    and two roundings for the scales."""
    k = 16384
    case = Experts(sizes, n=n, k=k, mode="fp8", scales="row", seed=17)
    got = product(ops, case, output_dtype=F32).double().cpu()
    out, spread = case.oracle()
    e = (16 + k // 512 + 3) * 2.0**-22
    assert ((got - out).abs() <= 2.0**-24 * out.abs() + e * spread).all()
