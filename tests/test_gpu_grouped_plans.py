"""Products on the kernel that they are meant for: CTA pairs in several turns, K shared by
clusters, single CTAs.  Which one a call takes is asked for, so that another choice of tiles
cannot leave one of them without tests."""

import ctypes

import pytest
import torch

from grouped_cases import Experts, check_product
from grouped_plans import DEV, assert_pairs, oracle, plan_of

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
MODES = [("bf16", "none"), ("fp16", "none"), ("int8", "row"), ("fp8", "row"), ("fp8", "block")]
# (sizes, n, k, tiles a pair takes on 74 pairs): N on and off the grid of 16-byte stores
PAIRS = [([2500], 2056, 2064, 2), ([1000, 3, 0, 1300, 257, 700], 2306, 1616, 3),
         ([600, 0, 1, 900], 1800, 2064, 1)]


@pytest.fixture(scope="module")
def ops():
    import m5kernels_b200 as m
    from m5kernels_b200 import _lib

    yield m
    assert _lib.device_status() == 0  # no bounded wait gave up


def product(ops, args, **kw):
    return ops.grouped_gemm(args["a"], args["b"], args["group_start"], args["mode"],
                            a_scales=args["a_scales"], b_scales=args["b_scales"], **kw)


@pytest.mark.parametrize("mode,scales", MODES)
@pytest.mark.parametrize("sizes,n,k,turns", PAIRS)
def test_pairs(ops, sizes, n, k, turns, mode, scales):
    """Every output type; NaN in the rows around the groups."""
    case = Experts(sizes, n=n, k=k, mode=mode, scales=scales, lead=3, behind=30, seed=31)
    args, want = case.on(DEV), oracle(case)
    outside = case.outside.to(DEV)
    for dtype in (BF16, F16, F32):
        assert_pairs(case, dtype, turns)
        got = product(ops, args, output_dtype=dtype)
        check_product(got, want[0].cpu(), want[1].cpu(), k)
        assert (got[outside] == 0).all()
        given = torch.full((case.rows, n), 5.0, dtype=dtype, device=DEV)
        product(ops, args, out=given)
        assert (given[outside] == 5.0).all() and torch.equal(given[~outside], got[~outside])


@pytest.mark.parametrize("mode,scales", MODES)
def test_views_on_pairs(ops, mode, scales):
    """Operands, scales and outputs of other strides and alignments."""
    case = Experts([600, 0, 900], n=1796, k=2064, mode=mode, scales=scales, seed=32)
    args = case.on(DEV)
    n, k = case.n, case.k
    wide = torch.zeros(case.rows, 2304, dtype=case.a.dtype, device=DEV)
    wide[:, 16:16 + k] = args["a"]
    stack = torch.zeros(3, n + 10, 2320, dtype=case.b.dtype, device=DEV)
    stack[:, 5:5 + n, 32:32 + k] = args["b"]
    other = dict(args, a=wide[:, 16:16 + k], b=stack[:, 5:5 + n, 32:32 + k])
    if scales != "none":
        for name in ("a_scales", "b_scales"):
            v = args[name]
            other[name] = (v.transpose(0, 1).contiguous().transpose(0, 1) if v.dim() > 1
                           else torch.stack([v, v], 1)[:, 1])
    for dtype in (BF16, F16, F32):
        assert_pairs(case, dtype)
        want = product(ops, args, output_dtype=dtype)
        assert torch.equal(product(ops, other, output_dtype=dtype), want)
        for more, at in ((60, 0), (11, 0), (11, 5), (8, 1)):
            buf = torch.full((case.rows + 2, n + more), 7.0, dtype=dtype, device=DEV)
            out = buf[1:-1, at:at + n]
            product(ops, other, out=out)
            assert torch.equal(out, want)
            out.fill_(7.0)
            assert (buf == 7.0).all()


@pytest.mark.parametrize("mode,scales", [m for m in MODES if m[0] != "int8"])
def test_nan_stays_in_its_row_and_channel_on_pairs(ops, mode, scales):
    case = Experts([2500], n=2056, k=2064, mode=mode, scales=scales, seed=33)
    assert_pairs(case, F32, 2)
    want = product(ops, case.on(DEV), output_dtype=F32)
    bad = torch.zeros_like(want, dtype=torch.bool)
    for row, at in ((13, 7), (255, 2063), (2499, 130)):
        case.a[row, at] = 0x7F if mode == "fp8" else float("nan")
        bad[row] = True
    for ch, at in ((200, 2050), (2055, 0)):
        case.b[0, ch, at] = 0x7F if mode == "fp8" else float("nan")
        bad[:, ch] = True
    if scales == "block":  # a scale that is not finite: that row
        case.a_scales[700, 16] = float("inf")
        bad[700] = True
    got = product(ops, case.on(DEV), output_dtype=F32)
    assert not torch.isfinite(got[bad]).any() and torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("starts,means", [
    ([-5, 700, 500, 900], [0, 700, 700, 900]), ([0, 900, 900, 1500], [0, 900, 900, 1500]),
    ([2**31 - 1, 0, 64, 1500], [1500] * 4), ([100, 1400, 50, 2**31 - 1], [100, 1400, 1400, 1500])])
@pytest.mark.parametrize("mode,scales", MODES)
def test_bounds_on_pairs(ops, starts, means, mode, scales):
    """Out of order and out of range."""
    case = Experts([600, 0, 900], n=1800, k=2064, mode=mode, scales=scales, seed=34)
    assert_pairs(case, BF16)
    case.group_start = torch.tensor(starts, dtype=torch.int32)
    got = product(ops, case.on(DEV), output_dtype=BF16)
    case.starts, case.sizes = means, [b - a for a, b in zip(means, means[1:])]
    out, spread = oracle(case)
    check_product(got, out.cpu(), spread.cpu(), case.k)


@pytest.mark.parametrize("m,n,k,turns", [(2500, 2056, 2064, 2), (1285, 4993, 1552, 2),
                                         (700, 4097, 2576, 1), (700, 2305, 2576, 0)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_block_gemm_on_pairs(ops, m, n, k, turns, dtype):
    """(And the last beside them: single CTAs in several turns.)"""
    case = Experts([m], n=n, k=k, mode="fp8", scales="block", seed=35)
    if turns:
        assert_pairs(case, dtype, turns)
    else:
        assert plan_of(case, dtype)[::2] == (1, 1)
    args = case.on(DEV)
    got = ops.block_gemm(args["a"], args["b"][0], args["a_scales"], args["b_scales"][0],
                         output_dtype=dtype)
    out, spread = oracle(case)
    check_product(got, out.cpu(), spread.cpu(), k)


@pytest.mark.parametrize("mode,scales", MODES)
def test_graphs_on_pairs(ops, mode, scales):
    """Replays follow the bounds, beside each other, behind a quantization on their stream."""
    tokens, n, k = 1500, 2056, 2064
    case = Experts([tokens // 2, 0, tokens - tokens // 2], n=n, k=k, mode=mode, scales=scales,
                   seed=36)
    assert_pairs(case, BF16)
    args = case.on(DEV)
    x = torch.randn(tokens, k, device=DEV)

    def step():
        if scales != "block":
            return product(ops, args, output_dtype=BF16)
        codes, a_scales = ops.block_quantize(x)
        return product(ops, dict(args, a=codes, a_scales=a_scales), output_dtype=BF16)

    step()
    graphs, outs = [], []
    for _ in range(2):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(step())
        graphs.append(graph)
    for bounds in ([0, 1, 2, tokens], [0, tokens, tokens, tokens], [0, 0, 20, 700],
                   [300, 900, 1100, 1100]):
        args["group_start"].copy_(torch.tensor(bounds, dtype=torch.int32))
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


def test_pairs_on_several_streams(ops):
    """Calls side by side, of one kind and of several, repeat to the bit."""
    cases = [Experts([1500 + i], n=2056, k=2064, mode=m, scales=sc, seed=37 + i)
             for i, (m, sc) in enumerate(MODES + [("fp8", "block")] * 2)]
    for case in cases:
        assert_pairs(case, F32)
    args = [c.on(DEV) for c in cases]
    want = [product(ops, a, output_dtype=F32) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    for _ in range(4):
        got = []
        for a, stream in zip(args, streams):
            with torch.cuda.stream(stream):
                got.append(product(ops, a, output_dtype=F32))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


# (rows, n, k, CTAs that share K) of one group, on 148 SMs
SHARED = [(3, 8192, 4096, 2), (40, 2500, 4096, 4), (3, 1000, 16384, 8), (64, 130, 8192, 8),
          (200, 2000, 2064, 2), (13, 9600, 4096, 1)]


@pytest.mark.parametrize("mode,scales", MODES)
@pytest.mark.parametrize("rows,n,k,shared", SHARED)
def test_shared_sums(ops, rows, n, k, shared, mode, scales):
    case = Experts([rows], n=n, k=k, mode=mode, scales=scales, seed=38)
    args, want = case.on(DEV), oracle(case)
    for dtype in (BF16, F16, F32):
        assert plan_of(case, dtype)[::2] == (1, shared)
        check_product(product(ops, args, output_dtype=dtype), want[0].cpu(), want[1].cpu(), k)


@pytest.mark.parametrize("mode,scales", MODES)
@pytest.mark.parametrize("rows,n,k", [(3, 200, 4096), (40, 9600, 528), (1500, 2056, 2064)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_c_calls_without_bounds(ops, rows, n, k, mode, scales, dtype):
    """group_start NULL: all rows are group 0's, for operands of every kind."""
    from m5kernels_b200 import _lib, grouped

    case = Experts([rows], n=n, k=k, mode=mode, scales=scales, seed=40)
    args = case.on(DEV)
    want = product(ops, args, output_dtype=dtype)
    out = torch.full_like(want, 3.0)
    fields = (0,) * 7
    if scales != "none":
        sa, sb = args["a_scales"], args["b_scales"]
        strides = ((*sa.stride(), *sb.stride()) if scales == "block"
                   else (*sa.stride(), 0, *sb.stride(), 0))
        fields = (sa.data_ptr(), sb.data_ptr(), *strides)
    record = grouped._PACK_GEMM.pack(
        args["a"].data_ptr(), args["b"].data_ptr(), _lib.MODE[mode], rows, 1, n, k, k, n * k, k, 0,
        scales == "block", *fields, out.data_ptr(), _lib.DTYPE_CODE[dtype], n, 1)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    _lib.check(_lib.lib().m5b_grouped_gemm(record, stream))
    assert torch.equal(out, want)


def test_plans_of_calls_that_are_refused(ops):
    from m5kernels_b200 import _lib
    from grouped_plans import plan

    for error, args in ((ValueError, (0, 1, 8, 64, "bf16", "none", BF16)),
                        (ValueError, (4, 1, 8, 64, "bf16", "block", BF16)),
                        (NotImplementedError, (4, 1025, 8, 64, "bf16", "none", BF16)),
                        (NotImplementedError, (4, 1, 8, 64, "bf16", "none", torch.int32))):
        with pytest.raises(error):
            plan(*args)
    assert _lib.lib().m5b_grouped_gemm_plan(None, None) == _lib.EINVAL
