"""fp32 results of long sums: parts of a sum are added in fp32, so that K does not cost accuracy."""

import pytest
import torch

from grouped_cases import Experts
from grouped_plans import DEV, oracle, plan_of

pytestmark = pytest.mark.gpu

F32 = torch.float32
MODES = [("bf16", "none"), ("fp16", "none"), ("fp8", "row"), ("fp8", "block")]


@pytest.fixture(scope="module")
def ops():
    import m5kernels_b200 as m

    return m


# Relative 2-norm of what fp32 results may be off.  A truncated sum loses 2^-24 of its magnitude an
# instruction, on average and always towards zero.  A part of 16 instructions, 1 / sqrt(P) of the
# result R in magnitude (P parts), loses 16 * 2^-24 * 0.6 R / sqrt(P); P of them, of random signs,
# 9.6 * 2^-24 R = 5.7e-7 R at any K, and P roundings to fp32 of growing sums 0.4 sqrt(P) 2^-24 R,
# 2e-7 at most here.  1e-6, then; without parts the whole K is one sum, whose losses grow with it
# (measured at K 16384: 4.9e-6).  E4M3 products fill fewer bits: 0.8e-7 measured, and 1.2e-6
# without parts; 4e-7.  Scaled blocks are parts of four instructions, P = K / 128 additions
# (0.4 sqrt(128) 2^-24 = 2.7e-7 at K 16384) and as many rounded products of scales (2^-25 each,
# less in the sum): 5e-7.
LIMIT = {"bf16": 1e-6, "fp16": 1e-6, "row": 4e-7, "block": 5e-7}


@pytest.mark.parametrize("mode,scales", MODES)
@pytest.mark.parametrize("k", [1024, 4096, 16384])
@pytest.mark.parametrize("sizes,n,ctas", [([40], 300, 1), ([300, 200], 300, 1), ([700], 300, 1),
                                          ([2500], 2056, 2)])
def test_fp32_results_do_not_lose_with_k(ops, sizes, n, ctas, k, mode, scales):
    if ctas == 2 and k == 1024:
        sizes = [4000]  # (pairs for block scales too)
    case = Experts(sizes, n=n, k=k, mode=mode, scales=scales, seed=39)
    assert plan_of(case, F32)[0] == ctas
    args = case.on(DEV)
    got = ops.grouped_gemm(args["a"], args["b"], args["group_start"], mode,
                           a_scales=args["a_scales"], b_scales=args["b_scales"])
    out = oracle(case)[0]
    off = ((got.double() - out).norm() / out.norm()).item()
    assert off <= LIMIT[mode if scales == "none" else scales]
