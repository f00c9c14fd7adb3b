"""Which kernel a grouped product takes, and 64-bit oracles on the GPU for those that are large."""

import ctypes

import torch

from grouped_cases import BLOCK, dequantized, values

DEV = "cuda"


def plan(rows, groups, n, k, mode, scales, dtype):
    """(CTAs of a tile: 2 a pair, its most rows, CTAs that share its K, CTAs in all)."""
    from m5kernels_b200 import _lib, grouped

    record = grouped._PACK_GEMM.pack(0, 0, _lib.MODE[mode], rows, groups, n, k, 0, 0, 0, 0,
                                     scales == "block", 0, 0, 0, 0, 0, 0, 0, 0,
                                     _lib.DTYPE_CODE[dtype], 0, 0)
    out = (ctypes.c_int64 * 4)()
    _lib.check(_lib.lib().m5b_grouped_gemm_plan(record, out))
    return tuple(out)


def plan_of(case, dtype):
    return plan(case.rows, len(case.sizes), case.n, case.k, case.mode, case.scales, dtype)


def assert_pairs(case, dtype, turns=1):
    """The product takes CTA pairs, and some pair takes `turns` tiles."""
    ctas, rows, splits, grid = plan_of(case, dtype)
    assert ctas == 2 and splits == 1
    tiles = sum(-(-s // rows) for s in case.sizes) * -(-case.n // 256)
    assert -(-tiles // (grid // 2)) >= turns


def oracle(case):
    """As Experts.oracle, on the GPU."""
    out = torch.zeros(case.rows, case.n, dtype=torch.float64, device=DEV)
    spread = torch.zeros_like(out)
    for e, rows in enumerate(case.sizes):
        if not rows:
            continue
        mine = slice(case.starts[e], case.starts[e + 1])
        a, b = case.a[mine].to(DEV), case.b[e].to(DEV)
        if case.scales == "block":
            a = dequantized(a, case.a_scales[mine].to(DEV), 1)
            b = dequantized(b, case.b_scales[e].to(DEV), BLOCK)
        else:
            a = values(a) if case.mode == "fp8" else a.double()
            b = values(b) if case.mode == "fp8" else b.double()
            if case.scales == "row":
                a = a * case.a_scales[mine, None].to(DEV).double()
                b = b * case.b_scales[e][:, None].to(DEV).double()
        out[mine], spread[mine] = a @ b.T, a.abs() @ b.abs().T
    return out, spread
