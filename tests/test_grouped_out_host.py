"""Outputs that the products refuse, without a GPU: rows that share memory."""

import pytest

FAKE = 1 << 20


@pytest.mark.parametrize("rows,n,out_row,refused", [
    (5, 8, 0, True), (5, 8, 7, True), (5, 8, -7, True), (5, 1, 0, True), (2, 64, 63, True),
    (1, 8, 0, False), (5, 8, 8, False), (5, 8, -8, False), (5, 1, 1, False)])
def test_rows_that_overlap(rows, n, out_row, refused):
    from m5kernels_b200 import _lib, grouped

    lib = _lib.lib()
    # (operands off the 16-byte grid: what is not refused for out is refused for them)
    record = grouped._PACK_GEMM.pack(
        FAKE + 8, FAKE, _lib.MODE["bf16"], rows, 1, n, 64, 64, 512, 64, FAKE, 0, 0, 0, 0, 0, 0, 0,
        0, FAKE, _lib.BF16, out_row, 0)
    code = lib.m5b_grouped_gemm(record, None)
    assert code == (_lib.EINVAL if refused else _lib.EUNSUPPORTED)
    assert (b"overlap" if refused else b"16-byte") in lib.m5b_last_error()
