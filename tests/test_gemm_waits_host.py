"""Waits of the GEMM's epilogue, read from its source, as in test_grouped_waits_host."""

import re

from test_grouped_waits_host import SOURCE

GEMM = SOURCE.with_name("gemm.cu")


def test_the_epilogue_votes_on_its_waits():
    """Waits of whole warps (the epilogue's, but for those of its one leading thread)."""
    text = re.sub(r"//[^\n]*", "", GEMM.read_text())
    body = text[text.index("const int prow = quarter * 32 + lane;"):]
    body = body[:body.index("tmem_dealloc")]
    calls = [m.start() for m in re.finditer(r"\bmbar_wait_bounded\(", body)]
    voted = [body[:at].rstrip().endswith("__all_sync(0xffffffffu,") for at in calls]
    alone = ["recv_ready" in body[at:at + 40] for at in calls]
    assert len(calls) == 4 and sum(alone) == 1
    assert all(v != a for v, a in zip(voted, alone))
