"""Waits of the grouped kernel, read from its source: what a wait that gives up leads to cannot be
run on a GPU without breaking a kernel."""

import re
from pathlib import Path

SOURCE = Path(__file__).resolve().parents[1] / "m5-max-kernels_b200" / "csrc" / "grouped_gemm.cu"


def waits(text):
    """(text before the call, headers of the blocks it stands in) of each wait of the kernel."""
    text = re.sub(r"//[^\n]*", "", text)
    text = text[text.index("grouped_gemm_kernel("):]
    depth, headers, at, found = 0, [], 0, []
    for m in re.finditer(r"[{};]|\bmbar_(?:wait|try_wait)\w*\(", text):
        token = m.group()
        if token == "{":
            headers.append(" ".join(text[at:m.start()].split()))
            depth += 1
        elif token == "}":
            headers.pop()
            depth -= 1
            if depth == 0:
                return found
        elif token != ";":
            before = text[at:m.start()].rstrip()
            if token == "mbar_wait_lean(":  # votes itself, see below
                before += "LEAN"
            found.append((before, list(headers)))
            continue
        at = m.end()


def test_waits_of_whole_warps_are_voted_on():
    """Lanes of a warp may see a barrier's end and the abort flag in either order.  A wait is one
    elected thread's, or its answer is made the warp's before the aligned instructions (tcgen05
    loads, votes, barriers of the cluster) that follow."""
    found = waits(SOURCE.read_text())
    assert len(found) >= 10
    alone = [h for _, h in found if any("elect_one()" in x for x in h)]
    assert len(alone) >= 5
    for before, headers in found:
        if not any("elect_one()" in x for x in headers):
            assert before.endswith("whole_warp(") or before.endswith("LEAN"), before
    assert re.search(r"bool whole_warp\(bool ok\) \{\s*return __all_sync\(0xffffffffu, ok\);",
                     SOURCE.read_text())


def test_the_lean_wait_leaves_by_votes():
    text = re.sub(r"//[^\n]*", "", SOURCE.read_text())
    body = text[text.index("bool mbar_wait_lean("):]
    body = body[:body.index("\n}")]
    conditions = [" ".join(c.split()) for c in re.findall(r"if \((.*)\) (?:return|\{)", body)]
    assert len(conditions) == 3 == body.count("return")
    assert all("whole_warp(" in c for c in conditions), conditions
