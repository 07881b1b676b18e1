"""Warps that meet in a named barrier give up a wait together or not at all.

A bounded wait that expires makes its warp leave for the end of the kernel.  Warps that poll apart can come to different verdicts (the limit passes
between two polls, or the error word was set before); one that goes on would then stand in the named barrier of the epilogue for good.  Checked
in the source: what it would take to see it on hardware is a hang."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "torchure_b200" / "csrc"


def _code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def _arguments(text, at):
    """The arguments of the call whose opening bracket is at ``at``."""
    parts, depth, begin = [], 0, at + 1
    for i in range(at, len(text)):
        depth += (text[i] in "([{") - (text[i] in ")]}")
        if depth == 0:
            return [p.strip() for p in [*parts, text[begin:i]]]
        if depth == 1 and text[i] == ",":
            parts.append(text[begin:i])
            begin = i + 1
    raise ValueError("unbalanced")


def test_epilogues_with_named_barriers_wait_with_one_verdict():
    text = _code("grouped_gemm_sm100.cu")
    calls = [m for m in re.finditer(r"\brows_epilogue<EPI>\(", text)]
    assert len(calls) == 2
    for call in calls:
        wait = [m for m in re.finditer(r"\bmbar_wait\w*\(", text[:call.start()])][-1]
        assert wait.group() == "mbar_wait_warps(", "the warps of the epilogue poll apart"
        barrier, threads = _arguments(text, wait.end() - 1)[-2:]
        assert _arguments(text, call.end() - 1)[4] == barrier and threads == "128"


def test_other_files_have_no_named_barrier_behind_a_verdict_of_one_warp():
    """Two files have named barriers besides: one in a role without waits, one whose warps go on whatever the verdict."""
    with_barriers = {p.name for p in CSRC.glob("*.cu") if "named_bar_sync(" in p.read_text()}
    assert with_barriers == {"gemm_sm100.cu", "elementwise.cu", "grouped_gemm_sm100.cu"}
    copy = _code("gemm_sm100.cu")
    begin = copy.index("ag_copy_phase(const GemmComm*")
    role = copy[begin:copy.index("template <bool A_MN", begin)]
    assert role.count("named_bar_sync(") == copy.count("named_bar_sync(") == 1 and "mbar_wait" not in role
    rows = _code("elementwise.cu")
    assert rows.count("named_bar_sync(") == 1
    before = rows[:rows.index("named_bar_sync(")]
    assert re.search(r"ok = mbar_wait_warp\([^;]*\) && ok;", before[before.rindex("mbar_wait") - 10:])


def test_the_helper_votes_over_the_barrier():
    text = _code("common.cuh")
    body = text[text.index("bool mbar_wait_warps("):]
    body = body[:body.index("\n}")]
    assert "mbar_wait_warp(" in body and "__syncwarp();" in body[:body.index("bar.red.and.pred")]


def test_dependents_are_let_in_behind_the_wait():
    """Kernels that read matrices before the kernel before has ended rely on it: whoever lets them in has waited, so that all that came before
    it on the stream, what wrote the matrices included, has ended."""
    seen = 0
    for path in CSRC.glob("*.cu"):
        text = _code(path.name)
        for m in re.finditer(r"\bpdl_launch_dependents\(\);", text):
            assert text[:m.start()].rstrip().endswith("pdl_wait();"), path.name
            seen += 1
    assert seen >= 20
