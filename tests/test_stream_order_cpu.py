"""Kernels of the paged serving step are launched as programmatic dependents: what their predecessor wrote is promised to a thread only behind
its own grid's griddepcontrol.wait.  Shown on the source, since a missing wait cannot be made to fail on demand."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "nomos_nvfp4_b200" / "csrc"


def kernels(name):
    """(kernel, body) of every __global__ function of a file, comments taken out."""
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    for m in re.finditer(r"__global__ void (?:__launch_bounds__\((?:[^()]|\([^()]*\))*\) )?(\w+)\([^{]*\{", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        yield m.group(1), text[m.end():at]


@pytest.mark.parametrize("name,count", [("paged_plan.cu", 1), ("paged_rows.cu", 4), ("paged_select.cu", 1), ("spec_verify.cu", 1)])
def test_every_path_waits_before_it_reads(name, count):
    """One wait per kernel, outside any branch, with nothing read through a pointer argument and no dependent let go before it."""
    found = list(kernels(name))
    assert len(found) == count
    for kernel, body in found:
        assert body.count("griddepcontrol.wait") == 1, kernel
        before = body[:body.index("griddepcontrol.wait")]
        assert before.count("{") == before.count("}"), f"{kernel}: the wait lies in a branch"
        assert "griddepcontrol.launch_dependents" not in before, kernel
        assert not re.search(r"__ldcg|append_rows<|page_bounds\(|\ba\.(slot_map|pages|src_\w+|p|q|tokens|n_draft)\s*[\[+]|\bp\.(seq_lens|n_new|held|free_count|row_seq|row_pos)\s*\[",
                             before), f"{kernel}: reads before the wait"
