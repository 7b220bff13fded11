"""What no run can show without the risk of a fault: rules that the kernels' source has to keep."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "ltq_research_b200" / "csrc"


def body(file: str, function: str) -> str:
    """The text of a function's definition, comments taken out."""
    text = re.sub(r"//[^\n]*", "", (CSRC / file).read_text())
    start = re.search(re.escape(function) + r"\([^;{]*\)\s*\{", text)
    assert start, f"{file} defines no {function}"
    depth, i = 1, start.end()
    while depth:
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        i += 1
    return text[start.end():i]


@pytest.mark.parametrize("file,function", [("ltq_embed.cu", "sort_cluster"), ("ltq_distill.cu", "distill_rows_kernel"),
                                           ("ltq_fp8_few.cu", "gemm_few_kernel")])
def test_other_ctas_have_started_before_their_memory_is_written(file, function):
    """A CTA of the cluster may be written to once it is known to run: a wait for the cluster's barrier comes before the first
    store into another CTA's shared memory."""
    code = body(file, function)
    stores = [m.start() for m in re.finditer(r"st_cluster_u32|st\.shared::cluster", code)]
    assert stores
    wait = code.find("cluster_wait")
    assert 0 <= wait < stores[0]


def test_bounded_waits_of_whole_warps_have_one_answer():
    """Lanes of a warp that took a wait's answer each for itself could part at its limit and then hang at the next instruction of
    the whole warp.  So a role of whole warps polls together.  Of the bf16 products only the epilogues are whole warps; their other roles
    are one lane."""
    for file, function in (("ltq_fp8_gemm.cu", "gemm_wide_kernel"), ("ltq_fp8_few.cu", "gemm_few_kernel")):
        assert not re.search(r"\bmbar_wait\(", body(file, function)), function
    assert "__all_sync(0xffffffffu, mbar_try_wait(" in body("tc_pipe.cuh", "mbar_wait_warp")
    for function in ("epilogue_tma", "epilogue"):
        assert not re.search(r"\bmbar_wait\(", body("ltq_gemm_tc.cu", function)), function
    persistent = (CSRC / "ltq_gemm_tc.cu").read_text().split("epilogue warps: lane quarter")[1]
    assert not re.search(r"\bmbar_wait\(", persistent.split("tcgen05.dealloc")[0])
