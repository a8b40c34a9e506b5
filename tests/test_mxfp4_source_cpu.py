"""Rules of the MXFP4 products' sources that no run shows while all goes well; no GPU needed."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "hrm-moe_b200" / "csrc"


def _roles(name):
    """{banner: code without comments} of the kernel's warp roles."""
    body = (CSRC / name).read_text()
    body = body[body.index("__global__"):body.index("- teardown")]
    parts = re.split(r"// -{6,} (.*)\n", body)
    return {parts[i].strip("- "): re.sub(r"//.*", "", parts[i + 1]) for i in range(1, len(parts), 2)}


@pytest.mark.parametrize("name", ["gemm_mxfp4.cu", "gemm_mxfp4_pair.cu"])
def test_whole_warps_agree_on_a_wait_that_gave_up(name):
    """A role that one elected thread runs waits by itself.  In one that a whole warp runs, a lane
    that gave up alone would leave the others at the warp's next synchronisation for good: there,
    every wait is the form whose answer the lanes share."""
    roles = _roles(name)
    assert {"producer", "MMA issuer", "scales of A", "epilogue"} <= set(roles)
    alone = r"\b(wait|mbar_wait_bounded|wait_cluster_bounded)\("
    shared = r"\b(wait_warp|mbar_wait_warp)\("
    for role, code in roles.items():
        if role == "setup":  # where the kernel defines its short forms
            continue
        if role in ("scales of A", "epilogue"):
            assert re.search(shared, code) and not re.search(alone, code), role
        else:
            start = re.search(r"if \((leader && )?elect_one\(\)\) \{", code)
            first = re.search(alone, code)
            assert start and first and start.start() < first.start(), role
            assert not re.search(shared, code), role
