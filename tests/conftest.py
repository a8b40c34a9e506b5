import pathlib
import sys

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]
for p in (str(ROOT), str(ROOT / "tests"), str(ROOT / "tests" / "golden")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 (sm_100a) GPU")


# Cases whose expected value is wrong, with the reason.  They stay as written and keep running;
# strict: one that passes again is reported.
WRONG_VALUES = {
    "test_gpu_11_mxfp4.py::test_experts_forward[5000-256-96-16-4]":
        "expects sum(w * bf16(e)) for calls over 8 MiB: each expert's output e rounded to bf16 before the "
        "sum, which is up to 2^-8 sum(w |e|) from the value, with room for 2^-8 |sum| only; the sum is fp32 "
        "(test_gpu_12_mxfp4_experts.py holds the same case to 64 bits)",
}


def pytest_collection_modifyitems(config, items):
    for item in items:
        for case, why in WRONG_VALUES.items():
            if item.nodeid.endswith(case):
                item.add_marker(pytest.mark.xfail(raises=AssertionError, strict=True, reason=why))
    try:
        import torch
        has_gpu = torch.cuda.is_available()
    except Exception:  # pragma: no cover
        has_gpu = False
    if has_gpu:
        return
    skip = pytest.mark.skip(reason="no CUDA device")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)
