import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
GOLDEN = os.path.join(ROOT, "tests", "golden")


# Tests of programs that oracle/build_oracle.py builds from the reference tree,
# and what they run under oracle/_ref (test_oracle.py and test_llama2_cpu.py
# skip theirs by themselves).
REFERENCE_PROGRAMS = {
    "test_reference_llama_forward_on_b200": ("pin/llama2_logits", "b200/llama2_logits", "b200/llama2_logits_vxmath"),
    "test_reference_llama_generates_the_cpu_text_on_b200": ("pin/llama", "b200/llama", "b200/llama_vxmath"),
}


def missing_reference_programs(test, built=os.path.join(ROOT, "oracle", "_ref")):
    return [p for p in REFERENCE_PROGRAMS.get(test, ()) if not os.path.exists(os.path.join(built, p))]


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 (sm_100) GPU")


def pytest_collection_modifyitems(config, items):
    for item in items:
        missing = missing_reference_programs(getattr(item, "originalname", None) or item.name)
        if missing:
            item.add_marker(pytest.mark.skip(
                reason=f"reference-built {', '.join(missing)} not present (python oracle/build_oracle.py)"))
    try:
        import torch
        have_gpu = torch.cuda.is_available()
    except Exception:  # pragma: no cover
        have_gpu = False
    if have_gpu:
        return
    skip = pytest.mark.skip(reason="no CUDA device")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(scope="session")
def oracle():
    sys.path.insert(0, os.path.join(ROOT, "oracle"))
    import oracle_py
    oracle_py.lib()
    return oracle_py
