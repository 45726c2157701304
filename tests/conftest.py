import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "oracle"), os.path.dirname(os.path.abspath(__file__))):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


@pytest.fixture(scope="session")
def oracle():
    import pyoracle

    pyoracle.lib()
    return pyoracle


# Cases that expect a wrong value, kept as they are and run: strict, so each has to go on failing for as long as it stands here.
_WRONG_VALUES = {
    ("test_gpu_session_head_optimizer.py", "test_updates", "treelstm"):
        "sizes the step of a block that takes E = 10 inputs to H outputs by sqrt(max(1, E / H)) instead of sqrt(max(1, H / E)); "
        "test_gpu_session_step_size.py holds the latter",
}


def pytest_collection_modifyitems(items):
    for item in items:
        spec = getattr(item, "callspec", None)
        if spec is None:
            continue
        why = _WRONG_VALUES.get((item.path.name, item.originalname, spec.params.get("model")))
        if why:
            item.add_marker(pytest.mark.xfail(reason=why, strict=True, raises=AssertionError))
