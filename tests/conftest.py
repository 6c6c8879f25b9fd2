import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG_DIR = os.path.join(ROOT, "hot-cold-neural-split-openinfer2_amd")
for p in (ROOT, PKG_DIR):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (gfx950) GPU and the built HIP library")
    config.addinivalue_line("markers", "slow: full-size CPU oracle runs")


# Cases whose expected value is wrong.  They stay as they are and run; what they
# should hold is tested in the file named beside them.
WRONG_VALUES = {
    # the loop that they compare with hands the packed tokens to
    # submit_cold_fetch as one sequence, so that the last packed token chooses the
    # neurons of every request; the batch's set is the mean over the requests' last
    # tokens (engine.py:274-283): test_gpu_packed_cold_set.py
    "test_gpu_paged_layers.py::test_step_equals_plain_loop[new1]": "predicts every request's cold set from the last packed token",
    "test_gpu_paged_layers.py::test_step_equals_plain_loop[new2]": "predicts every request's cold set from the last packed token",
}


def pytest_collection_modifyitems(items):
    for item in items:
        why = WRONG_VALUES.get(item.nodeid.split("/")[-1])
        if why:
            item.add_marker(pytest.mark.xfail(reason=why, strict=True))
