import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


# Tests whose expected pairs are wrong, kept as they are: score_oracle.distill has p - q for the gradient also where the teacher's masses do not come to
# one (every class named and some left over, or entries that have more than one together), which is not the slope of its own loss
# (test_teacher_oracle_cpu.py). Their inputs are held against the slope in test_gpu_distill_ends.py.
WRONG_PAIRS = {
    "test_gpu_class_scores.py::test_distill": ["8-1000-5-True", "9-257-9-True", "31-65-40-True", "100-16-10-True", "129-63-64-True", "300-300-128-True", "1000-40-32-True"],
    "test_gpu_class_scores.py::test_distill_far_scores": ["5-6"],
    "test_gpu_class_scores_large.py::test_distill_many_rows": ["33-16384-128"],
}


def pytest_collection_modifyitems(items):
    for item in items:
        test, _, case = item.nodeid.rsplit("/", 1)[-1].partition("[")
        if case[:-1] in WRONG_PAIRS.get(test, ()):
            item.add_marker(pytest.mark.xfail(raises=AssertionError, strict=True, reason="expects p - q where the loss's slope is M p - q, M not being one"))
