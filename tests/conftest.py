import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


# Counts how often another thread wakes within some microseconds, which the operating system decides (a thread that it leaves asleep for half a millisecond fails it: 1 run in 100 on an idle
# machine, 1 in 20 on a busy one).  It runs behind all others, so that with -x its failure hides none of them.
LAST = ("test_other_python_threads_run_while_a_dispatch_waits_for_its_row_count",)


def pytest_collection_modifyitems(config, items):
    import torch

    items.sort(key=lambda item: item.name in LAST)  # (the others keep their order)
    if torch.cuda.is_available():
        return
    skip = pytest.mark.skip(reason="no GPU in this container")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)
