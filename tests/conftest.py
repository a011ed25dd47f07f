import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


# Tests of the argument checks whose accepted calls get as far as a launch on made-up addresses, which fails where there is no GPU and must not
# happen where there is one.  What they ask is asked on a stand-in for the kernels' layer too (test_rows_accepted.py), on any machine.
LAUNCHES_ON_MADE_UP_ADDRESSES = {"test_rows_side_by_side_do_not_overlap"}


def pytest_collection_modifyitems(items):
    if os.path.exists("/dev/kfd"):
        for item in items:
            if item.name in LAUNCHES_ON_MADE_UP_ADDRESSES:
                item.add_marker(pytest.mark.skip(reason="would launch on made-up addresses"))


@pytest.fixture(scope="session")
def cutt():
    """The ctypes binding of libcutt.so; fails loudly when the library has not been built."""
    import cutt_amd
    cutt_amd.lib()
    return cutt_amd


@pytest.fixture(scope="session")
def oracle_mod():
    import oracle
    oracle.lib()
    return oracle
