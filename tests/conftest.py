import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")
    config.addinivalue_line("markers", "no_gpu: passes made-up addresses through all checks, which only a missing device stops; skipped where there is one")


def devices():
    import torch
    return torch.cuda.device_count()


def pytest_collection_modifyitems(items):
    made_up = [item for item in items if item.get_closest_marker("no_gpu") or item.name == "test_columns_of_one_row_are_apart"]
    if made_up and devices():
        for item in made_up:
            item.add_marker(pytest.mark.skip(reason="made-up addresses, and a device that would go there"))


@pytest.fixture(scope="session")
def oracle():
    from tests import oracle_api
    return oracle_api.load_oracle()


@pytest.fixture(scope="session")
def hq():
    """The product package on a GPU box; fails loudly if libhq.so is missing."""
    import torch
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    import hecbench_amd
    hecbench_amd.init()
    return hecbench_amd


@pytest.fixture
def tunable():
    """Sets launch-shape knobs of the library through hq_set_tunable and clears them afterwards."""
    from hecbench_amd import _lib
    lib = _lib.load()
    touched = []

    def set_(name, value):
        rc = lib.hq_set_tunable(name.encode(), int(value), 0)
        assert rc == 0, (name, rc)
        touched.append(name)

    yield set_
    for name in touched:
        lib.hq_set_tunable(name.encode(), 0, 1)
