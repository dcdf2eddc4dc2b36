import os
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if REPO not in sys.path:
    sys.path.insert(0, REPO)

import __graft_entry__  # noqa: E402


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200, sm_100a)")


# A test that compares with the reference's own code cannot run where that code was not compiled (its
# sources were absent at build time): it is skipped with that reason, whether it meets the missing
# library in a fixture or in its body.
def _skip_without_reference(outcome):
    missing = getattr(sys.modules.get("oracle"), "ReferenceMissing", ())
    if isinstance(outcome.exception, missing):
        try:
            pytest.skip(str(outcome.exception))
        except pytest.skip.Exception as e:
            outcome.force_exception(e)


@pytest.hookimpl(hookwrapper=True)
def pytest_fixture_setup():
    _skip_without_reference((yield))


@pytest.hookimpl(hookwrapper=True)
def pytest_pyfunc_call():
    _skip_without_reference((yield))


@pytest.fixture(scope="session")
def pkg():
    return __graft_entry__.load_package()


@pytest.fixture(scope="session")
def orc():
    return __graft_entry__.load_oracle()


@pytest.fixture(scope="session")
def cuda():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    return torch
