from __future__ import annotations

import sys
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]
if str(REPO) not in sys.path:
    sys.path.insert(0, str(REPO))

from tests import _reference  # noqa: E402

if not _reference.available():
    import __graft_entry__  # noqa: E402

    __graft_entry__.install_reference()


class _SkipWithoutReference:
    """Import hook of a checkout without the reference: what imports ``qwenquest`` is skipped (a module or
    a test), and what needs no reference runs."""

    def find_spec(self, name, path=None, target=None):
        if name == "qwenquest" or name.startswith("qwenquest."):
            pytest.skip("the reference package `qwenquest` is not installed", allow_module_level=True)
        return None


_reference_installed = _reference.available()
if _reference_installed:
    _reference.ensure_importable()
else:
    sys.meta_path.insert(0, _SkipWithoutReference())


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200) — run with -m gpu")


def pytest_report_header(config):
    if not _reference_installed:
        return "reference package `qwenquest`: NOT installed, the tests that run or import it are skipped"
    return "reference package `qwenquest`: installed"


#: tests that run the reference in a child process, out of the import hook's reach
_RUNS_REFERENCE = {"test_bench_contract.py"}


def pytest_collection_modifyitems(config, items):
    import torch

    if not _reference_installed:
        absent = pytest.mark.skip(reason="the reference package `qwenquest` is not installed")
        for item in items:
            if item.path.name in _RUNS_REFERENCE:
                item.add_marker(absent)
    if torch.cuda.is_available():
        return
    skip = pytest.mark.skip(reason="needs a CUDA device")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(scope="session")
def cuda_device():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda", 0)
