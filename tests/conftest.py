import shutil
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run with -m gpu on a B200)")


@pytest.fixture(autouse=True)
def _packages_do_not_stay(request):
    """A test's folder goes with it: packages hold every kernel, and those of the whole suite took 73 GB."""
    yield
    folder = request.node.funcargs.get("tmp_path")
    if folder is not None:
        shutil.rmtree(folder, ignore_errors=True)
