"""pytest configuration: registers the ``gpu`` marker and puts the package on sys.path."""
import json
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "mindspeed-rl_amd")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run on the GPU box with -m gpu)")


def pytest_collection_modifyitems(items):
    # it looks at the error text of a library that has refused nothing yet: in front of everything that has calls refused, whatever its file's name
    items.sort(key=lambda item: item.name != "test_library_exports_every_declared_symbol")


@pytest.fixture(scope="session")
def reference_vectors():
    with open(os.path.join(ROOT, "tests", "golden", "reference_vectors.json")) as f:
        return json.load(f)


@pytest.fixture(scope="session")
def oracle_vectors():
    with open(os.path.join(ROOT, "tests", "golden", "oracle_vectors.json")) as f:
        return json.load(f)
