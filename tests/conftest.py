import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run on the B200 box)")


@pytest.fixture(scope="session")
def built_libs():
    """Every kernel variant, compiled in-tree (a no-op when the binaries are current)."""
    from unimonomoe_b200 import build
    return build.build_all()


@pytest.fixture(scope="session")
def attention_lib():
    from unimonomoe_b200 import build
    return build.build_attention()


@pytest.fixture(scope="session")
def linear_lib():
    from unimonomoe_b200 import build
    return build.build_linear()


@pytest.fixture(scope="session")
def oracle():
    from oracle import cpu_oracle
    cpu_oracle.build()
    return cpu_oracle
