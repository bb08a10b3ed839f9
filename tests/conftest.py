"""Test configuration: the `gpu` marker and import paths.

Tests marked `gpu` need a HIP device and the in-tree library
(full-inference-engine_amd/fie_amd/_native/libfie_sampler.so, built by
`__graft_entry__.build()`); everything else runs on the CPU.
"""

import os
import sys

import pytest

_REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for sub in ("full-inference-engine_amd", "oracle"):
    p = os.path.join(_REPO, sub)
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a HIP device (MI355X) and the built library")


# Tests that expect a value that the definition does not give.  They stay as they are and run;
# the tests named beside them hold what the definition gives.
_WRONG_VALUES = {
    ("test_gpu_norm.py", "test_quantize_rows_is_the_ieee_quotient"):
        "takes the scale of a row with a NaN from its other elements; max|row| / 127 is NaN "
        "(test_gpu_quantize_values.py, test of the same name)",
}


def pytest_collection_modifyitems(items):
    for item in items:
        why = _WRONG_VALUES.get((item.path.name, getattr(item, "originalname", item.name)))
        if why:
            item.add_marker(pytest.mark.xfail(reason=why, raises=AssertionError, strict=True))


@pytest.fixture(scope="session")
def oracle_lib():
    import oracle

    oracle.build()
    return oracle
