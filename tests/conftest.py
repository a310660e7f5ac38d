import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "oracle")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (gfx950) GPU")


@pytest.fixture(scope="session")
def oracle():
    import oracle as _oracle

    _oracle.lib()
    return _oracle


# Expected to fail, strictly: what they expect is not the definition's value.  A beam whose 5000 logits are
# all L = -3.4e38 is uniform: each value is score - log 5000.  The test forms (score + L) -
# (L + log 5000) in 64 bits, where neither the score nor the logarithm is left beside L (a unit of
# L's last place is 2^75), and expects 0, above the beam's own score.  (fp16's L is -65504: right.)
# test_generate_edges_gpu.py::test_masked_rows holds such beams against the definition.
EXPECT_A_WRONG_VALUE = ("test_generate_ops_gpu.py::test_select_masks[dtype0]",
                        "test_generate_ops_gpu.py::test_select_masks[dtype2]")


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid.endswith(EXPECT_A_WRONG_VALUE):
            item.add_marker(pytest.mark.xfail(strict=True, raises=AssertionError,
                                              reason="expects 0 for score - log 5000"))
