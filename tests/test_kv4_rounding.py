"""What kv4_attention's own arithmetic adds to its results, the kernels' source under the HIP emulation: bounds that follow
from the types alone."""

import pytest

import _kv4_rounding as cases
import test_kv4


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    lib = test_kv4.emulated(tmp_path_factory.mktemp("kv4_rounding"), "kv4_attention.hip")
    return lambda *args: test_kv4.run(lib, *args)


@pytest.mark.parametrize("case", cases.SHAPES, ids=str)
@pytest.mark.parametrize("dtype", cases.DTYPES, ids=str)
def test_weights(run, case, dtype):
    cases.check_weights(run, case, dtype)
