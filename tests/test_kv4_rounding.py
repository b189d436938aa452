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


@pytest.mark.parametrize("case,down", [(cases.SHAPES[i], down) for i in range(4) for down in (14, 18, 22)] +
                         [(cases.SHAPES[1], 10), (cases.SHAPES[0], 26)], ids=str)
@pytest.mark.parametrize("dtype", cases.DTYPES, ids=str)
def test_far_elements(run, case, down, dtype):
    cases.check_far_elements(run, case, dtype, down)


def test_a_far_element_in_one_head(run):
    cases.check_far_elements(run, cases.SHAPES[1], cases.DTYPES[0], 20, rows=[3])


@pytest.mark.parametrize("dtype,mixed", [(cases.DTYPES[0], False), (cases.DTYPES[0], True), (cases.DTYPES[1], False)],
                         ids=str)
def test_small_numbers(run, dtype, mixed):
    cases.check_small_numbers(run, dtype, mixed)


@pytest.mark.parametrize("dtype", cases.DTYPES, ids=str)
def test_large_products(run, dtype):
    cases.check_large_products(run, cases.SHAPES[1], dtype, 120.0)
