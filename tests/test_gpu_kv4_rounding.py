"""What kv4_attention's own arithmetic adds to its results on the GPU: bounds that follow from the types alone."""

import pytest
import torch

import _kv4_rounding as cases

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def run(pkg):
    def call(q, cache, tables, lens):
        return pkg.ops().kv4_attention(*(t.to("cuda:0") for t in (q, *cache, tables, lens))).cpu()
    return call


@pytest.mark.parametrize("case", cases.SHAPES + [(9, 1, 32, 8, 128, 64, [1 + 300 * i for i in range(9)]),
                                                 (4, 16, 8, 2, 256, 32, [700] * 4)], ids=str)
@pytest.mark.parametrize("dtype", cases.DTYPES, ids=str)
def test_weights(run, case, dtype):
    cases.check_weights(run, case, dtype)


@pytest.mark.parametrize("case,down", [(cases.SHAPES[i], down) for i in range(4) for down in (14, 18, 22)] +
                         [(cases.SHAPES[1], 10), (cases.SHAPES[0], 26), ((3, 2, 8, 2, 128, 16, [900, 33, 2000]), 20),
                          ((2, 16, 32, 4, 256, 32, [300, 1200]), 20), ((70, 1, 8, 2, 64, 64, [300] * 70), 18)], ids=str)
@pytest.mark.parametrize("dtype", cases.DTYPES, ids=str)
def test_far_elements(run, case, down, dtype):
    cases.check_far_elements(run, case, dtype, down)


def test_a_far_element_in_one_head(run):
    cases.check_far_elements(run, cases.SHAPES[1], cases.DTYPES[0], 20, rows=[3])


@pytest.mark.parametrize("dtype,mixed", [(cases.DTYPES[0], False), (cases.DTYPES[0], True), (cases.DTYPES[1], False)],
                         ids=str)
def test_small_numbers(run, dtype, mixed):
    cases.check_small_numbers(run, dtype, mixed)


@pytest.mark.parametrize("large", [30.0, 120.0, 500.0])
@pytest.mark.parametrize("case", cases.SHAPES + [(9, 1, 32, 8, 128, 64, [1 + 300 * i for i in range(9)])], ids=str)
@pytest.mark.parametrize("dtype", cases.DTYPES, ids=str)
def test_large_products(run, case, large, dtype):
    """The products of 4-bit and 8-bit numbers that the device has keep some 18 bits of the largest."""
    cases.check_large_products(run, case, dtype, large)
