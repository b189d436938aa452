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
