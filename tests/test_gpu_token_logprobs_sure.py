"""Log probabilities and entropies of rows whose token is sure, on the GPU."""

import ctypes

import pytest
import torch

import _sure_rows as sure

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("n,first,parts", [(3000, 0, 1), (9001, 77, 0), (25000, 2500, 0), (128256, 70001, 1),
                                           (128256, 70001, 0), (25000, 4090, 3)], ids=str)
@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_two_tokens(pkg, n, first, parts, top, dtype):
    x, tokens = sure.two_tokens(n, dtype, first)
    lib = ctypes.CDLL(pkg.lib_path("token_logprobs"))
    lib.token_logprobs_tune(0, parts)
    try:
        got = pkg.ops().token_logprobs(x.cuda(), tokens.cuda(), top)
    finally:
        lib.token_logprobs_tune(0, 0)
    assert sure.near(got, x, tokens)


@pytest.mark.parametrize("n", [40, 700, 10007, 262144])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_sure_rows(pkg, n, dtype):
    x, tokens = sure.sure_rows(torch.Generator().manual_seed(n), 8, n, dtype)
    assert sure.near(pkg.ops().token_logprobs(x.cuda(), tokens.cuda(), 5), x, tokens)
