"""Log probabilities and entropies of rows whose token is sure, the kernels' own source under the HIP emulation."""

import pytest
import torch

import _sure_rows as sure
import test_token_logprobs
from test_token_logprobs import lib  # noqa: F401  (the emulated library)

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("n,first,parts", [(3000, 0, 1), (9001, 77, 0), (25000, 2500, 0), (25000, 4090, 3)], ids=str)
@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_two_tokens(lib, n, first, parts, top, dtype):  # noqa: F811
    x, tokens = sure.two_tokens(n, dtype, first)
    lib.token_logprobs_tune(0, parts)
    try:
        got = test_token_logprobs.run(lib, x, tokens, min(top, 2))
    finally:
        lib.token_logprobs_tune(0, 0)
    assert sure.near(got, x, tokens)


@pytest.mark.parametrize("n", [40, 700, 10007])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_sure_rows(lib, n, dtype):  # noqa: F811
    x, tokens = sure.sure_rows(torch.Generator().manual_seed(n), 8, n, dtype)
    assert sure.near(test_token_logprobs.run(lib, x, tokens, 2), x, tokens)
