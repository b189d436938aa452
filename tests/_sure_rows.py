"""Rows of logits whose token is sure, and how near their log probability and entropy have to be: they are as small as
the rest of the row, wherever that lies."""

import math

import torch

import _logprobs as ref

DISTANCES = [1, 3, 4, 7, 8, 33, 255, 256, 500, 511, 512, 1024, 2047, 2048, 8192, 20001]


def two_tokens(n, dtype, first=0):
    """One row to each distance that fits: 25 and 5, and nothing else."""
    fits = [d for d in DISTANCES if first + d < n]
    x = torch.full((2 * len(fits), n), -math.inf)
    tokens = torch.empty(2 * len(fits), dtype=torch.int64)
    for i, d in enumerate(fits):
        x[2 * i, first], x[2 * i, first + d], tokens[2 * i] = 25.0, 5.0, first
        x[2 * i + 1, first + d], x[2 * i + 1, first], tokens[2 * i + 1] = 25.0, 5.0, first + d
    return x.to(dtype), tokens


def sure_rows(g, rows, n, dtype):
    x = torch.randn(rows, n, generator=g) * 2.5
    tokens = torch.randint(0, n, (rows,), generator=g)
    x[torch.arange(rows), tokens] = 20.0 + 2.0 * torch.arange(rows)
    x[::2] = x[::2].masked_fill_(torch.rand(x[::2].shape, generator=g) < 0.9, -math.inf)
    x[torch.arange(rows), tokens] = 20.0 + 2.0 * torch.arange(rows)
    return x.to(dtype), tokens


def near(got, x, tokens):
    """With u = 2^-24: a weight is off by u (3 ln 2 |t| + 2) of itself at an exponent of |t| up to 150 (150 ln 2 below the
    largest nothing is left), up to 32 of them summed in fp32 by 32 u, and the results are rounded: 2^-15 of themselves. (A
    largest weight of 1 that is summed with them takes 2^-25 from each sum.) In fp64 a sum of 1 and more is rounded by 2^-53,
    some 200 times on the way from 250000 elements to a row's, here and in what it is held against: 2^-45."""
    want = ref.logprobs64(x, tokens, 0)
    return all(bool(((a.double().cpu() - b).abs() <= 2.0 ** -15 * b.abs() + 2.0 ** -45).all())
               for a, b in zip(got[:2], want[:2]))
