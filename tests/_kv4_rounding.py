"""What attention over the cache in 4 bits may add to its results, from the types alone, and the inputs that show it."""

import math

import torch

import _kv4 as kv4
import _serving as ref

DTYPES = [torch.bfloat16, torch.float16]
SHAPES = [(2, 1, 4, 2, 64, 8, [40, 330]), (1, 3, 8, 2, 128, 32, [500]), (1, 2, 4, 2, 96, 16, [150]),
          (1, 9, 4, 1, 256, 64, [200])]  # batch, seq, q heads, kv heads, head size, page, lengths


def attention64(q, cache, tables, lens):
    """(out, mass, extra): the formula in 64 bits, the weighted sum of the values' magnitudes, and what sums in fp32 add
    (attention64 of _serving, whose weights are rounded to q's type: here to fp32)."""
    block = cache[0].shape[2]
    k, v = (kv4.flat(kv4.decode(*cache[i:i + 2])) for i in (0, 2))
    none = torch.zeros(0, dtype=torch.int32)
    out, extra = ref.attention64(q.float(), k, v, none, 0, tables, lens, block)
    mass, _ = ref.attention64(q.float(), k, v.abs(), none, 0, tables, lens, block)
    return out, mass, extra


def check_weights(run, case, dtype):
    """Queries that two numbers of 4 bits hold. A weight in [2^e, 2^(e + 1)) is a bf16 number and what is left of it, 2^(e - 8)
    at most, so another off by half a step of that: 2^(e - 17), 2^-17 of the weight."""
    batch, seq, hq, hk, d, block, lens = case
    g = torch.Generator().manual_seed(d + seq)
    q, cache, tables, lens = kv4.inputs(g, dtype, batch, seq, hq, hk, d, block, lens)
    q = (q.float() * 8).round().clamp(-32, 32).div(8).to(dtype)  # of at most 6 bits, none below 2^-5 of the largest
    got = run(q, cache, tables, lens)
    out, mass, extra = attention64(q, cache, tables, lens)
    assert ref.near(got, out, extra + 2.0 ** -17 * mass)
