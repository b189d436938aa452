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
    """Queries of few bits. A weight in [2^e, 2^(e + 1)) is a bf16 number and what is left of it, 2^(e - 8)
    at most, so another off by half a step of that: 2^(e - 17), 2^-17 of the weight."""
    batch, seq, hq, hk, d, block, lens = case
    g = torch.Generator().manual_seed(d + seq)
    q, cache, tables, lens = kv4.inputs(g, dtype, batch, seq, hq, hk, d, block, lens)
    q = (q.float() * 8).round().clamp(-32, 32).div(8).to(dtype)  # of at most 6 bits, none below 2^-5 of the largest
    got = run(q, cache, tables, lens)
    out, mass, extra = attention64(q, cache, tables, lens)
    assert ref.near(got, out, extra + 2.0 ** -17 * mass)


def check_far_elements(run, case, dtype, down, rows=None):
    """Queries whose first element is 2^down above the others and meets keys that are zero there, their other elements
    large enough for scores of about 1 (of `rows` of the q heads; the others have no such element). The bound is an eighth
    of the type's half step, of what the weighted values add up to."""
    batch, seq, hq, hk, d, block, lens = case
    g = torch.Generator().manual_seed(d + down)
    top = 14 if dtype == torch.float16 else 0
    power = 127 - top + down - 1
    q, cache, tables, lens = kv4.inputs(g, dtype, batch, seq, hq, hk, d, block, lens)
    held = cache[1] != 255
    cache[1][held] = torch.randint(power - 1, power + 1, cache[1].shape, generator=g).to(torch.uint8)[held]
    cache[0][..., 0] &= 0xf0
    q = torch.randn(q.shape, generator=g).clamp(-4, 4) * 2.0 ** (top - down)
    q[:, :, slice(None) if rows is None else rows, 0] = 2.0 ** top
    q = q.to(dtype)
    got = run(q, cache, tables, lens)
    out, mass, extra = attention64(q, cache, tables, lens)
    assert ref.near(got, out, extra + ref.half_step(dtype) / 8 * mass)


def check_small_numbers(run, dtype, mixed):
    """Queries below the type's smallest normal number over large keys; or (bf16) one large element over keys below it,
    the others as in check_far_elements."""
    g = torch.Generator().manual_seed(31)
    q, cache, tables, lens = kv4.inputs(g, dtype, 1, 2, 4, 2, 64, 16, [90])
    held = cache[1] != 255
    low = torch.randint(0, 2, cache[1].shape, generator=g)
    small = -22 if dtype == torch.float16 else -128
    q = torch.randn(q.shape, generator=g).clamp(-4, 4)
    if mixed:
        q *= 2.0 ** 104
        q[..., 0] = 2.0 ** 126
        low[..., 0] += 1
        low[..., 1:] += 127 - 105
        cache[0][..., 0] = cache[0][..., 0] & 0xf0 | torch.randint(0, 2, cache[0].shape[:-1], generator=g).to(torch.uint8)
    else:
        q *= 2.0 ** small
        low += 126 - small if dtype == torch.float16 else 251
    cache[1][held] = low.clamp(0, 252).to(torch.uint8)[held]
    q = q.to(dtype)
    got = run(q, cache, tables, lens)
    out, mass, extra = attention64(q, cache, tables, lens)
    assert ref.near(got, out, extra + ref.half_step(dtype) / 8 * mass)


def check_large_products(run, case, dtype, large):
    """An element of the queries and the keys whose product is about `large` in every score, beside others of about 1: what
    sums in fp32 add to a score is small beside it, and the results show what else does."""
    batch, seq, hq, hk, d, block, lens = case
    g = torch.Generator().manual_seed(d + int(large))
    q, cache, tables, lens = kv4.inputs(g, dtype, batch, seq, hq, hk, d, block, lens, peak=1.0, power=(126, 128))
    held = cache[1] != 255
    cache[1][..., -1][held[..., -1]] = 129
    cache[0][..., -16:] &= 0x11                    # the last group: 0 or 0.5 of 2^2,
    cache[0][..., -1] = cache[0][..., -1] & 0x0f | 0x70  # its last element 6
    q[..., -32:-1] *= 0.25
    q[..., -1] = large * d ** 0.5 / 24
    got = run(q, cache, tables, lens)
    out, mass, extra = attention64(q, cache, tables, lens)
    assert ref.near(got, out, extra + ref.half_step(dtype) / 8 * mass)
