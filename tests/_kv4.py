"""The cache of keys and values in 4 bits and attention over it, in 64 bits, written from the definition, and the inputs
that their tests share."""

import math

import torch

import _serving as ref

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
MOST = {torch.bfloat16: 125, torch.float16: 13}  # the largest exponent of a scale


def encode(x):
    """x [..., D] -> (codes [..., D / 2], scales [..., D / 32]), by looking for the nearest of all values."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    bad = ~g.isfinite().all(-1, keepdim=True)
    g = torch.where(bad, 0.0, g)
    e = torch.full_like(top, -126)
    for n in range(-126, MOST[x.dtype]):  # the least e with top < 7 * 2^e
        e = torch.where(torch.ldexp(torch.tensor(7.0, dtype=torch.float64), torch.tensor(n)) <= top, n + 1.0, e)
    e = e.clamp_max(MOST[x.dtype])
    far = (torch.ldexp(g.abs(), -e)[..., None] - GRID).abs()
    near = far == far.amin(-1, keepdim=True)
    even = torch.tensor([1, 0, 1, 0, 1, 0, 1, 0], dtype=torch.bool)
    both = near.sum(-1, keepdim=True) > 1
    code = (near & (even | ~both)).int().argmax(-1) + 8 * torch.signbit(g).long()
    code = torch.where(bad, 0, code).flatten(-2)
    scale = torch.where(bad, 255, e + 127)[..., 0]
    return (code[..., ::2] | code[..., 1::2] << 4).to(torch.uint8), scale.to(torch.uint8)


def decode(codes, scales):
    """[..., D] in 64 bits; NaN where the scale is above 252."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    value = torch.where(c > 7, -GRID[c % 8], GRID[c % 8])
    power = torch.where(scales > 252, math.nan, torch.ldexp(torch.ones(()).double(), scales.double() - 127))
    return value * power.repeat_interleave(32, -1)


def flat(x):
    """A cache tensor [pages, Hk, block, n] by slots: [slots, Hk, n]."""
    return x.transpose(1, 2).flatten(0, 1)


def attention64(q, cache, tables, lens, scale=None):
    """attention64 of _serving over the cache's values, its bound with what the queries' terms add: in e4m3 with the row's
    largest at 2^7 at least, an element below 2^-6 is off by 2^-10 of a term that counts 2^-4, so by 2^-14, 2^-21 of the
    row's largest (two terms; of fp16 three, 2^-25); a score then by that times the sum of a key's magnitudes, and a
    weight and their sum by as much relative to them."""
    block = cache[0].shape[2]
    k, v = (flat(decode(*cache[i:i + 2])) for i in (0, 2))
    none = torch.zeros(0, dtype=torch.int32)
    out, extra = ref.attention64(q, k, v, none, 0, tables, lens, block, scale)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    off = 2.0 ** (-21 if q.dtype == torch.bfloat16 else -25) * q.double().abs().amax(-1, keepdim=True)
    off = off * k.nan_to_num().abs().sum(-1).max() * scale
    return out, extra + 2 * off * v.nan_to_num().abs().max()


def inputs(g, dtype, batch, seq, hq, hk, d, block, lens, spare=2, peak=1.5, power=(122, 127)):
    """Scattered pages for sequences of `lens` keys; pages of no table, and rows behind a length, are NaN."""
    each = max(1, max(-(-n // block) for n in lens))
    pages = batch * each + spare
    tables = torch.randperm(pages, generator=g)[:batch * each].int().view(batch, each)
    cache = []
    for _ in range(2):
        codes = torch.randint(0, 256, (pages, hk, block, d // 2), generator=g).to(torch.uint8)
        scales = torch.full((pages, hk, block, d // 32), 255, dtype=torch.uint8)
        for b, n in enumerate(lens):
            t = torch.arange(n)
            page, at = tables[b].long()[t // block], t % block
            scales[page, :, at] = torch.randint(*power, (n, hk, d // 32), generator=g).to(torch.uint8)
        cache += [codes, scales]
    q = (torch.randn(batch, seq, hq, d, generator=g) * peak).to(dtype)
    return q, cache, tables, torch.tensor(lens, dtype=torch.int32)


def rows(g, dtype, tokens, hk, d):
    """Keys or values whose groups have magnitudes from 2^-10 to 2^5, with zeros, ties and the type's extremes."""
    x = torch.randn(tokens, hk, d, generator=g) * torch.exp2(torch.randint(-10, 6, (tokens, hk, d // 32), generator=g)
                                                             .float()).repeat_interleave(32, -1)
    x = x.to(dtype)
    if tokens > 6:
        tie = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.99, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0,
                            4.0] * 2)
        x[0, 0, :32] = (tie * 2.0 ** -3).to(dtype)
        x[1, 0, :32] = 0.0
        x[2, 0, :32] = torch.finfo(dtype).tiny * torch.linspace(-3, 3, 32)
        x[3, 0, :32] = torch.finfo(dtype).max * torch.linspace(-1, 1, 32)
        x[4, 0, 32:64] = (tie * 7 / 6.9921875).to(dtype)
        x[5, 0, 32:64] = torch.finfo(dtype).smallest_normal / 4
    return x
