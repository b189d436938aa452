"""Causal attention of packed prompts in 64 bits, a query at a time, and the inputs that its tests share."""

import torch

import _serving as ref


def attention64(q, k, v, offsets, scale=None):
    """(out, extra) as attention64 of _serving: each prompt is a sequence of its own keys, every token a query of them. Its
    bound holds here as well: the same products, the same rounding of the weights."""
    out, extra = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    none = torch.zeros(0, dtype=torch.int32)
    offsets = [min(max(int(x), 0), q.shape[0]) for x in offsets]
    for a, b in zip(offsets, offsets[1:]):
        if b > a:
            table = torch.arange(b - a, dtype=torch.int32)[None]
            o, e = ref.attention64(q[a:b][None], k[a:b], v[a:b], none, 0, table, torch.tensor([b - a]), 1, scale)
            out[a:b], extra[a:b] = o[0], e[0]
    return out, extra


def inputs(g, dtype, lens, hq, hk, d, before=0, behind=0, peak=1.5):
    """q, k, v, offsets; rows of no prompt are NaN."""
    rows = before + sum(lens) + behind
    q, k, v = (torch.randn(rows, h, d, generator=g) * p for h, p in ((hq, peak), (hk, 1.0), (hk, 1.0)))
    for t in (q, k, v):
        t[:before], t[rows - behind:] = float("nan"), float("nan")
    offsets = torch.tensor([before] + lens).cumsum(0).int()
    return q.to(dtype), k.to(dtype), v.to(dtype), offsets
