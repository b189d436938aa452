"""Log probabilities with entropy and alternatives in 64 bits, and the rows that their tests share."""

import math

import torch


def logprobs64(x, tokens, top):
    """(logprobs, entropy, top_logprobs, top_indices), the sums in 64 bits; a row at a time."""
    out = [], [], [], []
    for row, token in zip(x.double(), tokens.tolist()):
        m = row.max()
        e = torch.exp(row - m)
        total = e.sum()
        nowhere = not bool(total > 0) or not math.isfinite(float(m))
        p = row - m - torch.log(total)
        out[0].append(0.0 if token < 0 else math.nan if nowhere or token >= row.numel() else float(p[token]))
        h = torch.log(total) - (e * (row - m).clamp_min(-1e30)).sum() / total
        out[1].append(math.nan if nowhere else float(h))
        # descending by value, +0 above -0, then by index
        order = sorted(range(row.numel()), key=lambda i: (-float(row[i]), bool(torch.signbit(row[i])), i))[:top] \
            if not nowhere and row.numel() < 3000 else None
        if order is None and not nowhere:
            key = row.float().view(torch.int32).long()
            key = torch.where(key < 0, key ^ 0x7fffffff, key)
            order = torch.sort(key, descending=True, stable=True).indices[:top].tolist()
        out[2].append([math.nan] * top if nowhere else [float(p[i]) for i in order])
        out[3].append([-1] * top if nowhere else order)
    f = lambda v, *shape: torch.tensor(v, dtype=torch.float64).view(*shape)
    n = len(out[0])
    return f(out[0], n), f(out[1], n), f(out[2], n, top), torch.tensor(out[3], dtype=torch.int64).view(n, top)


def near(got, want):
    """With u = 2^-24: an exponent t = (x - m) log2(e) is rounded twice and log2(e) is off by u of itself: off by 3 u |t|,
    and the exponential by 2 u more, so a weight by u (3 ln 2 |t| + 2) of itself, up to 32 of them summed in fp32 by 32 u.
    What is 150 ln 2 and more below a row's largest weighs nothing, so |t| counts up to 150. The logarithm of the sum is off
    by as much; the entropy's mean of t ln 2 by that times its own size (150 ln 2 at most) and twice; all rounded to fp32."""
    u = 2.0 ** -24
    rel, ok = u * (3 * math.log(2) * 150 + 2 + 32 + 4), True
    for a, b, by in zip(got, want, (1.0, 2 + 150 * math.log(2), 1.0)):
        d = (a.double().cpu() - b).abs()
        d = torch.where(a.double().cpu() == b, 0.0, d)  # infinities
        same = a.isnan().cpu() == b.isnan()
        ok = ok and bool(same.all()) and bool((d.nan_to_num(0.0) <= rel * by + u * b.abs().nan_to_num(0.0)).all())
    return ok


def logits(g, rows, n, dtype, scale=2.5):
    x = torch.randn(rows, n, generator=g) * scale
    return x.to(dtype), torch.randint(0, n, (rows,), generator=g)


def edge_rows(g, n, dtype):
    """Rows that masks, ties and the type's extremes leave."""
    low, inf = torch.finfo(dtype).min, float("inf")
    rows = []
    base = torch.randn(n, generator=g) * 2
    rows.append(torch.full((n,), 1.5))                             # all equal
    rows.append(torch.arange(n) * (8.0 / n))                       # ascending
    rows.append(-torch.arange(n) * (8.0 / n))                      # descending
    rows.append(torch.full((n,), low))                             # all masked by the lowest value
    rows.append(torch.where(torch.rand(n, generator=g) < 0.9, low, base))
    rows.append(torch.where(torch.rand(n, generator=g) < 0.9, -inf, base))
    one = torch.full((n,), -inf)
    one[n // 2] = 3.0
    rows.append(one)                                               # one token left
    rows.append(torch.full((n,), -inf))                            # none
    bad = base.clone()
    bad[n // 3] = float("nan")
    rows.append(bad)
    bad = base.clone()
    bad[n // 3] = inf
    rows.append(bad)
    sure = base.clone()
    sure[n - 1] = 40.0
    rows.append(sure)
    zero = torch.zeros(n)
    zero[::2] = -0.0
    rows.append(zero)
    rows.append(base.abs() * (torch.finfo(dtype).max / 16))        # large
    rows.append(base.round())                                      # many ties
    x = torch.stack(rows).to(dtype)
    tokens = torch.randint(0, n, (x.shape[0],), generator=g)
    tokens[6], tokens[1], tokens[2] = n // 2, -100, n
    return x, tokens
