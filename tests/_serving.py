"""The serving step's operators in 64 bits, written from their formulas, and the inputs that their tests share."""

import math

import torch

EPS = 1e-6


def half_step(dtype):
    """How far a rounding to dtype moves a value at most, relative to it."""
    return torch.finfo(dtype).eps / 2


def inv_freq_of(rotary, theta=10000.0):
    return 1.0 / (theta ** (torch.arange(0, rotary, 2, dtype=torch.int64).float() / max(1, rotary)))


def norm_rope64(x, position_ids, inv_freq, weight=None, eps=EPS):
    """x [B, S, H, D]: the norm of each head, its weight, the rotation of the first 2 len(inv_freq) elements."""
    x = x.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if weight is not None:
        x = x * weight.double()
    half = inv_freq.numel()
    angle = position_ids.double()[:, :, None, None] * inv_freq.double()
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), x[..., 2 * half:]), -1)


def norm_rope_error(x, weight=None, eps=EPS):
    """A bound of what fp32 arithmetic adds to a normed and rotated head, per head: with u = 2^-24, the sum of squares is
    off by at most (D + 8) u of itself, so its root's inverse by half that and 4 u; the products with it and the weight add
    2 u, sine and cosine 2^-23 each (the reduced angle's rounding and the polynomial's), and a pair's two products and
    sum 3 u. Each component is at most sqrt(2) of the pair's largest; all times the head's largest normed element."""
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    return math.sqrt(2) * ((x.shape[-1] + 8) / 2 + 4 + 2 + 4 + 3) * 2.0 ** -24 * y.abs().amax(-1, keepdim=True)


def near(got, want, extra):
    """Whether got, rounded once to its type, is within half a step of a value within `extra` of want. Half a step of
    the type's smallest normal is also allowed where values are below it (subnormal spacing)."""
    tiny = torch.finfo(got.dtype).tiny
    slack = half_step(got.dtype) * (want.abs() + extra).clamp_min(tiny) + extra
    return bool(((got.double() - want).abs() <= slack).all())


def verify64(target, draft, tokens, uniforms, lens=None):
    """The rule, a sequence at a time, with exact sums (math.fsum) of the weights."""
    batch, drafts = tokens.shape
    out, accepted = [], []
    vocabulary = target.shape[2]
    for b in range(batch):
        n = drafts if lens is None else min(max(int(lens[b]), 0), drafts)
        j = 0
        while j < n:
            x, u = int(tokens[b, j]), float(uniforms[b, j])
            if not 0 <= x < vocabulary:
                break
            q = 1.0 if draft is None else float(draft[b, j, x])
            if not u * q < float(target[b, j, x]):
                break
            j += 1
        p = [v if v > 0 else 0.0 for v in target[b, j].double().tolist()]
        w = p
        if j < n:
            if draft is None:
                w = list(p)
                if 0 <= int(tokens[b, j]) < vocabulary:
                    w[int(tokens[b, j])] = 0.0
            else:
                d = (target[b, j].double() - draft[b, j].double()).tolist()
                w = [v if v > 0 else 0.0 for v in d]
            if not math.fsum(w) > 0:
                w = p
        total, drawn = math.fsum(w), -1
        if total > 0:
            level, run = float(uniforms[b, drafts]) * total, []
            for i, v in enumerate(w):
                if v > 0:
                    run.append(v)
                    drawn = i
                    if math.fsum(run) > level if len(run) < 2000 else sum(run) > level:
                        break
        out.append([int(t) for t in tokens[b, :j]] + [drawn] + [-1] * (drafts - j))
        accepted.append(j)
    return torch.tensor(out).view(batch, drafts + 1), torch.tensor(accepted)


def verify_inputs(g, batch, drafts, vocabulary, dtype, proposed=True, ragged=False):
    logits = torch.randn(batch, drafts + 1, vocabulary, generator=g) * 2.5
    target = torch.softmax(logits, -1).to(dtype)
    near_by = logits[:, :drafts] + torch.randn(batch, drafts, vocabulary, generator=g) * 0.7
    draft = torch.softmax(near_by, -1).to(dtype) if proposed else None
    noise = torch.empty(near_by.shape).exponential_(generator=g).clamp_min(1e-20)
    tokens = (near_by - noise.log()).argmax(-1) if drafts else torch.zeros(batch, 0, dtype=torch.int64)
    lens = torch.randint(0, drafts + 1, (batch,), generator=g, dtype=torch.int32) if ragged else None
    return target, draft, tokens, torch.rand(batch, drafts + 1, generator=g), lens
