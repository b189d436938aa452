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


def attention64(q, k_cache, v_cache, prefix_table, prefix_len, block_tables, seq_lens, block_size, scale=None):
    """Attention of q [B, S, Hq, D] over the shared prefix and each sequence's own keys, a query at a time, and a bound
    of what the kernel's arithmetic adds to each value (fp32 sums, weights rounded to q's dtype):
    (out, extra), both fp64 [B, S, Hq, D].

    With w the weights and t the dtype's half step: a weight is rounded (t) after an exponential whose argument, a score of
    D products summed in fp32, is off by at most D u of the sum of its products' magnitudes (u = 2^-24), plus 8 u of
    itself and of the row's maximum for the scale and the subtraction, plus 4 u for the exponential itself; the same
    errors are in the sum of weights. Sums over n keys in fp32 add at most 2 n u. So each value is off by at most
    (2 (t + e) + 4 n u) sum w |v|, e the largest of the exponents' errors; weights below the smallest normal of fp16
    (2^-14) of a reference 2^7 up to 2^15 are off by 2^-25 2^-7 of the largest weight at most, summed over the keys."""
    batch, seq, hq, d = q.shape
    slots, hk = k_cache.shape[:2]
    scale = d ** -0.5 if scale is None else scale
    u = 2.0 ** -24

    def rows(table, n):
        n = min(max(int(n), 0), table.numel() * block_size)
        t = torch.arange(n, device=table.device)
        slot = table.long()[t // block_size] * block_size + t % block_size
        return slot, (slot >= 0) & (slot < slots), n

    out, extra = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    shared, there, _ = rows(prefix_table, prefix_len)
    shared = shared[there]
    for b in range(batch):
        mine, here, n = rows(block_tables[b], seq_lens[b])
        for i in range(seq):
            p = n - seq + i
            if p < 0:
                continue
            at = torch.cat((shared, mine[:p + 1][here[:p + 1]]))
            if not at.numel():
                continue
            k = k_cache[at].double().repeat_interleave(hq // hk, 1).transpose(0, 1).contiguous()  # hq, keys, d
            v = v_cache[at].double().repeat_interleave(hq // hk, 1).transpose(0, 1).contiguous()
            x = q[b, i].double()[:, :, None]
            s = torch.bmm(k, x)[..., 0] * scale
            off = torch.bmm(k.abs(), x.abs())[..., 0] * abs(scale) * d * u
            w = torch.softmax(s, -1)
            o = torch.bmm(w[:, None], v)[:, 0]
            mass = torch.bmm(w[:, None], v.abs())[:, 0]
            e = (off + 8 * u * (s.abs() + s.abs().amax(-1, keepdim=True)) + 4 * u).amax(-1, keepdim=True)
            rel = 2 * (half_step(q.dtype) + e) + 4 * at.numel() * u
            small = 2.0 ** -32 * v.abs().amax(1) * w.amax(-1, keepdim=True) * at.numel()
            out[b, i], extra[b, i] = o, rel * mass + small
    return out, extra


def attention_inputs(g, dtype, batch, seq, hq, hk, d, block, prefix, lens, device="cpu", spare=2, peak=1.5):
    """Scattered pages for a prefix of `prefix` keys and sequences of `lens` own keys; pages of no table hold NaN, and so
    does what lies behind a length."""
    nan = float("nan")
    each = max(1, max(-(-n // block) for n in lens))
    shared = -(-prefix // block)
    blocks = shared + batch * each + spare
    order = torch.randperm(blocks, generator=g).int()
    table, tables = order[:shared].clone(), order[shared:shared + batch * each].view(batch, each).clone()
    k = torch.full((blocks * block, hk, d), nan, dtype=torch.float32)
    v = torch.full((blocks * block, hk, d), nan, dtype=torch.float32)
    for one, n in [(table, prefix)] + [(tables[b], lens[b]) for b in range(batch)]:
        t = torch.arange(n)
        at = one.long()[t // block] * block + t % block
        k[at], v[at] = torch.randn(n, hk, d, generator=g), torch.randn(n, hk, d, generator=g)
    q = torch.randn(batch, seq, hq, d, generator=g) * peak
    return [t.to(device) for t in (q.to(dtype), k.to(dtype), v.to(dtype), table,
                                   torch.tensor([prefix], dtype=torch.int32), tables,
                                   torch.tensor(lens, dtype=torch.int32))] + [block]
