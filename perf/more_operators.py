"""The operators of a prompt's path and of a cache held in 4 bits: cases with their inputs, one pass of each (in plain
torch operations, or through the package's entry points), the work that a pass cannot do without, and its result in 64
bits.

A case is a dict of plain values; "op" names the operator:
  prompt_attention   causal attention of whole prompts, packed one behind the other, over their own keys
  kv4_append         keys and values written into a paged cache of 4-bit codes (e2m1) with a power of two to every 32 of
                     them, and the whole cache read back in 16 bits
  kv4_read           the keys and values of a context read back from such a cache
  kv4_attention      attention of each sequence's last tokens over its pages of such a cache
  token_logprobs     the log probability of a given token in every row of logits, the row's entropy, and its likeliest
                     alternatives

listed() is the fixed set, draw(rng) gives more of the same ranges. Every input is drawn on the GPU from the seed.
"""

import importlib
import math
import random

import torch

own = False

_PACKAGE = "cuda-kernels-optimized-for-rtx5090_amd"
_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_GROUP = 32                      # elements that share a power of two
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_MOST = {"bf16": 252, "fp16": 140}  # the largest scale byte: 6 times the scale is still finite in the type
_FLOPS = 2.3e12                  # of the largest prompt
_SCORES = 1 << 33                # of a padded batch of prompts


def listed():
    return [
        # three short questions that arrive together: latency
        {"name": "prompt_short", "op": "prompt_attention", "dtype": "bf16", "batch": 3, "longest": 100, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "packed": True, "padded": 0},
        # a batch of ragged prompts, 7 query heads to each key head, padded to a fixed number of rows
        {"name": "prompt_batch", "op": "prompt_attention", "dtype": "fp16", "batch": 24, "longest": 1401,
         "q_heads": 28, "kv_heads": 4, "head_dim": 64, "packed": False, "padded": 64},
        # one document of 16384 tokens: the largest
        {"name": "prompt_document", "op": "prompt_attention", "dtype": "bf16", "batch": 1, "longest": 16384,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "packed": True, "padded": 0},
        # one decode step of 64 sequences appended; the pages of what they hold are few
        {"name": "append_step", "op": "kv4_append", "dtype": "bf16", "tokens": 64, "kv_heads": 8, "head_dim": 128,
         "block": 16, "slots": 512, "packed": True},
        # a prompt of 16384 tokens appended, all of its keys and values read back
        {"name": "append_prompt", "op": "kv4_append", "dtype": "bf16", "tokens": 16384, "kv_heads": 8,
         "head_dim": 128, "block": 64, "slots": 16384, "packed": True},
        # 5000 tokens of a context on scattered pages, heads of 64, widened for a kernel that takes 16 bits
        {"name": "read_context", "op": "kv4_read", "dtype": "fp16", "tokens": 5000, "kv_heads": 4, "head_dim": 64,
         "block": 32},
        # one user's next token behind 32768 others: latency of a long context
        {"name": "kv4_single", "op": "kv4_attention", "dtype": "bf16", "batch": 1, "seq": 1, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "block": 64, "longest": 32768},
        # a decode step of 64 users, 2048 to 8192 tokens each
        {"name": "kv4_decode", "op": "kv4_attention", "dtype": "bf16", "batch": 64, "seq": 1, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "block": 64, "longest": 8192},
        # 33 users with four drafted tokens and the last one each, heads of 64 in groups of 7, small pages
        {"name": "kv4_drafts", "op": "kv4_attention", "dtype": "fp16", "batch": 33, "seq": 5, "q_heads": 28,
         "kv_heads": 4, "head_dim": 64, "block": 24, "longest": 1801},
        # the tokens drawn in a decode step of 64 users, with the 20 likeliest of each
        {"name": "logprobs_step", "op": "token_logprobs", "dtype": "bf16", "rows": 64, "vocabulary": 128256,
         "top": 20},
        # a prompt of 4096 tokens scored, with the 5 likeliest of each
        {"name": "logprobs_prompt", "op": "token_logprobs", "dtype": "bf16", "rows": 4096, "vocabulary": 128256,
         "top": 5},
        # an evaluation's continuations scored in fp32 over a vocabulary of odd size, no alternatives
        {"name": "logprobs_score", "op": "token_logprobs", "dtype": "fp32", "rows": 700, "vocabulary": 49999,
         "top": 0},
    ]


def _log(rng, low, high):
    """An integer from low to high, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["prompt_attention", "prompt_attention", "kv4_append", "kv4_read", "kv4_attention",
                     "kv4_attention", "token_logprobs", "token_logprobs"])
    if op == "token_logprobs":
        dtype, vocabulary = rng.choice(["fp32", "bf16", "fp16"]), _log(rng, 1000, 262144)
        return {"op": op, "dtype": dtype, "rows": _log(rng, 1, min(8192, 525_000_000 // vocabulary)),
                "vocabulary": vocabulary, "top": rng.choice([0, 1, rng.randint(2, 20), rng.randint(2, 64)])}
    kv_heads, case = rng.choice([1, 2, 4, 8]), {"op": op, "dtype": rng.choice(["bf16", "fp16"])}
    q_heads = kv_heads * rng.choice([1, 3, 4, 7, 8])
    if op == "prompt_attention":
        head_dim, longest = rng.choice([64, 80, 96, 128, 128, 192, 256]), _log(rng, 1, 16384)
        batch = min(64, 65536 // longest, int(_FLOPS / (2 * q_heads * head_dim * longest ** 2)),
                    _SCORES // (q_heads * longest ** 2))
        while batch < 1:
            longest //= 2
            batch = min(int(_FLOPS / (2 * q_heads * head_dim * longest ** 2)), _SCORES // (q_heads * longest ** 2))
        return {**case, "batch": _log(rng, 1, min(batch, 64)), "longest": longest, "q_heads": q_heads,
                "kv_heads": kv_heads, "head_dim": head_dim, "packed": rng.random() < 0.5,
                "padded": rng.choice([0, 0, 64])}
    case |= {"kv_heads": kv_heads, "head_dim": rng.choice([64, 96, 128, 128, 192, 256]),
             "block": rng.choice([1, 8, 16, 24, 32, 64, 128])}
    if op == "kv4_attention":
        seq = _log(rng, 1, 16)
        longest = _log(rng, seq, 32768)
        keys = min((1 << 29) // (kv_heads * case["head_dim"]), (1 << 29) // (seq * q_heads))  # of all sequences
        return {**case, "batch": _log(rng, 1, max(1, min(256, keys // longest))), "seq": seq, "q_heads": q_heads,
                "longest": longest}
    case["tokens"] = _log(rng, 1, (1 << 24) // (kv_heads * case["head_dim"]))
    if op == "kv4_append":
        case |= {"slots": case["tokens"] * 5 // 4 + 16, "packed": rng.random() < 0.5}
    return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _cache(case, g, slots):
    """A cache in use: [pages, heads, block, head_dim / 2] codes and [..., head_dim / 32] scales, for keys and values.
    The scales are those of about normal values."""
    pages = -(-slots // case["block"])
    shape = pages, case["kv_heads"], case["block"]
    t = {}
    for name in "kv":
        t[name + "_codes"] = torch.randint(0, 256, (*shape, case["head_dim"] // 2), generator=g, device="cuda",
                                           dtype=torch.uint8)
        t[name + "_scales"] = torch.randint(123, 127, (*shape, case["head_dim"] // _GROUP), generator=g,
                                            device="cuda", dtype=torch.uint8)
    return t


def _lengths(case):
    """A batch's prompts, from the longest to a quarter of it."""
    batch, longest = case["batch"], case["longest"]
    return [longest - i * (longest * 3 // 4) // max(1, batch - 1) for i in range(batch)]


def _prompt_input(case, g, seed, dtype):
    batch, longest, hq, hk, d = (case[n] for n in ("batch", "longest", "q_heads", "kv_heads", "head_dim"))
    lens = _lengths(case)  # known on the host, where the prompts are packed
    random.Random(seed).shuffle(lens)
    offsets = [0]
    for n in lens:
        offsets.append(offsets[-1] + n)
    rows = offsets[-1]
    if case["padded"]:
        rows = -(-(rows + 1) // case["padded"]) * case["padded"]
    if case["packed"]:
        q, k, v = _normal(g, (rows, hq + 2 * hk, d), dtype, 1.2).split([hq, hk, hk], dim=1)
    else:
        q, k, v = (_normal(g, (rows, h, d), dtype, 1.2) for h in (hq, hk, hk))
    return {"q": q, "k": k, "v": v, "cu_seqlens": torch.tensor(offsets, dtype=torch.int32, device="cuda"),
            "longest": longest}


def _append_input(case, g, dtype):
    tokens, hk, d = case["tokens"], case["kv_heads"], case["head_dim"]
    if case["packed"]:  # beside 4 query heads to each key head
        qkv = _normal(g, (tokens, 6 * hk, d), dtype, 1.2)
        k, v = qkv[:, 4 * hk:5 * hk], qkv[:, 5 * hk:]
    else:
        k, v = (_normal(g, (tokens, hk, d), dtype, 1.2) for _ in range(2))
    t = {"k": k, "v": v, **_cache(case, g, case["slots"])}
    slots = t["k_codes"].shape[0] * case["block"]
    t["slot_mapping"] = torch.randperm(slots, generator=g, device="cuda")[:tokens].contiguous()
    if tokens > 100:  # a padded prompt: its last tokens are not written
        t["slot_mapping"][-3:] = -1
    t["every_slot"] = torch.arange(slots, device="cuda")
    return t


def _read_input(case, g):
    tokens, block = case["tokens"], case["block"]
    t = _cache(case, g, tokens + 3 * block)
    table = torch.randperm(t["k_codes"].shape[0], generator=g, device="cuda")
    at = torch.arange(tokens, device="cuda")
    t["slots"] = table[at // block] * block + at % block
    return t


def _attention_input(case, g, dtype):
    batch, seq, hq, d = (case[n] for n in ("batch", "seq", "q_heads", "head_dim"))
    block, longest = case["block"], case["longest"]
    each = -(-longest // block)
    t = _cache(case, g, batch * each * block)
    t["block_tables"] = torch.randperm(batch * each, generator=g, device="cuda").int().view(batch, each)
    # each sequence's tokens, the step's among them; the first is the longest, and one place of a larger batch is idle
    t["seq_lens"] = torch.randint(max(seq, longest // 4), longest + 1, (batch,), generator=g, device="cuda").int()
    t["seq_lens"][0] = longest
    if batch > 8 and seq == 1:
        t["seq_lens"][3] = 0
    t["q"] = _normal(g, (batch, seq, hq, d), dtype, 1.2)
    return t


def _logits_input(case, g, dtype):
    rows, n = case["rows"], case["vocabulary"]
    logits = torch.randn((rows, n), generator=g, device="cuda") * 2.5
    # drawn from them, with a few that were not likely; one row in 16 is sure of its token
    noise = torch.empty_like(logits).exponential_(generator=g).clamp_min_(1e-20).log_()
    tokens = (logits - noise).argmax(-1)
    del noise
    tokens[::7] = torch.randint(0, n, tokens[::7].shape, generator=g, device="cuda")
    sure = torch.arange(0, rows, 16, device="cuda")
    logits[sure, tokens[sure]] += 25.0
    # a grammar leaves half of the vocabulary in one row in 8
    masked = torch.arange(3, rows, 8, device="cuda")
    logits[masked] = logits[masked].masked_fill_(
        torch.rand((masked.numel(), n), generator=g, device="cuda") < 0.5, float("-inf"))
    logits[masked, tokens[masked]] = 4.0
    return {"logits": logits.to(dtype), "tokens": tokens}


def _inputs(case, seed):
    g, dtype = _generator(seed), _DTYPES[case["dtype"]]
    if case["op"] == "prompt_attention":
        return _prompt_input(case, g, seed, dtype)
    if case["op"] == "kv4_append":
        return _append_input(case, g, dtype)
    if case["op"] == "kv4_read":
        return _read_input(case, g)
    return (_attention_input if case["op"] == "kv4_attention" else _logits_input)(case, g, dtype)


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = dict(case)
    if own:
        state["ops"] = importlib.import_module(_PACKAGE).ops()
    return state


def _prompt_plain(t):
    """The prompts padded to the longest: one batch of scores."""
    q, k, v, longest = t["q"], t["k"], t["v"], t["longest"]
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    group, offsets = hq // hk, t["cu_seqlens"].long()
    at = torch.arange(longest, device=q.device)
    there = at < (offsets[1:] - offsets[:-1])[:, None]                                       # batch, longest
    rows = torch.where(there, offsets[:-1, None] + at, 0)
    x = q[rows].float().view(*rows.shape, hk, group, d).permute(0, 2, 1, 3, 4).flatten(2, 3) * d ** -0.5
    y, z = k[rows].float().transpose(1, 2), v[rows].float().transpose(1, 2)                  # batch, hk, longest, d
    s = (x @ y.transpose(2, 3)).view(-1, hk, longest, group, longest)
    s.masked_fill_((at > at[:, None])[:, None], float("-inf"))
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    o = (s.flatten(2, 3) @ z).view(-1, hk, longest, group, d) / s.sum(-1, keepdim=True)
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    out[rows[there]] = o.transpose(1, 2).reshape(*rows.shape, hq, d)[there].to(q.dtype)
    return out


def _power(byte):
    """2^(byte - 127), exact."""
    return (byte.int() << 23).view(torch.float32)


def _codes(x, most):
    """The codes of x [..., D], two to a byte, and the scales of its groups."""
    groups = x.float().unflatten(-1, (-1, _GROUP))
    # the least power of two that leaves the largest below 7 (which 6 is within half a step of)
    scales = (((groups.abs().amax(-1).view(torch.int32) + 0x200000) >> 23) - 2).clamp(1, most)
    y = groups.abs() * _power(254 - scales)[..., None]
    codes = ((y > 0.25).int() + (y >= 0.75).int() + (y > 1.25).int() + (y >= 1.75).int() + (y > 2.5).int() +
             (y >= 3.5).int() + (y > 5.0).int() + 8 * torch.signbit(groups).int()).flatten(-2)
    return (codes[..., ::2] | codes[..., 1::2] << 4).to(torch.uint8), scales.to(torch.uint8)


def _values(codes, scales):
    """What codes [..., D / 2] stand for: [..., D] in 32 bits."""
    value = torch.tensor([*_VALUES, *(-v for v in _VALUES)], device=codes.device)
    both = torch.stack((value.repeat(16), value.repeat_interleave(16)), -1)                  # of a byte
    return (both[codes.int()].flatten(-2).unflatten(-1, (-1, _GROUP)) * _power(scales)[..., None]).flatten(-2)


def _of_slots(t, name, slots):
    block = t["k_codes"].shape[2]
    page, at = slots // block, slots % block
    return _values(t[name + "_codes"][page, :, at], t[name + "_scales"][page, :, at])


def _append_plain(t, case):
    slots = t["slot_mapping"]
    written = slots >= 0
    # a token that is not written repeats one that is
    token = torch.where(written, torch.arange(slots.numel(), device=slots.device), written.int().argmax())
    page, at = slots[token] // case["block"], slots[token] % case["block"]
    for name in "kv":
        codes, scales = _codes(t[name], _MOST[case["dtype"]])
        t[name + "_codes"][page, :, at] = codes[token]
        t[name + "_scales"][page, :, at] = scales[token]
    return tuple(_of_slots(t, name, t["every_slot"]).to(t["k"].dtype) for name in "kv")


def _attention_plain(t, case):
    q = t["q"]
    batch, seq, hq, d = q.shape
    hk, block = case["kv_heads"], case["block"]
    group = hq // hk
    tables = t["block_tables"].long()

    def keys(name):  # batch, hk, keys, d
        x = _values(t[name + "_codes"][tables], t[name + "_scales"][tables])
        return x.transpose(1, 2).flatten(2, 3)

    x = q.float().view(batch, seq, hk, group, d).transpose(1, 2).reshape(batch, hk, seq * group, d) * d ** -0.5
    s = x @ keys("k").transpose(2, 3)
    last = t["seq_lens"].long()[:, None] - seq + torch.arange(seq, device=q.device)          # each query's own place
    last = last.repeat_interleave(group, 1)[:, None, :, None]
    s.masked_fill_(torch.arange(s.shape[-1], device=q.device) > last, float("-inf"))
    top = s.amax(-1, keepdim=True)
    s = (s - torch.where(top == float("-inf"), 0.0, top)).exp_()
    out = torch.where(last >= 0, s @ keys("v") / s.sum(-1, keepdim=True), 0.0)               # an idle place: zeros
    return out.view(batch, hk, seq, group, d).transpose(1, 2).reshape(batch, seq, hq, d).to(q.dtype)


def _logprobs_plain(t, case):
    x, tokens, top = t["logits"].float(), t["tokens"], case["top"]
    off = x - x.amax(-1, keepdim=True)
    e = off.exp()
    total = e.sum(-1, dtype=torch.float64)
    log_total = total.log()
    entropy = log_total - torch.where(e > 0, e * off, 0.0).sum(-1, dtype=torch.float64) / total
    logprob = off.gather(-1, tokens[:, None])[:, 0] - log_total
    # the largest, and of equal ones the first: one integer that orders both
    bits = x.view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    order = (order << 32) - torch.arange(x.shape[1], device=x.device)
    index = -(order.topk(top, dim=-1).values & 0xffffffff) & 0xffffffff
    return logprob.float(), entropy.float(), (off.gather(-1, index) - log_total[:, None]).float(), index


def run(state):
    case, t = state["case"], state
    op = case["op"]
    cache = ("k_codes", "k_scales", "v_codes", "v_scales")
    if not own:
        if op == "prompt_attention":
            return _prompt_plain(t)
        if op == "kv4_append":
            return _append_plain(t, case)
        if op == "kv4_read":
            return tuple(_of_slots(t, name, t["slots"]).to(_DTYPES[case["dtype"]]) for name in "kv")
        return (_attention_plain if op == "kv4_attention" else _logprobs_plain)(t, case)
    ops = state["ops"]
    if op == "prompt_attention":
        return ops.prompt_attention(t["q"], t["k"], t["v"], t["cu_seqlens"])
    if op == "kv4_append":
        ops.kv4_append_(t["k"], t["v"], *(t[n] for n in cache), t["slot_mapping"])
        return ops.kv4_read(*(t[n] for n in cache), t["every_slot"], t["k"].dtype)
    if op == "kv4_read":
        return ops.kv4_read(*(t[n] for n in cache), t["slots"], _DTYPES[case["dtype"]])
    if op == "kv4_attention":
        return ops.kv4_attention(t["q"], *(t[n] for n in cache), t["block_tables"], t["seq_lens"])
    return ops.token_logprobs(t["logits"], t["tokens"], case["top"])


def work(case):
    op, size = case["op"], _BYTES[case["dtype"]]
    if op == "token_logprobs":
        n = case["rows"] * case["vocabulary"]
        return {"bytes": n * size + case["rows"] * (16 + 12 * case["top"]), "flops": 4 * n}
    hk, d = case["kv_heads"], case["head_dim"]
    packed = 2 * hk * (d // 2 + d // _GROUP)      # bytes of a token's keys and values in the cache
    if op == "prompt_attention":
        hq, lens = case["q_heads"], _lengths(case)
        tokens, squares = sum(lens), sum(n * (n + 1) for n in lens)
        return {"bytes": 2 * tokens * (hq + hk) * d * size, "flops": 2 * squares * hq * d}
    if op == "kv4_attention":
        hq = case["q_heads"]
        keys = case["longest"] * (1 + (case["batch"] - 1) * 5 / 8)
        return {"bytes": int(keys * packed + 2 * case["batch"] * case["seq"] * hq * d * size),
                "flops": int(4 * keys * case["seq"] * hq * d)}
    tokens, read = case["tokens"], case["tokens"]
    both = 2 * hk * d
    if op == "kv4_read":
        return {"bytes": tokens * (packed + both * size + 8), "flops": tokens * both}
    read = -(-case["slots"] // case["block"]) * case["block"]
    return {"bytes": tokens * (both * size + packed + 8) + read * (packed + both * size + 8),
            "flops": 4 * tokens * both + read * both}


def _prompt_exact(t):
    """A prompt and a key head at a time."""
    q, k, v = t["q"], t["k"], t["v"]
    group, d = q.shape[1] // k.shape[1], q.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    offsets = t["cu_seqlens"].tolist()
    for a, b in zip(offsets, offsets[1:]):
        hidden = torch.ones((b - a, b - a), dtype=torch.bool, device="cuda").triu_(1)
        for h in range(k.shape[1]):
            for i in range(h * group, (h + 1) * group):
                s = torch.mm(q[a:b, i].double(), k[a:b, h].double().t().contiguous()).mul_(1 / math.sqrt(d))
                out[a:b, i] = torch.mm(torch.softmax(s.masked_fill_(hidden, -math.inf), -1), v[a:b, h].double())
    return out


def _decoded(codes, scales):
    """e2m1 from its bits: with an exponent of 0 the mantissa counts halves, else 1 and half the mantissa times 2^(e - 1)."""
    nibbles = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double()
    sign = 1 - 2 * (nibbles >= 8).double()
    rest = nibbles % 8
    exponent, mantissa = torch.floor(rest / 2), rest % 2
    size = torch.where(exponent > 0, torch.ldexp(1 + mantissa / 2, exponent - 1), mantissa / 2)
    return sign * torch.ldexp(size, (scales.double() - 127).repeat_interleave(_GROUP, -1))


def _append_exact(t, case):
    """Of every group the values that are nearest, found among all that the codes can be."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    even = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device="cuda")  # even codes first: ties go to them
    written = t["slot_mapping"] >= 0
    slots, out = t["slot_mapping"][written], []
    for name in "kv":
        x = t[name][written].double().unflatten(-1, (-1, _GROUP))
        top = x.abs().amax(-1, keepdim=True)
        e = torch.floor(torch.log2(top.clamp_min(2.0 ** -140))) - 2
        e = torch.where(top >= torch.ldexp(torch.full_like(top, 7), e), e + 1, e).clamp(-126, _MOST[case["dtype"]] - 127)
        y = torch.ldexp(x.abs(), -e)
        best, far = torch.zeros_like(y), torch.full_like(y, math.inf)
        for v in grid[even].tolist():
            nearer = (y - v).abs() < far
            best, far = torch.where(nearer, v, best), torch.where(nearer, (y - v).abs(), far)
        values = torch.ldexp(best, e) * torch.where(x < 0, -1.0, 1.0)
        cache = _decoded(t[name + "_codes"], t[name + "_scales"]).transpose(1, 2).flatten(0, 1)
        cache[slots] = values.flatten(-2)
        out.append(cache)
    return tuple(out)


def _attention_exact(t, case):
    """A sequence at a time: its keys in order."""
    block, group = case["block"], case["q_heads"] // case["kv_heads"]
    batch, seq, hq, d = t["q"].shape
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(t["seq_lens"].tolist()):
        if not n:
            continue
        pages = t["block_tables"][b, :-(-n // block)].long()
        k, v = (_decoded(t[name + "_codes"][pages], t[name + "_scales"][pages]).transpose(0, 1).flatten(1, 2)[:, :n]
                for name in "kv")                                                            # heads, keys, d
        k = k.transpose(1, 2).contiguous()
        for i in range(max(0, seq - n), seq):
            seen = n - seq + i + 1
            q = t["q"][b, i].double().view(-1, group, d)
            w = torch.softmax(torch.bmm(q, k[:, :, :seen].contiguous()) / math.sqrt(d), -1)
            out[b, i] = torch.bmm(w, v[:, :seen].contiguous()).reshape(hq, d)
    return out


def _logprobs_exact(t, case):
    """Some rows at a time, the alternatives by a stable sort."""
    found = []
    for x, tokens in zip(t["logits"].split(256), t["tokens"].split(256)):
        p = torch.log_softmax(x.double(), -1)
        entropy = -(p.exp() * p.clamp_min(-1e300)).sum(-1)
        index = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        found.append((p[torch.arange(len(tokens), device="cuda"), tokens], entropy, torch.gather(p, 1, index), index))
    return tuple(torch.cat(parts) for parts in zip(*found))


def exact(case, seed):
    t = _inputs(case, seed)
    if case["op"] == "prompt_attention":
        return _prompt_exact(t)
    if case["op"] == "kv4_append":
        return _append_exact(t, case)
    if case["op"] == "kv4_read":
        block = case["block"]
        page, at = t["slots"] // block, t["slots"] % block
        return tuple(_decoded(t[n + "_codes"][page, :, at], t[n + "_scales"][page, :, at]) for n in "kv")
    return (_attention_exact if case["op"] == "kv4_attention" else _logprobs_exact)(t, case)
