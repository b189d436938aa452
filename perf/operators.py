"""The operators of a serving step with drafted tokens over a batch that shares a prompt: cases with their inputs, one
pass of each (in plain torch operations, or through the package's entry points), the work that a pass cannot do
without, and its result in 64 bits.

A case is a dict of plain values; "op" names the operator:
  qk_norm_rope             the RMS norm of every query and key head, its weight, and the rotation
  qk_norm_rope_kv          the same, the keys and values written into a paged cache on the way
  shared_prefix_attention  attention of a batch's last tokens over one paged prefix that all share and over each
                           sequence's own paged keys
  verify_drafts            which drafted tokens the target's probabilities keep, and the token drawn behind them

listed() is the fixed set, draw(rng) gives more of the same ranges. Every input is drawn on the GPU from the seed.
"""

import importlib
import math

import torch

own = False

_PACKAGE = "cuda-kernels-optimized-for-rtx5090_amd"
_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_THETA = 10000.0
_EPS = 1e-6
_FAR = 100000         # positions start below this: conversations and documents of up to 100k tokens
_FLOPS = 150e9        # of the largest attention case
_ROW_ELEMENTS = 1 << 26
_KEPT = 0.727         # share of the drafted tokens that the probabilities below keep


def listed():
    return [
        # a prefill of 4 x 4096 tokens, the projection's packed output split into 32 query and 8 key heads: the largest
        {"name": "norm_rope_prefill", "op": "qk_norm_rope", "dtype": "bf16", "batch": 4, "seq": 4096, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "rotary": 128, "packed": True, "weights": True},
        # a ragged chunk of a prefill, 7 query heads to each key head, half of each head rotated, no weights
        {"name": "norm_rope_partial", "op": "qk_norm_rope", "dtype": "fp16", "batch": 3, "seq": 701, "q_heads": 14,
         "kv_heads": 2, "head_dim": 64, "rotary": 32, "packed": False, "weights": False},
        # one decode step of 64 sequences, keys and values appended to the cache: latency
        {"name": "norm_rope_kv_decode", "op": "qk_norm_rope_kv", "dtype": "bf16", "batch": 64, "seq": 1,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "rotary": 128, "packed": True, "weights": True,
         "slots": 8192},
        # a chunk of 2048 prompt tokens with heads of 256, padded at the end, written into the cache
        {"name": "norm_rope_kv_chunk", "op": "qk_norm_rope_kv", "dtype": "bf16", "batch": 2, "seq": 1024,
         "q_heads": 16, "kv_heads": 4, "head_dim": 256, "rotary": 256, "packed": False, "weights": True,
         "slots": 4096},
        # a single user behind a system prompt of 2000 tokens: one token, few keys of its own; latency
        {"name": "attention_single", "op": "shared_prefix_attention", "dtype": "bf16", "batch": 1, "seq": 1,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "block": 16, "prefix": 2000, "longest": 200},
        # a decode step of 64 users behind one document of 8192 tokens
        {"name": "attention_decode", "op": "shared_prefix_attention", "dtype": "bf16", "batch": 64, "seq": 1,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "block": 16, "prefix": 8192, "longest": 1000},
        # 33 users with four drafted tokens and the last one each, an odd prompt, heads of 64 in groups of 7
        {"name": "attention_drafts", "op": "shared_prefix_attention", "dtype": "fp16", "batch": 33, "seq": 5,
         "q_heads": 28, "kv_heads": 4, "head_dim": 64, "block": 32, "prefix": 4999, "longest": 701},
        # long conversations without a shared prompt, each read once from its own pages: the cache's bandwidth
        {"name": "attention_own", "op": "shared_prefix_attention", "dtype": "bf16", "batch": 16, "seq": 1,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "block": 64, "prefix": 0, "longest": 8192},
        # 96 users with three drafted tokens each over a book of 20000 tokens: the largest
        {"name": "attention_book", "op": "shared_prefix_attention", "dtype": "bf16", "batch": 96, "seq": 4,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "block": 64, "prefix": 20000, "longest": 500},
        # one user, four drafted tokens, a vocabulary of 50000: latency
        {"name": "verify_single", "op": "verify_drafts", "dtype": "fp32", "batch": 1, "drafts": 4, "vocabulary": 50000,
         "proposed": True, "ragged": False},
        # 64 users with five drafted tokens and a vocabulary of 128256
        {"name": "verify_batch", "op": "verify_drafts", "dtype": "fp32", "batch": 64, "drafts": 5,
         "vocabulary": 128256, "proposed": True, "ragged": False},
        # drafts looked up in the prompt (they have no probabilities), up to three each, a vocabulary of odd size
        {"name": "verify_lookup", "op": "verify_drafts", "dtype": "bf16", "batch": 200, "drafts": 3,
         "vocabulary": 49999, "proposed": False, "ragged": True},
    ]


def _log(rng, low, high):
    """An integer from low to high, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["qk_norm_rope", "qk_norm_rope_kv", "shared_prefix_attention", "shared_prefix_attention",
                     "verify_drafts"])
    if op == "verify_drafts":
        dtype, drafts, vocabulary = rng.choice(["fp32", "bf16"]), rng.randint(1, 8), _log(rng, 1000, 262144)
        return {"op": op, "dtype": dtype, "batch": _log(rng, 1, min(256, 60_000_000 // (vocabulary * (drafts + 1)))),
                "drafts": drafts, "vocabulary": vocabulary, "proposed": rng.random() < 0.75,
                "ragged": rng.random() < 0.5}
    kv_heads = rng.choice([1, 2, 4, 8])
    case = {"op": op, "dtype": rng.choice(["bf16", "fp16"])}
    if op == "shared_prefix_attention":
        q_heads, head_dim = kv_heads * rng.choice([1, 3, 4, 7, 8]), rng.choice([64, 80, 96, 128, 128, 256])
        seq, block = _log(rng, 1, 16), rng.choice([1, 8, 16, 24, 32, 64, 128])
        prefix = 0 if rng.random() < 0.15 else _log(rng, 16, 32768)
        longest = _log(rng, seq, 8192)
        # within the largest case's operations, the inputs within 1 GiB and the scores within 4
        batch = min(256, int(_FLOPS / (4 * seq * q_heads * head_dim * (prefix + longest))),
                    (1 << 28) // (kv_heads * head_dim * longest), (1 << 30) // (seq * q_heads * (prefix + longest)))
        return {**case, "batch": _log(rng, 1, max(1, batch)), "seq": seq, "q_heads": q_heads, "kv_heads": kv_heads,
                "head_dim": head_dim, "block": block, "prefix": prefix, "longest": longest}
    q_heads = kv_heads * rng.choice([1, 3, 4, 7, 8])
    head_dim = rng.choice([64, 80, 96, 128, 128, 256])
    tokens = _log(rng, 1, _ROW_ELEMENTS // ((q_heads + 2 * kv_heads) * head_dim))
    batch = min(tokens, _log(rng, 1, 64))
    case |= {"batch": batch, "seq": min(16384, tokens // batch), "q_heads": q_heads, "kv_heads": kv_heads,
             "head_dim": head_dim, "rotary": head_dim // 2 if rng.random() < 0.25 else head_dim,
             "packed": rng.random() < 0.5, "weights": rng.random() < 0.75}
    if op == "qk_norm_rope_kv":
        case["slots"] = max(1024, case["batch"] * case["seq"] * 5 // 4)
    return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _heads_input(case, g, dtype):
    batch, seq, hq, hk, d = (case[n] for n in ("batch", "seq", "q_heads", "kv_heads", "head_dim"))
    if case["packed"]:
        qkv = _normal(g, (batch, seq, hq + 2 * hk, d), dtype, 1.5)
        q, k, v = qkv.split([hq, hk, hk], dim=2)
    else:
        q, k, v = (_normal(g, (batch, seq, h, d), dtype, 1.5) for h in (hq, hk, hk))
    # prefills start somewhere in a sequence; a decode step's sequences are each at a place of their own
    start = torch.randint(0, _FAR, (batch, 1), generator=g, device="cuda")
    rotary = case["rotary"]
    inv_freq = 1.0 / (_THETA ** (torch.arange(0, rotary, 2, dtype=torch.int64).float() / rotary))
    t = {"q": q, "k": k, "position_ids": (start + torch.arange(seq, device="cuda")[None, :]).contiguous(),
         "inv_freq": inv_freq.cuda(), "q_weight": None, "k_weight": None}
    if case["weights"]:
        t["q_weight"], t["k_weight"] = ((torch.rand(d, generator=g, device="cuda") + 0.5).to(dtype) for _ in range(2))
    if case["op"] == "qk_norm_rope_kv":
        tokens, slots = batch * seq, case["slots"]
        t["v"] = v
        mapping = torch.randperm(slots, generator=g, device="cuda")[:tokens].view(batch, seq)
        if seq > 8:  # a padded prefill: the last tokens of the first sequence are not written
            mapping[0, -3:] = -1
        t["slot_mapping"] = mapping.contiguous()
        t["k_cache"], t["v_cache"] = (_normal(g, (slots, hk, d), dtype) for _ in range(2))
    return t


def _attention_input(case, g, dtype):
    batch, seq, hq, hk, d = (case[n] for n in ("batch", "seq", "q_heads", "kv_heads", "head_dim"))
    block, prefix, longest = case["block"], case["prefix"], case["longest"]
    shared, each = -(-prefix // block), -(-longest // block)
    blocks = shared + batch * each
    order = torch.randperm(blocks, generator=g, device="cuda").int()
    # each sequence's own tokens, the step's among them; the first is the longest, and one place of a larger batch is idle
    lens = torch.randint(max(seq, longest // 4), longest + 1, (batch,), generator=g, device="cuda").int()
    lens[0] = longest
    if batch > 8 and seq == 1:
        lens[3] = 0
    return {"q": _normal(g, (batch, seq, hq, d), dtype, 1.5),
            "k_cache": _normal(g, (blocks * block, hk, d), dtype), "v_cache": _normal(g, (blocks * block, hk, d), dtype),
            "prefix_table": order[:shared].contiguous(),
            "prefix_len": torch.full((1,), prefix, dtype=torch.int32, device="cuda"),
            "block_tables": order[shared:].view(batch, each).contiguous(), "seq_lens": lens}


def _drafts_input(case, g, dtype):
    batch, drafts, n = case["batch"], case["drafts"], case["vocabulary"]
    logits = torch.randn((batch, drafts + 1, n), generator=g, device="cuda") * 2.5
    t = {"target_probs": torch.softmax(logits, -1).to(dtype), "draft_probs": None, "draft_lens": None}
    logits = logits[:, :drafts]
    if case["proposed"]:  # a smaller model's: near the target's, about _KEPT of its tokens are kept
        logits = logits + torch.randn(logits.shape, generator=g, device="cuda") * 0.7
        t["draft_probs"] = torch.softmax(logits, -1).to(dtype)
    else:  # tokens that the target itself finds likely
        logits = logits * 2
    noise = torch.empty(logits.shape, device="cuda").exponential_(generator=g).clamp_min_(1e-20)
    t["draft_tokens"] = (logits - noise.log()).argmax(-1)
    if case["ragged"]:
        t["draft_lens"] = torch.randint(0, drafts + 1, (batch,), generator=g, device="cuda").int()
    t["uniforms"] = torch.rand((batch, drafts + 1), generator=g, device="cuda")
    return t


def _inputs(case, seed):
    make = {"shared_prefix_attention": _attention_input, "verify_drafts": _drafts_input}.get(case["op"], _heads_input)
    return make(case, _generator(seed), _DTYPES[case["dtype"]])


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = dict(case)
    if own:
        state["ops"] = importlib.import_module(_PACKAGE).ops()
    return state


def _normed(x, weight):
    x = x.float()
    x = x * (1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS))
    return x if weight is None else x * weight.float()


def _rotated(x, cos, sin, dtype):
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), dim=-1).to(dtype)


def _heads_plain(t):
    angle = t["position_ids"].double()[..., None] * t["inv_freq"].double()  # far positions: in 64 bits
    cos, sin = angle.cos().float().unsqueeze(2), angle.sin().float().unsqueeze(2)
    dtype = t["q"].dtype
    q = _rotated(_normed(t["q"], t["q_weight"]), cos, sin, dtype)
    k = _rotated(_normed(t["k"], t["k_weight"]), cos, sin, dtype)
    if "v" not in t:
        return q, k
    slots = t["slot_mapping"].flatten()
    written = slots >= 0
    # a token that is not written repeats one that is
    token = torch.where(written, torch.arange(slots.numel(), device=slots.device), written.int().argmax())
    t["k_cache"][slots[token]] = k.flatten(0, 1)[token]
    t["v_cache"][slots[token]] = t["v"].flatten(0, 1)[token]
    return q, t["k_cache"], t["v_cache"]


def _pages(table, block):
    return (table.long()[..., None] * block + torch.arange(block, device=table.device)).flatten(-2)


def _attention_plain(t, case):
    q, block = t["q"], case["block"]
    batch, seq, hq, d = q.shape
    hk = case["kv_heads"]
    group = hq // hk
    q = q.float().view(batch, seq, hk, group, d) * d ** -0.5
    shared, each = _pages(t["prefix_table"], block), _pages(t["block_tables"], block)
    kp, vp = (t[n][shared].float().transpose(0, 1) for n in ("k_cache", "v_cache"))          # hk, prefix, d
    ko, vo = (t[n][each].float().transpose(1, 2) for n in ("k_cache", "v_cache"))            # batch, hk, own, d
    sp = q.permute(2, 0, 1, 3, 4).reshape(hk, batch * seq * group, d) @ kp.transpose(1, 2)
    sp = sp.masked_fill_(torch.arange(shared.numel(), device=q.device) >= t["prefix_len"], float("-inf"))
    so = q.permute(0, 2, 1, 3, 4).reshape(batch, hk, seq * group, d) @ ko.transpose(2, 3)
    last = t["seq_lens"].long()[:, None] - seq + torch.arange(seq, device=q.device)         # each query's own place
    last = last.repeat_interleave(group, 1)[:, None, :, None]
    so = so.masked_fill_(torch.arange(each.shape[1], device=q.device) > last, float("-inf"))
    top = so.amax(-1, keepdim=True)
    if shared.numel():
        tp = sp.amax(-1, keepdim=True).view(hk, batch, seq * group, 1).transpose(0, 1)
        top = torch.maximum(top, tp)
    top = torch.where(top == float("-inf"), 0.0, top)
    sp = (sp - top.transpose(0, 1).reshape(hk, batch * seq * group, 1)).exp_()
    so = (so - top).exp_()
    total = so.sum(-1, keepdim=True) + sp.sum(-1).view(hk, batch, seq * group, 1).transpose(0, 1)
    out = so @ vo + (sp @ vp).view(hk, batch, seq * group, d).transpose(0, 1)
    out = torch.where((last >= 0) & (total > 0), out / total, 0.0)                           # a padding query: zeros
    return out.view(batch, hk, seq, group, d).transpose(1, 2).reshape(batch, seq, hq, d).to(t["q"].dtype)


def _drafts_plain(t):
    target, draft, tokens, u = t["target_probs"], t["draft_probs"], t["draft_tokens"], t["uniforms"].double()
    batch, drafts = tokens.shape
    rows, places = torch.arange(batch, device=tokens.device), torch.arange(drafts + 1, device=tokens.device)
    lens = torch.full_like(rows, drafts) if t["draft_lens"] is None else t["draft_lens"].long()
    p = target[:, :drafts].gather(-1, tokens[..., None])[..., 0].double()
    q = 1.0 if draft is None else draft.gather(-1, tokens[..., None])[..., 0].double()
    kept = (u[:, :drafts] * q < p) & (places[:drafts] < lens[:, None])  # exact: two 24-bit values in 53 bits
    accepted = kept.long().cumprod(1).sum(1)
    refused = accepted.clamp_max(drafts - 1)
    row = target[rows, accepted].double()
    if draft is None:
        left = row.scatter(1, tokens[rows, refused][:, None], 0.0)
    else:
        left = (row - draft[rows, refused].double()).clamp_min_(0.0)
    left = torch.where((accepted < lens)[:, None] & (left.sum(-1, keepdim=True) > 0), left, row)
    sums = left.cumsum(-1)
    drawn = (sums <= u[:, drafts:] * sums[:, -1:]).sum(-1)
    out = torch.where(places < accepted[:, None], torch.nn.functional.pad(tokens, (0, 1)), -1)
    return torch.where(places == accepted[:, None], drawn[:, None], out), accepted


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        if op == "shared_prefix_attention":
            return _attention_plain(state, case)
        return _drafts_plain(state) if op == "verify_drafts" else _heads_plain(state)
    t, ops = state, state["ops"]
    if op == "qk_norm_rope":
        return ops.qk_norm_rope(t["q"], t["k"], t["position_ids"], t["inv_freq"], t["q_weight"], t["k_weight"], _EPS)
    if op == "qk_norm_rope_kv":
        q = ops.qk_norm_rope_kv_(t["q"], t["k"], t["v"], t["position_ids"], t["inv_freq"], t["k_cache"], t["v_cache"],
                                 t["slot_mapping"], t["q_weight"], t["k_weight"], _EPS)
        return q, t["k_cache"], t["v_cache"]
    if op == "shared_prefix_attention":
        return ops.shared_prefix_attention(t["q"], t["k_cache"], t["v_cache"], t["prefix_table"], t["prefix_len"],
                                           t["block_tables"], t["seq_lens"], case["block"])
    return ops.verify_drafts(t["target_probs"], t["draft_probs"], t["draft_tokens"], t["uniforms"], t["draft_lens"])


def work(case):
    op, size = case["op"], _BYTES[case["dtype"]]
    batch = case["batch"]
    if op == "verify_drafts":
        # one row of the target's probabilities for the drawn token, the draft's beside it where one was refused
        rows = 1 + (1 - _KEPT ** case["drafts"] if case["proposed"] else 0)
        n = case["vocabulary"] * batch
        return {"bytes": int(n * size * rows) + batch * (case["drafts"] + 1) * (2 * size + 20), "flops": int(3 * n * rows)}
    seq, hq, hk, d = (case[n] for n in ("seq", "q_heads", "kv_heads", "head_dim"))
    q, kv = batch * seq * hq * d, batch * seq * hk * d
    if op == "shared_prefix_attention":
        # own lengths are spread evenly from a quarter to the whole of the longest
        seen = case["prefix"] + case["longest"] * 5 // 8
        keys = case["prefix"] + batch * (case["longest"] * 5 // 8)
        return {"bytes": 2 * q * size + 2 * keys * hk * d * size, "flops": 4 * q * seen}
    streams = 2 * (q + kv) + (2 * kv if op == "qk_norm_rope_kv" else 0)
    return {"bytes": streams * size + batch * seq * 16, "flops": 8 * (q + kv)}


def _heads_exact(t):
    def norm_and_rotate(x, weight):
        x = x.double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + _EPS).sqrt()
        if weight is not None:
            x = x * weight.double()
        r = 2 * t["inv_freq"].numel()
        angle = torch.einsum("bs,i->bsi", t["position_ids"].double(), t["inv_freq"].double())[:, :, None, :]
        z = torch.polar(torch.ones_like(angle), angle) * torch.complex(x[..., : r // 2], x[..., r // 2: r])
        return torch.cat((z.real, z.imag, x[..., r:]), dim=-1)

    q, k = norm_and_rotate(t["q"], t["q_weight"]), norm_and_rotate(t["k"], t["k_weight"])
    if "v" not in t:
        return q, k
    kc, vc = t["k_cache"].double(), t["v_cache"].double()
    written = t["slot_mapping"] >= 0
    kc[t["slot_mapping"][written]] = k[written]
    vc[t["slot_mapping"][written]] = t["v"].double()[written]
    return q, kc, vc


def _attention_exact(t, case):
    """A sequence at a time: its keys in order, one softmax over all of them."""
    block, group = case["block"], case["q_heads"] // case["kv_heads"]
    prefix, lens = int(t["prefix_len"]), t["seq_lens"].tolist()
    batch, seq, hq, d = t["q"].shape
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")

    def rows(table, n):
        at = torch.arange(n, device="cuda")
        return table.long()[at // block] * block + at % block

    first = rows(t["prefix_table"], prefix)
    kp, vp = (t[n][first].double().permute(1, 2, 0).contiguous() for n in ("k_cache", "v_cache"))   # heads, d, keys
    for b, n in enumerate(lens):
        mine = rows(t["block_tables"][b], n)
        k, v = (torch.cat((c, t[name][mine].double().permute(1, 2, 0)), 2)
                for c, name in ((kp, "k_cache"), (vp, "v_cache")))
        for i in range(max(0, seq - n), seq):
            seen = prefix + n - seq + i + 1
            q = t["q"][b, i].double().view(-1, group, d)
            w = torch.softmax(torch.bmm(q, k[:, :, :seen].contiguous()) / math.sqrt(d), -1)
            out[b, i] = torch.bmm(w, v[:, :, :seen].transpose(1, 2).contiguous()).reshape(hq, d)
    return out


def _drafts_exact(t):
    """Not one operation for the whole batch: the rule as it is told, a sequence at a time."""
    tokens, u = t["draft_tokens"].tolist(), t["uniforms"].double().tolist()
    batch, drafts = t["draft_tokens"].shape
    lens = [drafts] * batch if t["draft_lens"] is None else t["draft_lens"].tolist()
    out, counts = [], []
    for b in range(batch):
        kept = 0
        while kept < lens[b]:
            x = tokens[b][kept]
            q = 1.0 if t["draft_probs"] is None else float(t["draft_probs"][b, kept, x])
            if not u[b][kept] * q < float(t["target_probs"][b, kept, x]):
                break
            kept += 1
        weights = t["target_probs"][b, kept].double()
        if kept < lens[b]:
            minus = torch.zeros_like(weights)
            if t["draft_probs"] is None:
                minus[tokens[b][kept]] = weights[tokens[b][kept]]
            else:
                minus = t["draft_probs"][b, kept].double()
            rest = torch.relu(weights - minus)
            weights = rest if float(rest.sum()) > 0 else weights
        sums = torch.cumsum(weights, 0)
        drawn = int(torch.searchsorted(sums, sums[-1:] * u[b][drafts], right=True))
        out.append(tokens[b][:kept] + [drawn] + [-1] * (drafts - kept))
        counts.append(kept)
    return torch.tensor(out, device="cuda"), torch.tensor(counts, device="cuda")


def exact(case, seed):
    t = _inputs(case, seed)
    if case["op"] == "shared_prefix_attention":
        return _attention_exact(t, case)
    return _drafts_exact(t) if case["op"] == "verify_drafts" else _heads_exact(t)
