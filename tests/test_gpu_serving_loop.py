"""The serving operators together, a request's whole way: prompts packed one behind the other attend over their own keys,
which are appended to a cache in 4 bits; then each step normalizes and rotates, appends and attends over the cache, draws a
token from the likeliest and reports its log probability. Every operator is held against its formula in 64 bits on the
inputs that it got, and the step as a captured graph against the eager one."""

import pytest
import torch

import _kv4
import _logprobs
import _prompts
import _serving as ref

pytestmark = pytest.mark.gpu
BF, I32 = torch.bfloat16, torch.int32

HQ, HK, D, BLOCK, VOCABULARY, TOP = 8, 2, 64, 32, 700, 5
LENS, PAGES, EACH = [37, 1, 64, 5], 17, 4  # 17 pages, 4 to a sequence: one belongs to none


class Model:
    """One layer's projections, and a head."""

    def __init__(self, dev):
        g = torch.Generator().manual_seed(2)

        def normal(*shape):
            return torch.randn(*shape, generator=g).to(dev)

        self.embed = normal(VOCABULARY, 96).to(BF)
        self.qkv = (normal(96, (HQ + 2 * HK) * D) / 96 ** 0.5).to(BF)
        self.head = (normal(HQ * D, VOCABULARY) * 3.0 / (HQ * D) ** 0.5).to(BF)
        self.inv = ref.inv_freq_of(D).to(dev)

    def heads(self, ops, tokens, place):
        """Of tokens [N] at `place`: q [N, HQ, D], k and v [N, HK, D], the last one a view of the packed projection."""
        x = (self.embed[tokens] @ self.qkv).view(-1, HQ + 2 * HK, D)
        q, k, v = x.split([HQ, HK, HK], dim=1)
        q, k = ops.qk_norm_rope(q[None], k[None], place[None], self.inv)
        return q[0], k[0], v

    def logits(self, attended):
        return attended.flatten(1) @ self.head


class Cache:
    def __init__(self, dev):
        """All NaN, in scattered pages."""
        self.parts = []
        for _ in range(2):
            self.parts.append(torch.zeros(PAGES, HK, BLOCK, D // 2, dtype=torch.uint8, device=dev))
            self.parts.append(torch.full((PAGES, HK, BLOCK, D // 32), 255, dtype=torch.uint8, device=dev))
        order = torch.randperm(PAGES, generator=torch.Generator().manual_seed(1)).to(I32)
        self.tables, self.free = order[:4 * EACH].view(4, EACH).to(dev), int(order[-1])

    def slots(self, sequence, place):
        return self.tables.long()[sequence, place // BLOCK] * BLOCK + place % BLOCK


def cpu(*tensors):
    return [t.cpu() for t in tensors]


def check_logprobs(logits, tokens, got):
    want = _logprobs.logprobs64(logits.cpu(), tokens.cpu(), TOP)
    assert torch.equal(got[3].cpu(), want[3]) and _logprobs.near(got[:3], want[:3])


def start(ops, m, c, g, dev):
    """The prompts' tokens, their attention and the cache with their keys; returns each prompt's last row of logits."""
    tokens = torch.randint(0, VOCABULARY, (sum(LENS) + 3,), generator=g).to(dev)  # three rows of padding
    sequence = torch.tensor([b for b, n in enumerate(LENS) for _ in range(n)] + [0] * 3, device=dev)
    place = torch.cat([torch.arange(n) for n in LENS + [3]]).to(dev)
    offsets = torch.tensor([0] + LENS).cumsum(0).to(I32).to(dev)
    slots = c.slots(sequence, place)
    slots[-3:] = -1
    q, k, v = m.heads(ops, tokens, place)
    attended = ops.prompt_attention(q, k, v, offsets)
    ops.kv4_append_(k, v, *c.parts, slots)
    return tokens, slots, (q, k, v), offsets, attended, m.logits(attended)


def test_requests(pkg):
    dev, ops, g = torch.device("cuda:0"), pkg.ops(), torch.Generator().manual_seed(3)
    m, c = Model(dev), Cache(dev)
    tokens, slots, heads, offsets, attended, logits = start(ops, m, c, g, dev)
    want, extra = _prompts.attention64(*cpu(*heads, offsets))
    assert ref.near(attended.cpu(), want, extra) and not attended[-3:].any()
    for side, x in enumerate(heads[1:]):
        codes, scales = _kv4.encode(x[:-3].cpu())
        assert torch.equal(_kv4.flat(c.parts[2 * side].cpu())[slots[:-3].cpu()], codes)
        assert torch.equal(_kv4.flat(c.parts[2 * side + 1].cpu())[slots[:-3].cpu()], scales)
    # the prompts' own tokens: each by the row before it, none by a prompt's last row
    said = torch.full_like(tokens, -1)
    for a, b in zip(offsets.tolist(), offsets.tolist()[1:]):
        said[a:b - 1] = tokens[a + 1:b]
    got = ops.token_logprobs(logits, said, TOP)
    check_logprobs(logits, said, got)
    assert not got[0][said < 0].any()

    last = logits[offsets[1:].long() - 1]
    lens = torch.tensor(LENS, dtype=I32, device=dev)
    told, sums = [[] for _ in LENS], torch.zeros(len(LENS), device=dev)
    for step in range(6):
        values, indices = ops.topk(last.float(), 20)
        drawn = ops.topk_sample(values, indices, torch.rand(len(LENS), generator=g).to(dev), 0.8, 0.9).long()
        got = ops.token_logprobs(last, drawn, TOP)
        check_logprobs(last, drawn, got)
        assert torch.equal(got[3], indices[:, :TOP].long())  # the same order as top-k's
        sums += got[0]
        place = lens.long()
        q, k, v = m.heads(ops, drawn, place)
        ops.kv4_append_(k, v, *c.parts, c.slots(torch.arange(len(LENS), device=dev), place))
        lens += 1
        attended = ops.kv4_attention(q[:, None], *c.parts, c.tables, lens)
        cache = cpu(*c.parts)
        want, extra = _kv4.attention64(q[:, None].cpu(), cache, c.tables.cpu(), lens.cpu())
        assert ref.near(attended.cpu(), want, extra)
        last = m.logits(attended[:, 0])
        for b, t in enumerate(drawn.tolist()):
            told[b].append(t)

    # what was read back is what the codes stand for, and a page of no sequence was never written
    every = torch.cat([c.slots(b, torch.arange(n, device=dev)) for b, n in enumerate(lens.tolist())])
    k, v = ops.kv4_read(*c.parts, every, BF)
    for x, side in ((k, 0), (v, 2)):
        assert torch.equal(x.cpu().double(), _kv4.flat(_kv4.decode(*cpu(*c.parts[side:side + 2])))[every.cpu()])
    assert (c.parts[1][c.free] == 255).all() and (c.parts[3][c.free] == 255).all()
    assert (sums <= 0).all()


def test_a_captured_step(pkg):
    """A decode step in one graph, replayed with other tokens and lengths: one sequence has just begun, one is not there."""
    dev, ops, g = torch.device("cuda:0"), pkg.ops(), torch.Generator().manual_seed(4)
    m, c = Model(dev), Cache(dev)
    start(ops, m, c, g, dev)
    n = len(LENS)
    tokens, uniforms = torch.zeros(n, dtype=torch.int64, device=dev), torch.zeros(n, device=dev)
    lens, slots = torch.ones(n, dtype=I32, device=dev), torch.full((n,), -1, device=dev)

    def step(parts):
        q, k, v = m.heads(ops, tokens, (lens.long() - 1).clamp_min(0))
        ops.kv4_append_(k, v, *parts, slots)
        attended = ops.kv4_attention(q[:, None], *parts, c.tables, lens)
        logits = m.logits(attended[:, 0])
        values, indices = ops.topk(logits.float(), 20)
        drawn = ops.topk_sample(values, indices, uniforms, 0.8, 0.9).long()
        return attended, drawn, *ops.token_logprobs(logits, drawn, TOP)

    step([t.clone() for t in c.parts])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(c.parts)
    for own in ([38, 2, 65, 0], [39, 3, 66, 6], [40, 1, 0, 7], [41, 2, 67, 8]):
        lens.copy_(torch.tensor(own))
        place = (lens.long() - 1).clamp_min(0)
        slots.copy_(torch.where(lens > 0, c.slots(torch.arange(n, device=dev), place), -1))
        tokens.copy_(torch.randint(0, VOCABULARY, (n,), generator=g))
        uniforms.copy_(torch.rand(n, generator=g))
        parts = [t.clone() for t in c.parts]
        want = step(parts)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip([*got, *c.parts], [*want, *parts]):
            assert torch.equal(x, y)
        assert not got[0][lens == 0].any() and got[0][lens > 0].any()
