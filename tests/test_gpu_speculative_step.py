"""The serving step's operators together: a step of speculative decoding for sequences behind one shared prompt. The
prompt's keys and values are appended by one call and read by all; each step normalizes and rotates the new queries and
keys, appends them to paged caches, attends, verifies the drafts and goes on behind the kept ones, over the refused ones'
slots. Every operator is held against its formula in 64 bits on the inputs that it got, the caches at the end against the
tokens that were kept."""

import pytest
import torch

import _serving as ref

pytestmark = pytest.mark.gpu
BF, I32 = torch.bfloat16, torch.int32

HQ, HK, D, BLOCK, DRAFTS, VOCABULARY = 8, 2, 64, 16, 3, 500
PROMPT, STEPS = 53, 4


class Model:
    """One layer's projections, and tokens for drafts."""

    def __init__(self, g, dev):
        def normal(*shape):
            return torch.randn(*shape, generator=g).to(dev)

        width = 96
        self.embed = normal(VOCABULARY, width).to(BF)
        self.qkv = (normal(width, (HQ + 2 * HK) * D) / width ** 0.5).to(BF)
        self.head = normal(HQ * D, VOCABULARY) * 3.0 / (HQ * D) ** 0.5
        self.q_weight, self.k_weight = ((normal(D) * 0.1 + 1.0).to(BF) for _ in range(2))
        self.inv = ref.inv_freq_of(D).to(dev)

    def heads(self, tokens):
        x = (self.embed[tokens] @ self.qkv).view(*tokens.shape, HQ + 2 * HK, D)
        return x.split([HQ, HK, HK], dim=2)  # views of the packed projection


class Caches:
    def __init__(self, batch, pages, dev):
        self.k, self.v = (torch.full((pages * BLOCK, HK, D), float("nan"), dtype=BF, device=dev) for _ in range(2))
        self.order = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(I32).to(dev)
        shared = (PROMPT + BLOCK - 1) // BLOCK
        self.table, own = self.order[:shared].contiguous(), self.order[shared:]
        self.tables = own[:batch * (own.numel() // batch)].view(batch, -1).contiguous()


def append(ops, m, c, heads, ids, slots):
    q, k, v = heads
    out = ops.qk_norm_rope_kv_(q, k, v, ids, m.inv, c.k, c.v, slots, m.q_weight, m.k_weight, ref.EPS)
    want = ref.norm_rope64(q.cpu(), ids.cpu(), m.inv.cpu(), m.q_weight.cpu())
    assert ref.near(out.cpu(), want, ref.norm_rope_error(q.cpu(), m.q_weight.cpu()))
    return out


def probabilities(m, attended):
    return torch.softmax(attended.flatten(2).float() @ m.head, -1)


def test_steps(pkg):
    dev, g, ops = torch.device("cuda:0"), torch.Generator().manual_seed(3), pkg.ops()
    batch, m = 3, Model(torch.Generator().manual_seed(2), dev)
    c = Caches(batch, 16, dev)
    prompt = torch.randint(0, VOCABULARY, (1, PROMPT), generator=g).to(dev)
    at = torch.arange(PROMPT, device=dev)
    append(ops, m, c, m.heads(prompt), at[None], (c.table.long()[at // BLOCK] * BLOCK + at % BLOCK)[None])
    length = torch.tensor([PROMPT], dtype=I32, device=dev)

    kept = [[int(t)] for t in torch.randint(0, VOCABULARY, (batch,), generator=g)]  # each sequence's own tokens
    for step in range(STEPS):
        # the last kept token and the drafts; their places behind the kept ones
        drafts = torch.randint(0, VOCABULARY, (batch, DRAFTS), generator=g)
        lens = torch.tensor([len(t) + DRAFTS for t in kept], dtype=I32, device=dev)
        tokens = torch.cat((torch.tensor([t[-1:] for t in kept]), drafts), 1).to(dev)
        place = lens[:, None].long() - DRAFTS - 1 + torch.arange(DRAFTS + 1, device=dev)
        slots = c.tables.long().gather(1, place // BLOCK) * BLOCK + place % BLOCK
        q = append(ops, m, c, m.heads(tokens), PROMPT + place, slots)
        attended = ops.shared_prefix_attention(q, c.k, c.v, c.table, length, c.tables, lens, BLOCK)
        want, extra = ref.attention64(q.cpu(), c.k.cpu(), c.v.cpu(), c.table.cpu(), length.cpu(), c.tables.cpu(),
                                      lens.cpu(), BLOCK)
        assert ref.near(attended.cpu(), want, extra)
        target = probabilities(m, attended)
        # drafts that the target likes, now and then: its own tokens, with probabilities near its own
        liked = torch.rand(batch, DRAFTS, generator=g) < 0.5
        chosen = torch.where(liked.to(dev), target[:, :DRAFTS].argmax(-1), drafts.to(dev))
        proposed = torch.softmax(target[:, :DRAFTS].log() + 0.2, -1) if step % 2 else None
        uniforms = torch.rand(batch, DRAFTS + 1, generator=g).to(dev)
        out, accepted = ops.verify_drafts(target, proposed, chosen, uniforms, None)
        rule = ref.verify64(target.cpu(), None if proposed is None else proposed.cpu(), chosen.cpu(), uniforms.cpu())
        assert torch.equal(out.cpu(), rule[0]) and torch.equal(accepted.cpu(), rule[1])
        # only drafts whose keys are in the cache can be kept: those that were chosen before the step
        for b in range(batch):
            n = 0
            while n < int(accepted[b]) and int(chosen[b, n]) == int(drafts[b, n]):
                n += 1
            kept[b] += [int(t) for t in drafts[b, :n]] + [int(out[b, n])]

    for b in range(batch):
        own = torch.tensor([kept[b][:-1]], device=dev)  # the last one's keys are not there yet
        place = torch.arange(own.shape[1], device=dev)
        slots = c.tables[b].long()[place // BLOCK] * BLOCK + place % BLOCK
        _, k, v = m.heads(own)
        want = ref.norm_rope64(k.cpu(), PROMPT + place[None].cpu(), m.inv.cpu(), m.k_weight.cpu())
        assert ref.near(c.k[slots].cpu(), want[0], ref.norm_rope_error(k.cpu(), m.k_weight.cpu())[0])
        assert torch.equal(c.v[slots], v[0])
    # a free page was never written
    assert c.k.view(-1, BLOCK, HK, D)[c.tables[:, -1].long()].isnan().all()


def test_a_captured_step(pkg):
    """The four calls of a step in one graph, replayed with other tokens, lengths and pages."""
    dev, ops = torch.device("cuda:0"), pkg.ops()
    batch, m = 3, Model(torch.Generator().manual_seed(2), dev)
    g = torch.Generator().manual_seed(5)
    c = Caches(batch, 20, dev)
    c.k.normal_(), c.v.normal_()
    length = torch.tensor([PROMPT], dtype=I32, device=dev)
    heads = [torch.zeros(batch, DRAFTS + 1, h, D, dtype=BF, device=dev) for h in (HQ, HK, HK)]
    place = torch.arange(DRAFTS + 1, device=dev).repeat(batch, 1)
    slots, lens = place.clone(), torch.full((batch,), DRAFTS + 1, dtype=I32, device=dev)
    chosen = torch.zeros(batch, DRAFTS, dtype=torch.int64, device=dev)
    uniforms = torch.zeros(batch, DRAFTS + 1, device=dev)

    def step(k_cache, v_cache):
        q = ops.qk_norm_rope_kv_(*heads, PROMPT + place, m.inv, k_cache, v_cache, slots, m.q_weight, m.k_weight, ref.EPS)
        attended = ops.shared_prefix_attention(q, k_cache, v_cache, c.table, length, c.tables, lens, BLOCK)
        target = probabilities(m, attended)
        return q, attended, target, *ops.verify_drafts(target, None, chosen, uniforms, None)

    step(c.k.clone(), c.v.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(c.k, c.v)
    for own in ([4, 4, 4], [20, 7, 33], [5, 40, 19]):
        lens.copy_(torch.tensor(own))
        place.copy_(lens[:, None].long() - DRAFTS - 1 + torch.arange(DRAFTS + 1, device=dev))
        slots.copy_(c.tables.long().gather(1, place // BLOCK) * BLOCK + place % BLOCK)
        for x, y in zip(heads, m.heads(torch.randint(0, VOCABULARY, (batch, DRAFTS + 1), generator=g).to(dev))):
            x.copy_(y)
        chosen.copy_(torch.randint(0, VOCABULARY, (batch, DRAFTS), generator=g))
        uniforms.copy_(torch.rand(batch, DRAFTS + 1, generator=g))
        k, v = c.k.clone(), c.v.clone()
        want = step(k, v)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        assert torch.equal(c.k, k) and torch.equal(c.v, v)
