"""verify_drafts on the GPU, through the package's function and the torch operator, against the rule told in plain
Python (small vocabularies) or in fp64 torch operations on the CPU (large ones)."""

import pytest
import torch

import _serving as ref

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def on(dev, *tensors):
    return [None if t is None else t.to(dev) for t in tensors]


def both(pkg, *args):
    a, b = pkg.verify_drafts(*args), pkg.ops().verify_drafts(*args)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    return a[0].cpu(), a[1].cpu()


def wide64(target, draft, tokens, u, lens):
    """The rule with running sums by cumsum in fp64."""
    batch, drafts = tokens.shape
    out, accepted = torch.full((batch, drafts + 1), -1), torch.zeros(batch, dtype=torch.int64)
    for b in range(batch):
        j, n = 0, drafts if lens is None else int(lens[b])
        while j < n and float(u[b, j]) * (1.0 if draft is None else float(draft[b, j, tokens[b, j]])) < \
                float(target[b, j, tokens[b, j]]):
            j += 1
        w = target[b, j].double()
        if j < n:
            w = w.clone()
            if draft is None:
                w[tokens[b, j]] = 0
            else:
                w = (w - draft[b, j].double()).clamp_min(0)
        c = w.cumsum(0)
        out[b, :j], accepted[b] = tokens[b, :j], j
        out[b, j] = int((c <= float(u[b, drafts]) * float(c[-1])).sum())
    return out, accepted


@pytest.mark.parametrize("vocabulary", [1, 3, 64, 1000, 4097])
@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("batch,drafts,proposed,ragged", [(1, 4, True, False), (9, 0, True, False), (33, 2, False, True),
                                                          (7, 5, True, True)])
def test_rule(pkg, dev, vocabulary, dtype, batch, drafts, proposed, ragged):
    g = torch.Generator().manual_seed(vocabulary + drafts)
    args = ref.verify_inputs(g, batch, drafts, vocabulary, dtype, proposed and drafts > 0, ragged)
    got, want = both(pkg, *on(dev, *args)), ref.verify64(*args)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("batch,drafts,vocabulary,dtype,proposed", [(1, 4, 128256, F32, True), (40, 3, 49999, BF, True),
                                                                    (300, 1, 50000, BF, False), (3, 2, 262145, F32, True),
                                                                    (1100, 1, 2000, F32, True)])
def test_large_vocabularies(pkg, dev, batch, drafts, vocabulary, dtype, proposed):
    g = torch.Generator().manual_seed(batch)
    args = ref.verify_inputs(g, batch, drafts, vocabulary, dtype, proposed)
    got, want = both(pkg, *on(dev, *args)), wide64(*args)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_strided_empty_and_nothing_drafted(pkg, dev):
    g = torch.Generator().manual_seed(1)
    target, draft, tokens, u, _ = on(dev, *ref.verify_inputs(g, 5, 3, 777, F32))
    want = both(pkg, target, draft, tokens, u)
    wide = torch.zeros(5, 4, 900, device=dev)
    wide[:, :, 5:782] = target
    turned = draft.permute(2, 0, 1).contiguous().permute(1, 2, 0)  # the vocabulary is not contiguous: copied
    got = both(pkg, wide[:, :, 5:782], turned, tokens, u)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # one sequence's probabilities for all
    got = both(pkg, target[:1].expand(5, 4, 777), draft[:1].expand(5, 3, 777), tokens, u)
    want = ref.verify64(*(t.cpu() for t in (target[:1].expand(5, 4, 777), draft[:1].expand(5, 3, 777), tokens, u)))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out, accepted = both(pkg, target[:0], draft[:0], tokens[:0], u[:0])
    assert out.shape == (0, 4) and accepted.shape == (0,)


def test_draws_follow_the_target(pkg, dev):
    """Verification leaves the target's distribution: over 2^17 sequences that share one target and one draft row, the
    first token's frequencies are within 6 standard deviations of the target's probabilities."""
    n, v = 1 << 17, 8
    g = torch.Generator().manual_seed(2)
    p, q = torch.rand(v, generator=g), torch.rand(v, generator=g)
    p, q = (p / p.sum()).to(dev), (q / q.sum()).to(dev)
    tokens = torch.multinomial(q.cpu(), n, replacement=True, generator=g)[:, None].to(dev)
    u = torch.rand(n, 2, generator=g).to(dev)
    out, accepted = pkg.ops().verify_drafts(p.expand(n, 2, v), q.expand(n, 1, v), tokens, u)
    share = torch.bincount(out[:, 0], minlength=v).double() / n
    assert ((share - p.double()).abs() <= 6 * (p * (1 - p) / n).sqrt().double()).all()
    kept = torch.minimum(p, q).sum().double()
    assert (accepted.double().mean() - kept).abs() <= 6 * (kept * (1 - kept) / n).sqrt()


def test_two_to_the_32_threads(pkg, dev):
    """2^22 rows, 16 waves to each. All share one target of 4096 x 2^-13 on every second of 8192 entries and 2^-1 on the
    last: sums and levels are exact, so the drawn entry is."""
    n, v = 1 << 22, 8192
    w = torch.zeros(v, dtype=torch.float64)
    w[::2], w[-1] = 2.0 ** -13, 0.5
    total = w.cumsum(0)
    assert float(total[-1]) == 1.0
    u = ((torch.arange(n, device=dev) * 40503) % (1 << 24)).float().div(1 << 24).view(n, 1)
    target = w.float().to(dev).view(1, 1, v).expand(n, 1, v)
    out, accepted = pkg.ops().verify_drafts(target, None, torch.zeros(n, 0, dtype=torch.int64, device=dev), u)
    want = torch.searchsorted(total.to(dev), u[:, 0].double(), right=True)
    assert torch.equal(out[:, 0], want) and (accepted == 0).all()


def test_captured_graphs_share_nothing(pkg, dev):
    """Two graphs captured on one stream, replayed on two at once and between eager calls."""
    ops = pkg.ops()
    sets = []
    for seed in (3, 4):
        g = torch.Generator().manual_seed(seed)
        args = on(dev, *ref.verify_inputs(g, 3, 3, 60000, F32))
        ops.verify_drafts(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.verify_drafts(*args)
        sets.append((args, graph, out, torch.cuda.Stream()))
    for turn in range(5):
        for args, graph, out, s in sets:
            args[3].uniform_()
        torch.cuda.synchronize()
        for args, graph, out, s in sets:
            with torch.cuda.stream(s):
                graph.replay()
        eager = [ops.verify_drafts(*args) for args, *_ in sets]
        torch.cuda.synchronize()
        for (args, graph, out, s), want in zip(sets, eager):
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
