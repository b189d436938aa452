"""token_logprobs on the GPU, through the package's function and the torch operator, against the formulas in 64 bits."""

import ctypes

import pytest
import torch

import _logprobs as ref

pytestmark = pytest.mark.gpu
F32, BF, FP = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def same(a, b):
    return all(torch.equal(x.nan_to_num(7.5), y.nan_to_num(7.5)) for x, y in zip(a, b))


def check(pkg, dev, x, tokens, top):
    got = pkg.ops().token_logprobs(x.to(dev), tokens.to(dev), top)
    assert same(pkg.token_logprobs(x.to(dev), tokens.to(dev), top), got)
    want = ref.logprobs64(x, tokens, top)
    assert torch.equal(got[3].cpu(), want[3])
    assert ref.near(got[:3], want[:3])
    return got


@pytest.mark.parametrize("rows,n,top", [(1, 1, 1), (2, 7, 7), (3, 8, 0), (2, 63, 5), (9, 2049, 20), (1, 9000, 64),
                                        (2, 49999, 3), (5, 128256, 20), (1, 262144, 64), (300, 1000, 1)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF, FP], ids=["fp32", "bf16", "fp16"])
def test_formula(pkg, dev, rows, n, top, dtype):
    g = torch.Generator().manual_seed(n)
    check(pkg, dev, *ref.logits(g, rows, n, dtype), top)


@pytest.mark.parametrize("n,top,parts", [(200, 20, 0), (2500, 64, 1), (2500, 5, 3), (20, 20, 0), (50001, 64, 20),
                                         (50001, 20, 1)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF, FP], ids=["fp32", "bf16", "fp16"])
def test_edge_rows(pkg, dev, n, top, parts, dtype):
    g = torch.Generator().manual_seed(n)
    lib = ctypes.CDLL(pkg.lib_path("token_logprobs"))
    lib.token_logprobs_tune(0, parts)
    try:
        check(pkg, dev, *ref.edge_rows(g, n, dtype), top)
    finally:
        lib.token_logprobs_tune(0, 0)


def test_lists_under_pressure(pkg, dev):
    """Trips that each beat all before, values that come up again, the largest at the end."""
    g, n = torch.Generator().manual_seed(5), 100000
    x = torch.stack([torch.arange(n) // 1024 * 1.0, torch.arange(n) % 7 * 1.0, (torch.randn(n, generator=g) * 3).round(),
                     torch.randn(n, generator=g) + torch.arange(n) / 8192, torch.arange(n) / 1000.0])
    for top in (1, 20, 64):
        for dtype in (BF, F32):
            check(pkg, dev, x.to(dtype), torch.tensor([0, 39999, 17, 5, 99999]), top)


def test_zeros_of_both_signs(pkg, dev):
    """+0 comes before -0, also where a list is full of the latter."""
    n = 40000
    x = torch.zeros(3, n).neg_()
    x[0, 30000::50], x[1, ::50], x[2, -1] = 0.0, 0.0, 0.0
    for dtype in (BF, F32):
        check(pkg, dev, x.to(dtype), torch.tensor([0, 50, n - 1]), 20)


def test_views_and_repeated_calls(pkg, dev):
    g = torch.Generator().manual_seed(6)
    whole = torch.randn(40, 5003, generator=g).to(BF).to(dev)
    tokens = torch.randint(0, 4990, (40,), generator=g).to(dev)
    view = whole[:, 3:5000]
    want = pkg.ops().token_logprobs(view.contiguous(), tokens, 9)
    flipped = view.t().contiguous().t()
    for x in (view, flipped, view):
        assert same(pkg.ops().token_logprobs(x, tokens, 9), want) and same(pkg.token_logprobs(x, tokens, 9), want)
    one = pkg.ops().token_logprobs(whole[:1, :1].expand(40, 1), torch.zeros_like(tokens), 1)
    assert not one[0].any() and not one[1].any() and not one[3].any()
    none = pkg.token_logprobs(view[:0], tokens[:0], 4)
    assert [tuple(t.shape) for t in none] == [(0,), (0,), (0, 4), (0, 4)]


def test_a_row_alone_and_in_a_batch(pkg, dev):
    """The parts of a row follow the batch; alternatives are the same, and numbers near the formula."""
    g = torch.Generator().manual_seed(7)
    x, tokens = ref.logits(g, 3000, 30000, BF)
    want = ref.logprobs64(x[:4], tokens[:4], 20)
    for rows in (4, 100, 3000):
        got = pkg.ops().token_logprobs(x[:rows].to(dev), tokens[:rows].to(dev), 20)
        assert torch.equal(got[3][:4].cpu(), want[3]) and ref.near([t[:4] for t in got[:3]], want[:3])


def test_captured_and_streams(pkg, dev):
    g = torch.Generator().manual_seed(8)
    sets = [[t.to(dev) for t in ref.logits(g, n, 70000, BF)] for n in (3, 5)]
    want = [pkg.ops().token_logprobs(*s, 20) for s in sets]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in sets]
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(pkg.ops().token_logprobs(*s, 20))
        graphs.append(graph)
    for turn in range(3):
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(outs, want))
        for s, o in zip(sets, range(2)):
            s[0].copy_(ref.logits(g, s[0].shape[0], 70000, BF)[0])
            want[o] = pkg.ops().token_logprobs(*s, 20)


def test_far_rows(pkg, dev):
    """Rows behind 2^32 bytes."""
    g = torch.Generator().manual_seed(9)
    rows = (1 << 32) // (2 * 131072) + 8
    x = torch.zeros(rows, 131072, dtype=BF, device=dev)
    last, tokens = ref.logits(g, 3, 131072, BF)
    x[-3:] = last.to(dev)
    all_tokens = torch.zeros(rows, dtype=torch.int64, device=dev)
    all_tokens[-3:] = tokens.to(dev)
    got = pkg.ops().token_logprobs(x, all_tokens, 5)
    want = ref.logprobs64(last, tokens, 5)
    assert torch.equal(got[3][-3:].cpu(), want[3]) and ref.near([t[-3:] for t in got[:3]], want[:3])
    assert torch.equal(got[3][0].cpu(), torch.arange(5))


def test_refusals(pkg, dev):
    x, tokens = torch.zeros(3, 50, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    for a in ((x.double(), tokens, 0), (x[0], tokens, 0), (x, tokens.int(), 0), (x, tokens[:2], 0), (x, tokens, -1),
              (x, tokens, 51), (torch.zeros(3, 100, device=dev), tokens, 65), (x, tokens.cpu(), 0), (x[:, :0], tokens, 0)):
        with pytest.raises(ValueError):
            pkg.token_logprobs(*a)
        with pytest.raises(RuntimeError):
            pkg.ops().token_logprobs(*a)
