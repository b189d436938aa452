"""shared_prefix_attention on the GPU, through the package's function and the torch operator, against the formula in 64
bits."""

import ctypes

import pytest
import torch

import _serving as ref

pytestmark = pytest.mark.gpu
BF, FP, I32 = torch.bfloat16, torch.float16, torch.int32


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def check(pkg, dev, args, scale=None):
    on = [t.to(dev) if torch.is_tensor(t) else t for t in args]
    got = pkg.ops().shared_prefix_attention(*on, scale)
    assert torch.equal(pkg.shared_prefix_attention(*on, scale=scale), got)
    want, extra = ref.attention64(*args, scale=scale)
    assert not got.isnan().any()
    assert ref.near(got.cpu(), want, extra), ((got.cpu().double() - want).abs() - extra).max()
    return got


CASES = [  # batch, seq, q heads, kv heads, head size, page, prefix, own lengths
    (1, 1, 32, 8, 128, 16, 2000, [150]), (1, 1, 4, 1, 128, 16, 100, [3]), (2, 1, 4, 2, 128, 16, 0, [40, 1]),
    (3, 1, 3, 3, 64, 8, 65, [0, 33, 7]), (2, 3, 7, 1, 64, 32, 31, [3, 50]), (2, 5, 14, 2, 80, 24, 33, [2, 37]),
    (1, 9, 8, 1, 96, 1, 70, [20]), (1, 2, 2, 1, 256, 16, 300, [9]), (1, 1, 2, 2, 192, 128, 17, [130]),
    (9, 1, 8, 1, 64, 16, 600, [1] * 9), (1, 40, 2, 1, 64, 16, 40, [77]), (12, 4, 8, 2, 128, 64, 1500, list(range(4, 400, 33))),
    (33, 2, 28, 4, 64, 32, 777, [5 + 3 * i for i in range(33)]), (5, 7, 16, 2, 256, 16, 999, [7, 8, 100, 257, 31]),
    (2, 150, 8, 2, 128, 16, 70, [150, 290]), (4, 1, 64, 1, 128, 16, 321, [9, 0, 64, 65])]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_formula(pkg, dev, case, dtype):
    batch, seq, hq, hk, d, block, prefix, lens = case
    g = torch.Generator().manual_seed(d + seq)
    check(pkg, dev, ref.attention_inputs(g, dtype, batch, seq, hq, hk, d, block, prefix, lens))


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("peak", [20.0, 0.0])
def test_peaked_and_flat_scores(pkg, dev, dtype, peak):
    g = torch.Generator().manual_seed(6)
    check(pkg, dev, ref.attention_inputs(g, dtype, 6, 2, 8, 2, 128, 16, 1300, [100, 700, 3, 2, 40, 64], peak=peak))


def test_lengths_and_bad_pages(pkg, dev):
    g = torch.Generator().manual_seed(2)
    q, k, v, table, length, tables, lens, block = ref.attention_inputs(g, BF, 3, 2, 4, 2, 64, 16, 600, [400, 300, 90])
    for prefix, own in ((0, [0, 0, 0]), (1, [1, 2, 3]), (590, [17, 300, 5]), (-7, [-1, 20, 30])):
        check(pkg, dev, [q, k, v, table, torch.tensor([prefix], dtype=I32), tables, torch.tensor(own, dtype=I32), block])
    table[1], table[3], tables[0, 2] = -1, 2 ** 31 - 1, -2 ** 31
    tables[1, 0] = k.shape[0] // block
    check(pkg, dev, [q, k, v, table, length, tables, lens, block], scale=0.2)
    check(pkg, dev, [q, k[:-5].contiguous(), v[:-5].contiguous(), table, length, tables, lens, block])
    none = torch.zeros(0, dtype=I32, device=dev)
    out = pkg.shared_prefix_attention(q[:0].to(dev), k.to(dev), v.to(dev), none, length.to(dev), tables[:0].to(dev),
                                      lens[:0].to(dev), block)
    assert out.shape == (0, 2, 4, 64)


@pytest.mark.parametrize("tiles,team", [(1, 1), (1, 4), (2, 0), (3, 1), (3, 2), (3, 4)], ids=str)
@pytest.mark.parametrize("d,block", [(64, 16), (80, 24), (96, 1), (128, 16), (192, 64), (256, 16)], ids=str)
def test_every_way(pkg, dev, d, block, tiles, team):
    """Tiles of 32 rows and shared ones, the prefix before the own keys, teams of waves: whatever the sizes would choose."""
    g = torch.Generator().manual_seed(d)
    args = ref.attention_inputs(g, BF, 7, 5, 18, 2, d, block, 450, [5, 6, 33, 64, 300, 17, 0])
    lib = ctypes.CDLL(pkg.lib_path("shared_prefix_attention"))
    try:
        for splits in (1, 3):
            for slot, value in enumerate((splits if tiles < 3 else 0, splits, tiles, team)):
                lib.prefix_attention_tune(slot, value)
            check(pkg, dev, args)
    finally:
        for slot in range(4):
            lib.prefix_attention_tune(slot, 0)


@pytest.mark.parametrize("tiles,team", [(1, 1), (2, 0), (3, 4)], ids=str)
@pytest.mark.parametrize("d,dtype,bad", [(64, FP, "nan"), (80, BF, "-inf"), (128, BF, "nan"), (192, FP, "inf"), (256, BF, "nan")],
                         ids=str)
def test_bad_values_reach_only_the_queries_that_see_them(pkg, dev, d, dtype, bad, tiles, team):
    """A NaN or infinite value of a step's own token is in its query and those behind it, in that one place of the head."""
    g, seq, lens = torch.Generator().manual_seed(13), 9, [45, 39, 3, 35, 300]
    q, k, v, table, length, tables, lens, block = ref.attention_inputs(g, dtype, 5, seq, 6, 2, d, 16, 40, lens)
    clean, reached = v.clone(), torch.zeros(q.shape, dtype=torch.bool)
    for b, t, c in [(0, 41, 3), (0, 44, d - 1), (1, 33, 17), (2, 1, 0), (3, 30, 9), (3, 32, 40), (4, 295, 5)]:
        slot = int(tables[b, t // block]) * block + t % block
        v[slot, 1, c], clean[slot, 1, c] = float(bad), 0.0
        reached[b, max(0, t - int(lens[b]) + seq):, 3:, c] = True
    want, extra = ref.attention64(q, k, clean, table, length, tables, lens, block)
    on = [t.to(dev) if torch.is_tensor(t) else t for t in (q, k, v, table, length, tables, lens, block)]
    lib = ctypes.CDLL(pkg.lib_path("shared_prefix_attention"))
    lib.prefix_attention_tune(2, tiles), lib.prefix_attention_tune(3, team)
    try:
        got = pkg.ops().shared_prefix_attention(*on).cpu()
    finally:
        lib.prefix_attention_tune(2, 0), lib.prefix_attention_tune(3, 0)
    assert not got[reached].isfinite().any()
    assert got[~reached].isfinite().all() and ref.near(got[~reached], want[~reached], extra[~reached])


def test_strided_queries(pkg, dev):
    g = torch.Generator().manual_seed(5)
    q, *rest = [t.to(dev) if torch.is_tensor(t) else t for t in
                ref.attention_inputs(g, BF, 2, 3, 4, 2, 64, 16, 50, [20, 30])]
    want = pkg.ops().shared_prefix_attention(q, *rest)
    packed = torch.full((2, 3, 8, 64), float("nan"), dtype=BF, device=dev)
    packed[:, :, 2:6] = q
    odd = torch.full((2 * 3 * 4 * 64 + 3,), float("nan"), dtype=BF, device=dev)
    odd[3:] = q.flatten()
    for view in (packed[:, :, 2:6], q.transpose(1, 2).contiguous().transpose(1, 2), odd[3:].view(2, 3, 4, 64),
                 q.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(pkg.ops().shared_prefix_attention(view, *rest), want)
        assert torch.equal(pkg.shared_prefix_attention(view, *rest), want)


def test_queries_with_odd_outer_strides(pkg, dev):
    """Rows of 769 elements: one sequence's stride is not used, two sequences' queries are copied."""
    g = torch.Generator().manual_seed(15)
    for batch in (1, 2):
        q, *rest = [t.to(dev) if torch.is_tensor(t) else t for t in
                    ref.attention_inputs(g, BF, batch, 3, 4, 2, 64, 16, 50, [20] * batch)]
        odd = torch.full((2, 769), float("nan"), dtype=BF, device=dev)[:, :768].unflatten(1, (3, 4, 64))[:batch]
        odd.copy_(q)
        assert odd.stride(0) == 769
        want = pkg.ops().shared_prefix_attention(q, *rest)
        assert torch.equal(pkg.ops().shared_prefix_attention(odd, *rest), want)
        assert torch.equal(pkg.shared_prefix_attention(odd, *rest), want)
    step = torch.empty_strided((2, 1, 4, 64), (256, 7, 64, 1), dtype=BF, device=dev)  # single tokens
    q, *rest = [t.to(dev) if torch.is_tensor(t) else t for t in ref.attention_inputs(g, BF, 2, 1, 4, 2, 64, 16, 50, [20, 3])]
    step.copy_(q)
    want = pkg.ops().shared_prefix_attention(q, *rest)
    assert torch.equal(pkg.ops().shared_prefix_attention(step, *rest), want)
    assert torch.equal(pkg.shared_prefix_attention(step, *rest), want)


def test_result_does_not_depend_on_the_batch_around_it(pkg, dev):
    """No atomics: the same call gives the same bits."""
    g = torch.Generator().manual_seed(7)
    args = [t.to(dev) if torch.is_tensor(t) else t for t in
            ref.attention_inputs(g, BF, 20, 3, 16, 4, 128, 16, 3000, [3 + 40 * i for i in range(20)])]
    want = pkg.ops().shared_prefix_attention(*args)
    for _ in range(5):
        assert torch.equal(pkg.ops().shared_prefix_attention(*args), want)


@pytest.mark.parametrize("seq", [1, 3])
def test_a_sequence_alone_and_in_larger_batches(pkg, dev, seq):
    """One sequence's queries within batches of 1 to 90, which are cut into other splits and tiles: each near the formula
    (their bits may differ), and the same call the same bits."""
    g = torch.Generator().manual_seed(17)
    lens = [3 + (37 * i) % 200 for i in range(90)]
    lens[0] = 130
    q, k, v, table, length, tables, seq_lens, block = ref.attention_inputs(g, BF, 90, seq, 8, 2, 128, 16, 1200, lens)
    want, extra = ref.attention64(q[:1], k, v, table, length, tables[:1], seq_lens[:1], block)
    on = [t.to(dev) for t in (q, k, v, table, length, tables, seq_lens)]
    for batch in (1, 2, 7, 30, 90):
        args = [t[:batch] if i in (0, 5, 6) else t for i, t in enumerate(on)]
        got = pkg.ops().shared_prefix_attention(*args, block)
        assert ref.near(got[:1].cpu(), want, extra)
        for _ in range(3):
            assert torch.equal(pkg.ops().shared_prefix_attention(*args, block), got)


def test_two_to_the_32_threads(pkg, dev):
    """2^24 single tokens and some more, of 1000 queries in turn, behind one prefix, each with the same few own keys: the
    parts' join and the own keys' tiles take 2^32 threads."""
    g, n, some = torch.Generator().manual_seed(16), (1 << 24) + 1000, 1000
    q, k, v, table, length, tables, lens, block = ref.attention_inputs(g, BF, some, 1, 1, 1, 64, 16, 40, [3] * some)
    tables[:] = tables[:1]
    few = [t.to(dev) for t in (q, k, v, table, length, tables, lens)]
    many = [t[torch.arange(n, device=dev) % some] if i in (0, 5, 6) else t for i, t in enumerate(few)]
    lib = ctypes.CDLL(pkg.lib_path("shared_prefix_attention"))
    want, extra = ref.attention64(q, k, v, table, length, tables, lens, block)
    for tiles in (1, 2, 3):
        lib.prefix_attention_tune(2, tiles), lib.prefix_attention_tune(3, 1)
        try:
            out = pkg.ops().shared_prefix_attention(*many, block)
        finally:
            lib.prefix_attention_tune(2, 0), lib.prefix_attention_tune(3, 0)
        first = out[:some].clone()
        assert ref.near(first.cpu(), want, extra)
        assert torch.equal(out[:n // some * some].view(-1, some, 64), first.view(1, some, 64).expand(n // some, some, 64))
        assert torch.equal(out[n // some * some:], first[:n % some])


def test_captured_lengths_follow(pkg, dev):
    """Two graphs of one call, their lengths and pages changed between replays, on two streams at once."""
    g = torch.Generator().manual_seed(8)
    ops, sets = pkg.ops(), []
    for n in (2, 3):
        args = [t.to(dev) if torch.is_tensor(t) else t for t in
                ref.attention_inputs(g, BF, n, 1, 8, 2, 128, 16, 900, [700] * n)]
        ops.shared_prefix_attention(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.shared_prefix_attention(*args)
        sets.append((args, graph, out, torch.cuda.Stream()))
    for prefix, own in ((900, 700), (0, 33), (431, 1), (1, 0), (900, 512)):
        for args, *_ in sets:
            args[0].normal_(), args[4].fill_(prefix), args[6].fill_(own)
        torch.cuda.synchronize()
        for args, graph, out, s in sets:
            with torch.cuda.stream(s):
                graph.replay()
        want = [ops.shared_prefix_attention(*args) for args, *_ in sets]
        torch.cuda.synchronize()
        for (args, graph, out, s), w in zip(sets, want):
            assert torch.equal(out, w)


def test_cache_behind_four_gigabytes(pkg, dev):
    """Pages whose bytes lie past 2^32 in each cache."""
    slots, hk, d, block = (1 << 24) + 4096, 1, 128, 16
    k = torch.zeros((slots, hk, d), dtype=BF, device=dev)
    v = torch.zeros((slots, hk, d), dtype=BF, device=dev)
    g = torch.Generator().manual_seed(9)
    last = slots // block - 1
    q, _, _, table, length, tables, lens, _ = ref.attention_inputs(g, BF, 2, 1, 4, 1, d, block, 40, [20, 5])
    pages = torch.tensor([last, last - 7, 3, last - 2, 5, last - 1, (1 << 24) // block - 1], dtype=I32)
    table, tables = pages[:3], pages[3:].view(2, 2)
    small_k, small_v = torch.randn(7 * block, hk, d, generator=g).to(BF), torch.randn(7 * block, hk, d, generator=g).to(BF)
    for i, page in enumerate(pages.tolist()):
        k[page * block:(page + 1) * block] = small_k[i * block:(i + 1) * block].to(dev)
        v[page * block:(page + 1) * block] = small_v[i * block:(i + 1) * block].to(dev)
    got = pkg.ops().shared_prefix_attention(q.to(dev), k, v, table.to(dev), length.to(dev), tables.to(dev), lens.to(dev),
                                            block)
    want, extra = ref.attention64(q, small_k, small_v, torch.arange(3), length, torch.arange(3, 7).view(2, 2), lens, block)
    assert ref.near(got.cpu(), want, extra)
