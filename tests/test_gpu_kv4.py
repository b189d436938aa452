"""The cache in 4 bits and attention over it on the GPU, through the package's functions and the torch operators, against
the definition in 64 bits."""

import ctypes

import pytest
import torch

import _kv4 as kv4
import _serving as ref

pytestmark = pytest.mark.gpu
BF, FP, I32 = torch.bfloat16, torch.float16, torch.int32


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def new_cache(pages, hk, block, d, dev):
    return [torch.full((pages, hk, block, n), 17, dtype=torch.uint8, device=dev) for n in (d // 2, d // 32) * 2]


def check_append(pkg, dev, k, v, slots, pages, block):
    hk, d = k.shape[1:]
    want = new_cache(pages, hk, block, d, "cpu")
    for x, i in ((k, 0), (v, 2)):
        codes, scales = kv4.encode(x)
        inside = (slots >= 0) & (slots < pages * block)
        s = slots[inside]
        want[i][s // block, :, s % block], want[i + 1][s // block, :, s % block] = codes[inside], scales[inside]
    caches = [new_cache(pages, hk, block, d, dev) for _ in range(2)]
    pkg.ops().kv4_append_(k.to(dev), v.to(dev), *caches[0], slots.to(dev))
    pkg.kv4_append(k.to(dev), v.to(dev), *caches[1], slots.to(dev))
    for cache in caches:
        for a, b in zip(cache, want):
            assert torch.equal(a.cpu(), b)
    for dtype in (BF, FP):
        got = pkg.ops().kv4_read(*caches[0], slots.to(dev), dtype)
        other = pkg.kv4_read(*caches[0], slots.to(dev), dtype)
        for a, b, i in zip(got, other, (0, 2)):
            values = kv4.flat(kv4.decode(*want[i:i + 2]))
            inside = (slots >= 0) & (slots < pages * block)
            full = torch.where(inside[:, None, None], values[slots.clamp(0, pages * block - 1)], 0.0).to(dtype)
            bits = lambda t: torch.where(t.isnan(), 1, t.view(torch.int16)).cpu()
            assert torch.equal(bits(a), bits(full)) and torch.equal(bits(a), bits(b))


@pytest.mark.parametrize("tokens,hk,d,block", [(1, 1, 64, 1), (9, 2, 64, 24), (17, 1, 96, 16), (40, 3, 128, 8),
                                               (333, 2, 192, 32), (100, 1, 256, 128), (2000, 8, 128, 64)], ids=str)
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_append_and_read(pkg, dev, tokens, hk, d, block, dtype):
    g = torch.Generator().manual_seed(d + tokens)
    k, v = kv4.rows(g, dtype, tokens, hk, d), kv4.rows(g, dtype, tokens, hk, d)
    if tokens > 6:
        k[6, 0, 5], v[6, hk - 1, 40] = float("nan"), float("-inf")
    pages = -(-tokens // block) + 1
    slots = torch.randperm(pages * block, generator=g)[:tokens]
    if tokens > 2:
        slots[1], slots[2] = -1, pages * block
    check_append(pkg, dev, k, v, slots, pages, block)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_every_16_bit_number(pkg, dev, dtype):
    """All patterns, each in a group of its own scale (with a larger number beside it) and alone."""
    x = torch.arange(-32768, 32768).to(torch.int16).view(dtype)
    alone = x.view(-1, 1, 1).expand(-1, 1, 64).contiguous()
    beside = alone.clone()
    beside[:, 0, 1::2] = (beside[:, 0, :1].float() * 5.3).to(dtype)
    check_append(pkg, dev, alone, beside, torch.arange(65536), 1024, 64)


def test_append_views(pkg, dev):
    g = torch.Generator().manual_seed(4)
    qkv = kv4.rows(g, BF, 50, 6, 128)
    want = new_cache(4, 2, 16, 128, dev)
    slots = torch.randperm(64, generator=g)[:50].to(dev)
    pkg.ops().kv4_append_(qkv[:, 2:4].contiguous().to(dev), qkv[:, 4:].contiguous().to(dev), *want, slots)
    on = qkv.to(dev)
    odd = torch.empty(50 * 6 * 128 + 1, dtype=BF, device=dev)[1:].view(50, 6, 128).copy_(on)
    flipped = on.transpose(0, 1).contiguous().transpose(0, 1)
    for t in (on, odd, flipped):
        for call in (pkg.ops().kv4_append_, pkg.kv4_append):
            cache = new_cache(4, 2, 16, 128, dev)
            call(t[:, 2:4], t[:, 4:], *cache, slots)
            assert all(torch.equal(a, b) for a, b in zip(cache, want))
    step = torch.empty_strided((1, 2, 128), (7, 128, 1), dtype=BF, device=dev).copy_(on[:1, :2])  # one token
    cache = new_cache(4, 2, 16, 128, dev)
    pkg.ops().kv4_append_(step, step, *cache, slots[:1])
    assert torch.equal(cache[0], cache[2])


def check(pkg, dev, q, cache, tables, lens, scale=None):
    on = [q.to(dev), *(t.to(dev) for t in cache), tables.to(dev), lens.to(dev)]
    got = pkg.ops().kv4_attention(*on, scale)
    assert torch.equal(pkg.kv4_attention(*on, scale=scale), got)
    want, extra = kv4.attention64(q, cache, tables, lens, scale)
    assert not got.isnan().any()
    assert ref.near(got.cpu(), want, extra), ((got.cpu().double() - want).abs() - extra).max()
    return got


CASES = [  # batch, seq, q heads, kv heads, head size, page, lengths
    (1, 1, 4, 1, 128, 16, [100]), (2, 1, 4, 2, 64, 1, [40, 1]), (3, 1, 3, 3, 64, 8, [0, 33, 700]),
    (2, 3, 7, 1, 96, 32, [3, 650]), (1, 9, 8, 1, 128, 24, [600]), (1, 2, 2, 1, 256, 16, [530]),
    (1, 5, 8, 2, 192, 128, [130]), (2, 12, 4, 2, 64, 16, [5, 77]), (1, 1, 32, 8, 128, 64, [5000]),
    (9, 1, 32, 8, 128, 64, [1 + 300 * i for i in range(9)]), (5, 4, 28, 4, 64, 24, [7, 1801, 4, 900, 33]),
    (70, 1, 8, 2, 128, 16, [17 * i % 700 for i in range(70)]), (2, 16, 32, 4, 256, 32, [300, 1200]),
    (1, 40, 4, 2, 96, 16, [1500])]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_formula(pkg, dev, case, dtype):
    batch, seq, hq, hk, d, block, lens = case
    g = torch.Generator().manual_seed(d + seq)
    check(pkg, dev, *kv4.inputs(g, dtype, batch, seq, hq, hk, d, block, lens))


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("peak", [20.0, 0.0])
def test_peaked_and_flat_scores(pkg, dev, dtype, peak):
    g = torch.Generator().manual_seed(6)
    check(pkg, dev, *kv4.inputs(g, dtype, 4, 2, 8, 2, 128, 16, [100, 700, 3, 2000], peak=peak))


@pytest.mark.parametrize("runs", [-1, 1, 2, 5, 17, 300])
@pytest.mark.parametrize("tiles", [1, 2])
def test_every_cut(pkg, dev, runs, tiles):
    g = torch.Generator().manual_seed(1)
    lib = ctypes.CDLL(pkg.lib_path("kv4_attention"))
    lib.kv4_attention_tune(0, runs), lib.kv4_attention_tune(1, tiles)
    try:
        for d in (64, 128, 256):
            check(pkg, dev, *kv4.inputs(g, BF, 5, 3, 12, 2, d, 16, [600, 0, 2, 300, 1100]))
    finally:
        lib.kv4_attention_tune(0, 0), lib.kv4_attention_tune(1, 0)


def test_lengths_and_bad_pages(pkg, dev):
    g = torch.Generator().manual_seed(2)
    q, cache, tables, lens = kv4.inputs(g, BF, 3, 2, 4, 2, 64, 16, [400, 700, 90])
    for own in ([1, 2, 3], [0, 0, 0], [-1, 20, 30]):
        check(pkg, dev, q, cache, tables, torch.tensor(own, dtype=I32))
    tables[0, 2], tables[1, 1], tables[2, 0] = -2 ** 31, 2 ** 31 - 1, cache[0].shape[0]
    check(pkg, dev, q, cache, tables, lens, scale=0.2)
    on = [t.to(dev) for t in (tables, lens)]
    assert not pkg.kv4_attention(q.to(dev), *(t[:0].to(dev) for t in cache), *on).any()
    out = pkg.kv4_attention(q[:0].to(dev), *(t.to(dev) for t in cache), on[0][:0], on[1][:0])
    assert out.shape == (0, 2, 4, 64)
    assert not pkg.kv4_attention(q.to(dev), *(t.to(dev) for t in cache), on[0][:, :0], on[1]).any()


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("d,block", [(64, 8), (128, 32), (256, 64)], ids=str)
def test_growing_scores(pkg, dev, d, block, dtype):
    """Scores that grow without bound along a context, so that no early one is a point for the later; a first slice that is
    absent altogether."""
    g = torch.Generator().manual_seed(12)
    q, cache, tables, lens = kv4.inputs(g, dtype, 2, 2, 4, 2, d, block, [700, 300], peak=1.0, power=(127, 128))
    for b, n in enumerate(lens.tolist()):
        t = torch.arange(n)
        cache[1][tables[b].long()[t // block], :, t % block] = (118 + t // 40).to(torch.uint8)[:, None, None]
    check(pkg, dev, q, cache, tables, lens)
    tables[0, :-(-32 // block)], tables[1, 1] = -1, -1
    check(pkg, dev, q, cache, tables, lens)


@pytest.mark.parametrize("d", [64, 96, 128, 192, 256])
def test_nan_reaches_only_the_queries_that_see_it(pkg, dev, d):
    g, seq = torch.Generator().manual_seed(5), 6
    q, cache, tables, lens = kv4.inputs(g, BF, 2, seq, 4, 2, d, 8, [45, 900])
    clean = [t.clone() for t in cache]
    reached = torch.zeros(q.shape, dtype=torch.bool)
    for b, t, group in ((0, 41, 0), (0, 44, d // 32 - 1), (1, 896, 1), (1, 897, 0)):
        cache[3][tables[b, t // 8], 1, t % 8, group] = 255
        clean[3][tables[b, t // 8], 1, t % 8, group] = 120
        reached[b, t - int(lens[b]) + seq:, 2:, 32 * group:32 * group + 32] = True
    want, extra = kv4.attention64(q, clean, tables, lens)
    cache[1][tables[0, 42 // 8], 0, 42 % 8, 0] = 254  # a key: all of the queries' elements
    key = torch.zeros(q.shape, dtype=torch.bool)
    key[0, 42 - 45 + seq:, :2] = True
    got = pkg.ops().kv4_attention(q.to(dev), *(t.to(dev) for t in cache), tables.to(dev), lens.to(dev)).cpu()
    assert got[reached | key].isnan().all()
    rest = ~(reached | key)
    assert ref.near(got[rest], want[rest], extra[rest])


def test_queries_of_any_size_and_stride(pkg, dev):
    g = torch.Generator().manual_seed(6)
    q, cache, tables, lens = kv4.inputs(g, BF, 2, 4, 4, 1, 64, 16, [70, 900])
    q[0, 0, 0], q[0, 0, 1], q[0, 0, 2] = 0.0, q[0, 0, 1] * 1e-30, q[0, 0, 2] * 2.0 ** -60
    q[0, 0, 3, :32] *= 2.0 ** -9
    want = check(pkg, dev, q, cache, tables, lens)
    on = [t.to(dev) for t in (*cache, tables, lens)]
    packed = torch.full((2, 4, 8, 64), float("nan"), dtype=BF, device=dev)
    packed[:, :, 2:6] = q.to(dev)
    odd = torch.empty(q.numel() + 3, dtype=BF, device=dev)[3:].view(q.shape).copy_(q)
    for view in (packed[:, :, 2:6], odd, odd.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(pkg.ops().kv4_attention(view, *on), want)
        assert torch.equal(pkg.kv4_attention(view, *on), want)
    for bad in (float("nan"), float("inf")):
        q[0, 2, 1, 5] = bad
        got = pkg.ops().kv4_attention(q.to(dev), *on)
        assert got[0, 2, 1].isnan().all()
        got[0, 2, 1] = want[0, 2, 1]
        assert torch.equal(got, want)


def test_repeated_calls_and_streams(pkg, dev):
    """The same call gives the same bits, also on two streams at once."""
    g = torch.Generator().manual_seed(7)
    args = [[q.to(dev), *(t.to(dev) for t in cache), tables.to(dev), lens.to(dev)] for q, cache, tables, lens in
            (kv4.inputs(g, BF, 5, 2, 16, 4, 128, 16, [700 + 300 * i for i in range(5)]) for _ in range(2))]
    want = [pkg.ops().kv4_attention(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(pkg.ops().kv4_attention(*a))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_captured_lengths_follow(pkg, dev):
    """A decode step captured: the append and the attention; lengths, slots and pages change between replays."""
    g = torch.Generator().manual_seed(8)
    q, cache, tables, lens = kv4.inputs(g, BF, 3, 1, 8, 2, 128, 16, [900, 40, 300], spare=4)
    cache[1][cache[1] == 255], cache[3][cache[3] == 255] = 120, 120
    ops, on = pkg.ops(), [t.to(dev) for t in cache]
    static = dict(q=q.to(dev), k=kv4.rows(g, BF, 3, 2, 128).to(dev), v=kv4.rows(g, BF, 3, 2, 128).to(dev),
                  slots=torch.full((3,), -1, device=dev), tables=tables.to(dev), lens=lens.to(dev))

    def step():
        ops.kv4_append_(static["k"], static["v"], *on, static["slots"])
        return ops.kv4_attention(static["q"], *on, static["tables"], static["lens"])

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(4):
        static["lens"].copy_(lens - 7 * n)
        at = (static["lens"] - 1).long()
        static["slots"].copy_(static["tables"].long().gather(1, at[:, None] // 16)[:, 0] * 16 + at % 16)
        static["k"].copy_(kv4.rows(g, BF, 3, 2, 128)), static["q"].copy_(torch.randn(q.shape, generator=g).to(BF))
        before = [t.clone() for t in on]
        graph.replay()
        torch.cuda.synchronize()
        got, after = out.clone(), [t.clone() for t in on]
        for t, b in zip(on, before):
            t.copy_(b)
        want = step()
        assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(after, on))
        exact, extra = kv4.attention64(static["q"].cpu(), [t.cpu() for t in on], tables, static["lens"].cpu())
        assert ref.near(got.cpu(), exact, extra)


def test_far_slots(pkg, dev):
    """A cache of more than 2^32 bytes of codes: its last pages."""
    pages, hk, block, d = (1 << 32) // (8 * 128 * 64) + 20, 8, 128, 128
    cache = [torch.zeros(pages, hk, block, n, dtype=torch.uint8, device=dev) for n in (d // 2, d // 32) * 2]
    g = torch.Generator().manual_seed(9)
    k, v = kv4.rows(g, BF, 200, hk, d), kv4.rows(g, BF, 200, hk, d)
    k[3], v[3] = 1.0, 1.0
    tables = torch.tensor([[pages - 1, pages - 3]], dtype=I32)
    at = torch.arange(200)
    slots = tables[0].long()[at // block] * block + at % block
    pkg.ops().kv4_append_(k.to(dev), v.to(dev), *cache, slots.to(dev))
    q = torch.randn(1, 1, 16, d, generator=g).to(BF)
    got = pkg.ops().kv4_attention(q.to(dev), *cache, tables.to(dev), torch.tensor([200], dtype=I32, device=dev))
    near_by = [t[[pages - 1, pages - 3]].cpu() for t in cache]
    want, extra = kv4.attention64(q, near_by, torch.tensor([[0, 1]], dtype=I32), torch.tensor([200], dtype=I32))
    assert ref.near(got.cpu(), want, extra)
    back = pkg.ops().kv4_read(*cache, slots.to(dev), BF)
    for x, y in zip(back, (k, v)):
        assert torch.equal(x.cpu().double(), kv4.decode(*kv4.encode(y)))


def test_refusals(pkg, dev):
    g = torch.Generator().manual_seed(8)
    q, cache, tables, lens = kv4.inputs(g, BF, 2, 1, 4, 2, 64, 16, [30, 20])
    q, tables, lens, cache = q.to(dev), tables.to(dev), lens.to(dev), [t.to(dev) for t in cache]
    k, slots = torch.zeros(3, 2, 64, dtype=BF, device=dev), torch.arange(3, device=dev)
    ops = pkg.ops()

    def both(first, second):
        with pytest.raises(ValueError):
            first()
        with pytest.raises(RuntimeError):
            second()

    def attention(**kw):
        a = dict(zip(("q", "k_codes", "k_scales", "v_codes", "v_scales", "block_tables", "seq_lens"),
                     (q, *cache, tables, lens)), **kw)
        both(lambda: pkg.kv4_attention(**a), lambda: ops.kv4_attention(**a))

    for kw in (dict(q=q.float()), dict(q=q[..., :48]), dict(q=q[:, :, :3]), dict(q=q[0]), dict(k_codes=cache[0][:, :1]),
               dict(k_codes=cache[0].transpose(1, 2)), dict(k_scales=cache[1][..., :1].contiguous()),
               dict(v_scales=cache[3][:-1]), dict(v_codes=cache[2].to(torch.int8)), dict(block_tables=tables.long()),
               dict(block_tables=tables[:1]), dict(seq_lens=lens[:1]), dict(seq_lens=lens.cpu()), dict(scale=0.0),
               dict(scale=float("nan"))):
        attention(**kw)

    def append(*a):
        both(lambda: pkg.kv4_append(*a), lambda: ops.kv4_append_(*a))

    append(k.float(), k, *cache, slots)
    append(k[:2], k, *cache, slots)
    append(k[:, :1], k[:, :1], *cache, slots)
    append(k, k, *cache, slots.int())
    append(k, k, *cache, slots[:2])
    append(k, k, cache[0], cache[1], cache[0], cache[3], slots)
    append(k, k, *cache, slots.cpu())
    whole = torch.zeros(2, 2, 16, 32, dtype=torch.uint8, device=dev)
    inside = whole.view(-1)[:768].view(BF).view(6, 1, 64)
    append(inside, inside, whole, torch.zeros(2, 2, 16, 2, dtype=torch.uint8, device=dev), whole.clone(),
           torch.zeros(2, 2, 16, 2, dtype=torch.uint8, device=dev), torch.arange(6, device=dev))
    both(lambda: pkg.kv4_read(*cache, slots.int()), lambda: ops.kv4_read(*cache, slots.int(), BF))
    both(lambda: pkg.kv4_read(*cache, slots, torch.float32), lambda: ops.kv4_read(*cache, slots, torch.float32))
