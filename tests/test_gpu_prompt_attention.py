"""prompt_attention on the GPU, through the package's function and the torch operator, against the formula in 64 bits."""

import ctypes

import pytest
import torch

import _prompts as prompts
import _serving as ref

pytestmark = pytest.mark.gpu
BF, FP, I32 = torch.bfloat16, torch.float16, torch.int32


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def check(pkg, dev, q, k, v, offsets, scale=None):
    on = [t.to(dev) for t in (q, k, v, offsets)]
    got = pkg.ops().prompt_attention(*on, scale)
    assert torch.equal(pkg.prompt_attention(*on, scale=scale), got)
    want, extra = prompts.attention64(q, k, v, offsets, scale)
    assert not got.isnan().any()
    assert ref.near(got.cpu(), want, extra), ((got.cpu().double() - want).abs() - extra).max()
    return got


CASES = [  # lengths, q heads, kv heads, head size
    ([1], 4, 1, 64), ([33], 3, 3, 64), ([5, 0, 70, 1], 4, 2, 128), ([40], 7, 1, 80), ([150, 3], 2, 1, 96),
    ([66, 31], 2, 2, 192), ([40, 65], 4, 1, 256), ([0, 0, 9], 8, 8, 128), ([700, 257, 512], 8, 2, 128),
    ([1025], 3, 1, 64), ([513, 300], 4, 4, 256), ([1, 2, 3, 4, 5, 6, 7] * 20, 4, 2, 128)]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_formula(pkg, dev, case, dtype):
    lens, hq, hk, d = case
    g = torch.Generator().manual_seed(d + len(lens))
    check(pkg, dev, *prompts.inputs(g, dtype, lens, hq, hk, d))


@pytest.mark.parametrize("waves", [0, 4, 8])
@pytest.mark.parametrize("d", [64, 80, 96, 128, 192, 256])
def test_every_form(pkg, dev, waves, d):
    g = torch.Generator().manual_seed(d)
    lib = ctypes.CDLL(pkg.lib_path("prompt_attention"))
    lib.prompt_attention_tune(0, waves)
    try:
        for group in (1, 3, 8):
            check(pkg, dev, *prompts.inputs(g, BF, [300, 64, 1, 31], 2 * group, 2, d, before=3, behind=9))
    finally:
        lib.prompt_attention_tune(0, 0)


def test_many_prompts_and_rows_of_none(pkg, dev):
    g = torch.Generator().manual_seed(3)
    lens = [(5 * i) % 13 if i % 4 else 0 for i in range(5000)]
    q, k, v, offsets = prompts.inputs(g, BF, lens[:300], 2, 1, 64, before=7, behind=70)
    got = check(pkg, dev, q, k, v, offsets)
    assert not got[:7].any() and not got[-70:].any()
    on = [t.to(dev) for t in (q, k, v)]
    for none in ([5, 5, 5], [0], [q.shape[0]], [-9, 0, -3]):  # no prompt at all
        assert not pkg.ops().prompt_attention(*on, torch.tensor(none, dtype=I32, device=dev)).any()
    q, k, v, offsets = prompts.inputs(g, BF, lens, 2, 1, 64)  # 64 * 64 prompts and more
    got = pkg.ops().prompt_attention(*(t.to(dev) for t in (q, k, v, offsets))).cpu()
    for a in (0, 4100, 4990):
        b = a + 9
        o = offsets[a:b + 1] - offsets[a]
        part = slice(int(offsets[a]), int(offsets[b]))
        want, extra = prompts.attention64(q[part], k[part], v[part], o)
        assert ref.near(got[part], want, extra)


def test_peaked_and_flat_scores(pkg, dev):
    g = torch.Generator().manual_seed(6)
    for dtype in (BF, FP):
        for peak in (20.0, 0.0):
            check(pkg, dev, *prompts.inputs(g, dtype, [600], 4, 1, 128, peak=peak))


@pytest.mark.parametrize("d,dtype,bad", [(64, FP, "nan"), (80, BF, "-inf"), (128, BF, "nan"), (192, FP, "nan"),
                                         (256, FP, "inf")], ids=str)
@pytest.mark.parametrize("waves", [0, 4])
def test_bad_values_reach_only_the_queries_that_see_them(pkg, dev, d, dtype, bad, waves):
    """A NaN or infinite value of a token is in its query and those behind it, in that one place of the head; also where
    the next prompt begins behind it."""
    g = torch.Generator().manual_seed(7)
    lens = [300, 41, 8, 100]
    q, k, v, offsets = prompts.inputs(g, dtype, lens, 6, 2, d)
    clean, reached = v.clone(), torch.zeros(q.shape, dtype=torch.bool)
    for b, t, c in ((0, 40, 3), (0, 299, d - 1), (0, 201, 7), (1, 0, 17), (2, 5, 0), (3, 64, 11)):
        at, end = int(offsets[b]) + t, int(offsets[b + 1])
        v[at, 1, c], clean[at, 1, c] = float(bad), 0.0
        reached[at:end, 3:, c] = True
    want, extra = prompts.attention64(q, k, clean, offsets)
    lib = ctypes.CDLL(pkg.lib_path("prompt_attention"))
    lib.prompt_attention_tune(0, waves)
    try:
        got = pkg.ops().prompt_attention(*(t.to(dev) for t in (q, k, v, offsets))).cpu()
    finally:
        lib.prompt_attention_tune(0, 0)
    assert not got[reached].isfinite().any()
    assert got[~reached].isfinite().all() and ref.near(got[~reached], want[~reached], extra[~reached])


def test_bad_keys_reach_only_the_queries_that_see_them(pkg, dev):
    g = torch.Generator().manual_seed(8)
    q, k, v, offsets = prompts.inputs(g, BF, [70, 41], 4, 2, 64)
    want, extra = prompts.attention64(q, k, v, offsets)
    k[50, 1, 7], k[80, 0, 3] = float("nan"), float("inf")
    reached = torch.zeros(q.shape, dtype=torch.bool)
    reached[50:70, 2:], reached[80:, :2] = True, True
    got = pkg.ops().prompt_attention(*(t.to(dev) for t in (q, k, v, offsets))).cpu()
    assert got[50:70, 2:].isnan().all() and ref.near(got[~reached], want[~reached], extra[~reached])


def test_views(pkg, dev):
    g = torch.Generator().manual_seed(5)
    q, k, v, offsets = prompts.inputs(g, BF, [200, 50], 4, 2, 64)
    want = check(pkg, dev, q, k, v, offsets, scale=0.3)
    on, offsets = [t.to(dev) for t in (q, k, v)], offsets.to(dev)
    packed = torch.cat(on, 1)
    odd = torch.empty(packed.numel() + 1, dtype=BF, device=dev)[1:].view(packed.shape).copy_(packed)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in on]
    wide = [torch.empty(t.numel() * 2, dtype=BF, device=dev).view(*t.shape[:2], 128)[..., ::2].copy_(t) for t in on]
    for parts in (packed.split([4, 2, 2], 1), odd.split([4, 2, 2], 1), heads_first, wide):
        assert torch.equal(pkg.ops().prompt_attention(*parts, offsets, 0.3), want)
        assert torch.equal(pkg.prompt_attention(*parts, offsets, scale=0.3), want)
    spaced = torch.arange(5, device=dev, dtype=I32).repeat_interleave(1)
    spaced[::2] = offsets
    assert torch.equal(pkg.ops().prompt_attention(*on, spaced[::2], 0.3), want)
    one = [t[:1].expand(1, *t.shape[1:]).as_strided((1, t.shape[1], 64), (7, 64, 1)) for t in on]  # a single token
    assert torch.equal(pkg.ops().prompt_attention(*one, torch.tensor([0, 1], dtype=I32, device=dev)).view(2, 2, 64)[:, 0],
                       one[2][0])
    none = pkg.prompt_attention(*(t[:0] for t in on), offsets)
    assert none.shape == (0, 4, 64)


def test_a_prompt_alone_and_packed(pkg, dev):
    """A prompt's bits do not depend on those around it, nor on the call."""
    g = torch.Generator().manual_seed(10)
    q, k, v, offsets = [t.to(dev) for t in prompts.inputs(g, BF, [130, 700, 65], 8, 2, 128)]
    whole = pkg.ops().prompt_attention(q, k, v, offsets)
    for _ in range(3):
        assert torch.equal(pkg.ops().prompt_attention(q, k, v, offsets), whole)
    lib = ctypes.CDLL(pkg.lib_path("prompt_attention"))
    lib.prompt_attention_tune(0, 4)
    try:
        packed = pkg.ops().prompt_attention(q, k, v, offsets)
        for a, b in ((0, 130), (130, 830), (830, 895)):
            alone = pkg.ops().prompt_attention(q[a:b], k[a:b], v[a:b], torch.tensor([0, b - a], dtype=I32, device=dev))
            assert torch.equal(alone, packed[a:b])
    finally:
        lib.prompt_attention_tune(0, 0)


def test_captured_offsets_follow_and_streams(pkg, dev):
    """Two graphs of padded batches on two streams at once, their prompts changed between replays."""
    g = torch.Generator().manual_seed(8)
    ops, sets = pkg.ops(), []
    for _ in range(2):
        args = [t.to(dev) for t in prompts.inputs(g, BF, [100, 200, 50], 8, 2, 128, behind=30)]
        args[:3] = [t.nan_to_num(0.5) for t in args[:3]]
        ops.prompt_attention(*args)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.prompt_attention(*args)
        sets.append((args, graph, out, torch.cuda.Stream()))
    for lens in ([100, 200, 50], [10, 0, 370], [380, 0, 0], [1, 1, 1]):
        for args, *_ in sets:
            args[3].copy_(torch.tensor([0] + lens).cumsum(0))
        torch.cuda.synchronize()
        for _, graph, _, stream in sets:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for args, _, out, _ in sets:
            assert torch.equal(out, ops.prompt_attention(*args))
            assert not out[sum(lens):].any()


def test_far_rows(pkg, dev):
    """Keys and queries behind 2^32 bytes: the last prompt of a long packed batch, and one whose own keys are that far
    apart."""
    g = torch.Generator().manual_seed(9)
    rows, hq, d = (1 << 31) // (6 * 128) + 2000, 4, 128
    packed = torch.zeros(rows, 6, d, dtype=BF, device=dev)
    q, k, v, offsets = prompts.inputs(g, BF, [300], hq, 1, d)
    packed[-300:] = torch.cat((q, k, v), 1).to(dev)
    parts = packed.split([4, 1, 1], 1)
    lens = [5000] * ((rows - 300) // 5000)
    lens += [rows - 300 - sum(lens), 300]
    got = pkg.ops().prompt_attention(*parts, torch.tensor([0] + lens, device=dev).cumsum(0).int())
    want, extra = prompts.attention64(q, k, v, offsets)
    assert ref.near(got[-300:].cpu(), want, extra) and not got[:-300].any()
    del packed, parts, got
    far = torch.zeros(300, 1 << 23, dtype=BF, device=dev)[:, :768].unflatten(1, (6, 128))
    far.copy_(torch.cat((q, k, v), 1))
    got = pkg.ops().prompt_attention(*far.split([4, 1, 1], 1), offsets.to(dev))
    assert ref.near(got.cpu(), want, extra)


def test_refusals(pkg, dev):
    g = torch.Generator().manual_seed(9)
    q, k, v, offsets = [t.to(dev) for t in prompts.inputs(g, BF, [3, 4], 4, 2, 64)]
    for a in ((q.float(), k, v, offsets), (q[..., :48], k[..., :48], v[..., :48], offsets), (q[:, :3], k, v, offsets),
              (q, k[:6], v, offsets), (q, k, v[:, :1], offsets), (q, k.half(), v, offsets), (q[0], k, v, offsets),
              (q, k, v, offsets.long()), (q, k, v, offsets[:0]), (q, k, v, offsets.cpu()), (q, k, v, offsets[None]),
              (q, k, v, offsets, 0.0), (q, k, v, offsets, float("nan"))):
        with pytest.raises(ValueError):
            pkg.prompt_attention(*a)
        with pytest.raises(RuntimeError):
            pkg.ops().prompt_attention(*a)
