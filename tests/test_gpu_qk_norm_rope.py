"""qk_norm_rope on the GPU, through the package's functions and the torch operators, against the formula in 64 bits."""

import pytest
import torch

import _serving as ref

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def inputs(dev, seed, dtype, batch, seq, hq, hk, d, rotary, weights=True, packed=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    one = lambda *s: (torch.randn(s, generator=g, device=dev) * 1.5).to(dtype)  # noqa: E731
    if packed:
        q, k, v = one(batch, seq, hq + 2 * hk, d).split([hq, hk, hk], 2)
    else:
        q, k, v = one(batch, seq, hq, d), one(batch, seq, hk, d), one(batch, seq, hk, d)
    ids = torch.randint(0, 1 << 20, (batch, seq), generator=g, device=dev)
    qw, kw = ((torch.rand(d, generator=g, device=dev) + 0.5).to(dtype) for _ in range(2)) if weights else (None, None)
    return q, k, v, ids, ref.inv_freq_of(rotary).to(dev), qw, kw


def right(got, x, ids, inv, w):
    return ref.near(got, ref.norm_rope64(x, ids, inv, w), ref.norm_rope_error(x, w))


SHAPES = [(1, 1, 32, 8, 128, 128), (64, 1, 32, 8, 128, 128), (3, 701, 14, 2, 64, 32), (2, 129, 16, 4, 256, 256),
          (5, 77, 7, 1, 80, 80), (1, 1000, 3, 3, 96, 48), (2, 63, 4, 4, 192, 192), (2, 33, 5, 2, 50, 50),
          (1, 17, 2, 1, 512, 256), (4, 1024, 32, 8, 128, 128), (1, 3, 200, 100, 64, 64),
          (3, 1399, 1, 1, 64, 64), (1, 4100, 2, 1, 128, 64), (2, 2051, 1, 1, 80, 40), (1, 4099, 1, 1, 256, 256)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("weights,packed", [(True, True), (False, False)])
def test_formula(pkg, dev, shape, dtype, weights, packed):
    q, k, v, ids, inv, qw, kw = inputs(dev, 1, dtype, *shape, weights=weights, packed=packed)
    outs = [pkg.qk_norm_rope(q, k, ids, inv, qw, kw), pkg.ops().qk_norm_rope(q, k, ids, inv, qw, kw)]
    for qo, ko in outs:
        assert right(qo, q, ids, inv, qw) and right(ko, k, ids, inv, kw)
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_cache(pkg, dev, shape):
    q, k, v, ids, inv, qw, kw = inputs(dev, 2, BF, *shape)
    batch, seq, hq, hk, d, _ = shape
    slots = batch * seq + 5
    mapping = torch.randperm(slots, device=dev)[:batch * seq].view(batch, seq).clone()
    mapping[0, -1] = -1
    if seq > 2:
        mapping[0, 0], mapping[0, 1] = slots, 1 << 40  # outside the cache: not written
    written = (mapping >= 0) & (mapping < slots)
    for call in (pkg.qk_norm_rope_kv, pkg.ops().qk_norm_rope_kv_):
        kc, vc = torch.full((slots, hk, d), 3.0, dtype=BF, device=dev), torch.full((slots, hk, d), 5.0, dtype=BF, device=dev)
        qo = call(q, k, v, ids, inv, kc, vc, mapping, qw, kw)
        assert right(qo, q, ids, inv, qw)
        at = mapping[written]
        assert ref.near(kc[at], ref.norm_rope64(k, ids, inv, kw)[written], ref.norm_rope_error(k, kw)[written])
        assert torch.equal(vc[at], v[written])
        others = torch.ones(slots, dtype=torch.bool, device=dev)
        others[at] = False
        assert (kc[others] == 3).all() and (vc[others] == 5).all()


def test_in_place_and_strided(pkg, dev):
    q, k, v, ids, inv, qw, kw = inputs(dev, 3, BF, 2, 9, 6, 2, 128, 128)
    want = pkg.qk_norm_rope(q, k, ids, inv, qw, kw)
    kept = v.clone()
    qo, ko = pkg.qk_norm_rope(q, k, ids, inv, qw, kw, inplace=True)
    assert qo is q and ko is k and torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, kept)
    # [B, H, S, D] tensors seen as [B, S, H, D], and a last dimension that is not contiguous
    q, k, v, ids, inv, qw, kw = inputs(dev, 4, BF, 2, 9, 6, 2, 128, 128, packed=False)
    want = pkg.qk_norm_rope(q, k, ids, inv, qw, kw)
    for turn in (lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
                 lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)):
        got = pkg.qk_norm_rope(turn(q), turn(k), ids, inv, qw, kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        got = pkg.ops().qk_norm_rope(turn(q), turn(k), ids, inv, qw, kw)
        assert torch.equal(got[0], want[0]) and got[0].is_contiguous()
    with pytest.raises(ValueError, match="in-place"):
        pkg.qk_norm_rope(q[:, :, :1].expand(2, 9, 6, 128), k, ids, inv, inplace=True)
    with pytest.raises(ValueError, match="one tensor"):
        pkg.qk_norm_rope(q, q, ids, inv, inplace=True)


def test_empty_and_another_stream(pkg, dev):
    q, k, v, ids, inv, qw, kw = inputs(dev, 5, FP, 2, 5, 4, 2, 64, 64)
    qo, ko = pkg.qk_norm_rope(q[:0], k[:0], ids[:0], inv)
    assert qo.shape == (0, 5, 4, 64) and ko.shape == (0, 5, 2, 64)
    want = pkg.qk_norm_rope(q, k, ids, inv, qw, kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = pkg.ops().qk_norm_rope(q, k, ids, inv, qw, kw)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_caches_without_slots_and_shared_memory(pkg, dev):
    q, k, v, ids, inv, qw, kw = inputs(dev, 8, BF, 2, 3, 4, 2, 64, 64)
    mapping = torch.zeros(2, 3, dtype=torch.int64, device=dev)
    none = torch.zeros(0, 2, 64, dtype=BF, device=dev)
    want = pkg.qk_norm_rope(q, k, ids, inv, qw, kw)[0]
    for call in (pkg.qk_norm_rope_kv, pkg.ops().qk_norm_rope_kv_):
        got = call(q, k, v, ids, inv, none, none.clone(), mapping, qw, kw)
        assert torch.equal(got, want)
        both = torch.zeros(9, 2, 64, dtype=BF, device=dev)
        with pytest.raises((ValueError, RuntimeError), match="share memory"):
            call(q, k, v, ids, inv, both[:-1], both[1:], mapping, qw, kw)
        with pytest.raises((ValueError, RuntimeError), match="share memory"):
            call(q, both[:6].view(2, 3, 2, 64), v, ids, inv, both, both.clone(), mapping, qw, kw)
        call(q, k, v, ids, inv, both[:4], both[4:8], mapping, qw, kw)


def test_two_to_the_32_threads(pkg, dev):
    """2^25 tokens of two heads of one element, a wave to each: y = x w / sqrt(x^2 + eps), or x w where eps is most."""
    n = (1 << 25) + 3
    q = (torch.arange(n, device=dev) % 509 - 254).to(BF).view(1, n, 1, 1)
    k = (torch.arange(n, device=dev) % 251 + 1).to(BF).view(1, n, 1, 1)
    ids, inv = torch.zeros(1, n, dtype=torch.int64, device=dev), torch.zeros(0, device=dev)
    qo, ko = pkg.ops().qk_norm_rope(q, k, ids, inv)
    for got, x in ((qo, q), (ko, k)):
        x = x.double()
        want = x / (x * x + ref.EPS).sqrt()  # 0, or 1 - 5e-7 and nearer to 1: one rounding
        assert torch.equal(got.double(), want.to(BF).double())


def test_too_many_heads(pkg, dev):
    q, k = (torch.zeros(1, 1, n, 1, dtype=BF, device=dev) for n in ((1 << 20) + 1, 1))
    ids, inv = torch.zeros(1, 1, dtype=torch.int64, device=dev), torch.zeros(0, device=dev)
    with pytest.raises(ValueError, match="too large"):
        pkg.qk_norm_rope(q, k, ids, inv)
    with pytest.raises(RuntimeError):
        pkg.ops().qk_norm_rope(q, k, ids, inv)


def test_captured(pkg, dev):
    q, k, v, ids, inv, qw, kw = inputs(dev, 6, BF, 4, 1, 8, 2, 128, 128)
    ops, slots = pkg.ops(), 16
    kc, vc = torch.zeros(slots, 2, 128, dtype=BF, device=dev), torch.zeros(slots, 2, 128, dtype=BF, device=dev)
    mapping = torch.tensor([[3], [1], [-1], [9]], device=dev)
    ops.qk_norm_rope_kv_(q, k, v, ids, inv, kc, vc, mapping, qw, kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo = ops.qk_norm_rope_kv_(q, k, v, ids, inv, kc, vc, mapping, qw, kw)
    for seed in (7, 8, 9):
        fresh = inputs(dev, seed, BF, 4, 1, 8, 2, 128, 128)
        for t, f in zip((q, k, v, ids), fresh):
            t.copy_(f)
        kc.zero_(), vc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = qo.clone(), kc.clone(), vc.clone()
        kc.zero_(), vc.zero_()
        want = ops.qk_norm_rope_kv_(q, k, v, ids, inv, kc, vc, mapping, qw, kw)
        assert torch.equal(got[0], want) and torch.equal(got[1], kc) and torch.equal(got[2], vc)
