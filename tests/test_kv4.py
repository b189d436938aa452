"""The cache in 4 bits and attention over it on the CPU: the kernels' own source under the HIP emulation against the
definition in 64 bits, the libraries' exports and argument codes, and the wrappers' refusals."""

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import _emu
import _kv4 as kv4
import _launches
import _serving as ref
from test_abi import declared, exported

BF, FP, I32 = torch.bfloat16, torch.float16, torch.int32
LL, P, I = ctypes.c_longlong, ctypes.c_void_p, ctypes.c_int


def bind(lib):
    if hasattr(lib, "kv4_append_launch"):
        lib.kv4_append_launch.argtypes = [P] * 8 + [LL] * 2 + [I] * 4 + [P]
        lib.kv4_read_launch.argtypes = [P] * 7 + [LL] * 2 + [I] * 4 + [P]
    else:
        lib.kv4_attention_work.argtypes, lib.kv4_attention_work.restype = [LL] * 2 + [I] * 3 + [LL] * 2, LL
        lib.kv4_attention_launch.argtypes = [P] * 9 + [LL, P] + [LL] * 3 + [I] * 3 + [LL] * 2 + [ctypes.c_float, I, P]
    return lib


def emulated(d, source):
    """The kernel source with the emulation's matrix.hpp and fp4.hpp in the place of csrc's."""
    kern = _emu.kernel_source(d, source)
    for name in ("matrix.hpp", "fp4.hpp"):
        shutil.copy(os.path.join(_emu.EMU, name), os.path.join(str(d), name))
    out, clang = os.path.join(str(d), "libemu.so"), _emu._clang()
    if clang is None:
        pytest.skip("clang++ (for the kernels' vector extensions on the host) is missing")
    proc = subprocess.run([clang, "-std=c++17", "-O1", "-fPIC", "-shared", "-U_FORTIFY_SOURCE", "-D_FORTIFY_SOURCE=0",
                           "-fno-strict-aliasing", "-w", "-pthread", "-I", _emu.EMU, "-I", str(d), kern, "-o", out],
                          capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-4000:]
    lib = bind(ctypes.CDLL(out))
    lib.emu_guarded.argtypes, lib.emu_guarded.restype = [ctypes.c_size_t], P
    return lib


@pytest.fixture(scope="module")
def cache_lib(tmp_path_factory):
    return emulated(tmp_path_factory.mktemp("kv4_cache"), "kv4_cache.hip")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    return emulated(tmp_path_factory.mktemp("kv4_attention"), "kv4_attention.hip")


def guarded(lib, t):
    """t copied between pages that cannot be touched."""
    t = t.contiguous()
    n = t.numel() * t.element_size()
    if not n:
        return t
    p = lib.emu_guarded(n)
    ctypes.memmove(p, t.data_ptr(), n)
    return torch.frombuffer((ctypes.c_char * n).from_address(p), dtype=t.dtype).view(t.shape)


def new_cache(pages, hk, block, d):
    return [torch.full((pages, hk, block, n), 17, dtype=torch.uint8) for n in (d // 2, d // 32) * 2]


@pytest.mark.parametrize("tokens,hk,d,block", [(1, 1, 64, 1), (9, 2, 64, 24), (17, 1, 96, 16), (40, 3, 128, 8),
                                               (33, 2, 192, 32), (16, 1, 256, 128)], ids=str)
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_append_and_read(cache_lib, tokens, hk, d, block, dtype):
    g = torch.Generator().manual_seed(d + tokens)
    k, v = kv4.rows(g, dtype, tokens, hk, d), kv4.rows(g, dtype, tokens, hk, d)
    if tokens > 6:
        k[6, 0, 5], v[6, hk - 1, 40] = float("nan"), float("-inf")
    pages = -(-tokens // block) + 1
    slots = torch.randperm(pages * block, generator=g)[:tokens]
    if tokens > 2:
        slots[1], slots[2] = -1, pages * block
    cache = [guarded(cache_lib, t) for t in new_cache(pages, hk, block, d)]
    dt = 1 if dtype == BF else 2
    sizes = tokens, pages, hk, d, block, dt, None
    ptrs = [guarded(cache_lib, t) for t in (k, v, slots)]
    call = lambda: cache_lib.kv4_append_launch(ptrs[0].data_ptr(), ptrs[1].data_ptr(), *(t.data_ptr() for t in cache),
                                               ptrs[2].data_ptr(), None, *sizes)
    assert call() == 0
    want = new_cache(pages, hk, block, d)
    for x, i in ((k, 0), (v, 2)):
        codes, scales = kv4.encode(x)
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < pages * block:
                want[i][s // block, :, s % block], want[i + 1][s // block, :, s % block] = codes[t], scales[t]
    for a, b in zip(cache, want):
        assert torch.equal(a, b)
    out = [guarded(cache_lib, torch.zeros(tokens, hk, d, dtype=dtype)) for _ in range(2)]
    assert cache_lib.kv4_read_launch(*(t.data_ptr() for t in cache), ptrs[2].data_ptr(), out[0].data_ptr(),
                                     out[1].data_ptr(), *sizes) == 0
    inside = (slots >= 0) & (slots < pages * block)
    for got, i in zip(out, (0, 2)):
        values = kv4.flat(kv4.decode(*cache[i:i + 2]))
        assert torch.equal(got[inside].double().nan_to_num(7e5), values[slots[inside]].nan_to_num(7e5))
        assert not got[~inside].any()


def test_a_group_is_off_by_a_fifth_at_most():
    g = torch.Generator().manual_seed(3)
    for dtype in (BF, FP):
        x = kv4.rows(g, dtype, 200, 1, 64)
        x[3] = 1.0
        x[2] = 2.0
        values = kv4.decode(*kv4.encode(x))
        off = (values - x.double()).abs().unflatten(-1, (-1, 32))
        top = x.double().abs().unflatten(-1, (-1, 32)).amax(-1)
        assert (off.amax(-1) <= torch.where(top < 2.0 ** -124, 2.0 ** -127, top / 5)).all()  # there 2^-126 is the scale


def test_append_strided(cache_lib):
    g = torch.Generator().manual_seed(4)
    qkv = kv4.rows(g, BF, 20, 6, 64)
    k, v = qkv[:, 2:4], qkv[:, 4:6]
    cache = [guarded(cache_lib, t) for t in new_cache(3, 2, 8, 64)]
    slots = torch.arange(20)
    assert cache_lib.kv4_append_launch(k.data_ptr(), v.data_ptr(), *(t.data_ptr() for t in cache), slots.data_ptr(),
                                       (LL * 4)(384, 64, 384, 64), 20, 3, 2, 64, 8, 1, None) == 0
    for x, i in ((k, 0), (v, 2)):
        codes, scales = kv4.encode(x)
        assert torch.equal(kv4.flat(cache[i])[:20], codes) and torch.equal(kv4.flat(cache[i + 1])[:20], scales)


def run(lib, q, cache, tables, lens, scale=None, strides=None):
    batch, seq, hq, d = q.shape
    pages, hk, block, _ = cache[0].shape
    sizes = hq, hk, d, tables.shape[1], block
    n = lib.kv4_attention_work(batch, seq, *sizes)
    assert n >= 0
    on = [q if strides else guarded(lib, q)] + [guarded(lib, t) for t in (*cache, tables, lens)]
    out = guarded(lib, torch.full((batch, seq, hq, d), 9.0, dtype=q.dtype))
    work = guarded(lib, torch.full((n // 4,), float("nan"))) if n else None
    ptrs = [t.data_ptr() if t.numel() else None for t in on] + [out.data_ptr(), work.data_ptr() if n else None]
    assert lib.kv4_attention_launch(*ptrs, n, strides and (LL * 3)(*strides), batch, seq, pages, *sizes,
                                    d ** -0.5 if scale is None else scale, 1 if q.dtype == BF else 2, None) == 0
    return out


def check(lib, q, cache, tables, lens, scale=None, **kw):
    got = run(lib, q, cache, tables, lens, scale, **kw)
    want, extra = kv4.attention64(q, cache, tables, lens, scale)
    assert not got.isnan().any()
    assert ref.near(got, want, extra), ((got.double() - want).abs() - extra).max()
    return got


CASES = [  # batch, seq, q heads, kv heads, head size, page, lengths
    (1, 1, 4, 1, 128, 16, [100]), (2, 1, 4, 2, 64, 1, [40, 1]), (3, 1, 3, 3, 64, 8, [0, 33, 700]),
    (2, 3, 7, 1, 96, 32, [3, 650]), (1, 9, 8, 1, 128, 24, [600]), (1, 2, 2, 1, 256, 16, [530]),
    (1, 5, 8, 2, 192, 128, [130]), (2, 12, 4, 2, 64, 16, [5, 77])]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_formula(lib, case, dtype):
    batch, seq, hq, hk, d, block, lens = case
    g = torch.Generator().manual_seed(d + seq)
    check(lib, *kv4.inputs(g, dtype, batch, seq, hq, hk, d, block, lens))


@pytest.mark.parametrize("runs", [-1, 1, 2, 5, 17])
@pytest.mark.parametrize("tiles", [1, 2])
def test_every_cut(lib, runs, tiles):
    g = torch.Generator().manual_seed(1)
    args = kv4.inputs(g, BF, 4, 3, 12, 2, 64, 16, [600, 0, 2, 300])
    lib.kv4_attention_tune(0, runs), lib.kv4_attention_tune(1, tiles)
    try:
        check(lib, *args)
    finally:
        lib.kv4_attention_tune(0, 0), lib.kv4_attention_tune(1, 0)


def test_many_sequences(lib):
    """More sequences than a wave has lanes, most of them idle or short."""
    g = torch.Generator().manual_seed(9)
    lens = [(37 * i) % 90 if i % 3 else 0 for i in range(150)]
    lens[70] = 520
    for runs in (-1, 3, 40):
        lib.kv4_attention_tune(0, runs)
        try:
            check(lib, *kv4.inputs(g, BF, 150, 1, 2, 1, 64, 16, lens))
        finally:
            lib.kv4_attention_tune(0, 0)


def test_lengths_and_bad_pages(lib):
    g = torch.Generator().manual_seed(2)
    q, cache, tables, lens = kv4.inputs(g, BF, 3, 2, 4, 2, 64, 16, [400, 700, 90])
    for own in ([1, 2, 3], [0, 0, 0], [-1, 1 << 30, 30]):
        now = torch.tensor(own, dtype=I32)
        clean = [t.clone() for t in cache]
        if max(own) > 700:
            for i in (1, 3):
                clean[i][clean[i] == 255] = 120
        check(lib, q, clean, tables, now)
    tables[0, 2], tables[1, 1], tables[2, 0] = -2 ** 31, 2 ** 31 - 1, cache[0].shape[0]
    check(lib, q, cache, tables, lens, scale=0.2)
    none = run(lib, q, [t[:0] for t in cache], tables, lens)
    assert not none.any()


@pytest.mark.parametrize("block", [8, 32])
def test_growing_scores(lib, block):
    """Scores that grow without bound along a context, so that no early one is a point for the later; a first slice that is
    absent altogether."""
    g = torch.Generator().manual_seed(12)
    q, cache, tables, lens = kv4.inputs(g, BF, 2, 2, 4, 2, 64, block, [500, 300], peak=1.0, power=(127, 128))
    for b, n in enumerate(lens.tolist()):
        t = torch.arange(n)
        cache[1][tables[b].long()[t // block], :, t % block] = (118 + t // 40).to(torch.uint8)[:, None, None]
    check(lib, q, cache, tables, lens)
    tables[0, :32 // block], tables[1, 1] = -1, -1
    check(lib, q, cache, tables, lens)


@pytest.mark.parametrize("d", [64, 96, 256])
def test_nan_reaches_only_the_queries_that_see_it(lib, d):
    g, seq = torch.Generator().manual_seed(5), 6
    q, cache, tables, lens = kv4.inputs(g, BF, 2, seq, 4, 2, d, 8, [45, 600])
    clean = [t.clone() for t in cache]
    reached = torch.zeros(q.shape, dtype=torch.bool)
    for b, t, group in ((0, 41, 0), (0, 44, d // 32 - 1), (1, 596, 1), (1, 597, 0)):
        cache[3][tables[b, t // 8], 1, t % 8, group] = 255
        clean[3][tables[b, t // 8], 1, t % 8, group] = 120
        reached[b, t - int(lens[b]) + seq:, 2:, 32 * group:32 * group + 32] = True
    want, extra = kv4.attention64(q, clean, tables, lens)
    # the values that are NaN are the only difference, in the elements that they reach
    got = run(lib, q, cache, tables, lens)
    assert got[reached].isnan().all() and ref.near(got[~reached], want[~reached], extra[~reached])
    cache[1][tables[0, 42 // 8], 0, 42 % 8, 0] = 254  # a key: all of the queries' elements
    got = run(lib, q, cache, tables, lens)
    assert got[0, 42 - 45 + seq:, :2].isnan().all()
    reached[0, 42 - 45 + seq:, :2] = True
    assert ref.near(got[~reached], want[~reached], extra[~reached])


def test_queries_of_any_size(lib):
    """Zeros, small and large queries, NaN in one of them."""
    g = torch.Generator().manual_seed(6)
    q, cache, tables, lens = kv4.inputs(g, BF, 1, 4, 4, 1, 64, 16, [70])
    q[0, 0, 0], q[0, 0, 1], q[0, 0, 2] = 0.0, q[0, 0, 1] * 1e-30, q[0, 0, 2] * 2.0 ** -60
    q[0, 0, 3, :32] *= 2.0 ** -9
    want = check(lib, q, cache, tables, lens)
    for bad in (float("nan"), float("inf")):
        q[0, 2, 1, 5] = bad
        got = run(lib, q, cache, tables, lens)
        assert got[0, 2, 1].isnan().all()
        got[0, 2, 1] = want[0, 2, 1]
        assert torch.equal(got, want)


def test_strided_queries(lib):
    g = torch.Generator().manual_seed(7)
    q, cache, tables, lens = kv4.inputs(g, BF, 2, 3, 4, 2, 64, 16, [70, 20])
    packed = torch.full((2, 3, 8, 64), float("nan"), dtype=BF)
    packed[:, :, 2:6] = q
    view = packed[:, :, 2:6]
    assert torch.equal(run(lib, view, cache, tables, lens, strides=view.stride()[:3]), run(lib, q, cache, tables, lens))


@pytest.mark.parametrize("op", ["kv4_cache", "kv4_attention"])
def test_exports(pkg, op):
    names = declared(op)
    assert {s for s in exported(pkg.lib_path(op)) if not s.startswith("_")} == set(names) and len(names) >= 2


def test_cache_codes(pkg):
    lib = bind(ctypes.CDLL(pkg.lib_path("kv4_cache")))
    good = dict(k=16, v=16, kc=16, ks=1, vc=16, vs=1, slots=8, strides=None, tokens=4, pages=2, heads=2, dim=64,
                block=16, dtype=1)

    def append(**kw):
        x = {**good, **kw}
        return lib.kv4_append_launch(*list(x.values())[:7], x["strides"], *list(x.values())[8:], None)

    def read(**kw):
        x = {**good, **kw}
        return lib.kv4_read_launch(x["kc"], x["ks"], x["vc"], x["vs"], x["slots"], x["k"], x["v"],
                                   *list(x.values())[8:], None)

    assert append(tokens=0) == 0 and read(tokens=0) == 0 and append(tokens=-3) == 0
    for bad in (dict(k=None), dict(v=None), dict(k=8), dict(kc=None), dict(ks=None), dict(vc=18), dict(slots=None),
                dict(heads=0), dict(heads=65537), dict(dim=80), dict(dim=0), dict(block=0), dict(dtype=0), dict(dtype=3),
                dict(pages=-1), dict(pages=1 << 27), dict(tokens=1 << 34)):
        assert append(**bad) == -1, bad
        assert read(**bad) == -1, bad
    for strides in ((63, 64, 64, 64), (128, 64, 128, 12)):
        assert append(strides=(LL * 4)(*strides)) == -1


def test_attention_codes(pkg):
    lib = bind(ctypes.CDLL(pkg.lib_path("kv4_attention")))
    good = dict(q=16, kc=16, ks=1, vc=16, vs=1, tables=4, lens=4, out=16, work=None, bytes=0, strides=None, batch=2, seq=1,
                pages=8, hq=4, hk=2, dim=64, blocks=4, block=16, scale=0.1, dtype=1)

    def launch(**kw):
        return lib.kv4_attention_launch(*{**good, **kw}.values(), None)

    assert launch(batch=0) == 0 and launch(seq=0) == 0
    for bad in (dict(q=None), dict(q=8), dict(out=None), dict(out=24), dict(lens=None), dict(tables=None), dict(kc=None),
                dict(vs=None), dict(vc=8), dict(hq=5), dict(hk=0), dict(hq=65538), dict(dim=80), dict(block=0),
                dict(block=(1 << 30) + 1), dict(hq=9, hk=9, block=1 << 28, pages=1, blocks=1), dict(blocks=1 << 27),
                dict(pages=1 << 28), dict(pages=-1), dict(scale=0.0), dict(scale=float("nan")), dict(scale=1e31), dict(dtype=0), dict(batch=1 << 29),
                dict(strides=(LL * 3)(256, 256, 63)), dict(strides=(LL * 3)(100, 256, 64)), dict(blocks=9999),
                dict(blocks=9999, work=8, bytes=1 << 30), dict(blocks=9999, work=16, bytes=100)):
        assert launch(**bad) == -1, bad
    assert lib.kv4_attention_work(0, 1, 4, 2, 64, 4, 16) == 0 and lib.kv4_attention_work(2, 1, 4, 2, 64, 4, 16) == 0
    assert lib.kv4_attention_work(2, 1, 5, 2, 64, 4, 16) == -1 and lib.kv4_attention_work(2, 1, 4, 2, 64, 9999, 16) > 0
    assert lib.kv4_attention_tune(99, 1) == -1


def test_launches(tmp_path_factory):
    """Large calls stay within what a launch may have."""
    rec = bind(_launches.build(tmp_path_factory.mktemp("kv4_launches"), "kv4_cache.hip"))
    for tokens, heads, dim in ((1, 1, 64), (1 << 21, 8, 256), (1 << 30, 8, 64), (1 << 17, 65536, 64)):
        code, made = _launches.launches(rec, lambda: rec.kv4_append_launch(16, 16, 16, 1, 16, 1, 8, None, tokens, 4, heads,
                                                                           dim, 16, 1, None))
        assert code == 0 and len(made) == 1 and all(_launches.accepted(m) for m in made)
        assert made[0][0] * made[0][1] >= -(-tokens // 32) * 2 * heads  # 32 tokens of a head each
    rec = bind(_launches.build(tmp_path_factory.mktemp("kv4_launches"), "kv4_attention.hip"))
    for batch, seq, hq, hk, blocks in ((1, 1, 8, 8, 1), (1 << 24, 1, 8, 8, 1), (1 << 20, 1, 32, 8, 1 << 20),
                                       (1, 1 << 20, 64, 1, 1 << 16)):
        n = rec.kv4_attention_work(batch, seq, hq, hk, 64, blocks, 16)
        assert n >= 0
        code, made = _launches.launches(rec, lambda: rec.kv4_attention_launch(
            16, 16, 1, 16, 1, 4, 4, 16, 16, n, None, batch, seq, 8, hq, hk, 64, blocks, 16, 0.1, 1, None))
        assert code == 0 and len(made) == (2 if n else 1) and all(_launches.accepted(m) for m in made)


def test_wrappers_refuse(pkg):
    g = torch.Generator().manual_seed(8)
    q, cache, tables, lens = kv4.inputs(g, BF, 2, 1, 4, 2, 64, 16, [30, 20])
    k, slots = torch.zeros(3, 2, 64, dtype=BF), torch.arange(3)
    with pytest.raises(ValueError):  # no CPU path
        pkg.kv4_append(k, k, *cache, slots)
    with pytest.raises(ValueError):
        pkg.kv4_read(*cache, slots)
    with pytest.raises(ValueError):
        pkg.kv4_attention(q, *cache, tables, lens)
    ops = pkg.ops()
    for call in (lambda: ops.kv4_append_(k, k, *cache, slots), lambda: ops.kv4_read(*cache, slots, BF),
                 lambda: ops.kv4_attention(q, *cache, tables, lens)):
        with pytest.raises((NotImplementedError, RuntimeError)):
            call()


def test_meta(pkg):
    ops, meta = pkg.ops(), dict(device="meta")
    cache = [torch.empty(4, 2, 16, n, dtype=torch.uint8, **meta) for n in (64, 4, 64, 4)]
    k, v = ops.kv4_read(*cache, torch.empty(7, dtype=torch.int64, **meta), FP)
    assert k.shape == v.shape == (7, 2, 128) and k.dtype == FP
    q = torch.empty(3, 2, 8, 128, dtype=BF, **meta)
    out = ops.kv4_attention(q, *cache, torch.empty(3, 5, dtype=I32, **meta), torch.empty(3, dtype=I32, **meta))
    assert out.shape == q.shape and out.dtype == BF
    kv = torch.empty(7, 2, 128, dtype=BF, **meta)
    ops.kv4_append_(kv, kv, *cache, torch.empty(7, dtype=torch.int64, **meta))
    schema = ops.kv4_append_.default._schema
    assert [a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write] == [
        "k_codes", "k_scales", "v_codes", "v_scales"]
