"""prompt_attention on the CPU: the kernels' own source under the HIP emulation against the formula in 64 bits, the
library's exports and argument codes, and the wrapper's refusals."""

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import _emu
import _launches
import _prompts as prompts
import _serving as ref
from test_abi import declared, exported

BF, FP, I32 = torch.bfloat16, torch.float16, torch.int32
LL, P, I = ctypes.c_longlong, ctypes.c_void_p, ctypes.c_int


def bind(lib):
    lib.prompt_attention_launch.argtypes = [P] * 6 + [LL] * 2 + [I] * 3 + [ctypes.c_float, I, P]
    return lib


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("prompts")
    kern = _emu.kernel_source(d, "prompt_attention.hip")
    shutil.copy(os.path.join(_emu.EMU, "matrix.hpp"), os.path.join(str(d), "matrix.hpp"))
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


def guarded(lib, t):
    """t copied between pages that cannot be touched."""
    t = t.contiguous()
    n = t.numel() * t.element_size()
    p = lib.emu_guarded(n)
    ctypes.memmove(p, t.data_ptr(), n)
    return torch.frombuffer((ctypes.c_char * n).from_address(p), dtype=t.dtype).view(t.shape)


def run(lib, q, k, v, offsets, scale=None, strides=None):
    tokens, hq, d = q.shape
    on = [t if strides else guarded(lib, t) for t in (q, k, v)] + [guarded(lib, offsets)]
    out = guarded(lib, torch.full((tokens, hq, d), 9.0, dtype=q.dtype))
    assert lib.prompt_attention_launch(*(t.data_ptr() for t in on), out.data_ptr(), strides and (LL * 6)(*strides), tokens,
                                       offsets.numel() - 1, hq, k.shape[1], d, d ** -0.5 if scale is None else scale,
                                       1 if q.dtype == BF else 2, None) == 0
    return out


def check(lib, q, k, v, offsets, scale=None, **kw):
    got = run(lib, q, k, v, offsets, scale, **kw)
    want, extra = prompts.attention64(q, k, v, offsets, scale)
    assert not got.isnan().any()
    assert ref.near(got, want, extra), ((got.double() - want).abs() - extra).max()
    return got


CASES = [  # lengths, q heads, kv heads, head size
    ([1], 4, 1, 64), ([33], 3, 3, 64), ([5, 0, 70, 1], 4, 2, 128), ([40], 7, 1, 80), ([150, 3], 2, 1, 96),
    ([66, 31], 2, 2, 192), ([40, 65], 4, 1, 256), ([0, 0, 9], 8, 8, 128)]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_formula(lib, case, dtype):
    lens, hq, hk, d = case
    g = torch.Generator().manual_seed(d + len(lens))
    check(lib, *prompts.inputs(g, dtype, lens, hq, hk, d))


@pytest.mark.parametrize("env", [{}, {"EMU_WAVE_AHEAD": "1"}], ids=["in turn", "waves ahead"])
@pytest.mark.parametrize("waves", [4, 8])
@pytest.mark.parametrize("d,length", [(64, 300), (96, 290), (128, 333)], ids=str)
def test_long_prompts(lib, monkeypatch, env, waves, d, length):
    """More than a ring of slices."""
    for name, value in env.items():
        monkeypatch.setenv(name, value)
    g = torch.Generator().manual_seed(length)
    lib.prompt_attention_tune(0, waves)
    try:
        check(lib, *prompts.inputs(g, BF, [length, 20], 2, 1, d))
    finally:
        lib.prompt_attention_tune(0, 0)


def test_many_prompts(lib):
    """More prompts than a wave has lanes, empty ones among them, rows of none around them."""
    g = torch.Generator().manual_seed(3)
    lens = [(5 * i) % 13 if i % 4 else 0 for i in range(150)]
    q, k, v, offsets = prompts.inputs(g, BF, lens, 2, 1, 64, before=7, behind=70)
    got = check(lib, q, k, v, offsets)
    assert not got[:7].any() and not got[-70:].any()


def test_rows_of_no_prompt(lib):
    g = torch.Generator().manual_seed(4)
    q, k, v, offsets = prompts.inputs(g, FP, [9, 4], 3, 3, 80, before=5, behind=40)
    check(lib, q, k, v, offsets)
    for offsets in ([5, 5, 5], [0], [58], [-9, 0, -3]):  # no prompt at all
        assert not run(lib, q, k, v, torch.tensor(offsets, dtype=I32)).any()
    # beyond the rows: cut to them
    q, k, v = (t.nan_to_num(0.25) for t in (q, k, v))
    check(lib, q, k, v, torch.tensor([-3, 20, 1 << 30], dtype=I32))


def test_offsets_in_any_order(lib):
    """Offsets that decrease leave the results open; nothing outside the tensors is touched for them."""
    g = torch.Generator().manual_seed(6)
    q, k, v, _ = prompts.inputs(g, BF, [160], 2, 1, 64)
    for batch in (8, 20, 63, 150):
        run(lib, q, k, v, torch.randint(-9, 170, (batch + 1,), generator=g).int())
        run(lib, q, k, v, torch.arange(160, 0, -1)[:batch + 1].int())


def test_strided_and_scale(lib):
    g = torch.Generator().manual_seed(5)
    q, k, v, offsets = prompts.inputs(g, BF, [20, 50], 4, 2, 64)
    packed = torch.cat((q, k, v), 1)
    parts = packed.split([4, 2, 2], 1)
    got = run(lib, *parts, offsets, scale=0.3, strides=[512, 64] * 3)
    assert torch.equal(got, check(lib, q, k, v, offsets, scale=0.3))


def test_peaked_and_flat_scores(lib):
    g = torch.Generator().manual_seed(6)
    for peak in (20.0, 0.0):
        check(lib, *prompts.inputs(g, FP, [130], 2, 1, 64, peak=peak))


@pytest.mark.parametrize("d,dtype,bad", [(64, FP, "nan"), (80, BF, "-inf"), (128, BF, "nan"), (256, FP, "inf")], ids=str)
def test_bad_values_reach_only_the_queries_that_see_them(lib, d, dtype, bad):
    """A NaN or infinite value of a token is in its query and those behind it, in that one place of the head; also where
    the next prompt begins behind it."""
    g = torch.Generator().manual_seed(7)
    lens = [70, 41, 8]
    q, k, v, offsets = prompts.inputs(g, dtype, lens, 6, 2, d)
    clean, reached = v.clone(), torch.zeros(q.shape, dtype=torch.bool)
    for b, t, c in ((0, 40, 3), (0, 69, d - 1), (1, 0, 17), (2, 5, 0)):
        at, end = int(offsets[b]) + t, int(offsets[b + 1])
        v[at, 1, c], clean[at, 1, c] = float(bad), 0.0
        reached[at:end, 3:, c] = True
    want, extra = prompts.attention64(q, k, clean, offsets)
    got = run(lib, q, k, v, offsets)
    assert not got[reached].isfinite().any()
    assert got[~reached].isfinite().all() and ref.near(got[~reached], want[~reached], extra[~reached])


def test_bad_keys_reach_only_the_queries_that_see_them(lib):
    g = torch.Generator().manual_seed(8)
    q, k, v, offsets = prompts.inputs(g, BF, [70, 41], 4, 2, 64)
    want, extra = prompts.attention64(q, k, v, offsets)
    k[50, 1, 7], k[80, 0, 3] = float("nan"), float("inf")
    reached = torch.zeros(q.shape, dtype=torch.bool)
    reached[50:70, 2:], reached[80:, :2] = True, True
    got = run(lib, q, k, v, offsets)
    assert got[50:70, 2:].isnan().all() and ref.near(got[~reached], want[~reached], extra[~reached])


def test_exports_and_codes(pkg):
    lib = bind(ctypes.CDLL(pkg.lib_path("prompt_attention")))
    names = declared("prompt_attention")
    assert {s for s in exported(pkg.lib_path("prompt_attention")) if not s.startswith("_")} == set(names)
    good = dict(q=16, k=16, v=16, offsets=4, out=16, strides=None, tokens=8, batch=2, hq=4, hk=2, dim=64, scale=0.1, dtype=1)

    def launch(**kw):
        return lib.prompt_attention_launch(*{**good, **kw}.values(), None)

    assert launch(tokens=0) == 0 and launch(tokens=-1) == 0
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(offsets=None), dict(out=None), dict(q=8), dict(k=24),
                dict(v=4), dict(out=8), dict(tokens=1 << 28), dict(batch=-1), dict(batch=1 << 29), dict(hq=3), dict(hk=0),
                dict(hq=65538), dict(dim=72), dict(scale=0.0), dict(scale=float("nan")), dict(dtype=0),
                dict(strides=(LL * 6)(256, 64, 128, 64, 128, 63)), dict(strides=(LL * 6)(256, 64, 1 << 24, 64, 128, 64)),
                dict(strides=(LL * 6)(100, 64, 128, 64, 128, 64))):
        assert launch(**bad) == -1, bad


def test_launches(tmp_path_factory):
    rec = bind(_launches.build(tmp_path_factory.mktemp("prompt_launches"), "prompt_attention.hip"))
    for tokens, batch, hq, hk in ((1, 0, 1, 1), (1 << 29, 1, 1, 1), (1 << 24, 1 << 24, 32, 8), (1 << 13, 1, 65536, 65536),
                                  (16384, 3, 32, 8)):
        code, made = _launches.launches(rec, lambda: rec.prompt_attention_launch(16, 16, 16, 4, 16, None, tokens, batch, hq,
                                                                                 hk, 64, 0.1, 1, None))
        assert code == 0 and len(made) == 1 and all(_launches.accepted(m) for m in made)


def test_wrapper_refuses_and_meta(pkg):
    g = torch.Generator().manual_seed(9)
    args = prompts.inputs(g, BF, [3, 4], 4, 2, 64)
    with pytest.raises(ValueError):  # no CPU path
        pkg.prompt_attention(*args)
    with pytest.raises((NotImplementedError, RuntimeError)):
        pkg.ops().prompt_attention(*args)
    out = pkg.ops().prompt_attention(*(t.to("meta") for t in args))
    assert out.shape == args[0].shape and out.dtype == BF
