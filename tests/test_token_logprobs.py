"""token_logprobs on the CPU: the kernels' own source under the HIP emulation against the formulas in 64 bits, the
library's exports and argument codes, and the wrapper's refusals."""

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import _emu
import _launches
import _logprobs as ref
from test_abi import declared, exported

F32, BF, FP = torch.float32, torch.bfloat16, torch.float16
CODE = {F32: 0, BF: 1, FP: 2}
LL, P, I = ctypes.c_longlong, ctypes.c_void_p, ctypes.c_int


def bind(lib):
    lib.token_logprobs_work.argtypes, lib.token_logprobs_work.restype = [LL] * 2 + [I] * 2, LL
    lib.token_logprobs_launch.argtypes = [P] * 7 + [LL] * 4 + [I] * 2 + [P]
    return lib


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("logprobs")
    kern = _emu.kernel_source(d, "token_logprobs.hip")
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
    if not n:
        return t
    p = lib.emu_guarded(n)
    ctypes.memmove(p, t.data_ptr(), n)
    return torch.frombuffer((ctypes.c_char * n).from_address(p), dtype=t.dtype).view(t.shape)


def run(lib, x, tokens, top, stride=None):
    rows, n = x.shape
    out = [guarded(lib, t) for t in (torch.full((rows,), 9.0), torch.full((rows,), 9.0), torch.full((rows, top), 9.0),
                                     torch.full((rows, top), 9))]
    size = lib.token_logprobs_work(rows, n, top, CODE[x.dtype])
    assert size >= 0
    work = guarded(lib, torch.full((size // 8,), float("nan"), dtype=torch.float64)) if size else None
    on, t = x if stride else guarded(lib, x), guarded(lib, tokens)
    assert lib.token_logprobs_launch(on.data_ptr(), t.data_ptr(), *(o.data_ptr() if o.numel() else None for o in out),
                                     work.data_ptr() if size else None, size, stride or n, rows, n, top,
                                     CODE[x.dtype], None) == 0
    return out


def check(lib, x, tokens, top, **kw):
    got, want = run(lib, x, tokens, top, **kw), ref.logprobs64(x, tokens, top)
    assert torch.equal(got[3], want[3])
    assert ref.near(got[:3], want[:3])
    return got


@pytest.mark.parametrize("rows,n,top", [(1, 1, 1), (2, 7, 7), (3, 8, 0), (2, 63, 5), (2, 2049, 20), (1, 9000, 64),
                                        (1, 33001, 3)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF, FP], ids=["fp32", "bf16", "fp16"])
def test_formula(lib, rows, n, top, dtype):
    g = torch.Generator().manual_seed(n)
    check(lib, *ref.logits(g, rows, n, dtype), top)


@pytest.mark.parametrize("n,top,parts", [(200, 20, 0), (2500, 64, 1), (2500, 5, 3), (20, 20, 0), (5000, 64, 20)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF, FP], ids=["fp32", "bf16", "fp16"])
def test_edge_rows(lib, n, top, parts, dtype):
    g = torch.Generator().manual_seed(n)
    lib.token_logprobs_tune(0, parts)
    try:
        check(lib, *ref.edge_rows(g, n, dtype), top)
    finally:
        lib.token_logprobs_tune(0, 0)


def test_lists_under_pressure(lib):
    """Trips that each beat all before, values that come up again, the largest at the end."""
    g, n = torch.Generator().manual_seed(5), 40000
    rows = [torch.arange(n) // 1024 * 1.0, torch.arange(n) % 7 * 1.0, (torch.randn(n, generator=g) * 3).round(),
            torch.randn(n, generator=g) + torch.arange(n) / 8192]
    x = torch.stack(rows)
    for top in (1, 20, 64):
        check(lib, x.to(BF), torch.tensor([0, 39999, 17, 5]), top)


def test_zeros_of_both_signs(lib):
    """+0 comes before -0, also where a list is full of the latter."""
    n = 40000
    x = torch.zeros(3, n).neg_()
    x[0, 30000::50], x[1, ::50], x[2, -1] = 0.0, 0.0, 0.0
    for dtype in (BF, F32):
        check(lib, x.to(dtype), torch.tensor([0, 50, n - 1]), 20)


def test_strided_and_unaligned_rows(lib):
    g = torch.Generator().manual_seed(6)
    whole = torch.randn(4, 1003, generator=g).to(BF)
    tokens = torch.tensor([0, 5, 996, 7])
    view = whole[:, 3:1000]
    got = run(lib, view, tokens, 4, stride=1003)
    want = run(lib, view.contiguous(), tokens, 4)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_exports_and_codes(pkg):
    lib = bind(ctypes.CDLL(pkg.lib_path("token_logprobs")))
    names = declared("token_logprobs")
    assert {s for s in exported(pkg.lib_path("token_logprobs")) if not s.startswith("_")} == set(names)
    good = dict(x=16, tokens=8, lp=4, h=4, tlp=4, ti=8, work=8, bytes=1 << 40, stride=100, rows=2, n=100, top=3, dtype=1)

    def launch(**kw):
        return lib.token_logprobs_launch(*{**good, **kw}.values(), None)

    assert launch(rows=0) == 0 and launch(rows=-1) == 0
    for bad in (dict(x=None), dict(x=17), dict(x=18, dtype=0), dict(tokens=None), dict(lp=None), dict(h=None),
                dict(tlp=None), dict(ti=None), dict(n=0), dict(n=(1 << 28) + 1), dict(top=-1), dict(top=65),
                dict(top=101), dict(dtype=3), dict(rows=(1 << 31) + 1), dict(n=1 << 20, work=None),
                dict(n=1 << 20, work=4), dict(n=1 << 20, bytes=8)):
        assert launch(**bad) == -1, bad
    assert lib.token_logprobs_work(0, 100, 3, 1) == 0 and lib.token_logprobs_work(5, 100, 200, 1) == -1
    assert lib.token_logprobs_work(1, 1 << 20, 3, 1) > 0


def test_launches(tmp_path_factory):
    rec = bind(_launches.build(tmp_path_factory.mktemp("logprobs_launches"), "token_logprobs.hip"))
    for rows, n in ((1, 1), (1, 1 << 28), (1 << 31, 1000), (1 << 30, 1 << 28), (100, 262144)):
        size = rec.token_logprobs_work(rows, n, 1, 1)
        code, made = _launches.launches(rec, lambda: rec.token_logprobs_launch(16, 8, 4, 4, 4, 8, 8, size, n, rows, n, 1, 1,
                                                                               None))
        assert code == 0 and len(made) == (2 if size else 1) and all(_launches.accepted(m) for m in made)


def test_wrapper_refuses_and_meta(pkg):
    x, tokens = torch.zeros(3, 50), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError):  # no CPU path
        pkg.token_logprobs(x, tokens)
    with pytest.raises((NotImplementedError, RuntimeError)):
        pkg.ops().token_logprobs(x, tokens, 3)
    out = pkg.ops().token_logprobs(x.to("meta"), tokens.to("meta"), 7)
    assert [tuple(t.shape) for t in out] == [(3,), (3,), (3, 7), (3, 7)] and out[3].dtype == torch.int64
