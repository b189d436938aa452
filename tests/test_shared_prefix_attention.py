"""shared_prefix_attention on the CPU: the kernels' own source under the HIP emulation against the formula in 64 bits
(head sizes and groups, page sizes, odd lengths, lengths of zero and one, steps of several tokens, bad pages, NaN behind
every length), the library's exports and argument codes, and the wrapper's refusals."""

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import _emu
import _launches
import _serving as ref
from test_abi import declared, exported

BF, FP, I32 = torch.bfloat16, torch.float16, torch.int32


def bind(lib):
    lib.prefix_attention_work.argtypes = [ctypes.c_longlong] * 2 + [ctypes.c_int] * 3 + [ctypes.c_longlong] * 3
    lib.prefix_attention_work.restype = ctypes.c_longlong
    lib.prefix_attention_launch.argtypes = [ctypes.c_void_p] * 10 + [ctypes.c_longlong] * 3 + [ctypes.c_int] * 3 + \
        [ctypes.c_longlong] * 3 + [ctypes.c_float, ctypes.c_int, ctypes.c_void_p]
    return lib


@pytest.fixture(scope="module")
def recorded(tmp_path_factory):
    return bind(_launches.build(tmp_path_factory.mktemp("attention_launches"), "shared_prefix_attention.hip"))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    """The kernel source with tests/emu/matrix.hpp in the place of csrc/matrix.hpp."""
    d = tmp_path_factory.mktemp("attention")
    kern = _emu.kernel_source(d, "shared_prefix_attention.hip")
    shutil.copy(os.path.join(_emu.EMU, "matrix.hpp"), os.path.join(str(d), "matrix.hpp"))
    out = os.path.join(str(d), "libattention.so")
    clang = _emu._clang()
    if clang is None:
        pytest.skip("clang++ (for the kernels' vector extensions on the host) is missing")
    proc = subprocess.run([clang, "-std=c++17", "-O1", "-fPIC", "-shared", "-U_FORTIFY_SOURCE", "-D_FORTIFY_SOURCE=0",
                           "-fno-strict-aliasing", "-w", "-pthread", "-I", _emu.EMU, "-I", str(d), kern, "-o", out],
                          capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-4000:]
    lib = bind(ctypes.CDLL(out))
    lib.emu_guarded.argtypes, lib.emu_guarded.restype = [ctypes.c_size_t], ctypes.c_void_p
    return lib


def guarded(lib, t):
    """t copied between pages that cannot be touched."""
    t = t.contiguous()
    n = t.numel() * t.element_size()
    if not n:
        return t
    p = lib.emu_guarded(n)
    ctypes.memmove(p, t.data_ptr(), n)
    raw = (ctypes.c_char * n).from_address(p)
    return torch.frombuffer(raw, dtype=t.dtype).view(t.shape)


def run(lib, q, k, v, table, length, tables, lens, block, scale=None, strides=None):
    batch, seq, hq, d = q.shape
    hk = k.shape[1]
    sizes = batch, seq, hq, hk, d, table.numel(), tables.shape[1], block
    n = lib.prefix_attention_work(*sizes)
    assert n >= 0
    inputs = [guarded(lib, t) for t in ((q if strides is None else q.contiguous()), k, v, table, length, tables, lens)]
    if strides is not None:
        inputs[0] = q
    work = guarded(lib, torch.full((n // 4 + 1,), float("nan"))[:n // 4]) if n else None
    out = guarded(lib, torch.full((batch, seq, hq, d), 9.0, dtype=q.dtype))
    ptrs = [t.data_ptr() if t.numel() else None for t in inputs] + [out.data_ptr(), work.data_ptr() if n else None]
    host = strides and (ctypes.c_longlong * 3)(*strides)
    assert lib.prefix_attention_launch(*ptrs, host, batch, seq, k.shape[0], hq, hk, d, table.numel(), tables.shape[1],
                                       block, d ** -0.5 if scale is None else scale, 1 if q.dtype == BF else 2, None) == 0
    return out


def check(lib, *args, **kw):
    got = run(lib, *args, **kw)
    kw.pop("strides", None)
    want, extra = ref.attention64(*args, **kw)
    assert not got.isnan().any()
    assert ref.near(got, want, extra), ((got.double() - want).abs() - extra).max()
    return got


CASES = [  # batch, seq, q heads, kv heads, head size, page, prefix, own lengths
    (1, 1, 4, 1, 128, 16, 100, [3]), (2, 1, 4, 2, 128, 16, 0, [40, 1]), (3, 1, 3, 3, 64, 8, 65, [0, 33, 7]),
    (2, 3, 7, 1, 64, 32, 31, [3, 50]), (2, 5, 14, 2, 80, 24, 33, [2, 37]), (1, 9, 8, 1, 96, 1, 70, [20]),
    (1, 2, 2, 1, 256, 16, 300, [9]), (1, 1, 2, 2, 192, 128, 17, [130]), (9, 1, 8, 1, 64, 16, 600, [1] * 9),
    (1, 40, 2, 1, 64, 16, 40, [77])]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_formula(lib, case, dtype):
    batch, seq, hq, hk, d, block, prefix, lens = case
    g = torch.Generator().manual_seed(d + seq)
    check(lib, *ref.attention_inputs(g, dtype, batch, seq, hq, hk, d, block, prefix, lens))


@pytest.mark.parametrize("prefix_splits,own_splits", [(1, 1), (2, 3), (5, 1), (200, 200)])
@pytest.mark.parametrize("tiles", [1, 2], ids=["32 rows", "256 rows"])
def test_every_split(lib, prefix_splits, own_splits, tiles):
    g = torch.Generator().manual_seed(1)
    args = ref.attention_inputs(g, BF, 2, 2, 4, 2, 64, 16, 777, [600, 300])
    for slot, value in enumerate((prefix_splits, own_splits, tiles)):
        lib.prefix_attention_tune(slot, value)
    try:
        check(lib, *args)
    finally:
        for slot in range(3):
            lib.prefix_attention_tune(slot, 0)


@pytest.mark.parametrize("team", [1, 2, 4])
@pytest.mark.parametrize("tiles", [1, 3], ids=["prefix apart", "prefix first"])
@pytest.mark.parametrize("d,lens", [(64, [200, 0, 3, 1]), (80, [40, 90]), (128, [33, 2, 31]), (256, [130, 70])], ids=str)
def test_teams(lib, d, lens, tiles, team):
    """Teams of waves over few and many slices, row tiles of a sequence that end in the middle (4 x 11 rows), rows that see
    no key or one, a bad page, and a prefix shorter than its table."""
    g = torch.Generator().manual_seed(7)
    q, k, v, table, length, tables, lens, block = ref.attention_inputs(g, BF, len(lens), 4, 11, 1, d, 8, 150, lens)
    table[3] = -1
    length -= 5
    tables[0, 0] = 1 << 30
    lib.prefix_attention_tune(2, tiles)
    lib.prefix_attention_tune(3, team)
    try:
        for splits in (1, 3):
            lib.prefix_attention_tune(1, splits)
            check(lib, q, k, v, table, length, tables, lens, block)
    finally:
        for slot in (1, 2, 3):
            lib.prefix_attention_tune(slot, 0)


@pytest.mark.parametrize("env", [{}, {"EMU_WAVE_AHEAD": "1"}], ids=["in turn", "waves ahead"])
@pytest.mark.parametrize("d", [64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("prefix", [1, 33, 64, 161, 700])
def test_wide_tiles(lib, monkeypatch, env, d, prefix):
    """Prefixes from one key to more than a ring of slices, pages that end anywhere, one of them bad."""
    for name, value in env.items():
        monkeypatch.setenv(name, value)
    g = torch.Generator().manual_seed(prefix)
    q, k, v, table, length, tables, lens, block = ref.attention_inputs(g, FP, 3, 2, 4, 1, d, 24, prefix, [2, 5, 9])
    if prefix > 600:
        table[7] = -1
    lib.prefix_attention_tune(0, 1)
    lib.prefix_attention_tune(2, 2)
    try:
        check(lib, q, k, v, table, length, tables, lens, block)
    finally:
        lib.prefix_attention_tune(0, 0)
        lib.prefix_attention_tune(2, 0)


def test_tables_longer_than_the_lengths_and_the_reverse(lib):
    g = torch.Generator().manual_seed(2)
    q, k, v, table, length, tables, lens, block = ref.attention_inputs(g, BF, 3, 2, 4, 2, 64, 16, 600, [400, 300, 90])
    for prefix, own in ((0, [0, 0, 0]), (1, [1, 2, 3]), (590, [17, 300, 5]), (-7, [-1, 20, 30])):
        check(lib, q, k, v, table, torch.tensor([prefix], dtype=I32), tables, torch.tensor(own, dtype=I32), block)
    # lengths beyond the tables count as the tables' whole: pages behind the keys hold NaN, so only full ones here
    k, v = k.nan_to_num(0.5), v.nan_to_num(0.25)
    check(lib, q, k, v, table, torch.tensor([10 ** 6], dtype=I32), tables, torch.tensor([2 ** 31 - 1, 500, 7], dtype=I32),
          block)


def test_bad_pages_count_as_absent(lib):
    g = torch.Generator().manual_seed(3)
    q, k, v, table, length, tables, lens, block = ref.attention_inputs(g, BF, 2, 1, 4, 2, 64, 16, 100, [70, 40])
    table[1], table[3], tables[0, 2] = -1, 2 ** 31 - 1, -2 ** 31
    tables[1, 0] = k.shape[0] // block  # the first page behind the cache
    check(lib, q, k, v, table, length, tables, lens, block)
    # a cache whose last page ends early: keys behind its end are absent
    check(lib, q, k[:-5].contiguous(), v[:-5].contiguous(), table, length, tables, lens, block)
    # nothing left at all, and a cache of no slots
    table.fill_(-1), tables.fill_(-1)
    assert (run(lib, q, k, v, table, length, tables, lens, block) == 0).all()
    assert (run(lib, q, k[:0], v[:0], table, length, tables, lens, block) == 0).all()


def test_no_prefix_table_and_one_part(lib):
    g = torch.Generator().manual_seed(4)
    args = ref.attention_inputs(g, FP, 2, 3, 4, 2, 96, 16, 0, [20, 2])
    assert args[3].numel() == 0
    got = check(lib, *args)
    assert (got[1, 0] == 0).all() and (got[1, 1] != 0).any()  # two own keys: the first of three queries stands before them


def test_strided_queries_and_scale(lib):
    g = torch.Generator().manual_seed(5)
    q, *rest = ref.attention_inputs(g, BF, 2, 3, 4, 2, 64, 16, 50, [20, 30])
    packed = torch.full((2, 3, 8, 64), float("nan"), dtype=BF)
    packed[:, :, 2:6] = q
    view = packed[:, :, 2:6]
    check(lib, view, *rest, strides=view.stride()[:3], scale=0.3)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    check(lib, turned, *rest, strides=turned.stride()[:3], scale=0.05)


def test_strides_of_single_ones(lib, pkg):
    """The stride of a dimension of one element is not used: it may be any number, and the query is taken as it lies."""
    in_vectors = pkg.candidate("shared_prefix_attention")._in_vectors
    for batch, seq, hq in ((1, 3, 4), (2, 1, 4), (2, 3, 1), (1, 1, 1)):
        g = torch.Generator().manual_seed(15)
        q, *rest = ref.attention_inputs(g, BF, batch, seq, hq, 1, 64, 16, 20, [9] * batch)
        strides = [s if n > 1 else 769 for s, n in zip(q.stride(), q.shape)][:3]
        odd = q.as_strided(q.shape, (*strides, 1))
        assert in_vectors(odd)
        check(lib, odd, *rest, strides=strides)
    wide = torch.zeros(2, 769, dtype=BF)[:, :768].unflatten(1, (3, 4, 64))
    assert wide[:1].stride(0) == 769 and in_vectors(wide[:1]) and not in_vectors(wide)
    assert not in_vectors(wide[1:])  # an odd address


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_peaked_and_flat_scores(lib, dtype):
    """Scores from -60 to 60, where the reference point has to move and most weights vanish, and scores all alike, where
    the output is the mean."""
    g = torch.Generator().manual_seed(6)
    check(lib, *ref.attention_inputs(g, dtype, 1, 2, 2, 1, 64, 16, 300, [100], peak=20.0))
    check(lib, *ref.attention_inputs(g, dtype, 1, 2, 2, 1, 64, 16, 300, [100], peak=0.0))


@pytest.mark.parametrize("tiles", [1, 2, 3], ids=["prefix apart", "shared tiles", "prefix first"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_idle_rows_beside_a_bad_prefix(lib, tiles, bad):
    """A NaN or infinite value in the prefix is in every row that sees it; a row before its sequence's first key sees
    nothing and is zero."""
    g = torch.Generator().manual_seed(11)
    args = ref.attention_inputs(g, BF, 3, 4, 4, 2, 64, 16, 40, [2, 0, 9])
    q, k, v, table, length, tables, lens, block = args
    v[int(table[1]) * block + 3] = bad
    lib.prefix_attention_tune(2, tiles)
    try:
        for team in (1, 4):
            lib.prefix_attention_tune(3, team)
            got = run(lib, *args)
            idle = torch.arange(4)[None] < 4 - lens[:, None]
            assert (got[idle] == 0).all() and not got[~idle].isfinite().any()
    finally:
        lib.prefix_attention_tune(2, 0)
        lib.prefix_attention_tune(3, 0)


@pytest.mark.parametrize("tiles,team", [(1, 1), (1, 4), (2, 1), (3, 2)], ids=str)
@pytest.mark.parametrize("d", [64, 80, 128, 192, 256])
@pytest.mark.parametrize("bad", ["nan", "-inf"])
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_bad_keys_reach_only_the_queries_that_see_them(lib, tiles, team, d, dtype, bad):
    """A NaN or infinite value of a step's own token is in its query and those behind it, in that one place of the head;
    queries before it are what they are without it. The step's keys begin in the middle of a slice, at its start and
    before it; one sequence has fewer keys than the step."""
    g, bad = torch.Generator().manual_seed(13), float(bad)
    seq, lens = 7, [45, 39, 3, 35]
    q, k, v, table, length, tables, lens, block = ref.attention_inputs(g, dtype, 4, seq, 6, 2, d, 16, 40, lens)
    slot = lambda b, t: int(tables[b, t // block]) * block + t % block  # noqa: E731
    clean, places = v.clone(), [(0, 41, 3), (0, 44, d - 1), (1, 33, 17), (2, 1, 0), (3, 30, 9), (3, 32, 40)]
    for b, t, c in places:
        v[slot(b, t), 1, c] = bad
        clean[slot(b, t), 1, c] = 0.0
    k[slot(0, 43), 0] = bad
    reached = torch.zeros(q.shape, dtype=torch.bool)
    for b, t, c in places:
        reached[b, max(0, t - int(lens[b]) + seq):, 3:, c] = True
    scored = torch.zeros(q.shape, dtype=torch.bool)  # a NaN score is in all of a head
    scored[0, 43 - 45 + seq:, :3] = True
    lib.prefix_attention_tune(2, tiles)
    lib.prefix_attention_tune(3, team)
    try:
        for splits in (1, 2):
            lib.prefix_attention_tune(1, splits)
            got = run(lib, q, k, v, table, length, tables, lens, block)
            k_clean = k.clone()
            k_clean[slot(0, 43), 0] = 0.0
            want, extra = ref.attention64(q, k_clean, clean, table, length, tables, lens, block)
            assert not got[reached].isfinite().any()
            rest = ~(reached | scored)
            assert got[rest].isfinite().all() and ref.near(got[rest], want[rest], extra[rest])
            idle = torch.arange(seq)[None] < seq - lens[:, None]
            assert (got[idle] == 0).all()
    finally:
        for slot_ in (1, 2, 3):
            lib.prefix_attention_tune(slot_, 0)


@pytest.mark.parametrize("prefix,own", [(0, 0), (40, 0), (0, 3)])
def test_tables_without_blocks(lib, prefix, own):
    """No blocks of a kind at all: without own blocks every query stands before its sequence's first key."""
    g = torch.Generator().manual_seed(12)
    q, k, v, table, length, tables, lens, block = ref.attention_inputs(g, BF, 2, 2, 4, 2, 64, 16, max(prefix, 1), [30, 20])
    table = table if prefix else table[:0]
    check(lib, q, k, v, table, length, tables[:, :own].contiguous(), lens, block)


def test_library_exports_the_header_and_codes(pkg):
    path = pkg.lib_path("shared_prefix_attention")
    assert {s for s in exported(path) if not s.startswith("_")} == set(declared("shared_prefix_attention"))
    lib = bind(ctypes.CDLL(path))
    p = 256
    good = dict(batch=2, seq=3, slots=64, hq=4, hk=2, d=64, pb=200, ob=2, block=16, dtype=1, scale=0.1)

    def code(pointers=(p,) * 9, strides=None, **change):
        a = {**good, **change}
        return lib.prefix_attention_launch(*pointers, strides, a["batch"], a["seq"], a["slots"], a["hq"], a["hk"], a["d"],
                                           a["pb"], a["ob"], a["block"], a["scale"], a["dtype"], None)

    assert code(batch=0) == 0 and code(seq=-1) == 0
    for change in (dict(d=72), dict(d=512), dict(hq=5), dict(hk=0), dict(hq=1), dict(block=0), dict(block=(1 << 30) + 1),
                   dict(pb=-1), dict(pb=1 << 26, block=17), dict(ob=1 << 31, block=1), dict(slots=-1), dict(slots=1 << 31),
                   dict(dtype=0), dict(batch=1 << 20, seq=1 << 10), dict(hq=1 << 17, hk=1)):
        assert code(**change) == -1, change
    for i in range(9):
        assert code(tuple(None if j == i else p for j in range(9))) == -1, i
    for i in (0, 1, 2, 7, 8):
        assert code(tuple(p + 8 if j == i else p for j in range(9))) == -1, i
    assert code(strides=(ctypes.c_longlong * 3)(128, 64, 4)) == -1
    for scale in (-0.1, 0.0, 1e-40, float("inf"), float("nan")):  # an absent key's -inf is scaled with the scores
        assert code(scale=scale) == -1
    sizes = 2, 3, 4, 2, 64
    assert lib.prefix_attention_work(*sizes, 2, 2, 0) == -1 and lib.prefix_attention_work(0, 3, 4, 2, 64, 2, 2, 16) == 0
    assert lib.prefix_attention_work(*sizes, 0, 2, 16) == 0 and lib.prefix_attention_work(*sizes, 200, 2, 16) > 0
    assert lib.prefix_attention_tune(99, 1) == -1


def test_too_small_a_workspace_is_refused(pkg, lib):
    """A buffer for the largest batch may be too small for a smaller one, which is cut into more parts."""
    real = bind(ctypes.CDLL(pkg.lib_path("shared_prefix_attention")))
    for one in (real, lib):
        one.prefix_attention_launch_sized.argtypes = [ctypes.c_void_p] * 9 + [ctypes.c_longlong, ctypes.c_void_p] + \
            [ctypes.c_longlong] * 3 + [ctypes.c_int] * 3 + [ctypes.c_longlong] * 3 + [ctypes.c_float, ctypes.c_int,
                                                                                      ctypes.c_void_p]
    need = [real.prefix_attention_work(b, 1, 32, 8, 128, 512, 64, 16) for b in range(1, 129)]
    below = [b for b in range(1, 128) if need[b - 1] > need[b]]
    assert below  # else the bytes grow throughout, and the header can say so
    p = 256
    for b in below:
        sizes = b, 1, 1 << 20, 32, 8, 128, 512, 64, 16, 0.1, 1, None
        assert real.prefix_attention_launch_sized(*(p,) * 9, need[b], None, *sizes) == -1
        assert real.prefix_attention_launch_sized(*(p,) * 9, need[b - 1] - 1, None, *sizes) == -1
    g = torch.Generator().manual_seed(14)
    q, k, v, table, length, tables, lens, block = args = ref.attention_inputs(g, BF, 2, 2, 4, 2, 64, 16, 300, [90, 200])
    sizes = 4, 2, 64, table.numel(), tables.shape[1], block
    lib.prefix_attention_tune(2, 1)
    try:
        n = lib.prefix_attention_work(2, 2, *sizes)
        assert n > 0
        work, out = guarded(lib, torch.zeros(n, dtype=torch.uint8)), torch.full_like(q, 9.0)
        pointers = [t.data_ptr() for t in (q, k, v, table, length, tables, lens, out, work)]
        for given, code in ((n - 1, -1), (0, -1), (n, 0)):
            assert lib.prefix_attention_launch_sized(*pointers, given, None, 2, 2, k.shape[0], *sizes, 0.125, 1,
                                                     None) == code
            assert code == 0 or (out == 9).all()
        assert torch.equal(out, run(lib, *args))
    finally:
        lib.prefix_attention_tune(2, 0)


@pytest.mark.parametrize("tiles", [0, 1, 2, 3])
@pytest.mark.parametrize("batch,seq,hq,hk,d,prefix,own", [
    (1 << 24, 1, 1, 1, 64, 1, 1), (1 << 26, 1, 1, 1, 64, 4, 4), (1 << 22, 1, 32, 8, 128, 100, 20), (1 << 25, 1, 8, 8, 256, 2, 2),
    (3, 1 << 24, 4, 1, 64, 2, 1 << 20), (1 << 24, 3, 16, 2, 96, 0, 2), (1 << 24, 3, 16, 2, 192, 2, 0), (1 << 29, 1, 1, 1, 64, 0, 1),
    ((1 << 30) - 1, 1, 1, 1, 64, 0, 1), (1 << 26, 1, 15, 15, 64, 1, 1), (2, 1, 8, 2, 64, 4, 4)], ids=str)
def test_grids_of_many_rows(recorded, batch, seq, hq, hk, d, prefix, own, tiles):
    """Launches of 2^32 threads and more, as a device takes them, every wave's number within 31 bits; or -1 and none."""
    p, sizes = 256, (hq, hk, d, prefix, own, 16)
    recorded.prefix_attention_tune(2, tiles)
    try:
        work = recorded.prefix_attention_work(batch, seq, *sizes)
        code, made = _launches.launches(recorded, lambda: recorded.prefix_attention_launch(
            *[p] * 9, None, batch, seq, 100, *sizes, 0.1, 1, None))
    finally:
        recorded.prefix_attention_tune(2, 0)
    assert (code == -1) == (work == -1)
    if code:
        assert code == -1 and not made and batch * hk >= 1 << 28  # more tiles of one row than waves that are numbered
        return
    assert made and all(_launches.accepted(one) for one in made)
    x, y, z, threads = made[0]
    assert x * y * z * (threads // 64) <= 1 << 31
    if work:
        x, y, z, threads = made[1]
        assert x * z >= batch * seq and y * 4 >= hq and threads == 256 and len(made) == 2
    else:
        assert len(made) == 1


class Stub:
    def __init__(self, shape, dtype, device="cuda:0"):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device(device)

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def is_contiguous(self):
        return True


USUAL = {"q": ((2, 3, 8, 64), BF), "k_cache": ((96, 2, 64), BF), "v_cache": ((96, 2, 64), BF), "prefix_table": ((2,), I32),
         "prefix_len": ((1,), I32), "block_tables": ((2, 2), I32), "seq_lens": ((2,), I32)}
REFUSED = [("q", (2, 3, 8, 64), torch.float32), ("q", (2, 3, 8, 72), BF), ("q", (6, 8, 64), BF), ("q", (2, 3, 7, 64), BF),
           ("q", (2, 3, 0, 64), BF), ("k_cache", (96, 2, 64), FP), ("k_cache", (96, 2, 128), BF), ("k_cache", (90, 2, 64), BF),
           ("k_cache", (96, 0, 64), BF), ("v_cache", (6, 16, 2, 64), BF), ("prefix_table", (2,), torch.int64),
           ("prefix_table", (1, 2), I32), ("prefix_len", (2,), I32), ("prefix_len", (1,), torch.int64),
           ("block_tables", (3, 2), I32), ("block_tables", (2, 2), torch.int64), ("seq_lens", (3,), I32),
           ("seq_lens", (2,), torch.int64)]


@pytest.mark.parametrize("change", REFUSED, ids=str)
def test_refusals(pkg, change):
    tensors = {n: Stub(*(change[1:] if n == change[0] else USUAL[n])) for n in USUAL}
    with pytest.raises(ValueError, match="shared_prefix_attention"):
        pkg.candidate("shared_prefix_attention").run({**tensors, "block_size": 16})


@pytest.mark.parametrize("name", list(USUAL))
@pytest.mark.parametrize("device", ["cpu", "cuda:1"])
def test_refuses_other_devices(pkg, name, device):
    tensors = {n: Stub(*USUAL[n], **({"device": device} if n == name else {})) for n in USUAL}
    with pytest.raises(ValueError, match="devices"):
        pkg.candidate("shared_prefix_attention").run({**tensors, "block_size": 16})


@pytest.mark.parametrize("block", [0, -1, 1 << 31])
def test_refuses_page_sizes(pkg, block):
    tensors = {n: Stub(*USUAL[n]) for n in USUAL}
    with pytest.raises(ValueError, match="block_size"):
        pkg.candidate("shared_prefix_attention").run({**tensors, "block_size": block})


@pytest.mark.parametrize("scale", [-1.0, 0.0, float("inf"), float("nan")])
def test_refuses_scales(pkg, scale):
    tensors = {n: Stub(*USUAL[n]) for n in USUAL}
    with pytest.raises(ValueError, match="scale"):
        pkg.candidate("shared_prefix_attention").run({**tensors, "block_size": 16, "scale": scale})


def test_operator_meta_and_cpu(pkg):
    ckopt = pkg.ops()
    args = [torch.empty(s, dtype=t) for s, t in USUAL.values()]
    out = ckopt.shared_prefix_attention(*(t.to("meta") for t in args), 16)
    assert out.shape == (2, 3, 8, 64) and out.dtype == BF
    with pytest.raises((NotImplementedError, RuntimeError)):
        ckopt.shared_prefix_attention(*args, 16)
