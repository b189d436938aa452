"""verify_drafts on the CPU: the kernel's own source under the HIP emulation against the rule told in plain Python (every
split of a row over workgroups, odd vocabularies, ragged drafts, tokens outside the vocabulary, rows with nothing left to
draw from), the library's exports and argument codes, and the wrapper's refusals."""

import ctypes

import pytest
import torch

import _emu
import _launches
import _serving as ref
from test_abi import declared, exported

BF, F32, I64, I32 = torch.bfloat16, torch.float32, torch.int64, torch.int32


def bind(lib):
    for name in ("verify_plan", "verify_work"):
        getattr(lib, name).argtypes = [ctypes.c_longlong, ctypes.c_longlong, ctypes.c_int]
        getattr(lib, name).restype = ctypes.c_longlong
    lib.verify_launch.argtypes = [ctypes.c_void_p] * 10 + [ctypes.c_longlong, ctypes.c_int, ctypes.c_longlong,
                                                           ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
    return lib


@pytest.fixture(scope="module")
def recorded(tmp_path_factory):
    return bind(_launches.build(tmp_path_factory.mktemp("verify_launches"), "verify_drafts.hip"))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    return bind(ctypes.CDLL(_emu.build_shared(tmp_path_factory.mktemp("verify"), "verify_drafts.hip", "libverify.so")))


def run(lib, target, draft, tokens, uniforms, lens=None, blocks=1, strides=None):
    batch, rows, vocabulary = target.shape
    code = 0 if target.dtype == F32 else 1
    out = torch.full((batch + 2, rows), -99)
    accepted = torch.full((batch + 2,), -99)
    work = torch.full((lib.verify_work(batch, vocabulary, code),), float("nan"), dtype=torch.float64)
    counters = torch.zeros(batch, dtype=I32)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    strides = strides and (ctypes.c_longlong * 4)(*strides)
    assert lib.verify_launch(ptr(target), ptr(draft), ptr(tokens), ptr(lens), ptr(uniforms), ptr(out[1:]),
                             ptr(accepted[1:]), ptr(work), ptr(counters), strides, batch, rows - 1, vocabulary, code,
                             blocks, None) == 0
    assert (counters == 0).all()
    assert (out[[0, -1]] == -99).all() and (accepted[[0, -1]] == -99).all()
    return out[1:-1], accepted[1:-1]


def check(lib, *args, **kw):
    got, want = run(lib, *args, **kw), ref.verify64(*args, **({"lens": kw["lens"]} if "lens" in kw else {}))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (got, want)


@pytest.mark.parametrize("vocabulary", [1, 2, 63, 257, 1024, 2049, 4999])
@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("drafts,proposed,ragged,blocks",
                         [(3, True, False, 1), (0, True, False, 1), (1, False, False, 2), (5, True, True, 3),
                          (4, False, True, 1)])
def test_rule(lib, vocabulary, dtype, drafts, proposed, ragged, blocks):
    g = torch.Generator().manual_seed(vocabulary + drafts)
    target, draft, tokens, u, lens = ref.verify_inputs(g, 6, drafts, vocabulary, dtype, proposed and drafts > 0, ragged)
    check(lib, target, draft, tokens, u, lens=lens, blocks=blocks)


@pytest.mark.parametrize("blocks", [1, 2, 5, 16])
def test_every_split_draws_the_same(lib, blocks):
    """The level on and beside the running sums of exactly representable weights: 2^-k steps, so every sum is exact."""
    vocabulary, batch = 8192, 24
    target = torch.zeros(batch, 2, vocabulary)
    target[:, 0] = 2.0 ** -13
    draft = torch.full((batch, 1, vocabulary), 2.0 ** -13)
    draft[:, :, ::2] = 0  # every second entry is left, by 2^-13: 4096 of them
    tokens = torch.full((batch, 1), 1)
    u = torch.full((batch, 2), 1 - 2.0 ** -24)
    target[:, 0, 1] = 0  # refused
    u[:, 1] = torch.tensor([0.0, 2.0 ** -12, 2.0 ** -12 - 2.0 ** -30, 2.0 ** -12 + 2.0 ** -30, 0.25, 0.5, 1 - 2.0 ** -24,
                            0.125, *torch.linspace(0, 0.999, 16).tolist()])
    check(lib, target, draft, tokens, u, blocks=blocks)


@pytest.mark.parametrize("env", [{"EMU_CONCURRENT": "1"}, {"EMU_CONCURRENT": "1", "EMU_WEAK": "1"}],
                         ids=["concurrent", "weak"])
def test_hand_off_between_workgroups(lib, monkeypatch, env):
    for name, value in env.items():
        monkeypatch.setenv(name, value)
    g = torch.Generator().manual_seed(9)
    for seed in range(3):
        target, draft, tokens, u, lens = ref.verify_inputs(g, 4, 2, 20000, F32)
        check(lib, target, draft, tokens, u, blocks=5)


def test_long_vocabularies_take_longer_segments(lib):
    g = torch.Generator().manual_seed(3)
    n = 1024 * 1024 + 77  # more than 1024 segments of 1024
    target = torch.rand(2, 2, n, generator=g)
    tokens = torch.tensor([[5], [n - 1]])
    u = torch.tensor([[0.0, 0.7], [0.999999, 0.2]])
    got = run(lib, target, None, tokens, u, blocks=2)
    for b, j in ((0, 1), (1, 0)):
        w = target[b, j].double().clone()
        if j == 0:
            assert float(u[b, 0]) >= float(target[b, 0, n - 1])
            w[n - 1] = 0
        c = w.cumsum(0)
        assert int(got[1][b]) == j
        assert int(got[0][b, j]) == int((c <= float(u[b, 1]) * float(c[-1])).sum())


def test_nothing_left_to_draw_from(lib):
    v = 300
    target, draft = torch.zeros(5, 2, v), torch.zeros(5, 1, v)
    tokens, u = torch.full((5, 1), 7), torch.full((5, 2), 0.5)
    target[0, 0, 9] = draft[0, 0, 9] = 1.0        # the draft leaves nothing: the target's own, 9
    target[1, 0] = float("nan")                    # no probability at all: -1
    target[2, 0, 7], target[2, 1] = 1.0, -0.5      # kept, and a row of negative values behind it: -1
    target[3, 0, 250], draft[3, 0, 7] = 0.25, 1.0  # one entry left
    target[4, 0, :] = float("nan")
    target[4, 0, 3] = 0.5                          # NaN counts as zero
    for blocks in (1, 2):
        out, accepted = run(lib, target, draft, tokens, u, blocks=blocks)
        assert out.tolist() == [[9, -1], [-1, -1], [7, -1], [250, -1], [3, -1]]
        assert accepted.tolist() == [0, 0, 1, 0, 0]


def test_tokens_outside_the_vocabulary_are_refused(lib):
    g = torch.Generator().manual_seed(4)
    target, draft, tokens, u, _ = ref.verify_inputs(g, 4, 3, 500, F32)
    tokens[0, 0], tokens[1, 1], tokens[2, 2], tokens[3, 0] = -1, 500, 1 << 40, -(1 << 62)
    u[:, :3] = 0
    check(lib, target, draft, tokens, u)
    check(lib, target, None, tokens, u)


def test_lens_are_taken_within_the_drafts(lib):
    g = torch.Generator().manual_seed(5)
    target, draft, tokens, u, _ = ref.verify_inputs(g, 4, 3, 500, F32)
    u[:, :3] = 0
    check(lib, target, draft, tokens, u, lens=torch.tensor([-5, 99, 0, 2], dtype=I32))


def test_many_drafts(lib):
    g = torch.Generator().manual_seed(6)
    target, draft, tokens, u, _ = ref.verify_inputs(g, 2, 130, 70, F32)  # more than one wave of drafts
    u[0, :130] = 0
    u[1, :128] = 0
    u[1, 128] = 1 - 2.0 ** -24
    check(lib, target, draft, tokens, u)


def test_strided_probabilities(lib):
    g = torch.Generator().manual_seed(7)
    target, draft, tokens, u, _ = ref.verify_inputs(g, 3, 2, 333, BF)
    big_t, big_d = torch.zeros(3, 5, 400, dtype=BF), torch.zeros(2, 3, 335, dtype=BF)
    big_t[:, 1:4, 3:336] = target
    big_d[:, :, 1:334] = draft.transpose(0, 1)
    t, d = big_t[:, 1:4, 3:336], big_d[:, :, 1:334].transpose(0, 1)
    got = run(lib, t, d, tokens, u, blocks=2, strides=(*t.stride()[:2], *d.stride()[:2]))
    want = ref.verify64(target, draft, tokens, u)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_library_exports_the_header_and_codes(pkg):
    path = pkg.lib_path("verify_drafts")
    assert {s for s in exported(path) if not s.startswith("_")} == set(declared("verify_drafts"))
    lib = bind(ctypes.CDLL(path))
    p = 256
    good = dict(batch=2, drafts=3, vocabulary=100, dtype=0, blocks=1)

    def code(pointers=(p,) * 9, **change):
        a = {**good, **change}
        return lib.verify_launch(*pointers, None, a["batch"], a["drafts"], a["vocabulary"], a["dtype"], a["blocks"], None)

    assert code(batch=0) == 0
    for change in (dict(drafts=-1), dict(drafts=65536), dict(vocabulary=0), dict(vocabulary=(1 << 28) + 1), dict(dtype=2),
                   dict(blocks=0), dict(blocks=257), dict(batch=(1 << 22) + 1)):
        assert code(**change) == -1, change
    for i in (0, 2, 4, 5, 6):
        assert code(tuple(None if j == i else p for j in range(9))) == -1
    for i in (7, 8):
        assert code(tuple(None if j == i else p for j in range(9)), blocks=2) == -1
    assert lib.verify_plan(1, 0, 0) == lib.verify_work(1, 0, 0) == lib.verify_plan(1, 5, 3) == -1
    assert lib.verify_work(0, 100, 0) == 0
    for batch in (1, 7, 300, 5000):
        for vocabulary in (1, 1000, 128256, 1 << 28):
            assert 1 <= lib.verify_plan(batch, vocabulary, 0) <= 256
            assert batch <= lib.verify_work(batch, vocabulary, 0) <= 1024 * batch


def test_counters_suffice_for_every_plan(pkg, lib):
    """The bindings keep this many counters: rows are split over workgroups only where there are fewer."""
    most = pkg.candidate("verify_drafts")._COUNTERS
    for dtype in (0, 1):
        for vocabulary in (1, 5000, 128256, 1 << 28):
            split = [b for b in range(1, 2 * most) if lib.verify_plan(b, vocabulary, dtype) > 1]
            assert len(split) == (max(split) if split else 0) <= 2 * 256 // 5
            assert all(lib.verify_plan(b, vocabulary, dtype) == 1 for b in (2 * most, 1 << 20, 1 << 22))


@pytest.mark.parametrize("dtype", [0, 1])
def test_a_workspace_for_the_largest_sizes_serves_smaller_ones(lib, dtype):
    segment = 1024 if dtype == 0 else 2048
    sizes = [1, 1000, segment, segment * 1024 - 1, segment * 1024, segment * 1024 + 1, segment * 1500, segment * 2048,
             segment * 2048 + 1, 1 << 28]
    work = [lib.verify_work(7, v, dtype) for v in sizes]
    assert work == sorted(work)
    # what a launch of more workgroups writes: a row of longer segments, between guard values
    g, v = torch.Generator().manual_seed(8), segment * 1024 + 1
    target = torch.rand(2, 1, v, generator=g).to(F32 if dtype == 0 else BF)
    n = lib.verify_work(2, v, dtype)
    buffer = torch.full((n + 2,), -5.0, dtype=torch.float64)
    u, out, accepted, counters = torch.rand(2, 1, generator=g), torch.zeros(2, 1, dtype=I64), torch.zeros(2, dtype=I64), \
        torch.zeros(2, dtype=I32)
    assert lib.verify_launch(target.data_ptr(), None, None, None, u.data_ptr(), out.data_ptr(), accepted.data_ptr(),
                             buffer[1:].data_ptr(), counters.data_ptr(), None, 2, 0, v, dtype, 3, None) == 0
    assert float(buffer[0]) == float(buffer[-1]) == -5.0


@pytest.mark.parametrize("batch,vocabulary,blocks", [(1 << 22, 5000, 1), (1 << 22, 128256, 256), (1 << 22, 1 << 28, 4),
                                                     (1 << 22, 10, 1), (3, 50000, 256)])
@pytest.mark.parametrize("draft", [None, 256])
def test_grids_of_many_rows(recorded, batch, vocabulary, blocks, draft):
    """Launches of 2^32 threads and more, as a device takes them."""
    p = 256
    call = lambda: recorded.verify_launch(p, draft, *[p] * 7, None, batch, 3, vocabulary, 0, blocks, None)  # noqa: E731
    code, made = _launches.launches(recorded, call)
    (x, y, z, threads), = made
    assert code == 0 and _launches.accepted(made[0]) and x * y * z >= batch * blocks


class Stub:
    def __init__(self, shape, dtype, device="cuda:0"):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device(device)

    def dim(self):
        return len(self.shape)


USUAL = {"target_probs": ((2, 4, 50), F32), "draft_probs": ((2, 3, 50), F32), "draft_tokens": ((2, 3), I64),
         "uniforms": ((2, 4), F32), "draft_lens": ((2,), I32)}
REFUSED = [("target_probs", (2, 4, 50), torch.float16), ("target_probs", (4, 50), F32), ("target_probs", (2, 0, 50), F32),
           ("target_probs", (2, 4, 0), F32), ("target_probs", (2, 3, 50), F32), ("draft_probs", (2, 3, 50), BF),
           ("draft_probs", (2, 4, 50), F32), ("draft_probs", (2, 3, 49), F32), ("draft_tokens", (2, 3), I32),
           ("draft_tokens", (2, 4), I64), ("uniforms", (2, 3), F32), ("uniforms", (2, 4), torch.float64),
           ("draft_lens", (3,), I32), ("draft_lens", (2,), I64)]


@pytest.mark.parametrize("change", REFUSED, ids=str)
def test_refusals(pkg, change):
    tensors = {n: Stub(*(change[1:] if n == change[0] else USUAL[n])) for n in USUAL}
    with pytest.raises(ValueError, match="verify_drafts"):
        pkg.candidate("verify_drafts").run(tensors)


@pytest.mark.parametrize("name", list(USUAL))
@pytest.mark.parametrize("device", ["cpu", "cuda:1"])
def test_refuses_other_devices(pkg, name, device):
    tensors = {n: Stub(*USUAL[n], **({"device": device} if n == name else {})) for n in USUAL}
    with pytest.raises(ValueError, match="devices"):
        pkg.candidate("verify_drafts").run(tensors)


def test_operator_meta_and_cpu(pkg):
    ckopt = pkg.ops()
    m = dict(device="meta")
    out, accepted = ckopt.verify_drafts(torch.empty(2, 4, 50, **m), None, torch.empty(2, 3, dtype=I64, **m),
                                        torch.empty(2, 4, **m))
    assert out.shape == (2, 4) and accepted.shape == (2,) and out.dtype == accepted.dtype == I64
    with pytest.raises((NotImplementedError, RuntimeError)):
        ckopt.verify_drafts(torch.zeros(2, 4, 50), None, torch.zeros(2, 3, dtype=I64), torch.zeros(2, 4))
