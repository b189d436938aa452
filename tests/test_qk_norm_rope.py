"""qk_norm_rope on the CPU: the kernels' own source under the HIP emulation against the formula in 64 bits (head sizes,
partial rotations, strided views, every split of the heads over waves, slots outside the cache), the library's exports
and argument codes, and the wrapper's refusals."""

import ctypes
import itertools

import pytest
import torch

import _emu
import _launches
import _serving as ref
from test_abi import declared, exported

BF, FP, I64 = torch.bfloat16, torch.float16, torch.int64


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("qk_norm_rope")
    return bind(ctypes.CDLL(_emu.build_shared(d, "qk_norm_rope.hip", "libqk.so")))


def bind(lib):
    lib.qk_norm_rope_launch.argtypes = [ctypes.c_void_p] * 9 + [ctypes.c_longlong] * 2 + [ctypes.c_int] * 5 + \
        [ctypes.c_float, ctypes.c_void_p]
    lib.qk_norm_rope_kv_launch.argtypes = [ctypes.c_void_p] * 12 + [ctypes.c_longlong] * 3 + [ctypes.c_int] * 5 + \
        [ctypes.c_float, ctypes.c_void_p]
    return lib


def strides(*tensors):
    return (ctypes.c_longlong * 12)(*(s for t in tensors for s in t.stride()[:3]))


def ptr(t):
    return None if t is None else t.data_ptr()


def inputs(seed, dtype, batch, seq, hq, hk, d, rotary, weights=True, packed=False, offset=0):
    g = torch.Generator().manual_seed(seed)

    def one(*shape):
        flat = torch.empty(offset + torch.Size(shape).numel(), dtype=dtype)[offset:]
        return flat.view(shape).copy_(torch.randn(shape, generator=g) * 1.5)

    if packed:
        q, k, v = one(batch, seq, hq + 2 * hk, d).split([hq, hk, hk], 2)
    else:
        q, k, v = one(batch, seq, hq, d), one(batch, seq, hk, d), one(batch, seq, hk, d)
    ids = torch.randint(0, 1 << 20, (batch, seq), generator=g)
    qw, kw = ((torch.rand(d, generator=g) + 0.5).to(dtype) for _ in range(2)) if weights else (None, None)
    return q, k, v, ids, ref.inv_freq_of(rotary), qw, kw


SHAPES = [  # batch, seq, q heads, kv heads, head size, rotary
    (1, 1, 4, 1, 128, 128), (2, 3, 5, 2, 128, 64), (1, 2, 3, 3, 80, 80), (1, 5, 7, 1, 96, 96), (1, 3, 14, 2, 64, 32),
    (1, 2, 4, 4, 256, 256), (1, 2, 2, 1, 192, 48), (1, 2, 2, 1, 48, 0), (1, 2, 3, 2, 32, 32), (1, 2, 2, 1, 50, 50),
    (2, 2, 2, 1, 9, 4), (1, 1, 1, 1, 1, 0), (1, 2, 1, 1, 512, 512), (1, 1, 40, 8, 128, 128), (1, 2, 3, 1, 128, 24),
          (2, 3, 5, 1, 80, 40), (1, 4, 2, 2, 24, 8), (3, 2, 1, 1, 64, 64), (1, 3, 9, 3, 128, 24)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("packed,weights", [(False, True), (True, False)])
def test_formula(lib, shape, dtype, packed, weights):
    batch, seq, hq, hk, d, rotary = shape
    q, k, v, ids, inv, qw, kw = inputs(1, dtype, *shape, weights=weights, packed=packed)
    qo, ko = torch.full((batch, seq, hq, d), 7.0, dtype=dtype), torch.full((batch, seq, hk, d), 7.0, dtype=dtype)
    assert lib.qk_norm_rope_launch(ptr(q), ptr(k), ptr(ids), ptr(inv), ptr(qw), ptr(kw), ptr(qo), ptr(ko),
                                   strides(q, k, qo, ko), batch, seq, hq, hk, d, rotary, 1 if dtype == BF else 2,
                                   ref.EPS, None) == 0
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        assert ref.near(got, ref.norm_rope64(x, ids, inv, w), ref.norm_rope_error(x, w))


@pytest.mark.parametrize("steps", [1, 2, 4])
@pytest.mark.parametrize("shape", [(1, 3, 10, 3, 128, 128), (2, 2, 5, 2, 256, 64), (1, 2, 70, 9, 64, 64),
                                   (2, 3, 11, 1, 80, 40)], ids=str)
def test_every_split_gives_the_same_bits(lib, steps, shape):
    batch, seq, hq, hk, d, rotary = shape
    q, k, v, ids, inv, qw, kw = inputs(2, BF, *shape)
    outs = []
    for n in (0, steps):
        lib.qk_norm_rope_tune(0, n)
        qo, ko = torch.zeros_like(q), torch.zeros_like(k)
        assert lib.qk_norm_rope_launch(ptr(q), ptr(k), ptr(ids), ptr(inv), ptr(qw), ptr(kw), ptr(qo), ptr(ko), None,
                                       batch, seq, hq, hk, d, rotary, 1, ref.EPS, None) == 0
        outs.append((qo, ko))
    lib.qk_norm_rope_tune(0, 0)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(*outs))


@pytest.mark.parametrize("shape", [(2, 7, 1, 1, 64, 64), (1, 5, 2, 1, 128, 64), (3, 3, 1, 1, 256, 256), (1, 9, 2, 2, 24, 8),
                                   (1, 3, 1, 1, 80, 40), (2, 1, 1, 1, 48, 0)], ids=str)
def test_few_heads(lib, shape):
    """Several tokens to a wave, the last wave's not all there, with and without the caches; the same bits as one by one."""
    batch, seq, hq, hk, d, rotary = shape
    q, k, v, ids, inv, qw, kw = inputs(10, FP, *shape, packed=True)
    slots = batch * seq + 2
    mapping = torch.randperm(slots, generator=torch.Generator().manual_seed(1))[:batch * seq].view(batch, seq)
    mapping[-1, -1] = slots
    outs = []
    for few in (2, 1):
        lib.qk_norm_rope_tune(2, few)
        qo, ko, qc = (torch.full(t.shape, 7.0, dtype=FP) for t in (q, k, q))
        kc, vc = (torch.full((slots, hk, d), c, dtype=FP) for c in (3.0, 5.0))
        assert lib.qk_norm_rope_launch(ptr(q), ptr(k), ptr(ids), ptr(inv), ptr(qw), ptr(kw), ptr(qo), ptr(ko),
                                       strides(q, k, qo, ko), batch, seq, hq, hk, d, rotary, 2, ref.EPS, None) == 0
        assert lib.qk_norm_rope_kv_launch(ptr(q), ptr(k), ptr(v), ptr(ids), ptr(inv), ptr(qw), ptr(kw), ptr(qc), ptr(kc),
                                          ptr(vc), ptr(mapping), strides(q, k, v, qc), batch, seq, slots, hq, hk, d,
                                          rotary, 2, ref.EPS, None) == 0
        outs.append((qo, ko, qc, kc, vc))
    lib.qk_norm_rope_tune(2, 0)
    for x, y in zip(*outs):
        assert torch.equal(x, y)
    assert ref.near(outs[1][0], ref.norm_rope64(q, ids, inv, qw), ref.norm_rope_error(q, qw))


@pytest.mark.parametrize("scalar", [0, 1])
@pytest.mark.parametrize("d,rotary", [(128, 128), (80, 32), (256, 256), (80, 40)])
def test_cache_rows_and_slots_outside(lib, scalar, d, rotary):
    batch, seq, hq, hk, slots = 2, 4, 3, 2, 11
    q, k, v, ids, inv, qw, kw = inputs(3, BF, batch, seq, hq, hk, d, rotary, packed=True)
    slot = torch.tensor([[3, 10, -1, 0], [11, 1 << 40, -(1 << 40), 5]])  # four of them outside: nothing written
    # a guard row on either side of each cache
    kc, vc = (torch.full((slots + 2, hk, d), c, dtype=BF) for c in (3.0, 5.0))
    qo = torch.zeros(batch, seq, hq, d, dtype=BF)
    lib.qk_norm_rope_tune(1, scalar)
    err = lib.qk_norm_rope_kv_launch(ptr(q), ptr(k), ptr(v), ptr(ids), ptr(inv), ptr(qw), ptr(kw), ptr(qo),
                                     ptr(kc[1:]), ptr(vc[1:]), ptr(slot), strides(q, k, v, qo), batch, seq, slots, hq,
                                     hk, d, rotary, 1, ref.EPS, None)
    lib.qk_norm_rope_tune(1, 0)
    assert err == 0
    assert ref.near(qo, ref.norm_rope64(q, ids, inv, qw), ref.norm_rope_error(q, qw))
    want, extra = ref.norm_rope64(k, ids, inv, kw).flatten(0, 1), ref.norm_rope_error(k, kw).flatten(0, 1)
    written = {3: 0, 10: 1, 0: 3, 5: 7}
    for row in range(slots + 2):
        token = written.get(row - 1)
        if token is None:
            assert (kc[row] == 3).all() and (vc[row] == 5).all()
        else:
            assert ref.near(kc[row], want[token], extra[token])
            assert torch.equal(vc[row], v.flatten(0, 1)[token])


@pytest.mark.parametrize("slots,code", [(0, 0), (1, -1)])
def test_no_cache_for_no_slots(lib, slots, code):
    q, k, v, ids, inv, qw, kw = inputs(9, BF, 1, 2, 3, 1, 64, 64)
    qo, mapping = torch.empty_like(q), torch.tensor([[0, 1]])
    assert lib.qk_norm_rope_kv_launch(ptr(q), ptr(k), ptr(v), ptr(ids), ptr(inv), ptr(qw), ptr(kw), ptr(qo), None, None,
                                      ptr(mapping), strides(q, k, v, qo), 1, 2, slots, 3, 1, 64, 64, 1, ref.EPS,
                                      None) == code
    assert code or ref.near(qo, ref.norm_rope64(q, ids, inv, qw), ref.norm_rope_error(q, qw))


@pytest.fixture(scope="module")
def recorded(tmp_path_factory):
    return bind(_launches.build(tmp_path_factory.mktemp("qk_launches"), "qk_norm_rope.hip"))


@pytest.mark.parametrize("batch,seq,hq,hk,d", [(1, 1 << 25, 1, 1, 1), (3, (1 << 31) // 3, 1, 1, 64), (1 << 20, 64, 64, 8, 100),
                                               (1 << 15, 1 << 15, 40, 8, 128), (1 << 12, 1 << 12, 1 << 13, 1 << 13, 1)])
@pytest.mark.parametrize("cached", [False, True])
def test_grids_of_many_heads(recorded, batch, seq, hq, hk, d, cached):
    """Launches of 2^32 threads and more, as a device takes them; a wave has at most four steps of 16 heads."""
    p = 256
    if cached:
        call = lambda: recorded.qk_norm_rope_kv_launch(*[p] * 11, None, batch, seq, 100, hq, hk, d, 0, 1, 1e-6, None)  # noqa: E731
    else:
        call = lambda: recorded.qk_norm_rope_launch(*[p] * 8, None, batch, seq, hq, hk, d, 0, 1, 1e-6, None)  # noqa: E731
    code, made = _launches.launches(recorded, call)
    heads = batch * seq * (hq + hk * (2 if cached else 1))
    if heads > 1 << 38:
        assert code == -1 and not made
    else:
        (x, y, z, threads), = made
        assert code == 0 and _launches.accepted(made[0]) and x * y * z * threads // 64 * 64 >= heads


def test_strides_of_single_ones_decide_nothing(recorded, lib):
    """One sequence's, one token's or one head's stride is not used: an odd one does not send the call to the kernel of
    any stride, and changes no result."""
    for batch, seq, hq, hk in ((1, 3, 8, 2), (3, 1, 8, 2), (3, 2, 1, 1), (1, 1, 1, 1)):
        q, k, v, ids, inv, qw, kw = inputs(11, BF, batch, seq, hq, hk, 128, 128)
        qo, ko = torch.zeros_like(q), torch.zeros_like(k)
        kc, vc = (torch.zeros(16, hk, 128, dtype=BF) for _ in range(2))
        mapping = torch.arange(batch * seq).view(batch, seq)
        odd = [[777 if n == 1 else s for s, n in zip(t.stride(), t.shape)][:3] for t in (q, k, v)]
        odd, even = ((ctypes.c_longlong * 12)(*sum(parts, [])) for parts in (
            odd + [list(qo.stride()[:3])], [list(t.stride()[:3]) for t in (q, k, v, qo)]))

        def call(one, st):
            return one.qk_norm_rope_kv_launch(ptr(q), ptr(k), ptr(v), ptr(ids), ptr(inv), ptr(qw), ptr(kw), ptr(qo), ptr(kc),
                                              ptr(vc), ptr(mapping), st, batch, seq, 16, hq, hk, 128, 128, 1, ref.EPS, None)

        recorded.qk_norm_rope_tune(1, 1)
        scalar = _launches.launches(recorded, lambda: call(recorded, even))
        recorded.qk_norm_rope_tune(1, 0)
        assert _launches.launches(recorded, lambda: call(recorded, odd)) == \
            _launches.launches(recorded, lambda: call(recorded, even))
        if hq > 1:
            assert _launches.launches(recorded, lambda: call(recorded, odd)) != scalar
        assert call(lib, even) == 0
        want = [t.clone() for t in (qo, kc, vc)]
        for t in (qo, kc, vc):
            t.zero_()
        assert call(lib, odd) == 0 and all(torch.equal(a, b) for a, b in zip((qo, kc, vc), want))


@pytest.mark.parametrize("d", [128, 50])
def test_in_place_on_a_packed_projection(lib, d):
    q, k, v, ids, inv, qw, kw = inputs(4, FP, 1, 3, 5, 2, d, d, packed=True)
    want = [(ref.norm_rope64(x, ids, inv, w), ref.norm_rope_error(x, w)) for x, w in ((q, qw), (k, kw))]
    kept = v.clone()
    assert lib.qk_norm_rope_launch(ptr(q), ptr(k), ptr(ids), ptr(inv), ptr(qw), ptr(kw), ptr(q), ptr(k),
                                   strides(q, k, q, k), 1, 3, 5, 2, d, d, 2, ref.EPS, None) == 0
    assert ref.near(q, *want[0]) and ref.near(k, *want[1]) and torch.equal(v, kept)


def test_tensors_off_the_16_byte_grid(lib):
    q, k, v, ids, inv, qw, kw = inputs(5, BF, 1, 2, 3, 1, 128, 128, offset=1)
    assert q.data_ptr() % 16
    qo, ko = torch.zeros(1, 2, 3, 128, dtype=BF), torch.zeros(1, 2, 1, 128, dtype=BF)
    assert lib.qk_norm_rope_launch(ptr(q), ptr(k), ptr(ids), ptr(inv), ptr(qw), ptr(kw), ptr(qo), ptr(ko), None, 1, 2,
                                   3, 1, 128, 128, 1, ref.EPS, None) == 0
    assert ref.near(qo, ref.norm_rope64(q, ids, inv, qw), ref.norm_rope_error(q, qw))


@pytest.mark.parametrize("d", [64, 40])
def test_special_values(lib, d):
    """A zero head stays zero, a NaN makes its head NaN (its pair partner's too), other heads are untouched by it."""
    q, k, v, ids, inv, qw, kw = inputs(6, BF, 1, 1, 4, 1, d, d, weights=False)
    q[0, 0, 0] = 0
    q[0, 0, 1, 3] = float("nan")
    qo, ko = torch.zeros_like(q), torch.zeros_like(k)
    assert lib.qk_norm_rope_launch(ptr(q), ptr(k), ptr(ids), ptr(inv), None, None, ptr(qo), ptr(ko), None, 1, 1, 4, 1,
                                   d, d, 1, ref.EPS, None) == 0
    assert (qo[0, 0, 0] == 0).all() and qo[0, 0, 1].isnan().all()
    assert ref.near(qo[:, :, 2:], ref.norm_rope64(q[:, :, 2:], ids, inv), ref.norm_rope_error(q[:, :, 2:]))


def test_far_positions_keep_their_phase(lib):
    """Angles up to 2^31: the phase is that of the exact product, not of its fp32 rounding (off by up to 2^6 there)."""
    d = 64
    q, k, v, _, inv, qw, kw = inputs(7, FP, 1, 6, 1, 1, d, d, weights=False)
    ids = torch.tensor([[0, 1, (1 << 24) + 1, (1 << 31) - 1, -(1 << 30) - 7, 999999937]])
    qo, ko = torch.zeros_like(q), torch.zeros_like(k)
    assert lib.qk_norm_rope_launch(ptr(q), ptr(k), ptr(ids), ptr(inv), None, None, ptr(qo), ptr(ko), None, 1, 6, 1, 1,
                                   d, d, 2, ref.EPS, None) == 0
    # pi/2 in two parts: 2^31 multiples of a remainder below 2^-107 and roundings of the angle's 2^-53
    extra = ref.norm_rope_error(q) + 2.0 ** 31 * 2.0 ** -53 * 4
    assert ref.near(qo, ref.norm_rope64(q, ids, inv), extra)


def test_library_exports_the_header_and_codes(pkg):
    path = pkg.lib_path("qk_norm_rope")
    symbols = {s for s in exported(path) if not s.startswith("_")}
    assert symbols == set(declared("qk_norm_rope"))
    lib = bind(ctypes.CDLL(path))
    p = 256  # never dereferenced: every call below returns before a launch
    good = dict(batch=2, seq=3, hq=4, hk=2, d=64, r=64, dtype=1)

    def code(pointers=(p,) * 8, **change):
        a = {**good, **change}
        return lib.qk_norm_rope_launch(*pointers, None, a["batch"], a["seq"], a["hq"], a["hk"], a["d"], a["r"],
                                       a["dtype"], 1e-6, None)

    assert code(batch=0) == 0 and code(seq=0) == 0
    for change in (dict(hq=0), dict(hk=-1), dict(d=0), dict(d=65537), dict(r=63), dict(r=66), dict(r=-2), dict(dtype=0),
                   dict(dtype=3), dict(batch=1 << 20, seq=1 << 12)):
        assert code(**change) == -1, change
    for i in (0, 1, 2, 3, 6, 7):  # the weights may be absent
        assert code(tuple(None if j == i else p for j in range(8))) == -1
    kv = [p] * 11
    args = lambda kv, slots: (*kv, None, 2, 3, slots, 4, 2, 64, 64, 1, 1e-6, None)  # noqa: E731
    assert lib.qk_norm_rope_kv_launch(*args(kv, -1)) == -1
    for i in (2, 8, 9, 10):
        assert lib.qk_norm_rope_kv_launch(*args([None if j == i else p for j in range(11)], 8)) == -1
    assert lib.qk_norm_rope_tune(99, 1) == -1


class Stub:
    def __init__(self, shape, dtype, device="cuda:0"):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device(device)

    def dim(self):
        return len(self.shape)


USUAL = {"q": ((2, 3, 8, 64), BF), "k": ((2, 3, 2, 64), BF), "position_ids": ((2, 3), I64),
         "inv_freq": ((32,), torch.float32), "q_weight": ((64,), BF), "k_weight": ((64,), BF)}
REFUSED = [("q", (2, 3, 8, 62), BF), ("q", (2, 4, 8, 64), BF), ("q", (6, 8, 64), BF), ("q", (2, 3, 8, 64), torch.float32),
           ("q", (2, 3, 0, 64), BF), ("k", (2, 3, 2, 64), FP), ("k", (2, 3, 0, 64), BF), ("k", (3, 3, 2, 64), BF),
           ("position_ids", (6,), I64), ("position_ids", (2, 3), torch.int32), ("inv_freq", (33,), torch.float32),
           ("inv_freq", (32,), BF), ("inv_freq", (32, 1), torch.float32), ("q_weight", (32,), BF),
           ("k_weight", (64,), torch.float32)]


@pytest.mark.parametrize("change", REFUSED, ids=str)
def test_refusals(pkg, change):
    name, shape, dtype = change
    tensors = {n: Stub(*(change[1:] if n == name else USUAL[n])) for n in USUAL}
    with pytest.raises(ValueError, match="qk_norm_rope"):
        pkg.candidate("qk_norm_rope").run(tensors)


@pytest.mark.parametrize("name,device", itertools.product(USUAL, ["cpu", "cuda:1"]))
def test_refuses_other_devices(pkg, name, device):
    tensors = {n: Stub(*USUAL[n], **({"device": device} if n == name else {})) for n in USUAL}
    with pytest.raises(ValueError, match="devices"):
        pkg.candidate("qk_norm_rope").run(tensors)


def test_shared_elements_are_seen(pkg):
    spread = pkg.candidate("qk_norm_rope")._spread
    x = torch.zeros(2, 3, 6, 8)
    assert spread(x) and spread(x[:, :, 1:3]) and spread(x.transpose(1, 2)) and spread(x[:1])
    assert not spread(x[:, :1].expand(2, 3, 6, 8)) and not spread(x.view(-1).as_strided((2, 2, 2, 8), (16, 8, 4, 1)))


def test_views_of_one_projection_are_apart(pkg):
    apart = pkg.candidate("qk_norm_rope")._apart
    x = torch.zeros(2, 3, 8, 16, dtype=BF)
    turned = torch.zeros(2, 8, 3, 16, dtype=BF).transpose(1, 2)  # heads before tokens
    for t in (x, turned):
        for part in (t, t[:1], t[:, :1], t[:1, :1]):
            q, k, v = part.split([4, 2, 2], 2)
            assert apart(q, k) and apart(k, q) and apart(q, v) and apart(k, v)
            assert apart(part[:, :, ::2], part[:, :, 1::2]) and apart(part[:, :, :4, :8], part[:, :, 2:, 8:])
            assert not apart(part[:, :, :4], part[:, :, 3:5]) and not apart(part[:, :, 3:5], part[:, :, :4])
            assert not apart(q, q) and not apart(q, q[:, :, :1].expand_as(k)) and not apart(part[:, :, ::2], part[:, :, 2:3])
    assert apart(x[:, :, :4], x.clone()) and apart(x[:1], x[1:]) and not apart(x[:, :2], x[:, 1:])
    assert apart(x[:0], x) and apart(x[:, :, :4], x[:, :, 4:5].expand(2, 3, 4, 16))
    flat = x.view(-1)  # the same memory half an element further on, seen as another period
    assert not apart(flat[:16 * 6].view(1, 2, 3, 16), flat[8:8 + 16 * 6].view(1, 3, 2, 16))


class OnGpu:
    """A CPU tensor that says it is on the GPU: refusals look at shapes, strides and addresses only."""

    def __init__(self, tensor):
        self.tensor, self.device = tensor, torch.device("cuda:0")

    def __getattr__(self, name):
        return getattr(self.tensor, name)


@pytest.mark.parametrize("cached", [False, True])
def test_in_place_refuses_shared_elements(pkg, cached):
    """q is written while k, and v where there are caches, are read."""
    x = torch.zeros(2, 3, 8, 64, dtype=BF)
    q, k, v = x.split([4, 2, 2], 2)
    rest = {"position_ids": torch.zeros(2, 3, dtype=I64), "inv_freq": torch.zeros(32), "inplace": True}
    if cached:
        rest |= {"k_cache": torch.zeros(9, 2, 64, dtype=BF), "v_cache": torch.zeros(9, 2, 64, dtype=BF),
                 "slot_mapping": torch.zeros(2, 3, dtype=I64)}

    def run(**tensors):
        pkg.candidate("qk_norm_rope").run({n: OnGpu(t) if torch.is_tensor(t) else t for n, t in (rest | tensors).items()})

    for bad in (q[:, :, :2], x[:, :, 3:5], x[:, :, :1].expand(2, 3, 2, 64)):
        with pytest.raises(ValueError, match="share"):
            run(q=q, k=bad, v=v)
        if cached:
            with pytest.raises(ValueError, match="share"):
                run(q=q, k=k, v=bad)


def test_cpu_tensors_refused_by_the_operators(pkg):
    ckopt = pkg.ops()
    q, ids = torch.zeros(1, 2, 2, 64, dtype=BF), torch.zeros(1, 2, dtype=I64)
    with pytest.raises((NotImplementedError, RuntimeError)):
        ckopt.qk_norm_rope(q, q, ids, torch.zeros(32))
    m = dict(device="meta", dtype=BF)
    q, k = torch.empty(1, 2, 8, 64, **m), torch.empty(1, 2, 2, 64, **m)
    qo, ko = ckopt.qk_norm_rope(q, k, ids.to("meta"), torch.empty(32, device="meta"))
    assert qo.shape == q.shape and ko.shape == k.shape and qo.dtype == BF
