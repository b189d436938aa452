"""How kv4_attention deals out the slices of sequences that share their pages and are as long as a table may be (2^30 keys),
the kernels' own source under the HIP emulation."""

import ctypes

import pytest

import _emu
import test_kv4

PROBE = """
namespace {
__global__ void look(Args a, long long at, long long* out) {
  const int lane = lane_id();
  long long before = 0;
  const long long total = all_slices(a, lane);
  const int b = sequence_at(a, at, before, lane);
  const Parts p = parts_of<64>(a, b, 0, lane);
  if (lane == 0) out[0] = total, out[1] = b, out[2] = before, out[3] = p.n, out[4] = p.stats - a.stats;
}
}  // namespace
extern "C" __attribute__((visibility("default"))) void look_at(const int* lens, int batch, int runs, long long at,
                                                               long long* out) {
  Args a{};
  a.lens = lens, a.batch = batch, a.runs = runs, a.blocks = 1, a.block_size = 1 << 30, a.seq = 1;
  a.q_heads = a.kv_heads = a.group = a.tiles = 1, a.tile_rows = kRows, a.by_group = divisor(1);
  hipLaunchKernelGGL(look, dim3(1), dim3(64), 0, nullptr, a, at, out);
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    plain = _emu.kernel_source

    def with_probe(d, source):
        path = plain(d, source)
        with open(path, "a") as f:
            f.write(PROBE)
        return path

    _emu.kernel_source = with_probe
    try:
        return test_kv4.emulated(tmp_path_factory.mktemp("kv4_long"), "kv4_attention.hip")
    finally:
        _emu.kernel_source = plain


@pytest.mark.parametrize("batch,runs", [(1, 7), (63, 40), (64, 41), (130, 100), (130, 1)])
def test_slices_of_long_sequences(lib, batch, runs):
    each = 1 << 25  # slices of a sequence
    lens = (ctypes.c_int * batch)(*[1 << 30] * batch)
    for b in {0, batch // 2, batch - 1}:
        at, out = b * each + 5, (ctypes.c_longlong * 5)()
        lib.look_at(lens, batch, runs, ctypes.c_longlong(at), out)
        run = -(-batch * each // runs)
        first, last = b * each // run, ((b + 1) * each - 1) // run
        assert list(out) == [batch * each, b, b * each, last - first + 1, (first + b) * 16]
