"""Which calls of kv4_attention have their keys dealt out evenly (they have a workspace)."""

import ctypes

import pytest

import test_kv4


@pytest.fixture(scope="module")
def work(pkg):
    lib = test_kv4.bind(ctypes.CDLL(pkg.lib_path("kv4_attention")))
    return lambda batch, keys, q_heads=32, kv_heads=8: lib.kv4_attention_work(batch, 1, q_heads, kv_heads, 128, keys // 64,
                                                                              64)


@pytest.mark.parametrize("batch,keys,kv_heads", [(128, 32768, 8), (128, 16384, 8), (256, 32768, 8), (64, 32768, 32),
                                                 (16, 32768, 8), (1, 8192, 8)], ids=str)
def test_one_long_sequence_does_not_bound_the_launch(work, batch, keys, kv_heads):
    """Tables as wide as this have room for a sequence that takes a workgroup several times as long as the whole launch."""
    assert work(batch, keys, kv_heads=kv_heads) > 0


@pytest.mark.parametrize("batch,keys", [(256, 512), (256, 4096), (128, 8192), (1, 1024)], ids=str)
def test_narrow_tables_have_no_second_launch(work, batch, keys):
    assert work(batch, keys) == 0


def test_the_workspace_is_bounded(work):
    """Parts of runs and of sequences, of 16 rows of 128 sums: sequences are no more than four times the runs of 512
    workgroups, so the rows are no more than 5 x 512 tiles (of 16 rows here, 32 at most)."""
    for batch in (1, 50, 256, 257, 1000, 30000):
        for keys in (512, 8192, 32768, 1 << 20):
            for kv_heads in (1, 8, 32):
                assert 0 <= work(batch, keys, kv_heads=kv_heads) <= 5 * 512 * 32 * (4 * 128 + 8)
