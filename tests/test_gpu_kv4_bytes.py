"""The cache in 4 bits on the GPU: every scale byte with every code, read in both types."""

import pytest
import torch

import _kv4 as kv4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_every_scale_byte_read(pkg, dtype):
    """bf16 holds every element; fp16 overflows to infinity and rounds below its smallest."""
    codes = torch.arange(16, dtype=torch.uint8).repeat(2)
    codes = (codes[::2] | codes[1::2] << 4).expand(1, 1, 256, 2, 16).flatten(3).contiguous()
    scales = torch.arange(256, dtype=torch.uint8)[:, None].expand(1, 1, 256, 2).contiguous()
    cache = [codes, scales, codes.flip(-1).contiguous(), scales.clone()]
    got = pkg.ops().kv4_read(*(t.cuda() for t in cache), torch.arange(256, device="cuda"), dtype)
    for x, i in zip(got, (0, 2)):
        want = kv4.flat(kv4.decode(*cache[i:i + 2])).to(dtype)
        x = x.cpu()
        assert torch.equal(x.isnan(), want.isnan())
        off = (x.nan_to_num(0, posinf=1e30, neginf=-1e30) != want.nan_to_num(0, posinf=1e30, neginf=-1e30))
        assert not off.any(), (off.nonzero()[:5], x[off][:5], want[off][:5])
