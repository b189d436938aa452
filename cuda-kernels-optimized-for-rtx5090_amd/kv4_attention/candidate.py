"""Attention of a batch's last tokens over each sequence's paged keys and values in 4 bits, served by this package's
MI355X library. No counterpart in the reference; the wrapper follows the contract of the others: run(inputs) over a dict
of tensors.

run(inputs) with q [B, S, Hq, D] in bf16 or fp16 (D 64, 96, 128, 192 or 256), the cache's k_codes, k_scales, v_codes and
v_scales (as kv4_cache writes them: uint8 [pages, Hk, block_size, D / 2] and [..., D / 32], contiguous), block_tables int32
[B, N] with seq_lens int32 [B], and optionally scale (1 / sqrt(D)) returns {"out"} [B, S, Hq, D]. Key t of a sequence is
row t % block_size of page block_tables[b, t // block_size]. Query i of sequence b stands at place seq_lens[b] - S + i: it
sees the keys up to its place, and is zero where its place is below zero.

The lengths stay on the device, so a captured call follows them from replay to replay. A q whose strides are whole
16-byte vectors is taken as it is.

Library: libkernel.so from the directory named by CKOPT_BUILD_DIR, or this package's build/kv4_attention/ when that
variable is unset. A missing library is an ImportError; there is no CPU path.

Errors: ValueError before any launch for an input the kernels do not take, RuntimeError carrying the HIP error code
when the launch reports one.
"""

import ctypes
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
_DTYPES = {torch.bfloat16: 1, torch.float16: 2}
_HEAD_DIMS = (64, 96, 128, 192, 256)
_MOST_KEYS = 1 << 30  # of a table
CACHE = ("k_codes", "k_scales", "v_codes", "v_scales")

LIB_PATH = os.path.join(os.environ.get("CKOPT_BUILD_DIR") or os.path.join(_HERE, "..", "build", "kv4_attention"),
                        "libkernel.so")
if not os.path.exists(LIB_PATH):
    raise ImportError(f"kv4_attention: no library at {LIB_PATH}; run make_libs.py first")
_lib = ctypes.CDLL(LIB_PATH)
_lib.kv4_attention_work.argtypes = [ctypes.c_longlong] * 2 + [ctypes.c_int] * 3 + [ctypes.c_longlong] * 2
_lib.kv4_attention_work.restype = ctypes.c_longlong
_lib.kv4_attention_launch.argtypes = [ctypes.c_void_p] * 9 + [ctypes.c_longlong, ctypes.c_void_p] + \
    [ctypes.c_longlong] * 3 + [ctypes.c_int] * 3 + [ctypes.c_longlong] * 2 + [ctypes.c_float, ctypes.c_int,
                                                                              ctypes.c_void_p]
_lib.kv4_attention_launch.restype = ctypes.c_int


def _in_vectors(q):
    """Whether the heads of q are whole 16-byte vectors where they lie."""
    return q.stride(3) == 1 and q.data_ptr() % 16 == 0 and \
        all(s % 8 == 0 or n == 1 for s, n in zip(q.stride()[:3], q.shape))


def _reject(q, cache, tables, lens, scale):
    """A short reason when these arguments cannot go to the kernels, else None."""
    if q.dtype not in _DTYPES or q.dim() != 4 or q.shape[3] not in _HEAD_DIMS or not 1 <= q.shape[2] <= 65536:
        return f"q {q.dtype} {tuple(q.shape)}"
    if any(t.dtype != torch.uint8 or t.dim() != 4 or not t.is_contiguous() for t in cache):
        return "a cache of " + ", ".join(f"{t.dtype} {tuple(t.shape)}" for t in cache)
    pages, heads, block, half = cache[0].shape
    if 2 * half != q.shape[3] or cache[2].shape != cache[0].shape or \
            any(t.shape != (pages, heads, block, half // 16) for t in cache[1::2]):
        return "a cache of " + ", ".join(str(tuple(t.shape)) for t in cache) + f" for heads of {q.shape[3]}"
    if heads < 1 or q.shape[2] % heads:
        return f"{q.shape[2]} query heads over {heads} kv heads"
    if tables.dtype != torch.int32 or tables.dim() != 2 or tables.shape[0] != q.shape[0] or \
            lens.dtype != torch.int32 or tuple(lens.shape) != (q.shape[0],):
        return f"block_tables {tables.dtype} {tuple(tables.shape)}, seq_lens {lens.dtype} {tuple(lens.shape)}"
    if not 1 <= block <= _MOST_KEYS or tables.shape[1] > _MOST_KEYS // block or pages * block >= 1 << 31:
        return f"{pages} pages of {block} with tables of {tables.shape[1]}"
    if scale is not None and not 1e-30 <= scale <= 1e30:
        return f"scale {scale}"
    tensors = (q, *cache, tables, lens)
    if any(t.device != q.device for t in tensors) or q.device.type != "cuda":
        return "devices " + ", ".join(str(t.device) for t in tensors)
    if any(t.data_ptr() % 16 for t in cache[::2]):
        return "codes that are not 16-byte aligned"
    return None


def run(inputs):
    q, cache = inputs["q"], [inputs[n] for n in CACHE]
    tables, lens, scale = inputs["block_tables"], inputs["seq_lens"], inputs.get("scale")
    reason = _reject(q, cache, tables, lens, scale)
    if reason:
        raise ValueError(f"kv4_attention candidate: {reason}")
    batch, seq, q_heads, head_dim = q.shape
    pages, kv_heads, block, _ = cache[0].shape
    with torch.cuda.device(q.device):
        if not _in_vectors(q):
            q = q.clone(memory_format=torch.contiguous_format)
        tables, lens = tables.contiguous(), lens.contiguous()
        out = torch.empty((batch, seq, q_heads, head_dim), dtype=q.dtype, device=q.device)
        sizes = q_heads, kv_heads, head_dim, tables.shape[1], block
        size = _lib.kv4_attention_work(batch, seq, *sizes)
        work = torch.empty(size, dtype=torch.uint8, device=q.device) if size > 0 else None
        err = _lib.kv4_attention_launch(
            q.data_ptr(), *(t.data_ptr() for t in cache), tables.data_ptr(), lens.data_ptr(), out.data_ptr(),
            None if work is None else work.data_ptr(), size, (ctypes.c_longlong * 3)(*q.stride()[:3]), batch, seq,
            pages, *sizes, head_dim ** -0.5 if scale is None else scale, _DTYPES[q.dtype],
            torch.cuda.current_stream(q.device).cuda_stream)
    if err == -1:
        raise ValueError(f"kv4_attention candidate: q {tuple(q.shape)} with tables of {tables.shape[1]} is too large")
    if err:
        raise RuntimeError(f"kernel launch failed: HIP error {err}")
    return {"out": out}
