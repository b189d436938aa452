"""Attention of a batch's last tokens over one paged prefix that all of it shares and over each sequence's own paged
keys, served by this package's MI355X library. No counterpart in the reference; the wrapper follows the contract of the
others: run(inputs) over a dict of tensors.

run(inputs) with q [B, S, Hq, D] in bf16 or fp16 (D 64, 80, 96, 128, 192 or 256), k_cache and v_cache (contiguous
[slots, Hk, D], as rope_kv and qk_norm_rope_kv write them), prefix_table int32 [P] with prefix_len int32 [1],
block_tables int32 [B, N] with seq_lens int32 [B], block_size, and optionally scale (1 / sqrt(D)) returns {"out"}
[B, S, Hq, D]. Key t of a table is in slot table[t // block_size] * block_size + t % block_size. Query i of sequence b
stands at own place seq_lens[b] - S + i: it sees the whole prefix and the own keys up to its place, and is zero where
its place is below zero. An empty prefix_table leaves plain paged attention.

The lengths stay on the device, so a captured call follows them from replay to replay. A q whose strides are whole
16-byte vectors is taken as it is.

Library: libkernel.so from the directory named by CKOPT_BUILD_DIR, or this package's build/shared_prefix_attention/ when
that variable is unset. A missing library is an ImportError; there is no CPU path.

Errors: ValueError before any launch for an input the kernels do not take, RuntimeError carrying the HIP error code
when the launch reports one.
"""

import ctypes
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
_DTYPES = {torch.bfloat16: 1, torch.float16: 2}
_HEAD_DIMS = (64, 80, 96, 128, 192, 256)
_MOST_KEYS = 1 << 30  # of a table

LIB_PATH = os.path.join(os.environ.get("CKOPT_BUILD_DIR") or
                        os.path.join(_HERE, "..", "build", "shared_prefix_attention"), "libkernel.so")
if not os.path.exists(LIB_PATH):
    raise ImportError(f"shared_prefix_attention: no library at {LIB_PATH}; run make_libs.py first")
_lib = ctypes.CDLL(LIB_PATH)
_lib.prefix_attention_work.argtypes = [ctypes.c_longlong] * 2 + [ctypes.c_int] * 3 + [ctypes.c_longlong] * 3
_lib.prefix_attention_work.restype = ctypes.c_longlong
_lib.prefix_attention_launch_sized.argtypes = [ctypes.c_void_p] * 9 + [ctypes.c_longlong, ctypes.c_void_p] + \
    [ctypes.c_longlong] * 3 + [ctypes.c_int] * 3 + [ctypes.c_longlong] * 3 + [ctypes.c_float, ctypes.c_int,
                                                                              ctypes.c_void_p]
_lib.prefix_attention_launch_sized.restype = ctypes.c_int


def _in_vectors(q):
    """Whether the heads of q are whole 16-byte vectors where they lie."""
    return q.stride(3) == 1 and q.data_ptr() % 16 == 0 and \
        all(s % 8 == 0 or n == 1 for s, n in zip(q.stride()[:3], q.shape))


def _reject(q, kc, vc, table, length, tables, lens, block, scale):
    """A short reason when these arguments cannot go to the kernels, else None."""
    if q.dtype not in _DTYPES or q.dim() != 4 or q.shape[3] not in _HEAD_DIMS or not 1 <= q.shape[2] <= 65536:
        return f"q {q.dtype} {tuple(q.shape)}"
    if any(c.dtype != q.dtype or c.dim() != 3 or c.shape[2] != q.shape[3] or not c.is_contiguous()
           for c in (kc, vc)) or kc.shape != vc.shape:
        return f"caches {kc.dtype} {tuple(kc.shape)}, {vc.dtype} {tuple(vc.shape)} (contiguous [slots, Hk, " \
               f"{q.shape[3]}] of q's dtype)"
    if kc.shape[1] < 1 or q.shape[2] % kc.shape[1]:
        return f"{q.shape[2]} query heads over {kc.shape[1]} kv heads"
    if table.dtype != torch.int32 or table.dim() != 1 or length.dtype != torch.int32 or tuple(length.shape) != (1,):
        return f"prefix_table {table.dtype} {tuple(table.shape)}, prefix_len {length.dtype} {tuple(length.shape)}"
    if tables.dtype != torch.int32 or tables.dim() != 2 or tables.shape[0] != q.shape[0] or \
            lens.dtype != torch.int32 or tuple(lens.shape) != (q.shape[0],):
        return f"block_tables {tables.dtype} {tuple(tables.shape)}, seq_lens {lens.dtype} {tuple(lens.shape)}"
    if not 1 <= block <= _MOST_KEYS or max(table.shape[0], tables.shape[1]) > _MOST_KEYS // block:
        return f"block_size {block} with tables of {table.shape[0]} and {tables.shape[1]} blocks"
    if scale is not None and not 1e-30 <= scale <= 1e30:
        return f"scale {scale}"
    tensors = (q, kc, vc, table, length, tables, lens)
    if any(t.device != q.device for t in tensors) or q.device.type != "cuda":
        return "devices " + ", ".join(str(t.device) for t in tensors)
    return None


def run(inputs):
    q, kc, vc = inputs["q"], inputs["k_cache"], inputs["v_cache"]
    table, length, tables, lens = (inputs[n] for n in ("prefix_table", "prefix_len", "block_tables", "seq_lens"))
    block, scale = int(inputs["block_size"]), inputs.get("scale")
    reason = _reject(q, kc, vc, table, length, tables, lens, block, scale)
    if reason is None and (kc.data_ptr() % 16 or vc.data_ptr() % 16):
        reason = "caches that are not 16-byte aligned"
    if reason:
        raise ValueError(f"shared_prefix_attention candidate: {reason}")
    batch, seq, q_heads, head_dim = q.shape
    with torch.cuda.device(q.device):
        if not _in_vectors(q):
            q = q.clone(memory_format=torch.contiguous_format)
        table, tables, lens = table.contiguous(), tables.contiguous(), lens.contiguous()
        out = torch.empty((batch, seq, q_heads, head_dim), dtype=q.dtype, device=q.device)
        sizes = q_heads, kc.shape[1], head_dim, table.shape[0], tables.shape[1], block
        size = _lib.prefix_attention_work(batch, seq, *sizes)
        work = torch.empty(size, dtype=torch.uint8, device=q.device) if size > 0 else None
        err = _lib.prefix_attention_launch_sized(
            q.data_ptr(), kc.data_ptr(), vc.data_ptr(), table.data_ptr(), length.data_ptr(), tables.data_ptr(),
            lens.data_ptr(), out.data_ptr(), None if work is None else work.data_ptr(), size,
            (ctypes.c_longlong * 3)(*q.stride()[:3]), batch, seq, kc.shape[0], *sizes,
            head_dim ** -0.5 if scale is None else scale, _DTYPES[q.dtype],
            torch.cuda.current_stream(q.device).cuda_stream)
    if err == -1:
        raise ValueError(f"shared_prefix_attention candidate: q {tuple(q.shape)} with {kc.shape[0]} slots is too large")
    if err:
        raise RuntimeError(f"kernel launch failed: HIP error {err}")
    return {"out": out}
