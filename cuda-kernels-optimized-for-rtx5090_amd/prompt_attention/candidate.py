"""Causal attention of whole prompts, packed one behind the other, over their own keys, served by this package's MI355X
library. No counterpart in the reference; the wrapper follows the contract of the others: run(inputs) over a dict of
tensors.

run(inputs) with q [T, Hq, D], k and v [T, Hk, D] in bf16 or fp16 (D 64, 80, 96, 128, 192 or 256), cu_seqlens int32 [B + 1]
and optionally scale (1 / sqrt(D)) returns {"out"} [T, Hq, D]. Prompt b is tokens cu_seqlens[b] to cu_seqlens[b + 1]; token
i of a prompt sees its tokens 0 to i. Tokens of no prompt (padding before the first offset or behind the last) are zeros.

The offsets stay on the device, so a captured call follows them from replay to replay. q, k and v whose strides are whole
16-byte vectors (the parts of a packed projection) are taken as they are.

Library: libkernel.so from the directory named by CKOPT_BUILD_DIR, or this package's build/prompt_attention/ when that
variable is unset. A missing library is an ImportError; there is no CPU path.

Errors: ValueError before any launch for an input the kernels do not take, RuntimeError carrying the HIP error code
when the launch reports one.
"""

import ctypes
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
_DTYPES = {torch.bfloat16: 1, torch.float16: 2}
_HEAD_DIMS = (64, 80, 96, 128, 192, 256)

LIB_PATH = os.path.join(os.environ.get("CKOPT_BUILD_DIR") or os.path.join(_HERE, "..", "build", "prompt_attention"),
                        "libkernel.so")
if not os.path.exists(LIB_PATH):
    raise ImportError(f"prompt_attention: no library at {LIB_PATH}; run make_libs.py first")
_lib = ctypes.CDLL(LIB_PATH)
_lib.prompt_attention_launch.argtypes = [ctypes.c_void_p] * 6 + [ctypes.c_longlong] * 2 + [ctypes.c_int] * 3 + [
    ctypes.c_float, ctypes.c_int, ctypes.c_void_p]
_lib.prompt_attention_launch.restype = ctypes.c_int


def _in_vectors(t):
    """Whether the heads of t are whole 16-byte vectors where they lie, its tokens no further apart than 2^23."""
    return t.stride(2) == 1 and t.data_ptr() % 16 == 0 and (t.shape[0] == 1 or t.stride(0) <= 1 << 23) and \
        all(s % 8 == 0 or n == 1 for s, n in zip(t.stride()[:2], t.shape))


def _reject(q, k, v, offsets, scale):
    """A short reason when these arguments cannot go to the kernel, else None."""
    if q.dtype not in _DTYPES or q.dim() != 3 or q.shape[2] not in _HEAD_DIMS or not 1 <= q.shape[1] <= 65536:
        return f"q {q.dtype} {tuple(q.shape)}"
    if any(t.dtype != q.dtype or t.dim() != 3 or t.shape[0] != q.shape[0] or t.shape[2] != q.shape[2]
           for t in (k, v)) or k.shape != v.shape:
        return f"k {k.dtype} {tuple(k.shape)}, v {v.dtype} {tuple(v.shape)} for q {q.dtype} {tuple(q.shape)}"
    if k.shape[1] < 1 or q.shape[1] % k.shape[1]:
        return f"{q.shape[1]} query heads over {k.shape[1]} kv heads"
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 1:
        return f"cu_seqlens {offsets.dtype} {tuple(offsets.shape)}"
    if scale is not None and not 1e-30 <= scale <= 1e30:
        return f"scale {scale}"
    tensors = (q, k, v, offsets)
    if any(t.device != q.device for t in tensors) or q.device.type != "cuda":
        return "devices " + ", ".join(str(t.device) for t in tensors)
    return None


def run(inputs):
    q, k, v, offsets, scale = (inputs.get(n) for n in ("q", "k", "v", "cu_seqlens", "scale"))
    reason = _reject(q, k, v, offsets, scale)
    if reason:
        raise ValueError(f"prompt_attention candidate: {reason}")
    tokens, q_heads, head_dim = q.shape
    with torch.cuda.device(q.device):
        q, k, v = (t if _in_vectors(t) else t.clone(memory_format=torch.contiguous_format) for t in (q, k, v))
        offsets = offsets.contiguous()
        out = torch.empty((tokens, q_heads, head_dim), dtype=q.dtype, device=q.device)
        strides = (ctypes.c_longlong * 6)(*(s for t in (q, k, v) for s in t.stride()[:2]))
        err = _lib.prompt_attention_launch(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), offsets.data_ptr(), out.data_ptr(), strides, tokens,
            offsets.shape[0] - 1, q_heads, k.shape[1], head_dim, head_dim ** -0.5 if scale is None else scale,
            _DTYPES[q.dtype], torch.cuda.current_stream(q.device).cuda_stream)
    if err == -1:
        raise ValueError(f"prompt_attention candidate: q {tuple(q.shape)} of {offsets.shape[0] - 1} prompts is too large")
    if err:
        raise RuntimeError(f"kernel launch failed: HIP error {err}")
    return {"out": out}
