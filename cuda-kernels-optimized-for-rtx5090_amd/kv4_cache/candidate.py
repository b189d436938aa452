"""A paged cache of keys and values in 4 bits, served by this package's MI355X library: appending tokens to it and
reading them back. No counterpart in the reference; the wrapper follows the contract of the others: run(inputs) over a
dict of tensors.

The cache: k_codes and v_codes uint8 [pages, Hk, block_size, D / 2], k_scales and v_scales uint8 [pages, Hk, block_size,
D / 32], all contiguous (D 64, 96, 128, 192 or 256); slot s is row s % block_size of page s // block_size. A byte of codes
holds elements 2 i (low half) and 2 i + 1 in e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6, bit 3 the sign), a scale byte b is the
2^(b - 127) that 32 elements share (above 252: a group of NaN).

run(inputs) with k and v [T, Hk, D] in bf16 or fp16, slot_mapping int64 [T] and the four cache tensors writes token t to
slot slot_mapping[t] (outside the cache: nothing; slots are distinct) and returns the cache's tensors. A group's scale is
the least power of two that leaves its largest magnitude below 7; its elements go to the nearest value, ties to the even
code; one with an infinity or a NaN becomes NaN. k and v whose strides are whole 16-byte vectors are taken as they are.

read(k_codes, k_scales, v_codes, v_scales, slots, dtype) returns (k, v) [T, Hk, D] of the slots int64 [T] (outside the
cache: zeros) in bf16 or fp16.

Library: libkernel.so from the directory named by CKOPT_BUILD_DIR, or this package's build/kv4_cache/ when that variable
is unset. A missing library is an ImportError; there is no CPU path.

Errors: ValueError before any launch for an input the kernels do not take, RuntimeError carrying the HIP error code
when the launch reports one.
"""

import ctypes
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
_DTYPES = {torch.bfloat16: 1, torch.float16: 2}
_HEAD_DIMS = (64, 96, 128, 192, 256)
CACHE = ("k_codes", "k_scales", "v_codes", "v_scales")

LIB_PATH = os.path.join(os.environ.get("CKOPT_BUILD_DIR") or os.path.join(_HERE, "..", "build", "kv4_cache"),
                        "libkernel.so")
if not os.path.exists(LIB_PATH):
    raise ImportError(f"kv4_cache: no library at {LIB_PATH}; run make_libs.py first")
_lib = ctypes.CDLL(LIB_PATH)
_lib.kv4_append_launch.argtypes = [ctypes.c_void_p] * 8 + [ctypes.c_longlong] * 2 + [ctypes.c_int] * 4 + [
    ctypes.c_void_p]
_lib.kv4_append_launch.restype = ctypes.c_int
_lib.kv4_read_launch.argtypes = [ctypes.c_void_p] * 7 + [ctypes.c_longlong] * 2 + [ctypes.c_int] * 4 + [ctypes.c_void_p]
_lib.kv4_read_launch.restype = ctypes.c_int


def _span(t):
    first = t.data_ptr()
    return first, first + t.element_size() * (1 + sum(s * (n - 1) for s, n in zip(t.stride(), t.shape)))


def _overlap(a, b):
    """Whether the memory from a's first to its last element meets b's."""
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def _in_vectors(t):
    """Whether the heads of t are whole 16-byte vectors where they lie."""
    return t.stride(2) == 1 and t.data_ptr() % 16 == 0 and \
        all(s % 8 == 0 or n == 1 for s, n in zip(t.stride()[:2], t.shape))


def reject_cache(cache, device):
    """A short reason when these are not the tensors of a cache on this device, else None."""
    codes, scales = cache[0], cache[1]
    if any(t.dtype != torch.uint8 or t.dim() != 4 or not t.is_contiguous() for t in cache):
        return "a cache of " + ", ".join(f"{t.dtype} {tuple(t.shape)}" for t in cache) + \
            " (contiguous uint8 [pages, Hk, block_size, ...])"
    if 2 * codes.shape[3] not in _HEAD_DIMS or scales.shape != (*codes.shape[:3], codes.shape[3] // 16) or \
            cache[2].shape != codes.shape or cache[3].shape != scales.shape or not 1 <= codes.shape[1] <= 65536 or \
            codes.shape[2] < 1 or codes.shape[0] * codes.shape[2] >= 1 << 31:
        return "a cache of " + ", ".join(str(tuple(t.shape)) for t in cache) + \
            f" (codes [pages, Hk, block_size, D / 2], scales [..., D / 32], D of {_HEAD_DIMS})"
    if any(t.device != device for t in cache) or device.type != "cuda":
        return "devices " + ", ".join(str(t.device) for t in (*cache, torch.empty(0, device=device)))
    if any(t.data_ptr() % 16 for t in (cache[0], cache[2])):
        return "codes that are not 16-byte aligned"
    return None


def _sizes(cache):
    pages, heads, block, half = cache[0].shape
    return pages, heads, 2 * half, block


def _launched(err, what):
    if err == -1:
        raise ValueError(f"kv4_cache candidate: {what} is too large")
    if err:
        raise RuntimeError(f"kernel launch failed: HIP error {err}")


def run(inputs):
    k, v, slots = inputs["k"], inputs["v"], inputs["slot_mapping"]
    cache = [inputs[n] for n in CACHE]
    reason = None
    if k.dtype not in _DTYPES or v.dtype != k.dtype or k.dim() != 3 or v.shape != k.shape:
        reason = f"k {k.dtype} {tuple(k.shape)}, v {v.dtype} {tuple(v.shape)}"
    elif slots.dtype != torch.int64 or slots.shape != k.shape[:1]:
        reason = f"slot_mapping {slots.dtype} {tuple(slots.shape)}"
    elif any(t.device != k.device for t in (v, slots)):
        reason = f"devices {k.device}, {v.device}, {slots.device}"
    reason = reason or reject_cache(cache, k.device)
    if reason is None and (cache[0].shape[1] != k.shape[1] or 2 * cache[0].shape[3] != k.shape[2]):
        reason = f"k {tuple(k.shape)} into a cache of {tuple(cache[0].shape)}"
    if reason is None and any(_overlap(a, b) for i, a in enumerate(cache) for b in (*cache[i + 1:], k, v, slots)):
        reason = "a cache that shares memory within itself or with k, v or slot_mapping"
    if reason:
        raise ValueError(f"kv4_cache candidate: {reason}")
    pages, heads, dim, block = _sizes(cache)
    with torch.cuda.device(k.device):
        k, v = (t if _in_vectors(t) else t.clone(memory_format=torch.contiguous_format) for t in (k, v))
        slots = slots.contiguous()
        strides = (ctypes.c_longlong * 4)(*k.stride()[:2], *v.stride()[:2])
        _launched(_lib.kv4_append_launch(k.data_ptr(), v.data_ptr(), *(t.data_ptr() for t in cache), slots.data_ptr(),
                                         strides, k.shape[0], pages, heads, dim, block, _DTYPES[k.dtype],
                                         torch.cuda.current_stream(k.device).cuda_stream), f"k {tuple(k.shape)}")
    return dict(zip(CACHE, cache))


def read(k_codes, k_scales, v_codes, v_scales, slots, dtype=torch.bfloat16):
    cache = (k_codes, k_scales, v_codes, v_scales)
    reason = reject_cache(cache, k_codes.device)
    if reason is None and (slots.dtype != torch.int64 or slots.dim() != 1 or slots.device != k_codes.device):
        reason = f"slots {slots.dtype} {tuple(slots.shape)} {slots.device}"
    if reason is None and dtype not in _DTYPES:
        reason = f"dtype {dtype}"
    if reason:
        raise ValueError(f"kv4_cache candidate: {reason}")
    pages, heads, dim, block = _sizes(cache)
    with torch.cuda.device(k_codes.device):
        slots = slots.contiguous()
        k, v = (torch.empty((slots.shape[0], heads, dim), dtype=dtype, device=k_codes.device) for _ in range(2))
        _launched(_lib.kv4_read_launch(*(t.data_ptr() for t in cache), slots.data_ptr(), k.data_ptr(), v.data_ptr(),
                                       slots.shape[0], pages, heads, dim, block, _DTYPES[dtype],
                                       torch.cuda.current_stream(k.device).cuda_stream), f"k {tuple(k.shape)}")
    return k, v
