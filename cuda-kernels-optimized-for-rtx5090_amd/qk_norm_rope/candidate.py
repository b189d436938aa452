"""RMS norm of every query and key head with the rotary embedding in the same pass, and the paged KV-cache append on top
of it, served by this package's MI355X library. No counterpart in the reference; the wrapper follows the contract of the
others: run(inputs) over a dict of tensors.

run(inputs) with q [B, S, Hq, D] and k [B, S, Hk, D] in bf16 or fp16, position_ids int64 [B, S] and inv_freq fp32 [r/2]
(r <= D: the first r elements of a head are rotated, i with i + r/2) returns {"q_out", "k_out"}. Optional: q_weight and
k_weight [D] of q's dtype, eps (1e-6), and inplace (q and k are overwritten and returned). Everything between the load
and the store of an element is fp32; the angles pos * inv_freq are not rounded.

With v [B, S, Hk, D], k_cache, v_cache (contiguous [slots, Hk, D]) and slot_mapping (int64 [B, S]) the normed and
rotated k and the untouched v go to the cache rows that slot_mapping names (a slot outside the cache: not written; no
two tokens may share a slot), and {"q_out", "k_cache", "v_cache"} is returned; inplace then overwrites q. In place, q
shares no element with k (nor v); views of one packed projection are told apart by their strides.

Tensors whose last dimension is contiguous are taken as they are, so the parts of a packed projection need no copy.

Library: libkernel.so from the directory named by CKOPT_BUILD_DIR, or this package's build/qk_norm_rope/ when that
variable is unset. A missing library is an ImportError; there is no CPU path.

Errors: ValueError before any launch for an input the kernels do not take, RuntimeError carrying the HIP error code
when the launch reports one.
"""

import ctypes
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
_DTYPES = {torch.bfloat16: 1, torch.float16: 2}

LIB_PATH = os.path.join(os.environ.get("CKOPT_BUILD_DIR") or os.path.join(_HERE, "..", "build", "qk_norm_rope"),
                        "libkernel.so")
if not os.path.exists(LIB_PATH):
    raise ImportError(f"qk_norm_rope: no library at {LIB_PATH}; run make_libs.py first")
_lib = ctypes.CDLL(LIB_PATH)
_lib.qk_norm_rope_launch.argtypes = [ctypes.c_void_p] * 9 + [ctypes.c_longlong] * 2 + [ctypes.c_int] * 5 + \
    [ctypes.c_float, ctypes.c_void_p]
_lib.qk_norm_rope_launch.restype = ctypes.c_int
_lib.qk_norm_rope_kv_launch.argtypes = [ctypes.c_void_p] * 12 + [ctypes.c_longlong] * 3 + [ctypes.c_int] * 5 + \
    [ctypes.c_float, ctypes.c_void_p]
_lib.qk_norm_rope_kv_launch.restype = ctypes.c_int


def _spread(t):
    """Whether no two elements of t share memory, by its strides."""
    reach = 0
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if stride <= reach:
            return False
        reach += stride * (size - 1)
    return True


def _overlap(a, b):
    """Whether the memory from a's first to its last element meets b's."""
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + t.element_size() *
                           (1 + sum(s * (n - 1) for s, n in zip(t.stride(), t.shape)))) for t in (a, b))
    return a0 < b1 and b0 < a1


def _apart(a, b):
    """Whether the strides of a and b, of one dtype, show that they share no element: their memory does not meet, or
    they are different parts of a period that the larger strides of both repeat (views of one packed projection)."""
    if not _overlap(a, b):
        return True
    shift, odd = divmod(b.data_ptr() - a.data_ptr(), a.element_size())
    dims = [[(st, n) for st, n in zip(t.stride(), t.shape) if n > 1] for t in (a, b)]
    for period in {st for d in dims for st, _ in d if st > 0} if not odd else ():
        if any(st >= period and st % period for d in dims for st, _ in d):
            continue
        length_a, length_b = (1 + sum(st * (n - 1) for st, n in d if st < period) for d in dims)
        if length_a <= shift % period and shift % period + length_b <= period:
            return True
    return False


def _reject(q, k, ids, inv_freq, weights, inplace):
    """A short reason when these tensors cannot go to the kernels, else None."""
    if q.dtype not in _DTYPES or k.dtype != q.dtype:
        return f"dtypes q {q.dtype}, k {k.dtype}"
    if ids.dtype != torch.int64 or q.dim() != 4 or k.dim() != 4 or ids.dim() != 2:
        return f"position_ids {ids.dtype} {tuple(ids.shape)}, q {tuple(q.shape)}, k {tuple(k.shape)}"
    if q.shape[:2] != ids.shape or k.shape[:2] != ids.shape or q.shape[3] != k.shape[3] or 0 in q.shape[2:] or \
            k.shape[2] == 0 or q.shape[3] > 65536:
        return f"shapes q {tuple(q.shape)}, k {tuple(k.shape)}, position_ids {tuple(ids.shape)}"
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or 2 * inv_freq.shape[0] > q.shape[3]:
        return f"inv_freq {inv_freq.dtype} {tuple(inv_freq.shape)}"
    for name, w in zip(("q_weight", "k_weight"), weights):
        if w is not None and (w.dtype != q.dtype or tuple(w.shape) != (q.shape[3],)):
            return f"{name} {w.dtype} {tuple(w.shape)}"
    tensors = [q, k, ids, inv_freq] + [w for w in weights if w is not None]
    if any(t.device != q.device for t in tensors) or q.device.type != "cuda":
        return "devices " + ", ".join(str(t.device) for t in tensors)
    if inplace and any(t.stride(3) != 1 or not _spread(t) for t in (q, k)):
        return "an in-place call needs q and k with a contiguous last dimension and no shared elements"
    return None


def _rows(t):
    return t if t.stride(3) == 1 else t.contiguous()


def _strides(*tensors):
    return (ctypes.c_longlong * 12)(*(s for t in tensors for s in t.stride()[:3]))


def run(inputs):
    q, k, ids, inv_freq = inputs["q"], inputs["k"], inputs["position_ids"], inputs["inv_freq"]
    weights = inputs.get("q_weight"), inputs.get("k_weight")
    inplace, cached = bool(inputs.get("inplace", False)), "k_cache" in inputs
    reason = _reject(q, k, ids, inv_freq, weights, inplace)
    if reason is None and inplace and not _apart(q, k):
        reason = "q and k are one tensor, or share elements"
    if reason is None and cached:
        v, kc, vc, slots = inputs["v"], inputs["k_cache"], inputs["v_cache"], inputs["slot_mapping"]
        if v.dtype != q.dtype or v.shape != k.shape or v.device != q.device:
            reason = f"v {v.dtype} {tuple(v.shape)} {v.device}"
        elif any(c.dtype != q.dtype or c.dim() != 3 or c.shape[1:] != k.shape[2:] or not c.is_contiguous()
                 or c.device != q.device for c in (kc, vc)) or kc.shape != vc.shape:
            reason = f"caches {tuple(kc.shape)} {tuple(vc.shape)} (contiguous [slots, {k.shape[2]}, {k.shape[3]}] " \
                     "of q's dtype)"
        elif _overlap(kc, vc) or any(_overlap(t, c) for t in (q, k, v) for c in (kc, vc)):
            reason = "caches that share memory with each other or with q, k or v"
        elif inplace and not _apart(q, v):
            reason = "q, which is overwritten, shares elements with v"
        elif slots.dtype != torch.int64 or slots.shape != ids.shape or slots.device != q.device:
            reason = f"slot_mapping {slots.dtype} {tuple(slots.shape)}"
    if reason:
        raise ValueError(f"qk_norm_rope candidate: {reason}")
    batch, seq, q_heads, head_dim = q.shape
    eps = float(inputs.get("eps", 1e-6))
    with torch.cuda.device(q.device):
        q, k, ids, inv_freq = _rows(q), _rows(k), ids.contiguous(), inv_freq.contiguous()
        weights = [None if w is None else w.contiguous() for w in weights]
        pointers = [None if w is None else w.data_ptr() for w in weights]
        sizes = q_heads, k.shape[2], head_dim, 2 * inv_freq.shape[0], _DTYPES[q.dtype], eps
        stream = torch.cuda.current_stream(q.device).cuda_stream
        q_out = q if inplace else torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if cached:
            v, slots = _rows(v), slots.contiguous()
            err = _lib.qk_norm_rope_kv_launch(q.data_ptr(), k.data_ptr(), v.data_ptr(), ids.data_ptr(),
                                              inv_freq.data_ptr(), *pointers, q_out.data_ptr(), kc.data_ptr(),
                                              vc.data_ptr(), slots.data_ptr(), _strides(q, k, v, q_out), batch, seq,
                                              kc.shape[0], *sizes, stream)
            out = {"q_out": q_out, "k_cache": kc, "v_cache": vc}
        else:
            k_out = k if inplace else torch.empty(k.shape, dtype=k.dtype, device=k.device)
            err = _lib.qk_norm_rope_launch(q.data_ptr(), k.data_ptr(), ids.data_ptr(), inv_freq.data_ptr(), *pointers,
                                           q_out.data_ptr(), k_out.data_ptr(), _strides(q, k, q_out, k_out), batch, seq,
                                           *sizes, stream)
            out = {"q_out": q_out, "k_out": k_out}
    if err == -1:
        raise ValueError(f"qk_norm_rope candidate: q {tuple(q.shape)} with {sizes[1]} kv heads is too large")
    if err:
        raise RuntimeError(f"kernel launch failed: HIP error {err}")
    return out
