"""Verification of drafted tokens against a target model's probabilities, served by this package's MI355X library. No
counterpart in the reference; the wrapper follows the contract of the others: run(inputs) over a dict of tensors.

run(inputs) with target_probs [B, S + 1, V] in fp32 or bf16, draft_tokens int64 [B, S], uniforms fp32 [B, S + 1] in
[0, 1) and optionally draft_probs [B, S, V] of target_probs' dtype and draft_lens int32 [B] (how many of a sequence's S
drafts count) returns {"tokens": int64 [B, S + 1], "accepted": int64 [B]}. Draft i is kept while uniforms[i] *
draft_probs[i, token] < target_probs[i, token]; behind the kept ones one token is drawn with the last uniform, from what
the refused draft's probabilities leave of the target's, or from the target's next row where all were kept. tokens holds
the kept drafts, the drawn token and -1. Without draft_probs the drafts count as certain (a prompt lookup, a greedy
draft model). Every comparison and sum is fp64: the result is that of the formula.

Probabilities with a contiguous last dimension are taken as they are.

Library: libkernel.so from the directory named by CKOPT_BUILD_DIR, or this package's build/verify_drafts/ when that
variable is unset. A missing library is an ImportError; there is no CPU path.

Errors: ValueError before any launch for an input the kernel does not take, RuntimeError carrying the HIP error code
when the launch reports one.
"""

import ctypes
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
_CODE = {torch.float32: 0, torch.bfloat16: 1}

LIB_PATH = os.path.join(os.environ.get("CKOPT_BUILD_DIR") or os.path.join(_HERE, "..", "build", "verify_drafts"),
                        "libkernel.so")
if not os.path.exists(LIB_PATH):
    raise ImportError(f"verify_drafts: no library at {LIB_PATH}; run make_libs.py first")
_lib = ctypes.CDLL(LIB_PATH)
for _name in ("verify_plan", "verify_work"):
    getattr(_lib, _name).argtypes = [ctypes.c_longlong, ctypes.c_longlong, ctypes.c_int]
    getattr(_lib, _name).restype = ctypes.c_longlong
_lib.verify_launch.argtypes = [ctypes.c_void_p] * 10 + [ctypes.c_longlong, ctypes.c_int, ctypes.c_longlong,
                                                        ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
_lib.verify_launch.restype = ctypes.c_int

# (device, stream) -> int32 zeros, which a launch leaves at zero; streams may overlap, so each has its own. Rows are
# split over workgroups only where they are few (verify_plan: fewer than two for every five CUs).
_counters = {}
_COUNTERS = 4096


def _counters_for(device, stream, rows):
    if torch.cuda.is_current_stream_capturing():
        # a captured launch clears counters of its own at every replay: two graphs that replay at once share none
        return torch.zeros(rows, dtype=torch.int32, device=device)
    if rows > _COUNTERS:
        raise RuntimeError(f"verify_drafts: {rows} rows of several workgroups each")
    c = _counters.get((device, stream))
    if c is None:
        c = _counters[device, stream] = torch.zeros(_COUNTERS, dtype=torch.int32, device=device)
    return c


def _reject(target, draft, tokens, uniforms, lens):
    """A short reason when these tensors cannot go to the kernel, else None."""
    if target.dtype not in _CODE or target.dim() != 3 or not 1 <= target.shape[1] <= 65536 or \
            not 1 <= target.shape[2] <= 1 << 28 or target.shape[0] > 1 << 22:
        return f"target_probs {target.dtype} {tuple(target.shape)}"
    batch, drafts = target.shape[0], target.shape[1] - 1
    if tokens.dtype != torch.int64 or tuple(tokens.shape) != (batch, drafts):
        return f"draft_tokens {tokens.dtype} {tuple(tokens.shape)}"
    if uniforms.dtype != torch.float32 or tuple(uniforms.shape) != (batch, drafts + 1):
        return f"uniforms {uniforms.dtype} {tuple(uniforms.shape)}"
    if draft is not None and (draft.dtype != target.dtype or tuple(draft.shape) != (batch, drafts, target.shape[2])):
        return f"draft_probs {draft.dtype} {tuple(draft.shape)}"
    if lens is not None and (lens.dtype != torch.int32 or tuple(lens.shape) != (batch,)):
        return f"draft_lens {lens.dtype} {tuple(lens.shape)}"
    tensors = [target, tokens, uniforms] + [t for t in (draft, lens) if t is not None]
    if any(t.device != target.device for t in tensors) or target.device.type != "cuda":
        return "devices " + ", ".join(str(t.device) for t in tensors)
    return None


def run(inputs):
    target, draft, lens = inputs["target_probs"], inputs.get("draft_probs"), inputs.get("draft_lens")
    tokens, uniforms = inputs["draft_tokens"], inputs["uniforms"]
    reason = _reject(target, draft, tokens, uniforms, lens)
    if reason:
        raise ValueError(f"verify_drafts candidate: {reason}")
    batch, rows, vocabulary = target.shape
    with torch.cuda.device(target.device):
        target = target if target.stride(2) == 1 else target.contiguous()
        if draft is not None:
            draft = draft if draft.stride(2) == 1 else draft.contiguous()
        tokens, uniforms = tokens.contiguous(), uniforms.contiguous()
        lens = None if lens is None else lens.contiguous()
        stream = torch.cuda.current_stream(target.device).cuda_stream
        code = _CODE[target.dtype]
        blocks = _lib.verify_plan(batch, vocabulary, code)
        work = counters = None
        if blocks > 1:
            work = torch.empty(_lib.verify_work(batch, vocabulary, code), dtype=torch.float64, device=target.device)
            counters = _counters_for(target.device, stream, batch)
        out = torch.empty((batch, rows), dtype=torch.int64, device=target.device)
        accepted = torch.empty((batch,), dtype=torch.int64, device=target.device)
        strides = (ctypes.c_longlong * 4)(*target.stride()[:2], *(draft.stride()[:2] if draft is not None else (0, 0)))
        pointers = [None if t is None else t.data_ptr() for t in (target, draft, tokens, lens, uniforms, out, accepted,
                                                                  work, counters)]
        if rows == 1:
            pointers[1] = None  # no drafts: nothing to read
        err = _lib.verify_launch(*pointers, strides, batch, rows - 1, vocabulary, code, blocks, stream)
    if err:
        raise RuntimeError(f"kernel launch failed: HIP error {err}")
    return {"tokens": out, "accepted": accepted}
