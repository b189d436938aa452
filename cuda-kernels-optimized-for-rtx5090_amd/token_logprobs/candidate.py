"""Log probabilities of given tokens with the entropy of their rows and the likeliest alternatives, served by this
package's MI355X library. No counterpart in the reference; the wrapper follows the contract of the others: run(inputs) over
a dict of tensors.

run(inputs) with logits [N, V] in fp32, bf16 or fp16, tokens int64 [N] and optionally top (0 to 64) returns {"logprobs"}
fp32 [N], {"entropy"} fp32 [N] in nats, {"top_logprobs"} fp32 [N, top] and {"top_indices"} int64 [N, top], of equal logits
the lowest index first (+0 above -0). A negative token (padding) has log probability 0, one beyond the vocabulary NaN; a row without a
distribution (a NaN, plus infinity, nothing above minus infinity) has NaN throughout and indices of -1. Rows may lie at
any distance.

Library: libkernel.so from the directory named by CKOPT_BUILD_DIR, or this package's build/token_logprobs/ when that
variable is unset. A missing library is an ImportError; there is no CPU path.

Errors: ValueError before any launch for an input the kernels do not take, RuntimeError carrying the HIP error code
when the launch reports one.
"""

import ctypes
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

LIB_PATH = os.path.join(os.environ.get("CKOPT_BUILD_DIR") or os.path.join(_HERE, "..", "build", "token_logprobs"),
                        "libkernel.so")
if not os.path.exists(LIB_PATH):
    raise ImportError(f"token_logprobs: no library at {LIB_PATH}; run make_libs.py first")
_lib = ctypes.CDLL(LIB_PATH)
_lib.token_logprobs_work.argtypes = [ctypes.c_longlong] * 2 + [ctypes.c_int] * 2
_lib.token_logprobs_work.restype = ctypes.c_longlong
_lib.token_logprobs_launch.argtypes = [ctypes.c_void_p] * 7 + [ctypes.c_longlong] * 4 + [ctypes.c_int] * 2 + [
    ctypes.c_void_p]
_lib.token_logprobs_launch.restype = ctypes.c_int


def _reject(logits, tokens, top):
    """A short reason when these arguments cannot go to the kernel, else None."""
    if logits.dtype not in _CODE or logits.dim() != 2 or not 1 <= logits.shape[1] <= 1 << 28 or \
            logits.shape[0] > 1 << 31:
        return f"logits {logits.dtype} {tuple(logits.shape)}"
    if tokens.dtype != torch.int64 or tokens.shape != logits.shape[:1]:
        return f"tokens {tokens.dtype} {tuple(tokens.shape)}"
    if not 0 <= top <= min(64, logits.shape[1]):
        return f"top {top} of {logits.shape[1]}"
    if tokens.device != logits.device or logits.device.type != "cuda":
        return f"devices {logits.device}, {tokens.device}"
    return None


def run(inputs):
    logits, tokens, top = inputs["logits"], inputs["tokens"], int(inputs.get("top", 0))
    reason = _reject(logits, tokens, top)
    if reason:
        raise ValueError(f"token_logprobs candidate: {reason}")
    rows, vocabulary = logits.shape
    code = _CODE[logits.dtype]
    with torch.cuda.device(logits.device):
        logits = logits if logits.stride(1) == 1 or vocabulary == 1 else logits.contiguous()
        tokens = tokens.contiguous()
        new = lambda shape, dtype: torch.empty(shape, dtype=dtype, device=logits.device)
        logprobs, entropy = new(rows, torch.float32), new(rows, torch.float32)
        top_logprobs, top_indices = new((rows, top), torch.float32), new((rows, top), torch.int64)
        size = _lib.token_logprobs_work(rows, vocabulary, top, code)
        work = new(size, torch.uint8) if size > 0 else None
        err = _lib.token_logprobs_launch(logits.data_ptr(), tokens.data_ptr(), logprobs.data_ptr(), entropy.data_ptr(),
                                         top_logprobs.data_ptr() if top else None,
                                         top_indices.data_ptr() if top else None,
                                         None if work is None else work.data_ptr(), size, logits.stride(0), rows,
                                         vocabulary, top, code, torch.cuda.current_stream(logits.device).cuda_stream)
    if err:
        raise RuntimeError(f"kernel launch failed: HIP error {err}")
    return {"logprobs": logprobs, "entropy": entropy, "top_logprobs": top_logprobs, "top_indices": top_indices}
