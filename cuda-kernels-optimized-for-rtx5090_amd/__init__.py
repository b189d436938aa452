"""MI355X-native LLM-inference kernels, hand-written in HIP for gfx950: softmax, RMSNorm, RoPE and top-k by rows, and a
serving step's head norms with the rotation, attention over a shared paged prefix, verification of drafts, attention of
packed prompts, a paged cache in 4 bits with its attention, and log probabilities of tokens.

The product is one C-ABI library per op, build/<op>/libkernel.so (make_libs.py), exporting the reference's entry
points (`launch`, and `plan` for top-k; declared in include/<op>.h) plus extensions; the serving step's export their
own. Two bindings sit above them: <op>/candidate.py mirrors the reference harness's `run(inputs)` wrapper for the op and
loads that library with ctypes (the functions below are conveniences over those wrappers), and torch_ops.py registers
the PyTorch-ROCm operators torch.ops.ckopt.* (build/torch/libckopt_torch.so) over the same entry points. Inputs must be
GPU tensors; there is no CPU fallback.
"""

import importlib.util
import os
import sys

from . import workloads  # noqa: F401  (named workloads: shapes, seeds, byte counts)

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
OPS = ("softmax", "rmsnorm", "rope", "topk", "qk_norm_rope", "verify_drafts", "shared_prefix_attention",
       "kv4_cache", "kv4_attention", "token_logprobs", "prompt_attention")
TORCH = ("torch",)   # the torch operators over the op libraries


def lib_path(op):
    """The in-tree library of an op (what a harness's CKOPT_BUILD_DIR would point at)."""
    return os.path.join(PKG_DIR, "build", op, "libkernel.so")


def build(ops=OPS + TORCH):
    """Compiles the libraries of the given ops (and the torch operators); returns {op: path}."""
    from . import make_libs
    return make_libs.build(ops)


def candidate(op):
    """The op's reference-style wrapper module, <op>/candidate.py, loaded by file path as the reference harness loads
    its candidates (it loads the op's library on first use)."""
    name = f"{__name__}_{op}_candidate"
    mod = sys.modules.get(name)
    if mod is None:
        spec = importlib.util.spec_from_file_location(name, os.path.join(PKG_DIR, op, "candidate.py"))
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        sys.modules[name] = mod
    return mod


def ops():
    """torch.ops.ckopt, with the operators registered (torch_ops.py)."""
    from . import torch_ops
    return torch_ops.load()


def softmax(x):
    """softmax(x) over the last dim; fp32 or bf16."""
    return candidate("softmax").run({"x": x})["y"]


def rmsnorm(x, weight=None, eps=1e-6):
    """RMSNorm over the last dim of a 2-D bf16/fp16 x, optionally times weight."""
    inputs = {"x": x, "eps": eps}
    if weight is not None:
        inputs["weight"] = weight
    return candidate("rmsnorm").run(inputs)["y"]


def rmsnorm_add(x, residual, weight=None, eps=1e-6, inplace=False):
    """Fused residual add + RMSNorm: returns (y, h) with h = x + residual (written over residual when inplace) and
    y = rmsnorm(h), times weight when given."""
    inputs = {"x": x, "residual": residual, "eps": eps, "inplace": inplace}
    if weight is not None:
        inputs["weight"] = weight
    out = candidate("rmsnorm").run(inputs)
    return out["y"], out["residual"]


def rope(q, k, position_ids, cos=None, sin=None, inv_freq=None, inplace=False):
    """RoPE of q [B, S, Hq, D] and k [B, S, Hk, D]: from a cos/sin cache, or on the fly from inv_freq."""
    inputs = {"q": q, "k": k, "position_ids": position_ids, "inplace": inplace}
    if inv_freq is not None:
        inputs["inv_freq"] = inv_freq
    else:
        inputs["cos"], inputs["sin"] = cos, sin
    out = candidate("rope").run(inputs)
    return out["q_out"], out["k_out"]


def rope_kv(q, k, v, position_ids, inv_freq, k_cache, v_cache, slot_mapping, inplace=False):
    """RoPE fused with the KV-cache write: returns q_out; the rotated k and v land in the cache rows slot_mapping
    picks ([slots, Hk, D] caches, updated in place; a negative slot writes nothing)."""
    out = candidate("rope").run({"q": q, "k": k, "v": v, "position_ids": position_ids, "inv_freq": inv_freq,
                                 "k_cache": k_cache, "v_cache": v_cache, "slot_mapping": slot_mapping,
                                 "inplace": inplace})
    return out["q_out"]


def topk(x, k=50):
    """The k largest entries of each row of a 2-D fp32/bf16 x, sorted descending, ties by lowest index."""
    out = candidate("topk").run({"x": x, "k": k})
    return out["values"], out["indices"]


def topk_sample(values, indices, uniforms, temperature=1.0, top_p=1.0):
    """Draws one index per row from a top-k list with temperature, nucleus cut and the caller's uniforms."""
    return candidate("topk").sample(values, indices, uniforms, temperature, top_p)


def qk_norm_rope(q, k, position_ids, inv_freq, q_weight=None, k_weight=None, eps=1e-6, inplace=False):
    """RMSNorm of every head of q [B, S, Hq, D] and k [B, S, Hk, D], times its weight [D] when given, and RoPE of the
    first 2 * len(inv_freq) elements, in one pass: returns (q_out, k_out)."""
    out = candidate("qk_norm_rope").run({"q": q, "k": k, "position_ids": position_ids, "inv_freq": inv_freq,
                                         "q_weight": q_weight, "k_weight": k_weight, "eps": eps, "inplace": inplace})
    return out["q_out"], out["k_out"]


def qk_norm_rope_kv(q, k, v, position_ids, inv_freq, k_cache, v_cache, slot_mapping, q_weight=None, k_weight=None,
                    eps=1e-6, inplace=False):
    """qk_norm_rope fused with the KV-cache write: returns q_out; k (normed and rotated) and v land in the cache rows
    slot_mapping picks ([slots, Hk, D] caches, updated in place; a slot outside them writes nothing)."""
    out = candidate("qk_norm_rope").run({"q": q, "k": k, "v": v, "position_ids": position_ids, "inv_freq": inv_freq,
                                         "k_cache": k_cache, "v_cache": v_cache, "slot_mapping": slot_mapping,
                                         "q_weight": q_weight, "k_weight": k_weight, "eps": eps, "inplace": inplace})
    return out["q_out"]


def verify_drafts(target_probs, draft_probs, draft_tokens, uniforms, draft_lens=None):
    """Which drafted tokens [B, S] the target's probabilities [B, S + 1, V] keep against the draft's [B, S, V] (None:
    certain), and the token drawn behind them, from uniforms [B, S + 1]: returns (tokens [B, S + 1], accepted [B])."""
    out = candidate("verify_drafts").run({"target_probs": target_probs, "draft_probs": draft_probs,
                                          "draft_tokens": draft_tokens, "uniforms": uniforms, "draft_lens": draft_lens})
    return out["tokens"], out["accepted"]


def shared_prefix_attention(q, k_cache, v_cache, prefix_table, prefix_len, block_tables, seq_lens, block_size,
                            scale=None):
    """Attention of q [B, S, Hq, D] over the prefix_len keys of the pages in prefix_table, which the batch shares, and
    over each sequence's own seq_lens keys in its row of block_tables, causal: returns [B, S, Hq, D]. The caches are
    [slots, Hk, D], slot = page * block_size + offset."""
    return candidate("shared_prefix_attention").run({
        "q": q, "k_cache": k_cache, "v_cache": v_cache, "prefix_table": prefix_table, "prefix_len": prefix_len,
        "block_tables": block_tables, "seq_lens": seq_lens, "block_size": block_size, "scale": scale})["out"]


def kv4_append(k, v, k_codes, k_scales, v_codes, v_scales, slot_mapping):
    """Writes k and v [T, Hk, D] into the slots [T] of a paged cache in 4 bits, updated in place: codes uint8 [pages, Hk,
    block_size, D / 2], scales uint8 [pages, Hk, block_size, D / 32]; a slot outside it writes nothing."""
    candidate("kv4_cache").run({"k": k, "v": v, "k_codes": k_codes, "k_scales": k_scales, "v_codes": v_codes,
                                "v_scales": v_scales, "slot_mapping": slot_mapping})


def kv4_read(k_codes, k_scales, v_codes, v_scales, slots, dtype=None):
    """The keys and values in the slots [T] of such a cache: (k, v) [T, Hk, D] in dtype (bf16)."""
    import torch
    return candidate("kv4_cache").read(k_codes, k_scales, v_codes, v_scales, slots, dtype or torch.bfloat16)


def kv4_attention(q, k_codes, k_scales, v_codes, v_scales, block_tables, seq_lens, scale=None):
    """Attention of q [B, S, Hq, D] over each sequence's seq_lens keys in the pages of such a cache that its row of
    block_tables names, causal: returns [B, S, Hq, D]."""
    return candidate("kv4_attention").run({
        "q": q, "k_codes": k_codes, "k_scales": k_scales, "v_codes": v_codes, "v_scales": v_scales,
        "block_tables": block_tables, "seq_lens": seq_lens, "scale": scale})["out"]


def token_logprobs(logits, tokens, top=0):
    """The log probabilities of tokens [N] in the rows of logits [N, V], the rows' entropies, and the `top` likeliest tokens
    of each: returns (logprobs [N], entropy [N], top_logprobs [N, top], top_indices [N, top])."""
    out = candidate("token_logprobs").run({"logits": logits, "tokens": tokens, "top": top})
    return out["logprobs"], out["entropy"], out["top_logprobs"], out["top_indices"]


def prompt_attention(q, k, v, cu_seqlens, scale=None):
    """Causal attention of whole prompts over their own keys, q [T, Hq, D], k and v [T, Hk, D] packed one behind the other
    at cu_seqlens int32 [B + 1]: returns [T, Hq, D], zeros for tokens of no prompt."""
    return candidate("prompt_attention").run({"q": q, "k": k, "v": v, "cu_seqlens": cu_seqlens, "scale": scale})["out"]
