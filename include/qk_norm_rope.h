/* qk_norm_rope: the RMS norm of every query and key head, its weight and the rotary embedding (rotate-half pairing) in
 * one pass over q[batch, seq, q_heads, head_dim] and k[batch, seq, kv_heads, head_dim] in bf16 (dtype 1) or fp16 (2),
 * and the same with the keys and values appended to a paged cache. Library: build/qk_norm_rope/libkernel.so. No
 * counterpart in the reference. Device pointers; asynchronous on `stream`; no allocation.
 *
 * For a head x at position p, in fp32 with one rounding at the end, r = rotary_dim:
 *   y = x * w / sqrt(mean(x^2) + eps)                                 (w = 1 where the weight is NULL)
 *   out[i]         = y[i] cos(a_i)         - y[i + r/2] sin(a_i)      i < r/2, a_i = p * inv_freq[i]
 *   out[i + r/2]   = y[i + r/2] cos(a_i)   + y[i] sin(a_i)
 *   out[i]         = y[i]                                             i >= r
 * The angle is the exact product of the int64 position and the fp32 frequency (formed in fp64, reduced by multiples
 * of pi/2, then rounded), so far positions keep their phase; rope_launch_freq rounds the product to fp32 as the
 * reference's cache does, and differs by that rounding.
 *
 * strides: a HOST array of element strides (batch, seq, head) for each tensor in the order the entry point names, or
 * NULL for contiguous ones; the last dimension is contiguous. Views of a packed projection need no copy. q_out may be q
 * and k_out may be k (with the same strides: in place); otherwise outputs do not overlap inputs.
 *
 * Return: 0 success (batch or seq <= 0 is a no-op), -1 invalid argument (batch * seq > 2^31 - 1 or over 2^38 heads of
 * all tokens, q_heads or kv_heads outside [1, 2^20], head_dim outside [1, 65536], rotary_dim odd, negative or >
 * head_dim, a dtype other than 1 and 2, a null tensor), otherwise the hipError_t of the launch. */
#ifndef ROWKERN_QK_NORM_ROPE_H
#define ROWKERN_QK_NORM_ROPE_H
#include <hip/hip_runtime_api.h>
#ifdef __cplusplus
extern "C" {
#endif

/* strides: q, k, q_out, k_out (12 values). inv_freq: fp32 [rotary_dim / 2]; may be NULL where rotary_dim is 0. */
int qk_norm_rope_launch(const void* q, const void* k, const void* ids, const float* inv_freq, const void* q_weight,
                        const void* k_weight, void* q_out, void* k_out, const long long* strides, long long batch,
                        long long seq, int q_heads, int kv_heads, int head_dim, int rotary_dim, int dtype, float eps,
                        hipStream_t stream);

/* strides: q, k, v, q_out (12 values). The normed and rotated k and the untouched v of a token go to row
 * slot_mapping[token] (int64 [batch, seq]) of k_cache and v_cache, both contiguous [slots, kv_heads, head_dim]; a
 * slot outside [0, slots) writes nothing for its token. No two tokens share a slot. The caches overlap neither each
 * other nor an input; they may be NULL where slots is 0. */
int qk_norm_rope_kv_launch(const void* q, const void* k, const void* v, const void* ids, const float* inv_freq,
                           const void* q_weight, const void* k_weight, void* q_out, void* k_cache, void* v_cache,
                           const void* slot_mapping, const long long* strides, long long batch, long long seq,
                           long long slots, int q_heads, int kv_heads, int head_dim, int rotary_dim, int dtype,
                           float eps, hipStream_t stream);

/* Tuning override for parameter sweeps. Slots: 0 steps per wave (1, 2 or 4), 1 forced scalar kernel (1),
 * 2 several tokens to a wave wherever their heads fit (1) or never (2).
 * Returns 0 or -1. */
int qk_norm_rope_tune(int slot, int value);

#ifdef __cplusplus
}
#endif
#endif
