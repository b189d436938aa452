/* prompt_attention: causal attention of whole prompts, packed one behind the other, over their own keys, with grouped
 * heads. bf16 (dtype 1) or fp16 (2). Library: build/prompt_attention/libkernel.so. No counterpart in the reference. Device
 * pointers; asynchronous on `stream`; no allocation.
 *
 * q [tokens, q_heads, head_dim], k and v [tokens, kv_heads, head_dim], out [tokens, q_heads, head_dim], contiguous; q head h
 * reads kv head h / (q_heads / kv_heads). cu_seqlens int32 [batch + 1], device memory, which may change between replays
 * of a captured graph: prompt b is tokens cu_seqlens[b] ... cu_seqlens[b + 1] - 1, none where the two are equal. Offsets do
 * not decrease; they are taken within [0, tokens]. Token i of a prompt sees its tokens 0..i:
 *   out = sum_j softmax_j(scale * q . k_j) v_j
 * in fp32, the weights rounded to the dtype before the products with v (and summed as rounded). Tokens before the first
 * offset and from the last one on (padding to a fixed number of rows) belong to no prompt: zeros are written for them. A
 * NaN or infinity in a key or value reaches the queries that see it and no others.
 *
 * strides: a HOST array of element strides (token and head of q, of k, of v), multiples of 8 (of sizes over 1), those of k's
 * and v's tokens at most 2^23, or NULL for contiguous; the last dimension is contiguous, so the parts of a packed
 * projection are taken as they are. All tensors are 16-byte aligned.
 *
 * Return: 0 success (tokens <= 0 is a no-op), -1 invalid argument (head_dim none of 64, 80, 96, 128, 192, 256; heads
 * outside [1, 65536] or q_heads no multiple of kv_heads; tokens * q_heads >= 2^30; batch < 0 or batch * kv_heads >= 2^29; a
 * scale outside [1e-30, 1e30]; a null or misaligned tensor; strides out of range), otherwise the hipError_t of the
 * launch. */
#ifndef ROWKERN_PROMPT_ATTENTION_H
#define ROWKERN_PROMPT_ATTENTION_H
#include <hip/hip_runtime_api.h>
#ifdef __cplusplus
extern "C" {
#endif

int prompt_attention_launch(const void* q, const void* k, const void* v, const void* cu_seqlens, void* out,
                            const long long* strides, long long tokens, long long batch, int q_heads, int kv_heads,
                            int head_dim, float scale, int dtype, hipStream_t stream);

/* Tuning override for parameter sweeps. Slot 0: waves of a workgroup (4, or 8 of 80 to 128 values). Returns 0 or -1. */
int prompt_attention_tune(int slot, int value);

#ifdef __cplusplus
}
#endif
#endif
