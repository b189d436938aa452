/* kv4_cache: a paged cache of keys and values in 4 bits: appending to it and reading from it. Library:
 * build/kv4_cache/libkernel.so. No counterpart in the reference. Device pointers; asynchronous on `stream`; no
 * allocation.
 *
 * The cache: codes uint8 [pages, kv_heads, block_size, head_dim / 2] and scales uint8 [pages, kv_heads, block_size,
 * head_dim / 32], contiguous, for keys and for values. Slot s is row s % block_size of page s / block_size. A byte of
 * codes holds elements 2 i (its low half) and 2 i + 1: bit 3 the sign, bits 2..0 one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (the
 * e2m1 of the OCP microscaling formats); a scale byte b stands for 2^(b - 127), shared by 32 elements, and b > 252 for a
 * group of NaN. An element is the product.
 *
 * kv4_append_launch: k and v [tokens, kv_heads, head_dim] in bf16 (dtype 1) or fp16 (2); token t goes to slot
 * slot_mapping[t] (int64; outside the cache: it writes nothing; two tokens of a call in one slot leave it undefined). A
 * group's scale is the least power of two that leaves its largest magnitude below 7, at least 2^-126 and at most 2^125
 * of bf16 or 2^13 of fp16 (what is above 6 times that is cut to it); its elements go to the nearest value, ties to the
 * even code. So an element that is not cut, of a group whose largest magnitude is 2^-124 at least, is off by at most a
 * fifth of that magnitude. A group with an infinity or a NaN becomes NaN (scale 255, codes 0). What other slots hold stays
 * as it is.
 * strides: a HOST array of element strides (token and head of k, then of v), multiples of 8 (of sizes over 1), or NULL
 * for contiguous; the last dimension is contiguous; k and v are 16-byte aligned, the codes 4-byte.
 *
 * kv4_read_launch: k and v [tokens, kv_heads, head_dim], contiguous, become the elements of slots[t] (int64; outside
 * the cache: zeros), rounded to dtype: bf16 holds every one, fp16 those of a cache that was written in fp16; what a cache
 * that was written in bf16 holds above fp16's largest number is read as infinity there.
 *
 * Return: 0 success (tokens <= 0 is a no-op), -1 invalid argument (head_dim none of 64, 96, 128, 192, 256; kv_heads
 * outside [1, 65536]; block_size < 1; pages * block_size > 2^31 - 1; tokens * kv_heads over about 2^34; a dtype other
 * than 1 and 2; a null or misaligned tensor; strides that are no multiples of 8), otherwise the hipError_t of the
 * launch. */
#ifndef ROWKERN_KV4_CACHE_H
#define ROWKERN_KV4_CACHE_H
#include <hip/hip_runtime_api.h>
#ifdef __cplusplus
extern "C" {
#endif

int kv4_append_launch(const void* k, const void* v, void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                      const void* slot_mapping, const long long* strides, long long tokens, long long pages,
                      int kv_heads, int head_dim, int block_size, int dtype, hipStream_t stream);

int kv4_read_launch(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                    const void* slots, void* k, void* v, long long tokens, long long pages, int kv_heads, int head_dim,
                    int block_size, int dtype, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
