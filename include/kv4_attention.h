/* kv4_attention: attention of the last `seq` tokens of each of `batch` sequences over their paged keys and values in 4
 * bits, in the format of kv4_cache.h. q and out in bf16 (dtype 1) or fp16 (2). Library: build/kv4_attention/
 * libkernel.so. No counterpart in the reference. Device pointers; asynchronous on `stream`; no allocation.
 *
 * q [batch, seq, q_heads, head_dim], out of the same shape, contiguous; codes [pages, kv_heads, block_size, head_dim /
 * 2] and scales [pages, kv_heads, block_size, head_dim / 32], contiguous; q head h reads kv head h / (q_heads /
 * kv_heads). Key t of sequence b is row t % block_size of page block_tables[b][t / block_size]: block_tables int32
 * [batch, blocks], seq_lens int32 [batch] the keys of each, the step's among them. Both are device memory and may change
 * between replays of a captured graph; lengths are taken within [0, blocks * block_size].
 *
 * Query i of sequence b stands at place p = seq_lens[b] - seq + i and sees keys 0..p:
 *   out = sum_j softmax_j(scale * q . k_j) v_j
 * in fp32, of the queries and the cache's values as they are; a weight is two bf16 numbers (off by at most 2^-17 of it) in
 * the products with v. A query with p < 0 (a sequence shorter than the step, an idle place of the
 * batch) gets zeros. A key whose page is outside [0, pages) counts as absent. What pages hold behind a length is not read
 * into the result. A group of keys that is NaN reaches the queries that see it, one of values those queries' 32 elements,
 * and no others.
 *
 * strides: a HOST array of q's element strides (batch, seq, head), multiples of 8 (of sizes over 1), or NULL for
 * contiguous; the last dimension is contiguous. q, out and the codes are 16-byte aligned.
 *
 * work: work_bytes bytes, at least kv4_attention_work() of these very sizes, 16-byte aligned, contents free; launches
 * that share it must be ordered. NULL where that is 0. Tables may be wider than what they hold, but how the work is cut is
 * chosen from the sizes alone, the tables taken for about 0.6 full: the keys are dealt out evenly, by the lengths on the
 * device, to as many workgroups as the device holds, which takes work and a second launch; or (work 0) each sequence has a
 * workgroup to a kv head and tile of rows, and the longest bounds the launch: where tables are narrow or sequences many.
 *
 * Return: 0 success (batch or seq <= 0 is a no-op), -1 invalid argument (head_dim none of 64, 96, 128, 192, 256; heads
 * outside [1, 65536] or q_heads no multiple of kv_heads; block_size outside [1, 2^30], kv_heads * block_size or pages *
 * block_size > 2^31 - 1, a table of more than 2^30 keys; batch * seq * q_heads >= 2^30; over 2^30 - 2^21 workgroups; a
 * scale outside [1e-30, 1e30]; a null or misaligned tensor; too small a workspace), otherwise the hipError_t of the
 * launch. */
#ifndef ROWKERN_KV4_ATTENTION_H
#define ROWKERN_KV4_ATTENTION_H
#include <hip/hip_runtime_api.h>
#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of workspace for these sizes on the current device; -1 for invalid ones. They do not grow with the sizes
 * throughout: a buffer for launches of several sizes has the most that any of them needs. */
long long kv4_attention_work(long long batch, long long seq, int q_heads, int kv_heads, int head_dim, long long blocks,
                             long long block_size);

int kv4_attention_launch(const void* q, const void* k_codes, const void* k_scales, const void* v_codes,
                         const void* v_scales, const void* block_tables, const void* seq_lens, void* out, void* work,
                         long long work_bytes, const long long* strides, long long batch, long long seq,
                         long long pages, int q_heads, int kv_heads, int head_dim, long long blocks,
                         long long block_size, float scale, int dtype, hipStream_t stream);

/* Tuning override for parameter sweeps. Slots: 0 runs that a kv head's slices are dealt out in (-1: a workgroup to a
 * sequence), 1 rows of a tile in sixteens (1, 2). Returns 0 or -1. */
int kv4_attention_tune(int slot, int value);

#ifdef __cplusplus
}
#endif
#endif
