/* shared_prefix_attention: attention of the last `seq` tokens of each of `batch` sequences over one paged prefix that
 * all of them share (a system prompt, a document) and over each sequence's own paged keys and values; the prefix is
 * read once for the batch. bf16 (dtype 1) or fp16 (2). Library: build/shared_prefix_attention/libkernel.so. No
 * counterpart in the reference. Device pointers; asynchronous on `stream`; no allocation.
 *
 * q [batch, seq, q_heads, head_dim], out of the same shape, contiguous; k_cache and v_cache [slots, kv_heads,
 * head_dim], contiguous (rope_kv_launch's and qk_norm_rope_kv_launch's caches); q head h reads kv head h / (q_heads /
 * kv_heads). Key t of a table is in slot table[t / block_size] * block_size + t % block_size: prefix_table int32
 * [prefix_blocks] holds the prefix's prefix_len[0] keys, row b of block_tables int32 [batch, own_blocks] the
 * seq_lens[b] keys that are sequence b's own, the step's among them. prefix_len (int32 [1]) and seq_lens (int32
 * [batch]) are device memory and may change between replays of a captured graph; they are taken within [0, blocks *
 * block_size].
 *
 * Query i of sequence b stands at own place p = seq_lens[b] - seq + i and sees the whole prefix and own keys 0..p:
 *   out = sum_j softmax_j(scale * q . k_j) v_j
 * in fp32, the weights rounded to the dtype before the products with v (and summed as rounded). A query with p < 0 (a
 * sequence shorter than the step, an idle place of the batch) gets zeros. A key whose slot is outside [0, slots)
 * counts as absent. What pages hold behind a length is not read into the result; a NaN or infinity in a key or value
 * reaches the queries that see it and no others.
 *
 * How the work is cut follows the sizes given here, the tables' width among them: it is made for tables that are mostly
 * full. Lengths far below the width are right, and slower than the same ones in narrow tables.
 *
 * strides: a HOST array of q's element strides (batch, seq, head), multiples of 8 (of sizes over 1), or NULL for
 * contiguous; the last dimension is contiguous. q, caches and out are 16-byte aligned.
 *
 * work: prefix_attention_work() bytes of these very sizes, 16-byte aligned, contents free; launches that share it must
 * be ordered. NULL where it is 0. The bytes do not grow with the sizes throughout (a smaller batch may be cut into more
 * parts): a buffer for launches of several sizes has the most that any of them needs. prefix_attention_launch_sized
 * takes the buffer's bytes and refuses one that is too small; prefix_attention_launch cannot tell.
 *
 * Return: 0 success (batch or seq <= 0 is a no-op), -1 invalid argument (head_dim none of 64, 80, 96, 128, 192, 256;
 * heads outside [1, 65536] or q_heads no multiple of kv_heads; block_size outside [1, 2^30] or a table of more than
 * 2^30 keys; slots outside [0, 2^31 - 1]; batch * seq * q_heads >= 2^30, or so many tiles of a sequence's kv head (32
 * rows or fewer, a wave or more each) that they take over 2^28 - 2^21 workgroups of four waves; a scale outside [1e-30,
 * 1e30]; a null or misaligned tensor; too small a workspace), otherwise the hipError_t of the launch. */
#ifndef ROWKERN_SHARED_PREFIX_ATTENTION_H
#define ROWKERN_SHARED_PREFIX_ATTENTION_H
#include <hip/hip_runtime_api.h>
#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of workspace for these sizes on the current device; -1 for invalid ones. */
long long prefix_attention_work(long long batch, long long seq, int q_heads, int kv_heads, int head_dim,
                                long long prefix_blocks, long long own_blocks, long long block_size);

int prefix_attention_launch(const void* q, const void* k_cache, const void* v_cache, const void* prefix_table,
                            const void* prefix_len, const void* block_tables, const void* seq_lens, void* out,
                            void* work, const long long* strides, long long batch, long long seq, long long slots,
                            int q_heads, int kv_heads, int head_dim, long long prefix_blocks, long long own_blocks,
                            long long block_size, float scale, int dtype, hipStream_t stream);

/* The same with the bytes that `work` has. */
int prefix_attention_launch_sized(const void* q, const void* k_cache, const void* v_cache, const void* prefix_table,
                                  const void* prefix_len, const void* block_tables, const void* seq_lens, void* out,
                                  void* work, long long work_bytes, const long long* strides, long long batch,
                                  long long seq, long long slots, int q_heads, int kv_heads, int head_dim,
                                  long long prefix_blocks, long long own_blocks, long long block_size, float scale,
                                  int dtype, hipStream_t stream);

/* Tuning override for parameter sweeps. Slots: 0 splits of the prefix, 1 of a sequence's own keys, 2 the prefix by
 * tiles of 32 rows (1) or 256 (2; 128 of head sizes over 128), or the prefix's keys before each sequence's own (3); 3
 * waves that share a split of a 32-row tile (1, 2, 4). Returns 0 or -1. */
int prefix_attention_tune(int slot, int value);

#ifdef __cplusplus
}
#endif
#endif
