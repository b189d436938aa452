/* token_logprobs: the log probability of a given token in each row of logits, the entropy of the row's distribution, and
 * its likeliest tokens with theirs. Library: build/token_logprobs/libkernel.so. No counterpart in the reference. Device
 * pointers; asynchronous on `stream`; no allocation.
 *
 * logits [rows, vocabulary] in fp32 (dtype 0), bf16 (1) or fp16 (2), rows row_stride elements apart, at any element
 * alignment; tokens int64 [rows]. With p = softmax of a row:
 *   logprobs fp32 [rows]: log p[token]; 0 for a negative token (padding), NaN for one beyond the vocabulary;
 *   entropy fp32 [rows]: -sum p log p, in nats, a logit of minus infinity adding nothing;
 *   top_logprobs fp32 and top_indices int64 [rows, top]: log p of the `top` largest logits, the largest first, of equal
 *   ones the lowest index first (+0 above -0).
 * A row without a distribution (a NaN, plus infinity, or nothing above minus infinity) has NaN for all of these, and
 * indices of -1. The sums are held in fp32 over 16 or 32 elements and in fp64 beyond, those around a row's largest in fp64
 * where little is left beside it (so the log probability of a token that is sure, and the entropy then, are off by at most
 * 2^-15 of themselves and 2^-45), and the logarithms are fp64.
 *
 * work: work_bytes bytes, at least token_logprobs_work() of these very sizes, 8-byte aligned, contents free; launches
 * that share it must be ordered. NULL where that is 0.
 *
 * Return: 0 success (rows <= 0 is a no-op), -1 invalid argument (rows > 2^31, vocabulary outside [1, 2^28], top outside
 * [0, 64] or above the vocabulary, a dtype other than 0, 1 and 2, a null or misaligned tensor, too small a workspace),
 * otherwise the hipError_t of the launch. */
#ifndef ROWKERN_TOKEN_LOGPROBS_H
#define ROWKERN_TOKEN_LOGPROBS_H
#include <hip/hip_runtime_api.h>
#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of workspace for these sizes on the current device (few rows are read by several workgroups each); -1 for
 * invalid ones. They do not grow with the sizes throughout. */
long long token_logprobs_work(long long rows, long long vocabulary, int top, int dtype);

int token_logprobs_launch(const void* logits, const void* tokens, float* logprobs, float* entropy, float* top_logprobs,
                          void* top_indices, void* work, long long work_bytes, long long row_stride, long long rows,
                          long long vocabulary, int top, int dtype, hipStream_t stream);

/* Tuning override for parameter sweeps. Slot 0: workgroups to a row. Returns 0 or -1. */
int token_logprobs_tune(int slot, int value);

#ifdef __cplusplus
}
#endif
#endif
