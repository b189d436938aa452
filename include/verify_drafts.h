/* verify_drafts: which drafted tokens a target model's probabilities keep, and the token drawn behind them (rejection
 * sampling of speculative decoding), from given uniforms. Library: build/verify_drafts/libkernel.so. No counterpart
 * in the reference. Device pointers; asynchronous on `stream`; no allocation.
 *
 * target [batch, drafts + 1, vocabulary] and draft [batch, drafts, vocabulary] are probabilities in fp32 (dtype 0) or
 * bf16 (1); tokens int64 [batch, drafts]; lens int32 [batch] or NULL (each sequence's number of drafts, taken within
 * [0, drafts]; all where NULL); uniforms fp32 [batch, drafts + 1] in [0, 1). For each sequence, n its number of
 * drafts:
 *   draft i < n is kept while uniforms[i] * draft[i][tokens[i]] < target[i][tokens[i]] (exactly, in fp64); j is the
 *   first that is not, n where all are;
 *   weights w = max(target[j] - draft[j], 0) where j < n, else target[n]; if w has no positive sum, target[j];
 *   drawn is the first index whose running sum of w is above uniforms[drafts] * sum(w), in fp64; -1 where w has no
 *   positive sum;
 *   out_tokens int64 [drafts + 1] = the j kept drafts, drawn, then -1; accepted int64 = j.
 * draft == NULL: drafts without probabilities (looked up, or a greedy draft model's): draft i is kept while
 * uniforms[i] < target[i][tokens[i]], and w is target[j] without the refused token. NaN and negative weights count as
 * zero; a token outside the vocabulary is refused.
 *
 * strides: a HOST array of element strides (batch and row of target, then of draft), or NULL for contiguous ones; the
 * vocabulary is contiguous. The other tensors are contiguous.
 *
 * A row is read by verify_plan()'s number of workgroups, which may be 1. More than one hand their sums over in `work`
 * (verify_work() doubles) and count their arrivals on counters[batch] (u32, zero on entry, left zero); launches that
 * share them must be ordered. Both may be NULL for one workgroup a row.
 *
 * Return: 0 success (batch <= 0 is a no-op), -1 invalid argument (drafts outside [0, 65535], vocabulary outside [1,
 * 2^28], batch > 2^22, blocks outside [1, 256], a dtype other than 0 and 1, a null tensor), otherwise the hipError_t
 * of the launch. */
#ifndef ROWKERN_VERIFY_DRAFTS_H
#define ROWKERN_VERIFY_DRAFTS_H
#include <hip/hip_runtime_api.h>
#ifdef __cplusplus
extern "C" {
#endif

/* The workgroups a row's read is worth, for verify_launch's `blocks`; -1 for invalid sizes. */
long long verify_plan(long long batch, long long vocabulary, int dtype);
/* The doubles of `work` that a launch of more than one workgroup a row needs; no fewer for a larger batch or vocabulary
 * of the same dtype. */
long long verify_work(long long batch, long long vocabulary, int dtype);

int verify_launch(const void* target, const void* draft, const void* tokens, const void* lens, const float* uniforms,
                  void* out_tokens, void* accepted, void* work, void* counters, const long long* strides,
                  long long batch, int drafts, long long vocabulary, int dtype, int blocks, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
