/* C ABI of the fused softmax cross-entropy (loss + d_logits) for sm_100a: libb200loss.so / libb200loss.a.
 *
 * Replaces cross_entropy_forward_backward of sarimahsan/transformer-cuda (include/kernels/loss.cuh:8-15,
 * src/kernels/loss.cu:24-125), the first call of the model's backward pass (src/model.cu:449). The C++
 * declaration with the reference's exact signature is include/kernels/loss.cuh; the entry points below are
 * the same launch with plain pointers and sizes, for bindings from other languages and for the parity tests.
 *
 * All pointers are device pointers on the current device unless stated otherwise; `stream` is a cudaStream_t
 * passed as void*. Logits and d_logits are FP32, row-major (rows x V), rows = B * T; targets are int32.
 * Return value: 0 on success, a negative B200LOSS_ERR_* otherwise; b200loss_last_error() describes the failure. */
#ifndef B200LOSS_H
#define B200LOSS_H

#ifdef __cplusplus
extern "C" {
#endif

#define B200LOSS_OK 0
#define B200LOSS_ERR_ARG (-1)   /* NULL pointer, non-positive size */
#define B200LOSS_ERR_CUDA (-2)  /* a CUDA runtime call failed */
#define B200LOSS_ERR_WAIT (-3)  /* a bounded wait inside an earlier launch ran out (see check_device_fault) */

/* d_logits[i, v] = (softmax(logits[i, :])[v] - (v == targets[i])) / rows, and, when `device_loss` is not NULL,
 * *device_loss = mean_i (logsumexp(logits[i, :]) - logits[i, targets[i]]). Asynchronous on `stream`; nothing is
 * copied to the host. d_logits may alias logits (each row is resident on chip before it is written).
 * The first call on a device, and the first call with more rows than any before it, allocates the row-loss scratch
 * (rows * 4 bytes) with cudaMalloc and therefore must not happen inside a stream capture. */
int b200loss_cross_entropy(const float* logits, const int* targets, float* d_logits, float* device_loss, int B, int T,
                           int V, void* stream);

/* Element types of the logits of the calls below. */
#define B200LOSS_F32 0
#define B200LOSS_BF16 1

/* Log-probabilities of given tokens, the entropy of every row and its most likely tokens; one read of the logits.
 * With y = logits[i, :] / temperature and p = softmax(y):
 *   logprobs[i] = ln p[targets[i]]; 0 where the target is not a token (below 0 or >= V: padding)
 *   entropy[i]  = -sum_v p[v] ln p[v], for every row
 *   stats[2 i]  = max_v logits[i, v], stats[2 i + 1] = ln sum_v exp(y[v] - max y): what the gradient needs
 *   top_tokens[i * top + k], top_logprobs[i * top + k]: the k-th largest logit's index and ln p, equal logits by the lower
 *   index; 0 <= top <= min(32, V), top = 0 writes none (both may then be NULL).
 * Logits are rows of V elements of `dtype` (B200LOSS_F32 or B200LOSS_BF16), row i at logits + i * row_stride elements, at
 * any alignment that fits the type; outputs are FP32 (int32 for tokens), sums are held in FP32. A logit of -inf is a token
 * that is not allowed (p = 0); in a row that allows none every log-probability is -inf and the entropy 0. A row with a NaN
 * or +inf gives NaN (a NaN ranks above every number among the alternatives). 1e-6 <= temperature <= 1e6. rows = 0 is a no-op.
 * Allocates nothing and holds no state: calls may overlap and be captured. No counterpart in the reference. */
int b200loss_token_logprobs(const void* logits, int dtype, long long row_stride, const int* targets, int rows, int V,
                            float temperature, float* logprobs, float* entropy, float* stats, int top, float* top_logprobs,
                            int* top_tokens, void* stream);

/* Gradient of sum_i grad_logprobs[i] * logprobs[i] + grad_entropy[i] * entropy[i] with regard to the logits:
 *   dlogits[i, v] = ( g ([v = target] - p[v]) - grad_entropy[i] p[v] (ln p[v] + entropy[i]) ) / temperature
 * with g = grad_logprobs[i], 0 where the target is not a token. `entropy` and `stats` are the forward's for the same
 * logits and temperature; grad_entropy may be NULL (none). dlogits has the logits' type, row i at i * d_row_stride; it may
 * be the logits' own buffer with the same stride, any other overlap is not allowed. A row that no gradient reaches (g and
 * grad_entropy[i] both 0) or that allows no token is written as zeros, whatever its logits hold. The alternatives carry no
 * gradient. */
int b200loss_token_logprobs_backward(const void* logits, int dtype, long long row_stride, const int* targets, const float* entropy,
                                     const float* stats, const float* grad_logprobs, const float* grad_entropy, int rows, int V,
                                     float temperature, void* dlogits, long long d_row_stride, void* stream);

/* Which kernel a call with these arguments takes: 0 = one pass over HBM, the row held in shared memory
 * (16-byte aligned buffers, 8 <= V <= b200loss_max_resident_vocab()), 1 = streaming kernel, two reads of the row. */
int b200loss_kernel_path(const float* logits, const float* d_logits, int V);
int b200loss_max_resident_vocab(void);

/* Waits for the device and returns 0 if no bounded wait has run out since the last call, else B200LOSS_ERR_WAIT
 * (and clears the record). */
int b200loss_check_device_fault(void);

/* Frees the per-device scratch. */
void b200loss_release(void);

/* Text of the last failure on the calling thread ("" if none). */
const char* b200loss_last_error(void);

#ifdef __cplusplus
}
#endif
#endif
