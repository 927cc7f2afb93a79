// Launch interface of the operators over the vocabulary (raw pointers and a stream, no tensor library types):
// log-probabilities of given tokens, preference and policy losses, embedding gradient in sorted token order.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

enum class Scalar : int { kBf16 = 0, kF16 = 1, kF32 = 2 };

// ---- ops/token_log_probs.cu
// Where row r of a batch of logits [outer, inner, V] lies: (r / inner) * outer_stride + (r % inner) * row_stride elements from the base.
struct RowMap {
  long long inner, outer_stride, row_stride;
};
// T rows of V logits with a unit inner stride. log_probs: fp32 [T]; entropy: fp32 [T] or null; lse: [T] pairs (largest logit m,
// log2 of sum 2^(logit_scale log2e (x - m))), the log-sum-exp as the backward pass takes it.
void token_log_probs_fwd(const void* logits, Scalar type, const void* labels, bool labels64, float* log_probs, float* entropy,
                         float2* lse, long long T, int V, RowMap map, float logit_scale, long long ignore_index, cudaStream_t stream);
// d_log_probs / d_entropy: fp32 with strides (elements, 0 for a broadcast value); d_entropy may be null. grad: 16-byte
// aligned rows, grad_stride elements apart.
void token_log_probs_bwd(const void* logits, Scalar type, const void* labels, bool labels64, const float2* lse,
                         const float* entropy, const float* d_log_probs, long long d_log_probs_stride, const float* d_entropy,
                         long long d_entropy_stride, void* grad, long long T, int V, RowMap map, long long grad_stride,
                         float logit_scale, long long ignore_index, cudaStream_t stream);

// The rows of a batch that a product has to cover. index == null: rows base, base + 1, ... of the batch, `rows` of them. Else the
// batch has been compacted to the rows whose label counts: compact row r is row index[r] of the batch, *count of them are live (known
// on the device only), and this launch covers the live ones among compact rows [base, base + rows).
struct LiveRows {
  const int* index;
  const int* count;
  int base, rows;
};
// index[0 .. *count) <- rows with a label in [0, V) other than ignore_index, in order; compact[r] <-
// x[index[r]] (bf16 rows of H, a multiple of 8 elements), zeros from *count on; outputs of the rows that do not count <- 0.
void vocab_compact_rows(const void* labels, bool labels64, long long ignore_index, int T, int V, const void* x, long long ldx, int H,
    int* index, int* count, void* compact, float* log_probs, float* entropy, float2* lse, cudaStream_t stream);
// Joins the statistics of `slices` column slices of the rows: stats[slice][live.rows] = (m, s, u, the label's logit if it lies in the
// slice), see softmax_stats.cuh. Ignored rows give 0.
void token_log_probs_join(const float* stats, int slices, int slice_width, const void* labels, bool labels64, float* log_probs,
    float* entropy, float2* lse, LiveRows live, int V, float logit_scale, long long ignore_index, cudaStream_t stream);

// ---- gemm/vocab_gemm_2sm.cu: logits = x [M, K] w [N, K]^T, bf16 operands with row strides that are multiples of 8 elements.
// x holds the rows of this launch; labels, lse and gradients are those of the whole batch.
constexpr int kVocabSlice = 128;  // columns per slice of the statistics
// logits: null, or fp32 [live.rows, N] with a row stride ldl that is a multiple of 4, which keeps the live rows' logits.
void vocab_gemm_stats(const void* x, const void* w, const void* labels, bool labels64, float* stats, float* logits, long long ldl,
    bool entropy, LiveRows live, int N, int K, long long ldx, long long ldw, float logit_scale, int* status, cudaStream_t stream);
// grad[live.rows, N] (bf16, row stride ldg, a multiple of 8): gradient of the logits, as token_log_probs_bwd defines it; rows behind
// the live ones are 0 up to the next multiple of 256.
void vocab_gemm_grad(const void* x, const void* w, const void* labels, bool labels64, const float2* lse, const float* entropy,
                     const float* d_log_probs, long long d_log_probs_stride, const float* d_entropy, long long d_entropy_stride,
                     void* grad, LiveRows live, int N, int K, long long ldx, long long ldw, long long ldg, float logit_scale,
                     long long ignore_index, int* status, cudaStream_t stream);

// The same from kept logits (fp32, row stride ldl), without a product.
void token_log_probs_grad_rows(const float* logits, long long ldl, const void* labels, bool labels64, const float2* lse,
    const float* entropy, const float* d_log_probs, long long d_log_probs_stride, const float* d_entropy, long long d_entropy_stride,
    void* grad, long long ldg, LiveRows live, int N, float logit_scale, long long ignore_index, cudaStream_t stream);

// ---- gemm/balanced_gemm_2sm.cu: C [live.rows, N] = A [live.rows, K] B [K, N], bf16, for few tiles and a long K. Tiles that several CTA
// pairs share leave fp32 partial tiles in `partials` (balanced_partials() words); balanced_rows puts the result together and writes live
// row r to row t of `out`, its place in the batch. lda, ldb and N: multiples of 8; C and out: rows of N.
long long balanced_partials();
void balanced_gemm(const void* A, const void* B, void* C, float* partials, LiveRows live, int N, int K, long long lda, long long ldb,
    int* status, cudaStream_t stream);
void balanced_rows(const void* C, const float* partials, LiveRows live, void* out, int N, int K, cudaStream_t stream);

// ---- gemm/gemm_bf16_2sm.cu: C [M, N] (+)= A [K, M]^T B [K, N] on CTA pairs, where the K rows are those of a compacted batch: the
// contraction ends at max(1, *count - base). Rows from there to the next multiple of 64 must be 0 in both operands.
void gemm_bf16_2sm_live(const void* A, const void* B, void* C, int M, int N, int K, long long lda, long long ldb, long long ldc,
    bool f32_accumulate, LiveRows live, int* status, cudaStream_t stream);

// ---- ops/preference.cu
// A packed batch of `sequences` sequences of per-token values: sequence i is tokens [cu[i], cu[i + 1]), or, without cu,
// [i * length, (i + 1) * length). mask (bytes, or null): tokens with 0 take no part and are not looked at. cu entries are
// clamped to [0, T].
struct PackedTokens {
  long long T;
  const int* cu;
  long long length;
  int sequences;
  const unsigned char* mask;
};
long long packed_partials(long long T, int sequences);  // fp32 words of the workspace that both losses take

enum class PreferenceKind : int { kSigmoid = 0, kHinge = 1, kIpo = 2 };
struct PreferenceArgs {
  PreferenceKind kind;
  float beta, label_smoothing;
  bool average;   // log-ratio of a sequence: mean over its tokens instead of the sum
  int reduction;  // 0 = loss per pair, 1 = sum, 2 = mean
};
// sequences = 2 * pairs, chosen first. loss: [pairs] or [1]; chosen, rejected: [pairs] = beta * log-ratio; slope: [2 * pairs] =
// d(loss) / d(log-prob of a token of that sequence). reference may be null (0).
void preference_loss_fwd(const float* log_probs, const float* reference, PackedTokens tokens, PreferenceArgs args, float* partials,
                         float* loss, float* chosen, float* rejected, float* slope, cudaStream_t stream);
// grad[t] = slope[sequence of t] * d_loss[pair * d_loss_stride], 0 for tokens that take no part.
void preference_loss_bwd(const float* slope, const float* d_loss, long long d_loss_stride, PackedTokens tokens, float* grad,
                         cudaStream_t stream);

struct PolicyArgs {
  double log_low, log_high;  // log(1 - clip_low), log(1 + clip_high): the clipping borders of log(ratio)
  float ratio_low, ratio_high;
  float dual_clip;           // 0: none
  float kl_coef;
  bool per_token_advantage;
  int reduction;             // 0 = sum, 1 = mean over tokens, 2 = mean over sequences of their token means
};
struct PolicyOut {
  float *loss, *kl, *clipped, *factor;  // one value each; factor: 1 / divisor of the reduction
};
// kl: mean KL estimate, clipped: share of tokens whose gradient is clipped; slope (or null): [T] d(token's loss) /
// d(log-prob); weight: [sequences] 1 / tokens of the sequence (reduction 2 only).
void policy_loss_fwd(const float* log_probs, const float* old_log_probs, const float* reference, const float* advantages,
    PackedTokens tokens, PolicyArgs args, float* partials, PolicyOut out, float* slope, float* weight, cudaStream_t stream);
// grad[t] = slope[t] * factor (* weight[sequence of t]) * d_loss, 0 for tokens that take no part.
void policy_loss_bwd(const float* slope, const float* factor, const float* weight, const float* d_loss, PackedTokens tokens,
    int reduction, float* grad, cudaStream_t stream);

// ---- ops/embedding_sorted.cu
constexpr int kStatusBadTokenId = 7;  // an id outside of [0, V): its output row is 0, it takes no part in the gradient
// out[t] = scale * weight[ids[t]]
void embedding_lookup(const void* weight, Scalar type, const void* ids, bool ids64, void* out, long long T, long long V, int H,
                      float scale, int* status, cudaStream_t stream);
// Bytes of the workspace of the gradient (256-byte aligned).
long long embedding_gradient_workspace(long long T, int H, Scalar type);
// dweight[v] = scale * sum of dout[t] over the tokens with id v, in an order that the ids and sizes fix. accumulate: dweight is fp32, is added to, and rows
// that no id names are not touched; else it has dout's type, is 16-byte aligned, and is written whole.
void embedding_gradient(const void* dout, Scalar type, const void* ids, bool ids64, void* dweight, bool accumulate, void* workspace,
                        long long T, long long V, int H, float scale, cudaStream_t stream);

}  // namespace b200
