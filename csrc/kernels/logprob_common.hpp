// Arguments of the token log-probability kernels (csrc/hip/hip_logprob.hip).
//
// For a row x of V logits, M = max x and L = log sum exp(x - M):
//
//   logprob(j) = (x_j - M) - L          entropy H = L - sum_j p_j (x_j - M),   p_j = exp(logprob(j))
//
// and, with upstream gradients g_lp (target t), g_H and g_k (alternatives j_k),
//
//   dx_j = g_lp (d_jt - p_j) + sum_k g_k (d_jjk - p_j) - g_H p_j (logprob(j) + H)
//
// M and L are kept apart for the backward pass: x_j - M is exact for the entries that matter, while x_j - (M + L)
// would round the sum to the spacing of the logits.
#pragma once

#include <cstddef>
#include <cstdint>

namespace pccl::kernels {

constexpr int kMaxTopLogprobs = 64;

struct LogprobArgs {
    const void *logits = nullptr; // rows of `vocab` elements, `row_stride` elements apart
    int64_t row_stride = 0;
    int64_t rows = 0;
    int64_t vocab = 0;
    const int64_t *targets = nullptr;
    int64_t ignore_index = -100;
    int top_k = 0;
    float *logprob = nullptr; // [rows]
    float *entropy = nullptr; // [rows]
    float *stats = nullptr;   // [rows, 3]: M, L, H for the backward pass (an empty row: -inf, 0, 0)
    float *top_logprob = nullptr;   // [rows, top_k]
    int64_t *top_index = nullptr;   // [rows, top_k]
};

struct LogprobGradArgs {
    LogprobArgs fwd;                // inputs and results of the forward call
    const float *g_logprob = nullptr; // upstream gradients, nullptr = zero
    const float *g_entropy = nullptr;
    const float *g_top = nullptr;
    void *d_logits = nullptr; // [rows, vocab], contiguous, the logits' type
};

} // namespace pccl::kernels
