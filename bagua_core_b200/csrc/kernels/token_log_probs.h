// Log probabilities of given tokens under rows of logits, with the rows' entropy and likeliest tokens, and the gradient (sm_100a).
//
//   lse = log sum exp(x_j)     log p_j = x_j - lse     log_prob = log p_target     entropy = -sum p_j log p_j
//   d x_j = a ([j = target] - p_j) - b p_j (log p_j + entropy)    for gradients a of log_prob and b of entropy
//
// The logits are read once in each direction; nothing of their size is kept between the two.  Sums are fp32.
//
//   * target == ignored: the row is not looked at; 0, 0, no alternatives (-inf, -1), gradient 0.
//   * a row of nothing but -inf: log_prob and alternatives' values -inf, entropy 0, gradient 0.
//   * a row with NaN or +inf: all NaN, alternatives -1.
//   * a target outside the vocabulary: log_prob NaN, gradient 0 (check_indices() in encoder_ops.h tells).
// No counterpart in the reference, which has no model code.
#pragma once

#include <cuda_runtime_api.h>

#include <cstdint>

#include "../common.h"

namespace bagua {
namespace token_log_probs {

constexpr int kMaxTop = 32;
constexpr int64_t kMaxVocab = 1ll << 30, kMaxRows = (1ll << 31) - 1;

struct Logits {
  const void* x;
  DType type;
  int64_t rows, vocab, stride;  // elements between rows
};
// What the backward pass needs of a row: largest value, 1 / sum exp(x - it), entropy - log of that sum, and whether it has a gradient.
struct RowStats {
  float top, inverse, offset, counts;
};

// top: 0 to kMaxTop alternatives, values and ids [rows, top], the likeliest first, equal ones in the order of their ids.  stats: [rows], or null.
void forward(const Logits& l, const int64_t* targets, int64_t ignored, int top, float* log_probs, float* entropy, float* top_values,
             int64_t* top_ids, RowStats* stats, cudaStream_t s);
// dx: rows `dx_stride` elements apart, as far from 16-byte borders as the logits' rows.  Gradients of log_probs and entropy, either of
// which may be null, lie `a_stride` and `b_stride` elements apart.
void backward(const Logits& l, const int64_t* targets, const RowStats* stats, const float* a, int64_t a_stride, const float* b, int64_t b_stride,
              void* dx, int64_t dx_stride, cudaStream_t s);

}  // namespace token_log_probs
}  // namespace bagua
