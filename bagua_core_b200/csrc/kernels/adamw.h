// AdamW over many tensors in one launch, its moments held in fp32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
//
// in fp32 whatever p and g are held in; p is rounded once.  1 - lr wd is held in two numbers: in one it would be off by half a step of fp32
// next to 1, a tenth of the decay for lr wd of 2e-7, in the same direction at every step.  No counterpart in the reference, which has no
// optimizer.
//
// Moments in 8 bits.  kMoment8Block neighbouring elements of a tensor share a scale for each moment, fp32: the block's largest value
// times fp32's 1/480 or 1/496, so that it has the largest code.  A code is a small floating point number: for m a sign, 4 bits of exponent and 3 of fraction
// (up to 480, down to 2^-9), for v, which has no sign, 4 and 4 (up to 496, down to 2^-10).
//
// Rounding is stochastic: of the two neighbouring values the upper one is taken with the probability that keeps the mean.  To the
// nearest, the second moment would never move: with b2 = 0.999 a step changes it by a thousandth, its neighbours are a thirtieth
// away.  The random bits are a hash of (seed, step, tensor, element): a step can be repeated.  A second moment that is not zero
// does not become zero, since the step divides by it: it is held at the smallest code, 2^-19 of its block's largest, or 2^-9.5 of the
// largest root.  The step itself uses both moments before they are rounded.
// Codes are those that the definition in 64 bits gives: a value that fp32 cannot tell from the border between two codes, given its
// random bits, is computed again, with its block, in 64 bits.  (Where a first moment is a small difference of large terms, fp32 may
// be further off than that.)  A code that went the other way would show for as long as moments are remembered, in the scales above all.
// A block in which a moment is not finite has the scale NaN and reads as NaN.
#pragma once

#include <cuda_runtime_api.h>

#include <cstdint>

#include "../common.h"

namespace bagua {
namespace adamw {

constexpr int kMoment8Block = 256;
inline int64_t moment8_blocks(int64_t n) { return (n + kMoment8Block - 1) / kMoment8Block; }

// What all elements of a parameter group have in common at a step.
struct Hyper {
  float keep, rest;    // 1 - lr wd, as the sum of two numbers
  float rate;          // lr / (1 - b1^t)
  float root;          // 1 / sqrt(1 - b2^t)
  float eps, b1, c1, b2, c2;  // c: 1 - b
  uint32_t random;     // 8 bits: what the tensors' keys come from
  double beta1, beta2; // 8 bits: b1 and b2 for what is computed in 64
};
struct GroupValues {
  double lr, b1, b2, eps, weight_decay;
};
Hyper hyper(const GroupValues& g, int64_t step, uint64_t seed);

struct Segment {
  void* p;
  const void* g;
  void *m, *v;   // fp32, or codes
  void* copy;    // p in bf16, or null
  float *m_scale, *v_scale;  // of codes: one for each block
  int64_t n;
  uint32_t index;  // its own number among the tensors of a step
  int16_t group;   // index of its hyperparameters
  int16_t lead;    // set by the GPU path: elements in front of the first four that all buffers hold as one piece; -1: there are none
};

// Which types a call's parameters and gradients have, and what its moments are held in.
struct Types {
  DType p, g;
  bool moments8;
};
// p in F32, F16 or BF16; g in p's type or F32, or any of them where p is F32.
bool supported(const Types& t);

namespace cuda {
// Steps all segments with the groups' hyperparameters, which lie on the host, or, with `on_device`, on the device; returns the number
// of kernels launched.
int step(const Types& t, const Segment* segs, int n, const Hyper* hypers, int groups, bool on_device, cudaStream_t s);
// hyper() of a step whose numbers, one for each group, lie on the device, for a captured step that is replayed; `out` is there too.
int hypers(const GroupValues* g, int groups, const int64_t* step, uint64_t seed, Hyper* out, cudaStream_t s);
// The values of moments held in 8 bits, in the type `out`.
struct Read8 {
  const uint8_t *m, *v;
  const float *m_scale, *v_scale;
  void *m_out, *v_out;
  int64_t n;
};
int read8(const Read8* segs, int n, DType out, cudaStream_t s);
}  // namespace cuda
namespace host {
void step(const Types& t, const Segment* segs, int n, const Hyper* hypers);
void read8(const cuda::Read8* segs, int n, DType out);
}  // namespace host

}  // namespace adamw
}  // namespace bagua
