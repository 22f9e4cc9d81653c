// AdamW steps of torch tensors: lists of them given to each call, or laid out once as a plan.
#pragma once

#include <ATen/ATen.h>

#include <optional>
#include <vector>

#include "../kernels/adamw.h"
#include "sgd_plan.h"

namespace bagua {
namespace trainer {

using TensorList = std::vector<at::Tensor>;
using TensorRefs = std::vector<const at::Tensor*>;  // that the caller holds

// The number of a step for each parameter group: known to the host, or int64 on the device that are read when the step runs.
struct StepNumbers {
  std::vector<int64_t> host;
  std::optional<at::Tensor> device;
};

// Tensors with their gradients, moments and, for moments in 8 bits, their scales [2, blocks]; `copy`: where they go in bf16.
class AdamWPlan {
 public:
  void add(const at::Tensor& p, const at::Tensor& g, const at::Tensor& m, const at::Tensor& v, const at::Tensor* scales, const at::Tensor* copy,
           int group);
  void reserve(size_t n) { segs_.reserve(n); }
  // Throws if a buffer that is written overlaps another one of the plan.
  void check_apart() const;
  // On the current stream of the tensors' device; returns the number of kernels launched.
  int step(const std::vector<adamw::GroupValues>& groups, const StepNumbers& numbers, uint64_t seed);
  // A buffer of fp32 gradients that zero_grad() clears, whole.
  void add_grad_buffer(const at::Tensor& g);
  void zero_grad(uint64_t stream) { grads_.zero(device_, stream); }
  // Keeps the tensors of the plan alive (a plan that lives for one call does not need it).
  bool keep = false;
  // The first tensor's number among those of a step.
  uint32_t first_index = 0;

 private:
  int device_ = -1;
  adamw::Types types_{};
  std::vector<adamw::Segment> segs_;
  GradBuffers grads_;
  TensorList keep_;
};

int adamw_step(const TensorRefs& p, const TensorRefs& g, const TensorRefs& m, const TensorRefs& v, const std::optional<TensorRefs>& scales,
               const std::optional<TensorRefs>& copies, const adamw::GroupValues& values, const StepNumbers& numbers, uint64_t seed,
               uint32_t first_index);

// The values of moments held in 8 bits, into m_out and v_out.
int adamw_read8(const TensorRefs& m, const TensorRefs& v, const TensorRefs& scales, const TensorRefs& m_out, const TensorRefs& v_out);

}  // namespace trainer
}  // namespace bagua
