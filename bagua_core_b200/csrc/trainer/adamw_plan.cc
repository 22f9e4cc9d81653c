#include "adamw_plan.h"

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

namespace bagua {
namespace trainer {

namespace {

bool real(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }
DType dtype_of(at::ScalarType t) { return t == at::kFloat ? DType::F32 : t == at::kHalf ? DType::F16 : DType::BF16; }

// Whether `t` has its elements where `p`, a tensor without gaps, has them.
bool same_layout(const at::Tensor& t, const at::Tensor& p) {
  return t.sizes() == p.sizes() && (t.strides() == p.strides() || (t.is_contiguous() && p.is_contiguous()));
}

void check_scales(const at::Tensor& scales, int64_t n, const at::Device& device) {
  BAGUA_CHECK(scales.scalar_type() == at::kFloat && scales.dim() == 2 && scales.size(0) == 2 && scales.size(1) == adamw::moment8_blocks(n) &&
                  (scales.size(1) <= 1 || scales.stride(1) == 1) && scales.device() == device,
              Tensor, "the scales of 8-bit moments of " << n << " elements are a float32 tensor [2, " << adamw::moment8_blocks(n)
                                                        << "] with neighbouring columns, on their device");
}

void check_values(const adamw::GroupValues& g) {
  BAGUA_CHECK(g.lr >= 0 && std::isfinite(g.lr) && g.eps >= 0 && std::isfinite(g.eps) && g.b1 >= 0 && g.b1 < 1 && g.b2 >= 0 && g.b2 < 1 &&
                  g.weight_decay >= 0 && std::isfinite(g.weight_decay),
              Tensor, "AdamW needs lr, eps and weight_decay of 0 or more and betas from 0 to below 1; got lr " << fmt_double(g.lr) << ", betas "
                          << fmt_double(g.b1) << " and " << fmt_double(g.b2) << ", eps " << fmt_double(g.eps) << ", weight_decay "
                          << fmt_double(g.weight_decay));
}

cudaStream_t stream_on(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

// A tensor's memory.  Those of a kind (all parameters, all gradients, ...) are a list.
struct Piece {
  uintptr_t from, to;
};
struct Pieces {
  std::vector<Piece> list;
  bool written = true;
  void add(const void* p, int64_t bytes) {
    if (p && bytes > 0) list.push_back({(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes});
  }
};
// Throws if a piece that is written overlaps another one.
void check_apart(std::vector<Pieces>& kinds) {
  constexpr const char* what = "a buffer that is written overlaps another one of the same call";
  auto before = [](const Piece& a, const Piece& b) { return a.from < b.from; };
  // Lists whose pieces follow each other, in a part of memory that no other list has: slices of flat buffers.  Seen without sorting them all.
  std::vector<Piece> whole;
  bool apart = true;
  for (const Pieces& k : kinds) {
    if (k.list.empty()) continue;
    for (size_t i = 1; i < k.list.size() && apart; ++i) apart = k.list[i].from >= k.list[i - 1].to;
    whole.push_back({k.list.front().from, k.list.back().to});
  }
  std::sort(whole.begin(), whole.end(), before);
  for (size_t i = 1; i < whole.size() && apart; ++i) apart = whole[i].from >= whole[i - 1].to;
  if (apart) return;
  struct Mixed : Piece {
    bool written;
  };
  std::vector<Mixed> all;
  for (const Pieces& k : kinds)
    for (const Piece& p : k.list) all.push_back({{p.from, p.to}, k.written});
  std::sort(all.begin(), all.end(), before);
  uintptr_t read = 0, written = 0;  // the furthest ends so far
  for (const Mixed& x : all) {
    BAGUA_CHECK(x.from >= written && (!x.written || x.from >= read), Tensor, what);
    (x.written ? written : read) = std::max(x.written ? written : read, x.to);
  }
}

// Lets autograd notice that a graph's values have changed since.
void note_written(const TensorRefs& list) {
  for (const at::Tensor* t : list)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

}  // namespace

void AdamWPlan::add(const at::Tensor& p, const at::Tensor& g, const at::Tensor& m, const at::Tensor& v,
                    const at::Tensor* scales, const at::Tensor* copy, int group) {
  BAGUA_CHECK((p.is_cuda() || p.is_cpu()) && real(p.scalar_type()) && real(g.scalar_type()) && p.layout() == at::kStrided, Tensor,
              "AdamW works on float32, float16 and bfloat16 tensors on a GPU or the host");
  const int device = p.is_cuda() ? (int)p.device().index() : -1;
  const bool moments8 = m.scalar_type() == at::kByte;
  const adamw::Types types{dtype_of(p.scalar_type()), dtype_of(g.scalar_type()), moments8};
  BAGUA_CHECK(adamw::supported(types), Tensor,
              "AdamW needs gradients of the parameters' type or float32, or float32 parameters; got " << p.scalar_type() << " and "
                                                                                                    << g.scalar_type());
  const at::ScalarType held = moments8 ? at::kByte : at::kFloat;
  BAGUA_CHECK(m.scalar_type() == held && v.scalar_type() == held, Tensor, "AdamW's moments are both float32, or both codes of 8 bits (uint8)");
  BAGUA_CHECK(!p.is_neg() && !g.is_neg() && !m.is_neg() && !v.is_neg(), Tensor,
              "AdamW needs tensors that hold their values as they are, not negated views");
  BAGUA_CHECK(p.is_non_overlapping_and_dense(), Tensor, "AdamW needs parameters without gaps between their elements");
  for (const at::Tensor* t : {&g, &m, &v})
    BAGUA_CHECK(t->layout() == at::kStrided && t->device() == p.device() && same_layout(*t, p), Tensor,
                "AdamW needs gradients and moments of the parameter's sizes and strides, on its device");
  BAGUA_CHECK(moments8 == (scales != nullptr), Tensor, "moments of 8 bits need scales, others have none");
  if (scales) check_scales(*scales, p.numel(), p.device());
  if (copy)
    BAGUA_CHECK(copy->scalar_type() == at::kBFloat16 && copy->device() == p.device() && same_layout(*copy, p) && !copy->is_neg(), Tensor,
                "the copy must be a bfloat16 tensor of the parameter's sizes and strides on its device");
  BAGUA_CHECK(segs_.empty() || (device == device_ && types.p == types_.p && types.g == types_.g && types.moments8 == types_.moments8), Tensor,
              "the tensors of an AdamW step are of one kind: one device, one type of parameters, of gradients and of moments");
  BAGUA_CHECK(group >= 0 && group < 32768, Tensor, "parameter group " << group << " is not one of the first 32768");
  device_ = device;
  types_ = types;
  adamw::Segment a{};
  a.p = p.data_ptr();
  a.g = g.data_ptr();
  a.m = m.data_ptr();
  a.v = v.data_ptr();
  a.copy = copy ? copy->data_ptr() : nullptr;
  if (scales) {
    a.m_scale = scales->data_ptr<float>();
    a.v_scale = a.m_scale + scales->stride(0);
  }
  a.n = p.numel();
  a.index = first_index + (uint32_t)segs_.size();
  a.group = (int16_t)group;
  segs_.push_back(a);
  if (!keep) return;
  keep_.insert(keep_.end(), {p, g, m, v});
  if (scales) keep_.push_back(*scales);
  if (copy) keep_.push_back(*copy);
}

void AdamWPlan::add_grad_buffer(const at::Tensor& g) {
  BAGUA_CHECK(g.scalar_type() == at::kFloat && g.is_contiguous() && (g.is_cuda() ? (int)g.device().index() : -1) == device_, Tensor,
              "gradients are zeroed as contiguous float32 buffers on the plan's device");
  grads_.add(g);
  keep_.push_back(g);
}

void AdamWPlan::check_apart() const {
  std::vector<Pieces> kinds(7);
  for (auto& k : kinds) k.list.reserve(segs_.size());
  kinds[1].written = false;
  const int64_t p = (int64_t)dtype_bytes(types_.p), g = (int64_t)dtype_bytes(types_.g), held = types_.moments8 ? 1 : 4;
  for (const auto& a : segs_) {
    const int64_t blocks = adamw::moment8_blocks(a.n) * 4;
    kinds[0].add(a.p, a.n * p);
    kinds[1].add(a.g, a.n * g);
    kinds[2].add(a.m, a.n * held);
    kinds[3].add(a.v, a.n * held);
    kinds[4].add(a.copy, a.n * 2);
    kinds[5].add(a.m_scale, blocks);
    kinds[6].add(a.v_scale, blocks);
  }
  trainer::check_apart(kinds);
}

int AdamWPlan::step(const std::vector<adamw::GroupValues>& groups, const StepNumbers& numbers, uint64_t seed) {
  if (segs_.empty()) return 0;
  for (const auto& g : groups) check_values(g);
  for (const auto& a : segs_) BAGUA_CHECK((size_t)a.group < groups.size(), Tensor, "no hyperparameters for parameter group " << a.group);
  auto hypers = [&](const std::vector<int64_t>& steps) {
    BAGUA_CHECK(steps.size() == groups.size(), Tensor, "AdamW needs a step's number for each parameter group");
    std::vector<adamw::Hyper> h;
    for (size_t k = 0; k < groups.size(); ++k) {
      BAGUA_CHECK(steps[k] >= 1, Tensor, "AdamW's steps are counted from 1, got " << steps[k]);
      h.push_back(adamw::hyper(groups[k], steps[k], seed));
    }
    return h;
  };
  if (numbers.device)
    BAGUA_CHECK(numbers.device->scalar_type() == at::kLong && numbers.device->is_contiguous() && numbers.device->numel() == (int64_t)groups.size() &&
                    (device_ < 0 ? numbers.device->is_cpu() : numbers.device->is_cuda() && (int)numbers.device->device().index() == device_),
                Tensor, "AdamW takes steps' numbers in a tensor as one int64 for each parameter group, on the parameters' device");
  if (device_ < 0) {
    std::vector<int64_t> steps = numbers.host;
    if (numbers.device) steps.assign(numbers.device->data_ptr<int64_t>(), numbers.device->data_ptr<int64_t>() + groups.size());
    adamw::host::step(types_, segs_.data(), (int)segs_.size(), hypers(steps).data());
    return 1;
  }
  const c10::cuda::CUDAGuard on((c10::DeviceIndex)device_);
  const cudaStream_t s = stream_on(device_);
  if (numbers.device) {
    const at::Tensor& t = *numbers.device;
    // the framework's memory, not this package's pool: a graph that is being captured keeps it
    const at::Tensor scratch = at::detail::empty_cuda({(int64_t)(groups.size() * sizeof(adamw::Hyper))}, at::kByte, t.device(), c10::nullopt);
    auto* h = (adamw::Hyper*)scratch.data_ptr();
    const int launches = adamw::cuda::hypers(groups.data(), (int)groups.size(), t.data_ptr<int64_t>(), seed, h, s);
    return launches + adamw::cuda::step(types_, segs_.data(), (int)segs_.size(), h, (int)groups.size(), true, s);
  }
  cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
  BAGUA_CUDA_CHECK(cudaStreamIsCapturing(s, &capturing));
  BAGUA_CHECK(capturing == cudaStreamCaptureStatusNone, Tensor,
              "a captured AdamW step needs its number on the device (an int64 tensor): a number of the host would be the same at every replay");
  const auto h = hypers(numbers.host);
  return adamw::cuda::step(types_, segs_.data(), (int)segs_.size(), h.data(), (int)h.size(), false, s);
}

int adamw_step(const TensorRefs& p, const TensorRefs& g, const TensorRefs& m, const TensorRefs& v, const std::optional<TensorRefs>& scales,
               const std::optional<TensorRefs>& copies, const adamw::GroupValues& values, const StepNumbers& numbers, uint64_t seed,
               uint32_t first_index) {
  const size_t n = p.size();
  BAGUA_CHECK(g.size() == n && m.size() == n && v.size() == n && (!scales || scales->size() == n) && (!copies || copies->size() == n), Tensor,
              "AdamW needs lists of one length");
  AdamWPlan plan;
  plan.first_index = first_index;
  plan.reserve(n);
  for (size_t k = 0; k < n; ++k)
    plan.add(*p[k], *g[k], *m[k], *v[k], scales ? (*scales)[k] : nullptr, copies ? (*copies)[k] : nullptr, 0);
  plan.check_apart();
  const int launches = plan.step({values}, numbers, seed);
  for (const TensorRefs* list : {&p, &m, &v}) note_written(*list);
  if (scales) note_written(*scales);
  if (copies) note_written(*copies);
  return launches;
}

int adamw_read8(const TensorRefs& m, const TensorRefs& v, const TensorRefs& scales, const TensorRefs& m_out, const TensorRefs& v_out) {
  const size_t n = m.size();
  BAGUA_CHECK(v.size() == n && scales.size() == n && m_out.size() == n && v_out.size() == n, Tensor, "reading moments needs lists of one length");
  if (n == 0) return 0;
  const at::ScalarType type = m_out[0]->scalar_type();
  const at::Device device = m[0]->device();
  BAGUA_CHECK((m[0]->is_cuda() || m[0]->is_cpu()) && real(type), Tensor,
              "moments on a GPU or the host are read into float32, float16 or bfloat16 tensors");
  std::vector<adamw::cuda::Read8> segs;
  std::vector<Pieces> kinds(6);
  for (auto& k : kinds) k.list.reserve(n);
  for (int k = 0; k < 4; ++k) kinds[k].written = false;
  segs.reserve(n);
  for (size_t k = 0; k < n; ++k) {
    BAGUA_CHECK(m[k]->scalar_type() == at::kByte && v[k]->scalar_type() == at::kByte && m_out[k]->scalar_type() == type &&
                    v_out[k]->scalar_type() == type,
                Tensor, "moments are read from codes of 8 bits (uint8) into tensors of one type");
    BAGUA_CHECK(m[k]->is_non_overlapping_and_dense() && m[k]->device() == device, Tensor,
                "moments are read from tensors without gaps, on one device");
    BAGUA_CHECK(!m[k]->is_neg() && !v[k]->is_neg() && !m_out[k]->is_neg() && !v_out[k]->is_neg(), Tensor,
                "moments are read from and into tensors that hold their values as they are, not negated views");
    for (const at::Tensor* t : {v[k], m_out[k], v_out[k]})
      BAGUA_CHECK(t->device() == device && same_layout(*t, *m[k]), Tensor, "moments and what they are read into have one size and layout, on one device");
    check_scales(*scales[k], m[k]->numel(), device);
    const float* s = scales[k]->data_ptr<float>();
    segs.push_back({m[k]->data_ptr<uint8_t>(), v[k]->data_ptr<uint8_t>(), s, s + scales[k]->stride(0), m_out[k]->data_ptr(), v_out[k]->data_ptr(),
                    m[k]->numel()});
    const int64_t bytes = m[k]->numel() * (int64_t)m_out[k]->element_size(), blocks = adamw::moment8_blocks(m[k]->numel()) * 4;
    kinds[0].add(segs.back().m, m[k]->numel());
    kinds[1].add(segs.back().v, m[k]->numel());
    kinds[2].add(segs.back().m_scale, blocks);
    kinds[3].add(segs.back().v_scale, blocks);
    kinds[4].add(segs.back().m_out, bytes);
    kinds[5].add(segs.back().v_out, bytes);
  }
  check_apart(kinds);
  int launches = 1;
  if (m[0]->is_cuda()) {
    const c10::cuda::CUDAGuard on(device);
    launches = adamw::cuda::read8(segs.data(), (int)n, dtype_of(type), stream_on((int)device.index()));
  } else {
    adamw::host::read8(segs.data(), (int)n, dtype_of(type));
  }
  note_written(m_out);
  note_written(v_out);
  return launches;
}

}  // namespace trainer
}  // namespace bagua
