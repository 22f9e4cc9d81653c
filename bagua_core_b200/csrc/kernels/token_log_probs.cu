// See token_log_probs.h.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "index_report.cuh"
#include "launch.cuh"
#include "token_log_probs.h"
#include "typed_vec.cuh"

namespace bagua {
namespace token_log_probs {

namespace {

namespace cg = cooperative_groups;
using namespace kernels;
using encoder_ops::IndexReport;
using encoder_ops::report_index;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr unsigned kFull = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kNoToken = 0x7fffffff;

__device__ __forceinline__ float exp2_fast(float x) {  // to 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// ---- exponents ----------------------------------------------------------------------------------
// exp(x - m) is taken as 2^d, d = x log2(e) - m log2(e), one multiply-add with the same rounded m log2(e) for all of a row, so that its
// rounding leaves the probabilities.  d is held above kFar, where 2^d is 0, so that 2^d d is too, also for x = -inf.  For an m at
// the ends of fp32's range, where the product would be infinite, and for m = -inf, the difference is taken first.
constexpr float kFar = -1000.f, kWide = 2e38f;
__device__ __forceinline__ bool within(float m) { return fabsf(m) < kWide; }
__device__ __forceinline__ float exponent(float x, float log_m) { return max_nan(__fmaf_rn(x, kLog2e, -log_m), kFar); }
__device__ __forceinline__ float exponent_wide(float x, float m) { return max_nan((x - (m == -INFINITY ? 0.f : m)) * kLog2e, kFar); }

// Largest value m of what was seen, sum of 2^d, sum of 2^d d.
struct Sums {
  float m, s, t;
};
// The sums of values with largest value `m`, for a larger one `to`: every d grows by the difference.
__device__ __forceinline__ void shift(Sums& a, float to) {
  const float d = max_nan(within(a.m) && within(to) ? __fmul_rn(a.m, kLog2e) - __fmul_rn(to, kLog2e) : (a.m - to) * kLog2e, kFar);
  const float f = exp2_fast(d);
  a.t = f * __fmaf_rn(d, a.s, a.t);
  a.s *= f;
  a.m = to;
}
__device__ __forceinline__ Sums combine(Sums a, Sums b) {
  if (b.m > a.m) {
    const Sums c = a;
    a = b;
    b = c;
  }
  if (b.m != -INFINITY) shift(b, a.m);  // (nothing but -inf: the sums are 0, or NaN)
  a.s += b.s;
  a.t += b.t;
  return a;
}
__device__ __forceinline__ Sums combine_warp(Sums a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = combine(a, Sums{__shfl_xor_sync(kFull, a.m, o), __shfl_xor_sync(kFull, a.s, o), __shfl_xor_sync(kFull, a.t, o)});
  return a;
}
template <int N>
__device__ __forceinline__ void add(Sums& a, const float (&x)[N], float largest) {
  if (largest > a.m) {
    if (a.m == -INFINITY)
      a.m = largest;
    else
      shift(a, largest);
  }
  if (within(a.m)) {
    const float log_m = __fmul_rn(a.m, kLog2e);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float d = exponent(x[k], log_m), e = exp2_fast(d);
      a.s += e;
      a.t = __fmaf_rn(e, d, a.t);
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float d = exponent_wide(x[k], a.m), e = exp2_fast(d);
      a.s += e;
      a.t = __fmaf_rn(e, d, a.t);
    }
  }
}

// ---- alternatives -------------------------------------------------------------------------------
// A warp keeps the 32 best it has seen, one a lane, the best first; equal values in the order of their ids.
struct Best {
  float value;
  int id;
};
__device__ __forceinline__ bool better(float v, int id, float than, int than_id) { return v > than || (v == than && id < than_id); }
__device__ __forceinline__ void insert(Best& b, float v, int id) {
  const int lane = (int)threadIdx.x & 31;
  const int at = __popc(__ballot_sync(kFull, better(b.value, b.id, v, id)));
  const float up = __shfl_up_sync(kFull, b.value, 1);
  const int up_id = __shfl_up_sync(kFull, b.id, 1);
  if (lane > at) {
    b.value = up;
    b.id = up_id;
  } else if (lane == at) {
    b.value = v;
    b.id = id;
  }
}
// The last of the `top` best, which a candidate has to be better than.
struct Bar {
  float value;
  int id;
};
__device__ __forceinline__ Bar bar_of(const Best& b, int top) { return Bar{__shfl_sync(kFull, b.value, top - 1), __shfl_sync(kFull, b.id, top - 1)}; }
// One candidate a lane.
__device__ __forceinline__ void offer(Best& b, Bar& bar, int top, float v, int id, bool valid) {
  unsigned mask = __ballot_sync(kFull, valid && better(v, id, bar.value, bar.id));
  while (mask) {
    const int from = __ffs(mask) - 1;
    mask &= mask - 1;
    const float cv = __shfl_sync(kFull, v, from);
    const int ci = __shfl_sync(kFull, id, from);
    if (!better(cv, ci, bar.value, bar.id)) continue;
    insert(b, cv, ci);
    bar = bar_of(b, top);
  }
}
// fp32 in the order of whole numbers, for a maximum over warps
__device__ __forceinline__ int ordered(float x) {
  const int b = __float_as_int(x);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }

// ---- forward ------------------------------------------------------------------------------------
template <typename T>
struct ForwardArgs {
  const T* x;
  int64_t stride, rows, ignored;
  const int64_t* targets;
  float *log_probs, *entropy, *top_values;
  int64_t* top_ids;
  RowStats* stats;
  IndexReport* report;
  int vocab, top;
};

// A row's results, from its sums and, lane by lane, its best; by one warp.
template <typename T, bool kTop>
__device__ __forceinline__ void finish(const ForwardArgs<T>& a, int64_t row, const T* x, int64_t target, const Sums& u, const Best& best) {
  const int lane = (int)threadIdx.x & 31;
  const bool none = u.m == -INFINITY && u.s == 0.f, known = target >= 0 && target < a.vocab;
  const float log_s = log2f(u.s);
  auto log_prob = [&](float v) {
    if (none || v == -INFINITY) return u.s == u.s ? -INFINITY : nanf("");
    if (!within(u.m) || !within(v)) return (v - u.m) - log_s * kLn2;  // a logit at the type's lowest value has a finite one
    return (__fmaf_rn(v, kLog2e, -__fmul_rn(u.m, kLog2e)) - log_s) * kLn2;
  };
  if constexpr (kTop) {
    if (lane < a.top) {
      const bool there = u.s == u.s && best.id != kNoToken;
      a.top_values[row * a.top + lane] = u.s == u.s ? (there ? log_prob(best.value) : -INFINITY) : nanf("");
      a.top_ids[row * a.top + lane] = there ? best.id : -1;
    }
  }
  if (lane != 0) return;
  const float inverse = 1.f / u.s;
  const float entropy = none ? 0.f : (log_s - u.t * inverse) * kLn2;
  a.log_probs[row] = known ? log_prob(to_float(x[target])) : nanf("");
  a.entropy[row] = entropy;
  if (!known) report_index(a.report, encoder_ops::kTarget, target);
  if (a.stats) a.stats[row] = RowStats{u.m, inverse, entropy - log_s * kLn2, known && !none ? 1.f : 0.f};
}
template <typename T, bool kTop>
__device__ __forceinline__ void finish_ignored(const ForwardArgs<T>& a, int64_t row) {
  const int lane = (int)threadIdx.x & 31;
  if constexpr (kTop) {
    if (lane < a.top) {
      a.top_values[row * a.top + lane] = -INFINITY;
      a.top_ids[row * a.top + lane] = -1;
    }
  }
  if (lane != 0) return;
  a.log_probs[row] = 0.f;
  a.entropy[row] = 0.f;
  if (a.stats) a.stats[row] = RowStats{0.f, 0.f, 0.f, 0.f};
}

// Elements in front of the first 16-byte border of a row, and whole vectors behind it.
template <typename T>
__device__ __forceinline__ int in_front(const T* x, int vocab) {
  return min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
}

// The sums and the best of a part of a row, by a group of threads: `part` of `parts` of its vectors, and with part 0 what lies in front of and behind
// them.  Four vectors of a thread are under way together.
constexpr int kAhead = 4;
template <typename T, bool kTop, int kGroup>
__device__ __forceinline__ void scan(const T* x, int vocab, int part, int parts, int top, int* gate, Sums& u, Best& best) {
  constexpr int kVec = 16 / sizeof(T), kN = kVec * kAhead;
  const int tid = (int)threadIdx.x % kGroup;
  const int front = in_front(x, vocab), vectors = (vocab - front) / kVec;
  const int lo = (int)((int64_t)vectors * part / parts), hi = (int)((int64_t)vectors * (part + 1) / parts);
  const uint4* v = reinterpret_cast<const uint4*>(x + front);
  u = Sums{-INFINITY, 0.f, 0.f};
  best = Best{-INFINITY, kNoToken};
  Bar bar{-INFINITY, kNoToken};
  if (part == 0) {
    const int behind = front + vectors * kVec, rest = vocab - behind + front;
    const int id = tid < front ? tid : behind + tid - front;
    const bool valid = tid < rest;
    const float one[1] = {valid ? to_float(x[id]) : -INFINITY};
    add(u, one, one[0]);
    if constexpr (kTop) offer(best, bar, top, one[0], id, valid);
  }
  for (int base = lo; base < hi; base += kAhead * kGroup) {
    uint4 raw[kAhead];
    bool in[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      in[k] = base + k * kGroup + tid < hi;
      if (in[k]) raw[k] = v[base + k * kGroup + tid];
    }
    float f[kN], largest = -INFINITY;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const T* e = reinterpret_cast<const T*>(&raw[k]);
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        f[k * kVec + j] = in[k] ? to_float(e[j]) : -INFINITY;
        largest = fmaxf(largest, f[k * kVec + j]);
      }
    }
    add(u, f, largest);
    if constexpr (kTop) {
      // another warp's bar: no value below it is among the row's best
      const float floor = gate ? unordered(*(volatile int*)gate) : -INFINITY;
      if (__any_sync(kFull, largest >= fmaxf(bar.value, floor))) {
#pragma unroll
        for (int k = 0; k < kN; ++k)
          offer(best, bar, top, f[k], front + (base + k / kVec * kGroup + tid) * kVec + k % kVec, in[k / kVec] && f[k] >= floor);
        if (gate && (threadIdx.x & 31) == 0) atomicMax(gate, ordered(bar.value));
      }
    }
  }
}

// A warp for each row.
template <typename T, bool kTop>
__global__ void __launch_bounds__(kThreads) forward_short_kernel(const __grid_constant__ ForwardArgs<T> a) {
  wait_for_predecessor();
  const int64_t row = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= a.rows) return;
  const int64_t target = a.targets[row];
  if (target == a.ignored) return finish_ignored<T, kTop>(a, row);
  Sums u;
  Best best;
  const T* x = a.x + row * a.stride;
  scan<T, kTop, 32>(x, a.vocab, 0, 1, a.top, nullptr, u, best);
  finish<T, kTop>(a, row, x, target, combine_warp(u), best);
}

// A block, or a cluster of blocks, for each row.
template <typename T, bool kTop>
__global__ void __launch_bounds__(kThreads) forward_kernel(const __grid_constant__ ForwardArgs<T> a, int parts) {
  __shared__ Sums s_sums[kWarps];
  __shared__ Best s_best[kTop ? kWarps : 1][32];
  __shared__ int s_gate;
  wait_for_predecessor();
  const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x / parts;
  const int part = (int)(blockIdx.x % parts);
  const int64_t target = a.targets[row];
  if (target == a.ignored) {  // all blocks of a cluster
    if (part == 0 && warp == 0) finish_ignored<T, kTop>(a, row);
    return;
  }
  if constexpr (kTop) {
    if (threadIdx.x == 0) s_gate = ordered(-INFINITY);
    __syncthreads();
  }
  Sums u;
  Best best;
  const T* x = a.x + row * a.stride;
  scan<T, kTop, kThreads>(x, a.vocab, part, parts, a.top, &s_gate, u, best);
  u = combine_warp(u);
  if (lane == 0) s_sums[warp] = u;
  if constexpr (kTop) s_best[warp][lane] = best;
  if (parts == 1)
    __syncthreads();
  else
    cg::this_cluster().sync();
  if (part == 0 && warp == 0) {
    Bar bar{-INFINITY, kNoToken};
    if constexpr (kTop) bar = bar_of(best, a.top);
    for (int p = 0; p < parts; ++p) {
      const Sums* sums = parts == 1 ? s_sums : cg::this_cluster().map_shared_rank(s_sums, p);
      const Best* bests = parts == 1 ? &s_best[0][0] : cg::this_cluster().map_shared_rank(&s_best[0][0], p);
      for (int w = 0; w < kWarps; ++w) {
        if (p == 0 && w == 0) continue;
        u = combine(u, sums[w]);
        if constexpr (kTop) {
          const Best c = bests[w * 32 + lane];
          offer(best, bar, a.top, c.value, c.id, lane < a.top && c.id != kNoToken);
        }
      }
    }
    finish<T, kTop>(a, row, x, target, u, best);
  }
  if (parts > 1) cg::this_cluster().sync();  // a block's shared memory is read by the first
}

// ---- backward -----------------------------------------------------------------------------------
template <typename T>
struct BackwardArgs {
  const T* x;
  T* dx;
  int64_t stride, dx_stride, rows;
  const int64_t* targets;
  const RowStats* stats;
  const float *a, *b;
  int64_t a_stride, b_stride;
  int vocab;
};
// d x_j = -p_j (a + b (log p_j + entropy)) = -2^d (A + B d), with what d leaves of log p_j and the sum in A and B.
struct Coefficients {
  float m, log_m, A, B;
  __device__ __forceinline__ float operator()(float x) const {
    const float d = within(m) ? exponent(x, log_m) : exponent_wide(x, m);
    return -exp2_fast(d) * __fmaf_rn(B, d, A);
  }
};
template <typename T, int kGroup>
__device__ __forceinline__ void backward_part(const BackwardArgs<T>& g, int64_t row, int part, int parts) {
  constexpr int kVec = 16 / sizeof(T);
  const int tid = (int)threadIdx.x % kGroup;
  const T* x = g.x + row * g.stride;
  T* dx = g.dx + row * g.dx_stride;
  const int front = in_front(x, g.vocab), vectors = (g.vocab - front) / kVec;
  const int lo = (int)((int64_t)vectors * part / parts), hi = (int)((int64_t)vectors * (part + 1) / parts);
  const uint4* v = reinterpret_cast<const uint4*>(x + front);
  uint4* dv = reinterpret_cast<uint4*>(dx + front);
  const int behind = front + vectors * kVec, rest = g.vocab - behind + front;
  const int id = tid < front ? tid : behind + tid - front;  // outside the vectors, with part 0
  const RowStats st = g.stats[row];
  if (st.counts == 0.f) {
    for (int i = lo + tid; i < hi; i += kGroup) dv[i] = make_uint4(0, 0, 0, 0);
    if (part == 0 && tid < rest) dx[id] = from_float<T>(0.f);
    return;
  }
  const float a = g.a ? g.a[row * g.a_stride] : 0.f, b = g.b ? g.b[row * g.b_stride] : 0.f;
  const Coefficients c{st.top, __fmul_rn(st.top, kLog2e), st.inverse * __fmaf_rn(b, st.offset, a), st.inverse * b * kLn2};
  const int target = (int)g.targets[row];
  for (int base = lo; base < hi; base += kAhead * kGroup) {
    uint4 raw[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (base + k * kGroup + tid < hi) raw[k] = v[base + k * kGroup + tid];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = base + k * kGroup + tid;
      if (i >= hi) continue;
      T* e = reinterpret_cast<T*>(&raw[k]);
      const int first = front + i * kVec;
#pragma unroll
      for (int j = 0; j < kVec; ++j) e[j] = from_float<T>(c(to_float(e[j])));
      dv[i] = raw[k];
      if (target >= first && target < first + kVec) dx[target] = from_float<T>(c(to_float(x[target])) + a);
    }
  }
  if (part == 0 && tid < rest) dx[id] = from_float<T>(c(to_float(x[id])) + (id == target ? a : 0.f));
}
template <typename T>
__global__ void __launch_bounds__(kThreads) backward_short_kernel(const __grid_constant__ BackwardArgs<T> g) {
  wait_for_predecessor();
  const int64_t row = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row < g.rows) backward_part<T, 32>(g, row, 0, 1);
}
template <typename T>
__global__ void __launch_bounds__(kThreads) backward_kernel(const __grid_constant__ BackwardArgs<T> g, int parts) {
  wait_for_predecessor();
  backward_part<T, kThreads>(g, (int64_t)blockIdx.x / parts, (int)(blockIdx.x % parts), parts);
}

// Up to so many values, a warp takes a row.
constexpr int64_t kShort = 1024;

// Blocks of a cluster for a row: enough for two blocks on each SM, as long as each has a vector for every thread.
template <typename T>
int forward_parts(int64_t rows, int64_t vocab) {
  int parts = 1;
  const int64_t vectors = vocab * (int64_t)sizeof(T) / 16;
  while (parts < 8 && rows * parts < 2 * 148 && vectors / (2 * parts) >= kThreads) parts *= 2;
  return parts;
}

template <typename F>
void typed(DType t, F&& f) {
  switch (t) {
    case DType::F32: f((float*)nullptr); return;
    case DType::F16: f((__half*)nullptr); return;
    case DType::BF16: f((__nv_bfloat16*)nullptr); return;
    default: throw BaguaError(ErrorKind::Tensor, std::string("token_log_probs: unsupported type ") + dtype_name(t));
  }
}
void check(const Logits& l) {
  BAGUA_CHECK(l.rows > 0 && l.rows <= kMaxRows && l.vocab > 0 && l.vocab <= kMaxVocab, Tensor,
              "token_log_probs: " << l.rows << " rows of " << l.vocab << " logits");
}

template <typename T, bool kTop>
void launch_forward(const ForwardArgs<T>& a, cudaStream_t s) {
  if (a.vocab <= kShort) {
    launch_overlapped(forward_short_kernel<T, kTop>, dim3((unsigned)((a.rows + kWarps - 1) / kWarps)), dim3(kThreads), s, a);
    return;
  }
  const int parts = forward_parts<T>(a.rows, a.vocab);
  if (parts == 1)
    launch_overlapped(forward_kernel<T, kTop>, dim3((unsigned)a.rows), dim3(kThreads), s, a, 1);
  else
    launch_clusters(forward_kernel<T, kTop>, (int)a.rows, parts, dim3(kThreads), s, a, parts);
}

}  // namespace

void forward(const Logits& l, const int64_t* targets, int64_t ignored, int top, float* log_probs, float* entropy, float* top_values,
             int64_t* top_ids, RowStats* stats, cudaStream_t s) {
  check(l);
  BAGUA_CHECK(top >= 0 && top <= kMaxTop && top <= l.vocab, Tensor, "token_log_probs: " << top << " alternatives of " << l.vocab);
  typed(l.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const ForwardArgs<T> a{(const T*)l.x, l.stride,  l.rows, ignored, targets, log_probs, entropy, top_values, top_ids, stats, encoder_ops::index_report(),
                           (int)l.vocab,  top};
    top ? launch_forward<T, true>(a, s) : launch_forward<T, false>(a, s);
  });
}

void backward(const Logits& l, const int64_t* targets, const RowStats* stats, const float* a, int64_t a_stride, const float* b, int64_t b_stride,
              void* dx, int64_t dx_stride, cudaStream_t s) {
  check(l);
  typed(l.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    BAGUA_CHECK(((uintptr_t)l.x - (uintptr_t)dx) % 16 == 0 && (l.rows == 1 || (l.stride - dx_stride) * (int64_t)sizeof(T) % 16 == 0), Tensor,
                "token_log_probs: the gradient's rows lie differently from the logits'");
    const BackwardArgs<T> g{(const T*)l.x, (T*)dx, l.stride, dx_stride, l.rows, targets, stats, a, b, a_stride, b_stride, (int)l.vocab};
    if (l.vocab <= kShort) {
      launch_overlapped(backward_short_kernel<T>, dim3((unsigned)((l.rows + kWarps - 1) / kWarps)), dim3(kThreads), s, g);
      return;
    }
    const int64_t vectors = l.vocab * (int64_t)sizeof(T) / 16;
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(vectors / (kThreads * kAhead), ((1ll << 31) - 1) / l.rows));
    launch_overlapped(backward_kernel<T>, dim3((unsigned)(l.rows * parts)), dim3(kThreads), s, g, (int)parts);
  });
}

}  // namespace token_log_probs
}  // namespace bagua
