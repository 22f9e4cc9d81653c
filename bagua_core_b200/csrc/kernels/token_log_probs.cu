// See token_log_probs.h.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

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

// ---- parts of a row -----------------------------------------------------------------------------
// Elements in front of the first 16-byte border, whole vectors, elements behind them; `part` of `parts` of the vectors is lo .. hi.
struct RowParts {
  int front, behind, rest, lo, hi;  // rest: elements outside the vectors
};
template <typename T>
__device__ __forceinline__ RowParts row_parts(const T* x, int vocab, int part, int parts) {
  constexpr int kVec = 16 / sizeof(T);
  RowParts r;
  r.front = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
  const int vectors = (vocab - r.front) / kVec;
  r.behind = r.front + vectors * kVec;
  r.rest = vocab - r.behind + r.front;
  r.lo = (int)((int64_t)vectors * part / parts);
  r.hi = (int)((int64_t)vectors * (part + 1) / parts);
  return r;
}

// ---- alternatives -------------------------------------------------------------------------------
// The `top` largest of a group of threads' values, equal ones in the order of their ids, -inf and NaN not among them.
//
// A list kept along the way costs ten times the pass itself (64 rows of 131072, 20 alternatives: 98 us).  Here the first
// pass leaves each thread's largest value, which the sums have anyway.  The top-th largest of those is a floor: that many values at
// least are not below it, and in rows that are not ordered hardly more.  A second pass, from L2, collects the values that
// reach the floor, and those few are put in order by counting, for each, the better ones.
struct Best {
  float value;
  int id;
};
__device__ __forceinline__ bool better(const Best& a, const Best& b) { return a.value > b.value || (a.value == b.value && a.id < b.id); }
constexpr int kNoToken = 0x7fffffff;
constexpr int kRoom = 256;  // candidates of a group; where more reach the floor (equal values), they are taken a few at a time

template <int kGroup>
__device__ __forceinline__ void sync_group() {
  if constexpr (kGroup == 32)
    __syncwarp();
  else
    __syncthreads();
}
template <int kGroup>
struct TopScratch {
  float largest[kGroup];
  Best found[kRoom];
  int count;
  float floor;
};

// Calls f(value, id) for the elements of a thread's part of a row.
template <typename T, int kGroup, typename F>
__device__ __forceinline__ void each_value(const T* x, int vocab, int part, int parts, F&& f) {
  constexpr int kVec = 16 / sizeof(T);
  const int tid = (int)threadIdx.x % kGroup;
  const RowParts r = row_parts(x, vocab, part, parts);
  if (part == 0 && tid < r.rest) {
    const int id = tid < r.front ? tid : r.behind + tid - r.front;
    const float v[1] = {to_float(x[id])};
    f(v, id);
  }
  const uint4* v = reinterpret_cast<const uint4*>(x + r.front);
#pragma unroll 4
  for (int i = r.lo + tid; i < r.hi; i += kGroup) {
    const uint4 raw = v[i];
    const T* e = reinterpret_cast<const T*>(&raw);
    float w[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) w[j] = to_float(e[j]);
    f(w, r.front + i * kVec);
  }
}

// The group's best into best[0 .. top), kNoToken where there are no more; `largest`: of this thread's values.  All threads of the group.
template <typename T, int kGroup>
__device__ __forceinline__ void choose(const T* x, int vocab, int part, int parts, int top, float largest, TopScratch<kGroup>& s, Best* best) {
  const int tid = (int)threadIdx.x % kGroup;
  s.largest[tid] = largest;
  if (tid == 0) s.count = 0;
  sync_group<kGroup>();
  {
    int before = 0;
#pragma unroll 8
    for (int k = 0; k < kGroup; ++k) before += s.largest[k] > largest || (s.largest[k] == largest && k < tid);
    if (before == top - 1) s.floor = largest;
  }
  sync_group<kGroup>();
  const float floor = s.floor;
  each_value<T, kGroup>(x, vocab, part, parts, [&](const auto& v, int id) {
    constexpr int n = sizeof(v) / sizeof(float);
    float most = v[0];
#pragma unroll
    for (int j = 1; j < n; ++j) most = fmaxf(most, v[j]);
    if (most >= floor && most > -INFINITY) {
#pragma unroll
      for (int j = 0; j < n; ++j)
        if (v[j] >= floor && v[j] > -INFINITY) {
          const int at = atomicAdd(&s.count, 1);
          if (at < kRoom) s.found[at] = Best{v[j], id + j};
        }
    }
  });
  sync_group<kGroup>();
  const int count = s.count;
  if (count <= kRoom) {
    for (int k = tid; k < top; k += kGroup) best[k] = Best{-INFINITY, kNoToken};
    sync_group<kGroup>();
    for (int k = tid; k < count; k += kGroup) {
      const Best mine = s.found[k];
      int before = 0;
      for (int o = 0; o < count; ++o) before += better(s.found[o], mine);
      if (before < top) best[before] = mine;
    }
    sync_group<kGroup>();
    return;
  }
  // Too many of one value: one alternative after the other, each the best behind the one before.
  Best last{INFINITY, -1};
  for (int k = 0; k < top; ++k) {
    Best mine{-INFINITY, kNoToken};
    each_value<T, kGroup>(x, vocab, part, parts, [&](const auto& v, int id) {
      constexpr int n = sizeof(v) / sizeof(float);
#pragma unroll
      for (int j = 0; j < n; ++j) {
        const Best c{v[j], id + j};
        if (v[j] > -INFINITY && better(last, c) && better(c, mine)) mine = c;
      }
    });
    s.found[tid] = mine;
    sync_group<kGroup>();
    for (int o = 0; o < kGroup; ++o)
      if (better(s.found[o], mine)) mine = s.found[o];
    if (tid == 0) best[k] = mine;
    last = mine;
    sync_group<kGroup>();
  }
}

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

// A row's results, by one warp, from its sums and its best, of which lane k has the k-th.
template <typename T, bool kTop>
__device__ __forceinline__ void finish(const ForwardArgs<T>& a, int64_t row, const T* x, int64_t target, const Sums& u, Best best) {
  const int lane = (int)threadIdx.x & 31;
  const bool none = u.m == -INFINITY && u.s == 0.f, known = target >= 0 && target < a.vocab;
  const float log_s = log2f(u.s);
  auto log_prob = [&](float v) {
    if (none || v == -INFINITY) return u.s == u.s ? -INFINITY : nanf("");
    if (!within(u.m) || !within(v)) return (v - u.m) - log_s * kLn2;  // a logit at the type's lowest value has a finite one
    return (__fmaf_rn(v, kLog2e, -__fmul_rn(u.m, kLog2e)) - log_s) * kLn2;
  };
  if constexpr (kTop) {
    // fewer tokens than asked for: the first of those at -inf, which are among the row's first `top`
    const int found = __popc(__ballot_sync(kFull, lane < a.top && best.id != kNoToken));
    const unsigned gone = __ballot_sync(kFull, lane < a.top && to_float(x[min(lane, a.vocab - 1)]) == -INFINITY);
    if (lane >= found && lane < a.top) best = Best{-INFINITY, (int)__fns(gone, 0, lane - found + 1)};
    if (lane < a.top) {
      a.top_values[row * a.top + lane] = u.s == u.s ? log_prob(best.value) : nanf("");
      a.top_ids[row * a.top + lane] = u.s == u.s ? best.id : -1;
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

// The sums of a part of a row, by a group of threads: with part 0 also of what lies outside its vectors.  Four vectors of a thread are under way
// together.
constexpr int kAhead = 4;
template <typename T, int kGroup>
__device__ __forceinline__ Sums scan(const T* x, int vocab, int part, int parts) {
  constexpr int kVec = 16 / sizeof(T), kN = kVec * kAhead;
  const int tid = (int)threadIdx.x % kGroup;
  const RowParts r = row_parts(x, vocab, part, parts);
  const uint4* v = reinterpret_cast<const uint4*>(x + r.front);
  Sums u{-INFINITY, 0.f, 0.f};
  if (part == 0 && tid < r.rest) {
    const float one[1] = {to_float(x[tid < r.front ? tid : r.behind + tid - r.front])};
    add(u, one, fmaxf(-INFINITY, one[0]));
  }
  for (int base = r.lo + tid; base < r.hi; base += kAhead * kGroup) {
    uint4 raw[kAhead];
    bool in[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      in[k] = base + k * kGroup < r.hi;
      if (in[k]) raw[k] = v[base + k * kGroup];
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
  }
  return u;
}

// A warp for each row.
template <typename T, bool kTop>
__global__ void __launch_bounds__(kThreads) forward_short_kernel(const __grid_constant__ ForwardArgs<T> a) {
  __shared__ TopScratch<32> s_top[kTop ? kWarps : 1];
  __shared__ Best s_best[kTop ? kWarps : 1][32];
  wait_for_predecessor();
  const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * kWarps + warp;
  if (row >= a.rows) return;
  const int64_t target = a.targets[row];
  if (target == a.ignored) return finish_ignored<T, kTop>(a, row);
  const T* x = a.x + row * a.stride;
  const Sums u = scan<T, 32>(x, a.vocab, 0, 1);
  Best best{-INFINITY, kNoToken};
  if constexpr (kTop) {
    choose<T, 32>(x, a.vocab, 0, 1, a.top, u.m, s_top[warp], s_best[warp]);
    if (lane < a.top) best = s_best[warp][lane];
  }
  finish<T, kTop>(a, row, x, target, combine_warp(u), best);
}

// A block, or a cluster of blocks, for each row.
constexpr int kMaxParts = 8;
template <typename T, bool kTop>
__global__ void __launch_bounds__(kThreads) forward_kernel(const __grid_constant__ ForwardArgs<T> a, int parts) {
  __shared__ Sums s_sums[kWarps];
  __shared__ TopScratch<kTop ? kThreads : 1> s_top;
  __shared__ Best s_best[kTop ? 32 : 1];
  __shared__ Best s_all[kTop ? kMaxParts * 32 : 1];
  wait_for_predecessor();
  const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x / parts;
  const int part = (int)(blockIdx.x % parts);
  const int64_t target = a.targets[row];
  if (target == a.ignored) {  // all blocks of a cluster
    if (part == 0 && warp == 0) finish_ignored<T, kTop>(a, row);
    return;
  }
  const T* x = a.x + row * a.stride;
  Sums u = scan<T, kThreads>(x, a.vocab, part, parts);
  if constexpr (kTop) choose<T, kThreads>(x, a.vocab, part, parts, a.top, u.m, s_top, s_best);
  u = combine_warp(u);
  if (lane == 0) s_sums[warp] = u;
  if (parts == 1)
    __syncthreads();
  else
    cg::this_cluster().sync();
  if (part == 0) {
    Best best{-INFINITY, kNoToken};
    if constexpr (kTop) {
      if (parts == 1) {
        if (warp == 0 && lane < a.top) best = s_best[lane];
      } else {
        // warp p brings part p's best; each finds its place among all of them
        Best mine{-INFINITY, kNoToken};
        if (warp < parts && lane < a.top) mine = cg::this_cluster().map_shared_rank(s_best, warp)[lane];
        s_all[threadIdx.x] = mine;
        __syncthreads();
        int before = 0;
        for (int p = 0; p < parts; ++p)
          for (int k = 0; k < a.top; ++k) before += better(s_all[p * 32 + k], mine);
        __syncthreads();
        if (threadIdx.x < 32) s_all[threadIdx.x] = Best{-INFINITY, kNoToken};
        __syncthreads();
        if (mine.id != kNoToken && before < a.top) s_all[before] = mine;
        __syncthreads();
        if (warp == 0 && lane < a.top) best = s_all[lane];
      }
    }
    if (warp == 0) {
      // the sums of up to 64 warps, in the same tree whatever their number
      Sums all{-INFINITY, 0.f, 0.f};
      for (int k = lane; k < parts * kWarps; k += 32) {
        const Sums* from = parts == 1 ? s_sums : cg::this_cluster().map_shared_rank(s_sums, k / kWarps);
        all = combine(all, from[k % kWarps]);
      }
      finish<T, kTop>(a, row, x, target, combine_warp(all), best);
    }
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
  const RowParts r = row_parts(x, g.vocab, part, parts);
  const int front = r.front, lo = r.lo, hi = r.hi, rest = r.rest;
  const uint4* v = reinterpret_cast<const uint4*>(x + front);
  uint4* dv = reinterpret_cast<uint4*>(dx + front);
  const int id = tid < front ? tid : r.behind + tid - front;  // outside the vectors, with part 0
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
  while (parts < kMaxParts && rows * parts < 2 * 148 && vectors / (2 * parts) >= kThreads) parts *= 2;
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
