// See token_log_probs.h.
//
// Forward: one pass over a row, running maximum and sums in each thread's registers, joined once at the row's end.  A row is a warp's, a
// block's or a cluster's, by its length and the number of rows.  Bound by memory for long rows (2000 of 131072 in bf16: 86 us, 6.1
// TB/s; 4096 of 32003 in fp32: 84 us, 6.2), for rows of some tens of KB also by what a block does once a row (4096 of 30522 in bf16:
// 46 us, 5.4 TB/s; the exponentials alone take 28), for few rows by latency (one of 30522: 3.6 us, with 5 alternatives 7).
// Backward: reads and writes each logit once, 4096 of 30522 in bf16 in 80 us, 6.2 TB/s.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "clusters.h"
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

__device__ __forceinline__ Pair exp2_fast(Pair p) {
  const float2 f = halves(p);
  return pair(exp2_fast(f.x), exp2_fast(f.y));
}

// ---- elements -----------------------------------------------------------------------------------
// A 16-byte vector of logits: its largest value, and its values as pairs, held at or above kHeld.  A type of 16 bits is compared two
// at a time, before it is widened: comparing is what these passes have fewest instructions a cycle for.
template <typename T>
struct Elements;
template <>
struct Elements<float> {
  static constexpr int kPairs = 2;
  static constexpr float kHeld = -1e38f, kNear = 0x1p20f;
  static constexpr uint32_t kMasked = 0xff800000u;  // words of -inf
  __device__ static float largest(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  __device__ static void pairs(const uint4& v, Pair (&p)[kPairs]) {
    p[0] = pair(__uint_as_float(v.x), __uint_as_float(v.y));
    p[1] = pair(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  __device__ static uint32_t held(uint32_t w) { return __float_as_uint(max_nan(__uint_as_float(w), kHeld)); }
  __device__ static uint4 narrow(const Pair (&p)[kPairs]) {
    const float2 a = halves(p[0]), b = halves(p[1]);
    return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
  }
};
template <typename T, typename T2>
struct Elements16 {
  static constexpr int kPairs = 4;
  __device__ static T2 two(uint32_t w) { return *reinterpret_cast<const T2*>(&w); }
  __device__ static float largest(const uint4& v) {
    const T2 m = __hmax2(__hmax2(two(v.x), two(v.y)), __hmax2(two(v.z), two(v.w)));
    return fmaxf(to_float(m.x), to_float(m.y));
  }
  __device__ static uint32_t held(uint32_t w, uint32_t least) {
    const T2 m = __hmax2_nan(two(w), two(least));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
};
template <>
struct Elements<__half> : Elements16<__half, __half2> {
  static constexpr float kHeld = -65504.f, kNear = 6e4f;
  static constexpr uint32_t kMasked = 0xfc00fc00u;
  __device__ static uint32_t held(uint32_t w) { return Elements16::held(w, 0xfbfffbffu); }
  __device__ static void pairs(const uint4& v, Pair (&p)[kPairs]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = __half22float2(two(w[k]));
      p[k] = pair(f.x, f.y);
    }
  }
  __device__ static uint4 narrow(const Pair (&p)[kPairs]) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = halves(p[k]);
      const __half2 h = __floats2half2_rn(f.x, f.y);
      w[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Elements<__nv_bfloat16> : Elements16<__nv_bfloat16, __nv_bfloat162> {
  static constexpr float kHeld = -1e38f, kNear = 0x1p20f;
  static constexpr uint32_t kMasked = 0xff80ff80u;
  __device__ static uint32_t held(uint32_t w) { return Elements16::held(w, 0xfe96fe96u); }  // -9.97e37
  __device__ static void pairs(const uint4& v, Pair (&p)[kPairs]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = pair(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
  }
  __device__ static uint4 narrow(const Pair (&p)[kPairs]) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = halves(p[k]);
      const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
      w[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <typename T>
__device__ __forceinline__ uint4 held(const uint4& v) {
  return make_uint4(Elements<T>::held(v.x), Elements<T>::held(v.y), Elements<T>::held(v.z), Elements<T>::held(v.w));
}

// ---- exponents ----------------------------------------------------------------------------------
// exp(x - m) is taken as 2^d, d = x log2(e) - m log2(e), one multiply-add with the same rounded m log2(e) for all of a row, so that its
// rounding, the same in every d, leaves the probabilities.  It is 2^-4 at most for |m| below kNear; at 1e10 it would be 440, and no 2^d in
// range.  x is held above -inf before, so that d is finite and 2^d d is 0 where 2^d is.  For any other m (in fp16: next to the ends of its
// range; NaN and infinities too) the difference x - m is taken first ("wide"): two instructions more an element.
constexpr float kFar = -1000.f;
template <typename T>
__device__ __forceinline__ bool within(float m) { return fabsf(m) < Elements<T>::kNear; }
__device__ __forceinline__ float exponent_wide(float x, float m) { return max_nan((x - (m == -INFINITY ? 0.f : m)) * kLog2e, kFar); }
__device__ __forceinline__ Pair exponent_wide(Pair x, float m) {
  const float2 f = halves(x);
  return pair(exponent_wide(f.x, m), exponent_wide(f.y, m));
}

// Largest value m of what was seen, sum of 2^d, sum of 2^d d.
struct Sums {
  float m, s, t;
};
// The factor of sums of values with largest value `m`, for a larger one `to`, and by how much every d grows: what the two take off x log2(e),
// rounded or not, as the form of each has it.
template <typename T>
__device__ __forceinline__ float shift_sums(float m, float to, float* d) {
  const float l = __fmul_rn(m, kLog2e), l_to = __fmul_rn(to, kLog2e);
  const bool near = within<T>(m), near_to = within<T>(to);
  *d = max_nan(near ? (near_to ? l - l_to : __fmaf_rn(-to, kLog2e, l)) : near_to ? __fmaf_rn(m, kLog2e, -l_to) : (m - to) * kLog2e, kFar);
  return exp2_fast(*d);
}
// The sums of a warp's lanes: all are moved to the largest m, then added.  (Nothing but -inf in a lane: its sums are 0, or NaN.)
template <typename T>
__device__ __forceinline__ Sums combine_warp(Sums a) {
  float m = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
  if (a.m != -INFINITY) {
    float d;
    const float f = shift_sums<T>(a.m, m, &d);
    a.t = f * __fmaf_rn(d, a.s, a.t);
    a.s *= f;
  }
  a.m = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(kFull, a.s, o);
    a.t += __shfl_xor_sync(kFull, a.t, o);
  }
  return a;
}
// A thread's sums, two of each.
struct Running {
  float m = -INFINITY;
  Pair s = 0, t = 0;  // (0: two zeros)
  __device__ __forceinline__ Sums sums() const {
    const float2 a = halves(s), b = halves(t);
    return Sums{m, a.x + a.y, b.x + b.y};
  }
};
template <typename T, int N>
__device__ __forceinline__ void accumulate(Running& a, const uint4 (&v)[N], float largest) {
  using E = Elements<T>;
  if (largest > a.m) {
    if (a.m != -INFINITY) {
      float d;
      const float f = shift_sums<T>(a.m, largest, &d);
      a.t = mul(pair(f, f), fma(pair(d, d), a.s, a.t));
      a.s = mul(pair(f, f), a.s);
    }
    a.m = largest;
  }
  if (within<T>(a.m)) {
    const float l = -__fmul_rn(a.m, kLog2e);
    const Pair log2e = pair(kLog2e, kLog2e), less = pair(l, l);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      Pair x[E::kPairs];
      E::pairs(held<T>(v[k]), x);
#pragma unroll
      for (int j = 0; j < E::kPairs; ++j) {
        const Pair d = fma(x[j], log2e, less), e = exp2_fast(d);
        a.s = add(a.s, e);
        a.t = fma(e, d, a.t);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      Pair x[E::kPairs];
      E::pairs(v[k], x);
#pragma unroll
      for (int j = 0; j < E::kPairs; ++j) {
        const Pair d = exponent_wide(x[j], a.m), e = exp2_fast(d);
        a.s = add(a.s, e);
        a.t = fma(e, d, a.t);
      }
    }
  }
}

// ---- parts of a row -----------------------------------------------------------------------------
// Elements in front of the first 16-byte border, whole vectors, elements behind them; a part of the vectors is lo .. hi, and its group of
// threads has the elements outside the vectors if it is the first.
struct RowPart {
  int front, behind, rest, lo, hi;  // rest: elements outside the vectors, 0 if they are another part's
  __device__ __forceinline__ int outside(int k) const { return k < front ? k : behind + k - front; }
};
// Part `part` of 2^shift equal ones.
template <typename T>
__device__ __forceinline__ RowPart row_part(const T* x, int vocab, int part, int shift) {
  constexpr int kVec = 16 / sizeof(T);
  RowPart r;
  r.front = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
  const int vectors = (vocab - r.front) / kVec;
  r.behind = r.front + vectors * kVec;
  r.rest = part == 0 ? vocab - r.behind + r.front : 0;
  r.lo = (int)((int64_t)vectors * part >> shift);
  r.hi = (int)((int64_t)vectors * (part + 1) >> shift);
  return r;
}

// A thread has this many vectors of a row under way together, a turn.
constexpr int kAhead = 4;
// Turns that share one of the kSteps largest values that a thread leaves.
template <int kGroup>
constexpr int kSteps = kGroup == 32 ? 2 : 16;
template <int kGroup>
__device__ __forceinline__ int turns_of_step(const RowPart& r) {
  const int turns = (r.hi - r.lo + kAhead * kGroup - 1) / (kAhead * kGroup);
  return turns > kSteps<kGroup> ? (turns + kSteps<kGroup> - 1) / kSteps<kGroup> : 1;
}

// ---- alternatives -------------------------------------------------------------------------------
// The `top` largest of a group of threads' values, equal ones in the order of their ids, -inf and NaN not among them.
//
// A list kept along the way costs ten times the pass itself (64 rows of 131072, 20 alternatives: 90 us; now 15, without them 7).
// Here the pass leaves the largest value of every few vectors of a thread.  From the threads' largest ones comes a floor that at least
// `top` values reach, and in rows that are not ordered few more: the least, over the warps, of the top / warps-th largest of a warp's lanes.  The vectors
// whose largest value reaches the floor are read again, the values that do are collected, and put in order by counting, for each, the
// better ones.  Where that collects too many, as in a row with a few hundred tokens left, all neighbours, the floor is the top-th largest of all
// threads' values, and where that does too, values being equal, one alternative is looked for after the other.
//
// A candidate is one number: its value in the order of whole numbers, then its id from the last to the first.
using Key = unsigned long long;
constexpr Key kNoKey = 0;
__device__ __forceinline__ Key key_of(float v, int id) {
  const uint32_t b = __float_as_uint(v + 0.f);  // (-0 is 0)
  return (Key)(b ^ ((uint32_t)((int)b >> 31) | 0x80000000u)) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float value_of(Key k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float(b ^ ((b >> 31) - 1u | 0x80000000u));
}
__device__ __forceinline__ int id_of(Key k) { return (int)~(uint32_t)k; }
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
  Key found[kRoom];
  int reach[kRoom];  // the first vectors of steps with a value that reaches the floor
  float step[kSteps<kGroup>][kGroup];
  float floor[kGroup / 32], largest[kGroup];
  int count, steps;
};

// Calls f(value, id) for the elements of a thread's share of a part.
template <typename T, int kGroup, typename F>
__device__ __forceinline__ void each_value(const T* x, const RowPart& r, F&& f) {
  constexpr int kVec = 16 / sizeof(T);
  const int tid = (int)threadIdx.x % kGroup;
  if (tid < r.rest) f(to_float(x[r.outside(tid)]), r.outside(tid));
  for (int i = r.lo + tid; i < r.hi; i += kGroup) {
    const int first = r.front + i * kVec;
#pragma unroll
    for (int j = 0; j < kVec; ++j) f(to_float(x[first + j]), first + j);
  }
}

// Collects the values of a part that reach the floor, and returns how many there are, kRoom + 1 for any number above kRoom, of which not all are in
// s.found.  `largest`: of this thread's values.  All threads of the group; s.count and s.steps are 0.
template <typename T, int kGroup>
__device__ __forceinline__ int collect(const T* x, const RowPart& r, float floor, float largest, TopScratch<kGroup>& s) {
  constexpr int kVec = 16 / sizeof(T);
  const int tid = (int)threadIdx.x % kGroup;
  // the steps that reach the floor, dealt out to all threads: a thread's own would wait for one another
  const int vectors = turns_of_step<kGroup>(r) * kAhead;
  if (largest >= floor && largest > -INFINITY) {
    if (tid < r.rest) {
      const float v = to_float(x[r.outside(tid)]);
      if (v >= floor && v > -INFINITY) {
        const int at = atomicAdd(&s.count, 1);
        if (at < kRoom) s.found[at] = key_of(v, r.outside(tid));
      }
    }
    int step = 0;
    for (int base = r.lo + tid; base < r.hi; base += vectors * kGroup, ++step) {
      if (!(s.step[step][tid] >= floor)) continue;
      const int at = atomicAdd(&s.steps, 1);
      if (at < kRoom) s.reach[at] = base;
    }
  }
  sync_group<kGroup>();
  const int steps = s.steps;
  if (steps <= kRoom) {
    for (int k = tid; k < steps * vectors; k += kGroup) {
      const int i = s.reach[k / vectors] + k % vectors * kGroup;
      if (i >= r.hi) continue;
      const uint4 raw = reinterpret_cast<const uint4*>(x + r.front)[i];
      if (!(Elements<T>::largest(raw) >= floor)) continue;
      const T* e = reinterpret_cast<const T*>(&raw);
      int n = 0;
#pragma unroll
      for (int j = 0; j < kVec; ++j) n += to_float(e[j]) >= floor && to_float(e[j]) > -INFINITY;
      if (n == 0) continue;
      int at = atomicAdd(&s.count, n);
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (to_float(e[j]) >= floor && to_float(e[j]) > -INFINITY) {
          if (at < kRoom) s.found[at] = key_of(to_float(e[j]), r.front + i * kVec + j);
          ++at;
        }
    }
  }
  sync_group<kGroup>();
  return steps <= kRoom ? min(s.count, kRoom + 1) : kRoom + 1;
}

// The group's best into best[0 .. top), kNoKey where there are no more; `largest`: of this thread's values.  All threads of the group.
template <typename T, int kGroup>
__device__ __forceinline__ void choose(const T* x, const RowPart& r, int top, float largest, TopScratch<kGroup>& s, Key* best) {
  constexpr int kGroupWarps = kGroup / 32;
  const int tid = (int)threadIdx.x % kGroup, lane = tid & 31;
  {
    int before = 0;  // lanes with larger values, or equal ones in front
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      const float v = __shfl_sync(kFull, largest, k);
      before += (int)(v > largest) | ((int)(v == largest) & (int)(k < lane));
    }
    if (before == (top - 1) / kGroupWarps) s.floor[tid >> 5] = largest;
  }
  if (tid == 0) s.count = s.steps = 0;
  for (int k = tid; k < top; k += kGroup) best[k] = kNoKey;
  if constexpr (kGroupWarps > 1) s.largest[tid] = largest;
  sync_group<kGroup>();
  float floor = s.floor[0];
#pragma unroll
  for (int k = 1; k < kGroupWarps; ++k) floor = fminf(floor, s.floor[k]);
  int count = collect<T, kGroup>(x, r, floor, largest, s);
  if constexpr (kGroupWarps > 1) {
    if (count > kRoom) {
      sync_group<kGroup>();  // everybody has read the counts
      int before = 0;
#pragma unroll 8
      for (int k = 0; k < kGroup; ++k) before += (int)(s.largest[k] > largest) | ((int)(s.largest[k] == largest) & (int)(k < tid));
      if (before == top - 1) s.floor[0] = largest;
      if (tid == 0) s.count = s.steps = 0;
      sync_group<kGroup>();
      const float higher = s.floor[0];
      if (higher > floor) count = collect<T, kGroup>(x, r, higher, largest, s);
    }
  }
  if (count <= kRoom) {
    // four lanes share a candidate
    for (int base = 0; base < count; base += kGroup / 4) {
      const int k = base + tid / 4;
      const Key mine = s.found[min(k, count - 1)];
      int before = 0;
#pragma unroll 4
      for (int o = tid % 4; o < count; o += 4) before += s.found[o] > mine;
      before += __shfl_xor_sync(kFull, before, 1);
      before += __shfl_xor_sync(kFull, before, 2);
      if (tid % 4 == 0 && k < count && before < top) best[before] = mine;
    }
    sync_group<kGroup>();
    return;
  }
  Key last = ~0ull;
  for (int k = 0; k < top; ++k) {
    Key mine = kNoKey;
    each_value<T, kGroup>(x, r, [&](float v, int id) {
      const Key c = key_of(v, id);
      if (v > -INFINITY && c < last && c > mine) mine = c;
    });
    s.found[tid] = mine;
    sync_group<kGroup>();
#pragma unroll 8
    for (int o = 0; o < kGroup; ++o) mine = max(mine, s.found[o]);
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
__device__ __forceinline__ void finish(const ForwardArgs<T>& a, int64_t row, const T* x, int64_t target, float at_target, const Sums& u, Key best) {
  const int lane = (int)threadIdx.x & 31;
  const bool none = u.m == -INFINITY && u.s == 0.f, known = target >= 0 && target < a.vocab;
  const float log_s = log2f(u.s);
  auto log_prob = [&](float v) {
    if (none || v == -INFINITY) return u.s == u.s ? -INFINITY : nanf("");
    if (!within<T>(u.m) || v <= Elements<T>::kHeld) return (v - u.m) - log_s * kLn2;  // a logit at the type's lowest value has a finite one
    return (__fmaf_rn(v, kLog2e, -__fmul_rn(u.m, kLog2e)) - log_s) * kLn2;
  };
  if constexpr (kTop) {
    const int found = __popc(__ballot_sync(kFull, lane < a.top && best != kNoKey));
    float v = value_of(best);
    int id = id_of(best);
    if (found < a.top) {  // the first of those at -inf, which are among the row's first `top`
      unsigned gone = __ballot_sync(kFull, lane < a.top && to_float(x[min(lane, a.vocab - 1)]) == -INFINITY);
      for (int k = found; k < lane; ++k) gone &= gone - 1;
      if (lane >= found) {
        v = -INFINITY;
        id = gone ? __ffs(gone) - 1 : -1;
      }
    }
    if (lane < a.top) {
      a.top_values[row * a.top + lane] = u.s == u.s ? log_prob(v) : nanf("");
      a.top_ids[row * a.top + lane] = u.s == u.s ? id : -1;
    }
  }
  if (lane != 0) return;
  const float inverse = 1.f / u.s;
  const float entropy = none ? 0.f : (log_s - u.t * inverse) * kLn2;
  a.log_probs[row] = known ? log_prob(at_target) : nanf("");
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

// The sums of a part of a row, by a group of threads.  With kTop, steps[k][thread] becomes the largest value of the thread's k-th step.
template <typename T, bool kTop, int kGroup>
__device__ __forceinline__ Sums scan(const T* x, const RowPart& r, float (*steps)[kGroup]) {
  const int tid = (int)threadIdx.x % kGroup;
  const uint4* v = reinterpret_cast<const uint4*>(x + r.front);
  constexpr uint32_t masked = Elements<T>::kMasked;
  const uint4 none = make_uint4(masked, masked, masked, masked);
  Running u;
  auto load = [&](uint4 (&raw)[kAhead], int base) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) raw[k] = base + k * kGroup < r.hi ? v[base + k * kGroup] : none;
  };
  uint4 next[kAhead];
  load(next, r.lo + tid);
  if (tid < r.rest) {
    T e = x[r.outside(tid)];
    uint32_t w = masked;
    if constexpr (sizeof(T) == 4)
      w = __float_as_uint(e);
    else
      w = (masked & 0xffff0000u) | *reinterpret_cast<const uint16_t*>(&e);
    const uint4 one[1] = {make_uint4(w, masked, masked, masked)};
    accumulate<T>(u, one, Elements<T>::largest(one[0]));
  }
  const int turns = kTop ? turns_of_step<kGroup>(r) : 0;
  int turn = 0, step = 0;
  float step_largest = -INFINITY;
  for (int base = r.lo + tid; base < r.hi; base += kAhead * kGroup) {
    uint4 raw[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) raw[k] = next[k];
    load(next, base + kAhead * kGroup);  // the next turn's are on their way while this one is computed
    float largest = Elements<T>::largest(raw[0]);
#pragma unroll
    for (int k = 1; k < kAhead; ++k) largest = fmaxf(largest, Elements<T>::largest(raw[k]));
    accumulate<T>(u, raw, largest);
    if constexpr (kTop) {
      step_largest = fmaxf(step_largest, largest);
      steps[step][tid] = step_largest;
      if (++turn == turns) {
        turn = 0;
        ++step;
        step_largest = -INFINITY;
      }
    }
  }
  return u.sums();
}

// A warp for each row.
template <typename T, bool kTop>
__global__ void __launch_bounds__(kThreads) forward_short_kernel(const __grid_constant__ ForwardArgs<T> a) {
  __shared__ TopScratch<32> s_top[kTop ? kWarps : 1];
  __shared__ Key s_best[kTop ? kWarps : 1][32];
  wait_for_predecessor();
  const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * kWarps + warp;
  if (row >= a.rows) return;
  const int64_t target = a.targets[row];
  if (target == a.ignored) return finish_ignored<T, kTop>(a, row);
  const T* x = a.x + row * a.stride;
  const float at_target = target >= 0 && target < a.vocab ? to_float(x[target]) : 0.f;  // asked for now, needed last
  const RowPart r = row_part(x, a.vocab, 0, 0);
  const Sums u = scan<T, kTop, 32>(x, r, s_top[kTop ? warp : 0].step);
  Key best = kNoKey;
  if constexpr (kTop) {
    choose<T, 32>(x, r, a.top, u.m, s_top[warp], s_best[warp]);
    if (lane < a.top) best = s_best[warp][lane];
  }
  finish<T, kTop>(a, row, x, target, at_target, combine_warp<T>(u), best);
}

// A block, or a cluster of 2^shift blocks, for each row.
constexpr int kMaxParts = 8;
template <typename T, bool kTop, int kGroup>
__global__ void __launch_bounds__(kGroup) forward_kernel(const __grid_constant__ ForwardArgs<T> a, int shift) {
  constexpr int kGroupWarps = kGroup / 32;
  __shared__ Sums s_sums[kGroupWarps];
  __shared__ TopScratch<kGroup> s_top;
  __shared__ Key s_best[kTop ? 32 : 1], s_all[kTop ? kMaxParts * 32 : 1], s_joined[32];
  wait_for_predecessor();
  const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5, parts = 1 << shift;
  const int64_t row = blockIdx.x >> shift;
  const int part = (int)blockIdx.x & (parts - 1);
  const int64_t target = a.targets[row];
  const T* x = a.x + row * a.stride;
  // With few rows nothing is gained by not looking at one, and its logits come sooner without a look at the target.
  if (shift == 0 && target == a.ignored) {
    if (warp == 0) finish_ignored<T, kTop>(a, row);
    return;
  }
  const RowPart r = row_part(x, a.vocab, part, shift);
  Sums u = scan<T, kTop, kGroup>(x, r, s_top.step);
  if (shift > 0 && target == a.ignored) {  // all blocks of a cluster
    if (part == 0 && warp == 0) finish_ignored<T, kTop>(a, row);
    return;
  }
  const float at_target = part == 0 && target >= 0 && target < a.vocab ? to_float(x[target]) : 0.f;  // asked for now, needed last
  if constexpr (kTop) choose<T, kGroup>(x, r, a.top, u.m, s_top, s_best);
  u = combine_warp<T>(u);
  if (lane == 0) s_sums[warp] = u;
  if (shift == 0)
    __syncthreads();
  else
    cg::this_cluster().sync();
  if (part == 0) {
    Key best = kNoKey;
    if constexpr (kTop) {
      if (shift == 0) {
        if (warp == 0 && lane < a.top) best = s_best[lane];
      } else {
        // the parts' best, each of which finds its place among all of them
        for (int p = warp; p < parts; p += kGroupWarps) s_all[p * 32 + lane] = lane < a.top ? cg::this_cluster().map_shared_rank(s_best, p)[lane] : kNoKey;
        if (threadIdx.x < 32) s_joined[threadIdx.x] = kNoKey;
        __syncthreads();
        for (int p = warp; p < parts; p += kGroupWarps) {
          // how many of each part's, which are in order, are better: found by halves, the parts side by side
          const Key mine = s_all[p * 32 + lane];
          int place[kMaxParts] = {};
          for (int step = a.top > 8 ? 16 : 4; step > 0; step /= 2)
#pragma unroll
            for (int q = 0; q < kMaxParts; ++q)
              if (q < parts && s_all[q * 32 + place[q] + step - 1] > mine) place[q] += step;
          int before = 0;
#pragma unroll
          for (int q = 0; q < kMaxParts; ++q)
            if (q < parts) before += place[q] + (s_all[q * 32 + place[q]] > mine);
          if (mine != kNoKey && before < a.top) s_joined[before] = mine;
        }
        __syncthreads();
        if (warp == 0) best = s_joined[lane];
      }
    }
    if (warp == 0) {
      // the sums of up to 64 warps
      Sums all{-INFINITY, 0.f, 0.f};
      if (shift == 0) {
        if (lane < kGroupWarps) all = s_sums[lane];
      } else {
        Sums two[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int w = lane + 32 * k;
          two[k] = w < parts * kGroupWarps ? cg::this_cluster().map_shared_rank(s_sums, w / kGroupWarps)[w % kGroupWarps] : Sums{-INFINITY, 0.f, 0.f};
        }
        all.m = fmaxf(two[0].m, two[1].m);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float d = 0.f;
          const float f = two[k].m == -INFINITY ? 1.f : shift_sums<T>(two[k].m, all.m, &d);
          all.t += f * __fmaf_rn(d, two[k].s, two[k].t);
          all.s += f * two[k].s;
        }
      }
      finish<T, kTop>(a, row, x, target, at_target, combine_warp<T>(all), best);
    }
  }
  if (shift > 0) cg::this_cluster().sync();  // a block's shared memory is read by the first
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
// d x_j = -p_j (a + b (log p_j + entropy)) = 2^d A + 2^d d B, with the sum and what d leaves of log p_j in A and B.  2^d d comes first: d is
// -1.4e38 at masked tokens, where its product with B would be infinite, and NaN once it met the 2^d that is 0.
template <typename T>
struct Coefficients {
  float m, A, B;
  __device__ __forceinline__ void operator()(const uint4& v, Pair (&g)[Elements<T>::kPairs]) const {
    const Pair a = pair(A, A), b = pair(B, B);
    if (within<T>(m)) {
      const float l = -__fmul_rn(m, kLog2e);
      const Pair log2e = pair(kLog2e, kLog2e), less = pair(l, l);
      Elements<T>::pairs(held<T>(v), g);
#pragma unroll
      for (int k = 0; k < Elements<T>::kPairs; ++k) {
        const Pair d = fma(g[k], log2e, less), e = exp2_fast(d);
        g[k] = fma(mul(e, d), b, mul(e, a));
      }
    } else {
      Elements<T>::pairs(v, g);
#pragma unroll
      for (int k = 0; k < Elements<T>::kPairs; ++k) {
        const Pair d = exponent_wide(g[k], m), e = exp2_fast(d);
        g[k] = fma(mul(e, d), b, mul(e, a));
      }
    }
  }
  __device__ __forceinline__ float operator()(T x) const {
    uint4 v = make_uint4(Elements<T>::kMasked, Elements<T>::kMasked, Elements<T>::kMasked, Elements<T>::kMasked);
    *reinterpret_cast<T*>(&v) = x;
    Pair g[Elements<T>::kPairs];
    (*this)(v, g);
    return halves(g[0]).x;
  }
};
template <typename T, int kGroup>
__device__ __forceinline__ void backward_part(const BackwardArgs<T>& g, int64_t row, int part, int shift) {
  constexpr int kVec = 16 / sizeof(T);
  const int tid = (int)threadIdx.x % kGroup;
  const T* x = g.x + row * g.stride;
  T* dx = g.dx + row * g.dx_stride;
  const RowPart r = row_part(x, g.vocab, part, shift);
  const uint4* v = reinterpret_cast<const uint4*>(x + r.front);
  uint4* dv = reinterpret_cast<uint4*>(dx + r.front);
  const RowStats st = g.stats[row];
  const float a = g.a ? g.a[row * g.a_stride] : 0.f, b = g.b ? g.b[row * g.b_stride] : 0.f;
  const int target = (int)g.targets[row];
  if (st.counts == 0.f) {
    for (int i = r.lo + tid; i < r.hi; i += kGroup) dv[i] = make_uint4(0, 0, 0, 0);
    if (tid < r.rest) dx[r.outside(tid)] = from_float<T>(0.f);
    return;
  }
  uint4 next[kAhead];
  auto load = [&](int base) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (base + k * kGroup < r.hi) next[k] = v[base + k * kGroup];
  };
  load(r.lo + tid);
  const Coefficients<T> c{st.top, -st.inverse * __fmaf_rn(b, st.offset, a), -st.inverse * b * kLn2};
  for (int base = r.lo + tid; base < r.hi; base += kAhead * kGroup) {
    uint4 raw[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) raw[k] = next[k];
    load(base + kAhead * kGroup);  // the next turn's are on their way while this one is computed
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = base + k * kGroup;
      if (i >= r.hi) continue;
      Pair d[Elements<T>::kPairs];
      c(raw[k], d);
      dv[i] = Elements<T>::narrow(d);
      const int first = r.front + i * kVec;
      if (target >= first && target < first + kVec) dx[target] = from_float<T>(c(x[target]) + a);
    }
  }
  if (tid < r.rest) {
    const int id = r.outside(tid);
    dx[id] = from_float<T>(c(x[id]) + (id == target ? a : 0.f));
  }
}
template <typename T>
__global__ void __launch_bounds__(kThreads) backward_short_kernel(const __grid_constant__ BackwardArgs<T> g) {
  wait_for_predecessor();
  const int64_t row = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row < g.rows) backward_part<T, 32>(g, row, 0, 0);
}
template <typename T>
__global__ void __launch_bounds__(kThreads) backward_kernel(const __grid_constant__ BackwardArgs<T> g, int shift) {
  wait_for_predecessor();
  backward_part<T, kThreads>(g, (int64_t)(blockIdx.x >> shift), (int)blockIdx.x & ((1 << shift) - 1), shift);
}

// Up to so many values, a warp takes a row.
constexpr int64_t kShort = 1024;
// Many rows of few bytes go to blocks of half as many threads: more rows are under way, and the blocks' joint steps at a row's end cost less.  us with
// 128 / 256 threads: 4096 rows of 30522 in bf16 46.5 / 49.1, with 20 alternatives 63 / 79; but 517 such rows 9.6 / 9.0, 2000 of 32003 in
// fp32 47.9 / 44.0, 2000 of 131072 in bf16 88.2 / 85.9.
constexpr int64_t kManyRows = 4 * 148, kSmallRow = 64 << 10;

// Blocks of a cluster for a row, as a power of two: enough for two blocks on each SM, as long as each has a vector for every thread.
template <typename T>
int forward_shift(int64_t rows, int64_t vocab) {
  int shift = 0;
  const int64_t vectors = vocab * (int64_t)sizeof(T) / 16;
  while ((1 << shift) < kMaxParts && rows << shift < 2 * 148 && vectors >> (shift + 1) >= kThreads) ++shift;
  return shift;
}
// Blocks for a row: two for each SM, as in the forward pass.  (Eight: 517 rows of 30522 in bf16 12.1 us instead of 9.5, 148 of 131072 alike.)
template <typename T>
int backward_shift(int64_t rows, int64_t vocab) {
  int shift = 0;
  const int64_t vectors = vocab * (int64_t)sizeof(T) / 16;
  while (rows << shift < 2 * 148 && vectors >> (shift + 1) >= kThreads) ++shift;
  return shift;
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
  int shift = forward_shift<T>(a.rows, a.vocab);
  if (shift > 0)
    for (int fit = fitting_cluster((const void*)forward_kernel<T, kTop, kThreads>, 1 << shift, kThreads, 0, s); 1 << shift > fit;) --shift;
  if (shift > 0)
    launch_clusters(forward_kernel<T, kTop, kThreads>, (int)a.rows, 1 << shift, dim3(kThreads), s, a, shift);
  else if (a.rows >= kManyRows && (int64_t)a.vocab * (int64_t)sizeof(T) <= kSmallRow)
    launch_overlapped(forward_kernel<T, kTop, kThreads / 2>, dim3((unsigned)a.rows), dim3(kThreads / 2), s, a, 0);
  else
    launch_overlapped(forward_kernel<T, kTop, kThreads>, dim3((unsigned)a.rows), dim3(kThreads), s, a, 0);
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
    const int shift = backward_shift<T>(l.rows, l.vocab);
    launch_overlapped(backward_kernel<T>, dim3((unsigned)(l.rows << shift)), dim3(kThreads), s, g, shift);
  });
}

}  // namespace token_log_probs
}  // namespace bagua
