// See adamw.h.  Streams over memory: with fp32 parameters, gradients and moments 28 bytes an element, 16 with moments in 8 bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <vector>

#include "adamw.h"
#include "adamw_math.h"
#include "launch.cuh"

namespace bagua {
namespace adamw {

namespace {

using kernels::launch_overlapped;
using kernels::wait_for_predecessor;

constexpr int kThreads = 256;

// Segments are cut into tiles, a block each; the table of them travels with the launch.  A launch's parameters may take 32,764
// bytes; a step of few tensors takes the small table, whose 4 KB reach the GPU sooner.
constexpr int kGroups = 8;
template <int N>
struct Table {
  Segment seg[N];
  Hyper hyper[kGroups];
  const Hyper* on_device;  // instead of `hyper`, where the step's number lies on the device
  uint32_t first_tile[N + 1];
  int n;
};
constexpr int kFew = 44, kMany = 400;
static_assert(sizeof(Table<kFew>) <= 4096 && sizeof(Table<kMany>) <= 32764, "launch parameters");

template <typename First>
__device__ __forceinline__ int find_segment(const First& first_tile, int n, uint32_t tile) {
  int lo = 0, hi = n;  // first_tile[lo] <= tile < first_tile[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first_tile[mid] <= tile)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Four neighbouring elements, as one access where their address is a multiple of their size.
template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T x[4];
};
template <typename T>
__device__ __forceinline__ void load4(const T* at, float (&f)[4]) {
  const Four<T> v = *reinterpret_cast<const Four<T>*>(at);
#pragma unroll
  for (int k = 0; k < 4; ++k) f[k] = to_float(v.x[k]);
}
template <typename T>
__device__ __forceinline__ void store4(T* at, const float (&f)[4]) {
  Four<T> v;
#pragma unroll
  for (int k = 0; k < 4; ++k) v.x[k] = from_float<T>(f[k]);
  *reinterpret_cast<Four<T>*>(at) = v;
}
template <typename T>
__device__ __forceinline__ bool fours(const T* p) {
  return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0;
}

// ---- moments in fp32 ----------------------------------------------------------------------------
constexpr int kTile32 = kThreads * 4;
template <typename P, typename G, int N>
__global__ void __launch_bounds__(kThreads) step32_kernel(const __grid_constant__ Table<N> table) {
  wait_for_predecessor();
  const int k = find_segment(table.first_tile, table.n, blockIdx.x);
  const Segment& a = table.seg[k];
  const Hyper h = table.on_device ? table.on_device[a.group] : table.hyper[a.group];
  P* p = (P*)a.p;
  const G* g = (const G*)a.g;
  float *m = (float*)a.m, *v = (float*)a.v;
  auto* copy = (__nv_bfloat16*)a.copy;
  const int64_t base = (int64_t)(blockIdx.x - table.first_tile[k]) * kTile32;
  if (base + kTile32 <= a.n && fours(p) && fours(g) && fours(m) && fours(v) && fours(copy)) {
    const int64_t i = base + threadIdx.x * 4;
    float pv[4], gv[4], mv[4], vv[4];
    load4(p + i, pv);
    load4(g + i, gv);
    load4(m + i, mv);
    load4(v + i, vv);
#pragma unroll
    for (int e = 0; e < 4; ++e) update(h, pv[e], gv[e], mv[e], vv[e]);
    store4(p + i, pv);
    store4(m + i, mv);
    store4(v + i, vv);
    if (copy) store4(copy + i, pv);
  } else {
    const int64_t end = min(base + kTile32, a.n);
    for (int64_t i = base + threadIdx.x; i < end; i += kThreads) {
      float pv = to_float(p[i]), mv = m[i], vv = v[i];
      update(h, pv, to_float(g[i]), mv, vv);
      p[i] = from_float<P>(pv);
      m[i] = mv;
      v[i] = vv;
      if (copy) copy[i] = __float2bfloat16_rn(pv);
    }
  }
}

// ---- moments in 8 bits --------------------------------------------------------------------------
// A warp takes a block of elements that share their scales, eight to a lane: the largest value of a block is a reduction over the
// warp's registers, and each element is read and written once.  Lanes hold two runs of four, so that the 32 loads of a run are one
// piece of memory; elements of an address that no vector fits are taken one by one, lane by lane.
constexpr int kTile8 = kThreads / 32 * kMoment8Block;
template <typename P, typename G, int N>
__global__ void __launch_bounds__(kThreads) step8_kernel(const __grid_constant__ Table<N> table) {
  wait_for_predecessor();
  const int k = find_segment(table.first_tile, table.n, blockIdx.x);
  const Segment& a = table.seg[k];
  const int lane = (int)threadIdx.x & 31;
  const int64_t block = (int64_t)(blockIdx.x - table.first_tile[k]) * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t base = block * kMoment8Block;
  if (base >= a.n) return;
  const Hyper h = table.on_device ? table.on_device[a.group] : table.hyper[a.group];
  P* p = (P*)a.p;
  const G* g = (const G*)a.g;
  uint8_t *m = (uint8_t*)a.m, *v = (uint8_t*)a.v;
  auto* copy = (__nv_bfloat16*)a.copy;
  const float ms = a.m_scale[block], vs = a.v_scale[block];
  const bool vec = base + kMoment8Block <= a.n && fours(p) && fours(g) && fours(m) && fours(v) && fours(copy);
  // element e of run r: base + at(r, e)
  const int run = vec ? lane * 4 : lane, run_step = 128, step = vec ? 1 : 32;
  const int n = (int)min((int64_t)kMoment8Block, a.n - base);
  float pv[2][4], gv[2][4], mv[2][4], vv[2][4];
  uint32_t mc[2], vc[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t i = base + r * run_step + run;
    if (vec) {
      load4(p + i, pv[r]);
      load4(g + i, gv[r]);
      mc[r] = *reinterpret_cast<const uint32_t*>(m + i);
      vc[r] = *reinterpret_cast<const uint32_t*>(v + i);
    } else {
      mc[r] = vc[r] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = r * run_step + run + e * 32 < n;
        pv[r][e] = in ? to_float(p[i + e * 32]) : 0.f;
        gv[r][e] = in ? to_float(g[i + e * 32]) : 0.f;
        mc[r] |= (in ? (uint32_t)m[i + e * 32] : 0u) << (8 * e);
        vc[r] |= (in ? (uint32_t)v[i + e * 32] : 0u) << (8 * e);
      }
    }
  }
  uint32_t top_m = 0, top_v = 0;
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      mv[r][e] = decode1((mc[r] >> (8 * e)) & 0xffu, ms);
      vv[r][e] = decode2((vc[r] >> (8 * e)) & 0xffu, vs);
      update(h, pv[r][e], gv[r][e], mv[r][e], vv[r][e]);
      // an element behind the end leaves the scales alone
      const bool in = vec || r * run_step + run + e * step < n;
      top_m = max(top_m, in ? float_bits(mv[r][e]) & 0x7fffffffu : 0u);
      top_v = max(top_v, in ? float_bits(vv[r][e]) & 0x7fffffffu : 0u);
    }
  const uint32_t key = segment_key(h.random, a.index);
  float per_m, per_v;
  const float new_ms = block_scale(__reduce_max_sync(0xffffffffu, top_m), kLargest1, &per_m);
  const float new_vs = block_scale(__reduce_max_sync(0xffffffffu, top_v), kLargest2, &per_v);
  if (lane == 0) {
    a.m_scale[block] = new_ms;
    a.v_scale[block] = new_vs;
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t i = base + r * run_step + run;
    mc[r] = vc[r] = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t random = random_bits(key, i + e * step);
      mc[r] |= encode1(mv[r][e], per_m, random) << (8 * e);
      vc[r] |= encode2(vv[r][e], per_v, random) << (8 * e);
    }
    if (vec) {
      store4(p + i, pv[r]);
      *reinterpret_cast<uint32_t*>(m + i) = mc[r];
      *reinterpret_cast<uint32_t*>(v + i) = vc[r];
      if (copy) store4(copy + i, pv[r]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (r * run_step + run + e * 32 >= n) continue;
        p[i + e * 32] = from_float<P>(pv[r][e]);
        m[i + e * 32] = (uint8_t)(mc[r] >> (8 * e));
        v[i + e * 32] = (uint8_t)(vc[r] >> (8 * e));
        if (copy) copy[i + e * 32] = __float2bfloat16_rn(pv[r][e]);
      }
    }
  }
}

template <typename P, typename G, bool kMoments8, int N>
void launch(const Segment* segs, int n, const Hyper* hypers, int groups, const Hyper* on_device, cudaStream_t s) {
  constexpr int64_t tile = kMoments8 ? kTile8 : kTile32;
  Table<N> t;
  t.n = n;
  t.on_device = on_device;
  t.first_tile[0] = 0;
  for (int k = 0; k < n; ++k) {
    t.seg[k] = segs[k];
    t.first_tile[k + 1] = t.first_tile[k] + (uint32_t)((segs[k].n + tile - 1) / tile);
  }
  for (int k = 0; k < groups; ++k) t.hyper[k] = hypers[k];
  if constexpr (kMoments8)
    launch_overlapped(step8_kernel<P, G, N>, dim3(t.first_tile[n]), dim3(kThreads), s, t);
  else
    launch_overlapped(step32_kernel<P, G, N>, dim3(t.first_tile[n]), dim3(kThreads), s, t);
}

template <typename P, typename G, bool kMoments8>
int steps(const Segment* segs, int n, const Hyper* hypers, int groups, bool on_device, cudaStream_t s) {
  int launches = 0;
  std::vector<Segment> part;
  std::vector<Hyper> h;
  std::vector<int> of;  // hyperparameters' places in `h`, by group
  constexpr int64_t most = (int64_t)1 << 40;  // elements of a launch: its tiles are counted in 31 bits
  int64_t elements = 0;
  auto flush = [&] {
    if (part.empty()) return;
    if ((int)part.size() <= kFew)
      launch<P, G, kMoments8, kFew>(part.data(), (int)part.size(), h.data(), (int)h.size(), on_device ? hypers : nullptr, s);
    else
      launch<P, G, kMoments8, kMany>(part.data(), (int)part.size(), h.data(), (int)h.size(), on_device ? hypers : nullptr, s);
    ++launches;
    part.clear();
    h.clear();
    of.assign((size_t)groups, -1);
    elements = 0;
  };
  of.assign((size_t)groups, -1);
  for (int k = 0; k < n; ++k) {
    if (segs[k].n == 0) continue;
    const size_t group = (size_t)segs[k].group;
    if ((int)part.size() == kMany || (!on_device && of[group] < 0 && (int)h.size() == kGroups) || elements + segs[k].n > most) flush();
    if (!on_device && of[group] < 0) {
      of[group] = (int)h.size();
      h.push_back(hypers[group]);
    }
    part.push_back(segs[k]);
    if (!on_device) part.back().group = of[group];
    elements += segs[k].n;
  }
  flush();
  return launches;
}

template <typename P, typename G>
int steps(bool moments8, const Segment* segs, int n, const Hyper* hypers, int groups, bool on_device, cudaStream_t s) {
  return moments8 ? steps<P, G, true>(segs, n, hypers, groups, on_device, s) : steps<P, G, false>(segs, n, hypers, groups, on_device, s);
}

// ---- moments read back --------------------------------------------------------------------------
struct ReadTable {
  cuda::Read8 seg[kMany];
  uint32_t first_tile[kMany + 1];
  int n;
};
static_assert(sizeof(ReadTable) <= 32764, "launch parameters");
constexpr int kReadTile = kThreads * 4 * 4;
template <typename T>
__global__ void __launch_bounds__(kThreads) read8_kernel(const __grid_constant__ ReadTable table) {
  wait_for_predecessor();
  const int k = find_segment(table.first_tile, table.n, blockIdx.x);
  const cuda::Read8& a = table.seg[k];
  T *m = (T*)a.m_out, *v = (T*)a.v_out;
  const int64_t base = (int64_t)(blockIdx.x - table.first_tile[k]) * kReadTile;
  if (base + kReadTile <= a.n && fours(a.m) && fours(a.v) && fours(m) && fours(v)) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t i = base + (r * kThreads + threadIdx.x) * 4;
      const uint32_t mc = *reinterpret_cast<const uint32_t*>(a.m + i), vc = *reinterpret_cast<const uint32_t*>(a.v + i);
      const float ms = a.m_scale[i / kMoment8Block], vs = a.v_scale[i / kMoment8Block];
      float mv[4], vv[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        mv[e] = decode1((mc >> (8 * e)) & 0xffu, ms);
        vv[e] = decode2((vc >> (8 * e)) & 0xffu, vs);
      }
      store4(m + i, mv);
      store4(v + i, vv);
    }
  } else {
    const int64_t end = min(base + kReadTile, a.n);
    for (int64_t i = base + threadIdx.x; i < end; i += kThreads) {
      m[i] = from_float<T>(decode1(a.m[i], a.m_scale[i / kMoment8Block]));
      v[i] = from_float<T>(decode2(a.v[i], a.v_scale[i / kMoment8Block]));
    }
  }
}

// One thread for each group.
struct GroupTable {
  GroupValues g[kThreads / 2];
};
__global__ void hypers_kernel(const __grid_constant__ GroupTable table, int n, const int64_t* step, uint64_t seed, Hyper* out) {
  wait_for_predecessor();
  const int k = (int)threadIdx.x;
  if (k < n) out[k] = make_hyper(table.g[k], step[k], seed);
}

}  // namespace

namespace cuda {

int hypers(const GroupValues* g, int groups, const int64_t* step, uint64_t seed, Hyper* out, cudaStream_t s) {
  constexpr int most = kThreads / 2;
  int launches = 0;
  for (int at = 0; at < groups; at += most, ++launches) {
    GroupTable t;
    const int n = std::min(most, groups - at);
    for (int k = 0; k < n; ++k) t.g[k] = g[at + k];
    launch_overlapped(hypers_kernel, dim3(1), dim3(most), s, t, n, step + at, seed, out + at);
  }
  return launches;
}

int step(const Types& t, const Segment* segs, int n, const Hyper* hypers, int groups, bool on_device, cudaStream_t s) {
  BAGUA_CHECK(supported(t), Tensor, "AdamW: unsupported types " << dtype_name(t.p) << " and " << dtype_name(t.g));
  if (t.p == DType::F32) {
    if (t.g == DType::F32) return steps<float, float>(t.moments8, segs, n, hypers, groups, on_device, s);
    if (t.g == DType::F16) return steps<float, __half>(t.moments8, segs, n, hypers, groups, on_device, s);
    return steps<float, __nv_bfloat16>(t.moments8, segs, n, hypers, groups, on_device, s);
  }
  if (t.p == DType::F16) {
    if (t.g == DType::F32) return steps<__half, float>(t.moments8, segs, n, hypers, groups, on_device, s);
    return steps<__half, __half>(t.moments8, segs, n, hypers, groups, on_device, s);
  }
  if (t.g == DType::F32) return steps<__nv_bfloat16, float>(t.moments8, segs, n, hypers, groups, on_device, s);
  return steps<__nv_bfloat16, __nv_bfloat16>(t.moments8, segs, n, hypers, groups, on_device, s);
}

int read8(const Read8* segs, int n, DType out, cudaStream_t s) {
  int launches = 0;
  for (int at = 0; at < n;) {
    ReadTable t;
    t.n = 0;
    t.first_tile[0] = 0;
    for (; at < n && t.n < kMany; ++at) {
      if (segs[at].n == 0) continue;
      const int64_t tiles = t.first_tile[t.n] + (segs[at].n + kReadTile - 1) / kReadTile;
      if (tiles >= (int64_t)1 << 31) break;  // never the first: a tensor has fewer
      t.seg[t.n] = segs[at];
      t.first_tile[++t.n] = (uint32_t)tiles;
    }
    if (t.n == 0) continue;
    const dim3 grid(t.first_tile[t.n]);
    switch (out) {
      case DType::F32: launch_overlapped(read8_kernel<float>, grid, dim3(kThreads), s, t); break;
      case DType::F16: launch_overlapped(read8_kernel<__half>, grid, dim3(kThreads), s, t); break;
      case DType::BF16: launch_overlapped(read8_kernel<__nv_bfloat16>, grid, dim3(kThreads), s, t); break;
      default: throw BaguaError(ErrorKind::Tensor, std::string("moments are not read into ") + dtype_name(out));
    }
    ++launches;
  }
  return launches;
}

}  // namespace cuda
}  // namespace adamw
}  // namespace bagua
