// See adamw.h.  Streams over memory: with fp32 parameters, gradients and moments 28 bytes an element, 16 with moments in 8 bits.
// 131 M elements, twenty calls in a row, the best of nine such: 526 us with fp32 moments (6.97 TB/s, above the rate of a copy), 320 with
// 8 bits (6.6 TB/s; instructions are issued in three quarters of all cycles), 120 to read those into bf16 (6.6 TB/s).  Figures below
// are taken alike.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>
#include <vector>

#include "adamw.h"
#include "adamw_math.h"
#include "launch.cuh"
#include "typed_vec.cuh"

namespace bagua {
namespace adamw {

namespace {

using kernels::fma;
using kernels::from_float;
using kernels::halves;
using kernels::launch_overlapped;
using kernels::mul;
using kernels::Pair;
using kernels::pair;
using kernels::to_float;
using kernels::wait_for_predecessor;

constexpr int kThreads = 256;

// Segments are cut into tiles, a block each; the table of them travels with the launch.  A launch's parameters may take 32,764
// bytes; steps of fewer tensors take smaller tables, which reach the GPU sooner.
constexpr int kGroups = 8;
template <int N>
struct Table {
  Segment seg[N];
  Hyper hyper[kGroups];
  const Hyper* on_device;  // instead of `hyper`, where the step's number lies on the device
  uint32_t first_tile[N + 1];
  int n;
};
constexpr int kFew = 44, kSome = 128, kMany = 400;
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
  // tiles begin behind the lead, which the first one takes too
  const int lead = max((int)a.lead, 0);
  const int64_t tile = blockIdx.x - table.first_tile[k], base = lead + tile * kTile32;
  auto one = [&](int64_t i) {
    float pv = to_float(p[i]), mv = m[i], vv = v[i];
    update(h, pv, to_float(g[i]), mv, vv);
    p[i] = from_float<P>(pv);
    m[i] = mv;
    v[i] = vv;
    if (copy) copy[i] = __float2bfloat16_rn(pv);
  };
  if (a.lead >= 0 && base + kTile32 <= a.n) {
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
    for (int64_t i = base + threadIdx.x; i < end; i += kThreads) one(i);
  }
  if (tile == 0 && threadIdx.x < lead && threadIdx.x < a.n) one(threadIdx.x);
}

// ---- moments in 8 bits --------------------------------------------------------------------------
// A warp takes a block of elements that share their scales, eight to a lane: the largest value of a block is a reduction over the
// warp's registers, and each element is read and written once.  Lanes hold two runs of four, so that the 32 loads of a run are one
// piece of memory; elements of an address that no vector fits are taken one by one, lane by lane (131 M elements: 562 us instead of 320).
//
// With 16 bytes an element instead of 28, instructions count as much as bytes (at 89 an element 67 M elements took 234 us).
// So two elements are computed by one instruction where there is one; the square root and the reciprocal are the hardware's (within 2^-22 each: a
// parameter is off by that part of its update); the moments' betas go into the factor that decodes them, and both directions of coding take
// one factor.  A block with a scale beyond kPlainScale, or an eps so small that a subnormal square root counts next to
// it, goes the longer way.  2.3 % of the blocks hold codes that fp32 leaves open (256 elements, each with 2^-15 and 2^-14 of the random
// bits near a border).  Coding takes byte permutations where it can: with shifts and masks 131 M elements took 358 us where they took 316
// (bf16 parameters and gradients: 364, 306).  The weight decay's second factor made 320 of those, and 310.
// Blocks on an SM: so many leave 40 registers a thread and a few spilled ones.  131 M elements take 320 us, with five (48 registers)
// 341, seven (32) 347: the loads of waiting warps are worth more than the spills cost.  A warp that took two blocks in turn held
// more registers over the turn than it had (434 us where one took 362).
constexpr int kResident8 = 6;
constexpr int kTile8 = kThreads / 32 * kMoment8Block;
constexpr float kPlainEps = 1e-10f;
template <bool kPlain>
__device__ __forceinline__ float root_of(float x) {
  float y;
  if constexpr (kPlain)
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  else
    asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool kPlain>
__device__ __forceinline__ float reciprocal_of(float x) {
  float y;
  if constexpr (kPlain)
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  else
    asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Byte e of a word of codes as a code's bits (code1_bits, code2_bits).
__device__ __forceinline__ float word1_bits(uint32_t w, int e) { return __uint_as_float((uint32_t)((int)(w << (24 - 8 * e)) >> 4) & 0x87f00000u); }
__device__ __forceinline__ float word2_bits(uint32_t w, int e) {
  return __uint_as_float((e < 3 ? w << (19 - 8 * e) : w >> 5) & 0x07f80000u);
}
// The largest magnitude, or NaN.
__device__ __forceinline__ float largest(float a, float b, float c) {
  float y;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ Pair both(float x) { return pair(x, x); }
__device__ __forceinline__ uint32_t top_bytes(const uint32_t (&x)[4]) {
  return __byte_perm(__byte_perm(x[0], x[1], 0x0073), __byte_perm(x[2], x[3], 0x0073), 0x5410);
}
static_assert(kSlack == 16, "whole numbers of the random bits' steps, which the short way counts");

// A block's codes and scales in 64 bits, by the whole warp: 2.3 % of them.  (131 M elements take 320 us with two elements at a time, 323
// with one.)
template <typename G>
__device__ __forceinline__ void code_in_64_bits(const Segment& a, const Hyper& h, uint32_t key, int64_t block) {
  const int lane = (int)threadIdx.x & 31;
  const int64_t base = block * kMoment8Block;
  const int n = (int)min((int64_t)kMoment8Block, a.n - base);
  const G* g = (const G*)a.g + base;
  uint8_t *m = (uint8_t*)a.m + base, *v = (uint8_t*)a.v + base;
  const float ms = a.m_scale[block], vs = a.v_scale[block];
  float top1 = 0.f, top2 = 0.f;
#pragma unroll 2
  for (int i = lane; i < n; i += 32) {
    top1 = fmaxf(top1, (float)fabs(first64(h, to_float(g[i]), m[i], ms)));
    top2 = fmaxf(top2, (float)second64(h, to_float(g[i]), v[i], vs));
  }
  double per1, per2;
  const float new_ms = scale64(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top1))), kLargest1, &per1);
  const float new_vs = scale64(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top2))), kLargest2, &per2);
  if (lane == 0) {  // (all lanes have read the old ones)
    a.m_scale[block] = new_ms;
    a.v_scale[block] = new_vs;
  }
#pragma unroll 2
  for (int i = lane; i < n; i += 32) {
    const uint32_t random = random_bits(key, base + i);
    const float gi = to_float(g[i]);
    m[i] = (uint8_t)first_code64(first64(h, gi, m[i], ms), per1, random);
    v[i] = (uint8_t)second_code64(second64(h, gi, v[i], vs), per2, random);
  }
}

// Whether the block's codes and scales are settled, and written, too.
template <typename P, typename G, bool kVec>
__device__ __forceinline__ bool step8_block(const Segment& a, const Hyper& h, uint32_t key, int64_t block) {
  const int lane = (int)threadIdx.x & 31;
  const int64_t base = block * kMoment8Block;
  P* p = (P*)a.p + base;
  const G* g = (const G*)a.g + base;
  uint8_t *m = (uint8_t*)a.m + base, *v = (uint8_t*)a.v + base;
  auto* copy = (__nv_bfloat16*)a.copy;
  const float ms = a.m_scale[block], vs = a.v_scale[block];
  const int n = kVec ? kMoment8Block : (int)min((int64_t)kMoment8Block, a.n - base);
  auto at = [&](int r, int e) { return r * 128 + (kVec ? lane * 4 + e : e * 32 + lane); };  // element e of run r
  float pv[2][4], gv[2][4], mv[2][4], vv[2][4];
  uint32_t mc[2], vc[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if constexpr (kVec) {
      load4(p + at(r, 0), pv[r]);
      load4(g + at(r, 0), gv[r]);
      mc[r] = *reinterpret_cast<const uint32_t*>(m + at(r, 0));
      vc[r] = *reinterpret_cast<const uint32_t*>(v + at(r, 0));
    } else {
      mc[r] = vc[r] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = at(r, e);
        pv[r][e] = i < n ? to_float(p[i]) : 0.f;
        gv[r][e] = i < n ? to_float(g[i]) : 0.f;
        mc[r] |= (i < n ? (uint32_t)m[i] : 0u) << (8 * e);
        vc[r] |= (i < n ? (uint32_t)v[i] : 0u) << (8 * e);
      }
    }
  }
  float top_m = 0.f, top_v = 0.f;
  auto step = [&](auto plain) {
    constexpr bool kPlain = decltype(plain)::value;
    const Pair km = both(__fmul_rn(h.b1, ms) * (kPlain ? kUp : 1.f)), kv = both(__fmul_rn(h.b2, vs) * (kPlain ? kUp : 1.f));
    const Pair c1 = both(h.c1), c2 = both(h.c2), root = both(h.root), eps = both(h.eps), rate = both(-h.rate);
    const Pair keep = both(h.keep), rest = both(h.rest);
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        Pair mb = pair(word1_bits(mc[r], e), word1_bits(mc[r], e + 1)), vb = pair(word2_bits(vc[r], e), word2_bits(vc[r], e + 1));
        if constexpr (!kPlain) {
          mb = mul(mb, both(kUp));
          vb = mul(vb, both(kUp));
        }
        // (moments() and parameter() of two elements)
        const Pair gg = pair(gv[r][e], gv[r][e + 1]);
        const Pair mm = fma(c1, gg, mul(mb, km)), v2 = fma(mul(c2, gg), gg, mul(vb, kv));
        const float2 vf = halves(v2), mf = halves(mm);
        const float2 d = halves(fma(pair(root_of<kPlain>(vf.x), root_of<kPlain>(vf.y)), root, eps));
        const Pair per = pair(reciprocal_of<kPlain>(d.x), reciprocal_of<kPlain>(d.y));
        const Pair pp = pair(pv[r][e], pv[r][e + 1]);
        const float2 pf = halves(fma(pp, keep, fma(pp, rest, mul(mul(rate, mm), per))));
        pv[r][e] = pf.x;
        pv[r][e + 1] = pf.y;
        mv[r][e] = mf.x;
        mv[r][e + 1] = mf.y;
        vv[r][e] = vf.x;
        vv[r][e + 1] = vf.y;
        // (an element behind the end leaves the scales alone)
        if (kVec || at(r, e + 1) < n) {
          top_m = largest(top_m, mf.x, mf.y);
          top_v = largest(top_v, vf.x, vf.y);
        } else if (at(r, e) < n) {
          top_m = largest(top_m, mf.x, mf.x);
          top_v = largest(top_v, vf.x, vf.x);
        }
      }
  };
  if (ms < kPlainScale && vs < kPlainScale && h.eps >= kPlainEps)
    step(std::true_type{});
  else
    step(std::false_type{});
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if constexpr (kVec) {
      store4(p + at(r, 0), pv[r]);
      if (copy) store4(copy + base + at(r, 0), pv[r]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = at(r, e);
        if (i >= n) continue;
        p[i] = from_float<P>(pv[r][e]);
        if (copy) copy[base + i] = __float2bfloat16_rn(pv[r][e]);
      }
    }
  }
  float per_m, per_v;
  const float new_ms = block_scale(__reduce_max_sync(0xffffffffu, float_bits(top_m)), kLargest1, &per_m);
  const float new_vs = block_scale(__reduce_max_sync(0xffffffffu, float_bits(top_v)), kLargest2, &per_v);
  bool near = false;
  const uint32_t random = random_base(key, base) + (uint32_t)at(0, 0) * kStride;
  auto bits_of = [&](int r, int e) { return mix(random + (uint32_t)(at(r, e) - at(0, 0)) * kStride); };
  if (new_ms < kPlainScale && new_vs < kPlainScale) {
    // sum1(), sum2(), cut1() and cut2() with all bits moved up, so that codes are bytes 3 and the bits that are cut off begin with bytes
    // 2 and 1: bytes are put together by one instruction.  No sum overflows: y is at most three steps of fp32 above the largest code.
    const Pair fm = both(per_m * kDown), fv = both(per_v * kDown);
    uint32_t near1 = ~0u, near2 = ~0u;  // of two codes each: above1() and above2() in units of the random bits
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      uint32_t t1[4], t2[4];
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const float2 y1 = halves(mul(pair(mv[r][e], mv[r][e + 1]), fm)), y2 = halves(mul(pair(vv[r][e], vv[r][e + 1]), fv));
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const uint32_t bits = bits_of(r, e + o);
          t1[e + o] = (float_bits(o ? y1.y : y1.x) << 4) + __byte_perm(bits, 0x80u, 0x5104);
          t2[e + o] = (float_bits(o ? y2.y : y2.x) << 5) + __byte_perm(bits, 0x80u, 0x5324);
          if (!kVec && at(r, e + o) >= n) t1[e + o] = t2[e + o] = 0x800000u;
          t1[e + o] |= float_bits(mv[r][e + o]) & 0x80000000u;
        }
        near1 = __viaddmin_u16x2(__byte_perm(t1[e], t1[e + 1], 0x6521), kSlack / 16 * 0x10001u, near1);
        near2 = __viaddmin_u16x2(__byte_perm(t2[e], t2[e + 1], 0x6521), kSlack / 8 * 0x10001u, near2);
      }
      mc[r] = top_bytes(t1);
      vc[r] = top_bytes(t2);
      if ((vc[r] - 0x01010101u) & ~vc[r] & 0x80808080u)  // seldom: a code 0, which stands for nothing but 0
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (vv[r][e] > 0 && !(vc[r] >> (8 * e) & 0xffu)) vc[r] |= 1u << (8 * e);
    }
    near = (near1 & 0xffffu) < kSlack / 8 || near1 >> 16 < kSlack / 8 || (near2 & 0xffffu) < kSlack / 4 || near2 >> 16 < kSlack / 4;
  } else {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      uint32_t c1[4], c2[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // each by its own scale
        const uint32_t bits = bits_of(r, e);
        const uint32_t s1 = sum1(scaled(fabsf(mv[r][e]), per_m, new_ms < kPlainScale), bits);
        const uint32_t s2 = sum2(scaled(vv[r][e], per_v, new_vs < kPlainScale), bits);
        c1[e] = cut1(s1, mv[r][e]) << 24;
        c2[e] = cut2(s2, vv[r][e]) << 24;
        near |= (kVec || at(r, e) < n) && (above1(s1) < kNear1 || above2(s2) < kNear2);
      }
      mc[r] = top_bytes(c1);
      vc[r] = top_bytes(c2);
    }
  }
  if (__any_sync(0xffffffffu, near) && new_ms < INFINITY && new_vs < INFINITY) {
    return false;
  }
  if (lane == 0) {
    a.m_scale[block] = new_ms;
    a.v_scale[block] = new_vs;
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if constexpr (kVec) {
      *reinterpret_cast<uint32_t*>(m + at(r, 0)) = mc[r];
      *reinterpret_cast<uint32_t*>(v + at(r, 0)) = vc[r];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = at(r, e);
        if (i >= n) continue;
        m[i] = (uint8_t)(mc[r] >> (8 * e));
        v[i] = (uint8_t)(vc[r] >> (8 * e));
      }
    }
  }
  return true;
}
template <typename P, typename G, int N>
__global__ void __launch_bounds__(kThreads, kResident8) step8_kernel(const __grid_constant__ Table<N> table) {
  wait_for_predecessor();
  const int k = find_segment(table.first_tile, table.n, blockIdx.x);
  const Segment& a = table.seg[k];
  const Hyper h = table.on_device ? table.on_device[a.group] : table.hyper[a.group];
  const uint32_t key = segment_key(h.random, a.index);
  const bool vec = fours((P*)a.p) && fours((const G*)a.g) && fours((uint8_t*)a.m) && fours((uint8_t*)a.v) && fours((__nv_bfloat16*)a.copy);
  const int64_t block = (int64_t)(blockIdx.x - table.first_tile[k]) * (kTile8 / kMoment8Block) + (threadIdx.x >> 5);
  if (block * kMoment8Block >= a.n) return;
  const bool settled = vec && (block + 1) * kMoment8Block <= a.n ? step8_block<P, G, true>(a, h, key, block) : step8_block<P, G, false>(a, h, key, block);
  if (!settled) code_in_64_bits<G>(a, table.on_device ? table.on_device[a.group] : table.hyper[a.group], key, block);
}

// Buffers that start anywhere, slices of flat ones, for instance: how many elements further all of them hold four as one piece.  (60 M elements
// one by one take 390 us, four at a time 263.)
template <typename P, typename G>
int lead_of(const Segment& a) {
  for (int k = 0; k < 4; ++k) {
    auto fits = [k](const void* p, size_t element) { return ((uintptr_t)p + k * element) % (4 * element) == 0; };
    if (fits(a.p, sizeof(P)) && fits(a.g, sizeof(G)) && fits(a.m, 4) && fits(a.v, 4) && (!a.copy || fits(a.copy, 2))) return k;
  }
  return -1;
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
    int64_t n_tiled = segs[k].n;
    if constexpr (!kMoments8) {
      const int lead = lead_of<P, G>(segs[k]);
      t.seg[k].lead = (int16_t)lead;
      if (lead > 0) n_tiled = std::max<int64_t>(1, n_tiled - lead);  // (a tile takes the lead where there is no more)
    }
    t.first_tile[k + 1] = t.first_tile[k] + (uint32_t)((n_tiled + tile - 1) / tile);
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
    else if ((int)part.size() <= kSome)
      launch<P, G, kMoments8, kSome>(part.data(), (int)part.size(), h.data(), (int)h.size(), on_device ? hypers : nullptr, s);
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
    if (!on_device) part.back().group = (int16_t)of[group];
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
template <int N>
struct ReadTable {
  cuda::Read8 seg[N];
  uint32_t first_tile[N + 1];
  int n;
};
static_assert(sizeof(ReadTable<kMany>) <= 32764, "launch parameters");
// (Vectors up to the last whole one: 79 tensors of 9.9 M elements that end anywhere take 11.5 us; tiles that end early element by
// element 22.6.)
constexpr int kReadVecs = 2, kReadTile = kThreads * 8 * kReadVecs;
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) read8_kernel(const __grid_constant__ ReadTable<N> table) {
  wait_for_predecessor();
  const int k = find_segment(table.first_tile, table.n, blockIdx.x);
  const cuda::Read8& a = table.seg[k];
  T *m = (T*)a.m_out, *v = (T*)a.v_out;
  const int64_t base = (int64_t)(blockIdx.x - table.first_tile[k]) * kReadTile;
  auto one = [&](int64_t i) {
    m[i] = from_float<T>(decode1(a.m[i], a.m_scale[i / kMoment8Block]));
    v[i] = from_float<T>(decode2(a.v[i], a.v_scale[i / kMoment8Block]));
  };
  if ((((uintptr_t)a.m | (uintptr_t)a.v) % 8 | ((uintptr_t)m | (uintptr_t)v) % 16) == 0) {
    uint2 mc[kReadVecs], vc[kReadVecs];
    float ms[kReadVecs], vs[kReadVecs];
#pragma unroll
    for (int r = 0; r < kReadVecs; ++r) {
      const int64_t i = base + (r * kThreads + threadIdx.x) * 8;
      if (i + 8 > a.n) continue;
      mc[r] = *reinterpret_cast<const uint2*>(a.m + i);
      vc[r] = *reinterpret_cast<const uint2*>(a.v + i);
      ms[r] = a.m_scale[i / kMoment8Block];
      vs[r] = a.v_scale[i / kMoment8Block];
    }
#pragma unroll
    for (int r = 0; r < kReadVecs; ++r) {
      const int64_t i = base + (r * kThreads + threadIdx.x) * 8;
      if (i + 8 > a.n) {  // the last elements, those of one vector that is not whole
        for (int64_t k = i; k < a.n; ++k) one(k);
        continue;
      }
      float mv[8], vv[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        mv[e] = word1_bits(e < 4 ? mc[r].x : mc[r].y, e % 4) * kUp * ms[r];
        vv[e] = word2_bits(e < 4 ? vc[r].x : vc[r].y, e % 4) * kUp * vs[r];
      }
      kernels::store8(m + i, kernels::narrow8<T>(mv));
      kernels::store8(v + i, kernels::narrow8<T>(vv));
    }
  } else {
    const int64_t end = min(base + kReadTile, a.n);
    for (int64_t i = base + threadIdx.x; i < end; i += kThreads) one(i);
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
  auto read = [&](auto size, int from, int count) {
    ReadTable<decltype(size)::value> t;
    t.n = 0;
    t.first_tile[0] = 0;
    for (int k = from; k < from + count; ++k) {
      if (segs[k].n == 0) continue;
      t.seg[t.n] = segs[k];
      t.first_tile[t.n + 1] = t.first_tile[t.n] + (uint32_t)((segs[k].n + kReadTile - 1) / kReadTile);
      ++t.n;
    }
    if (t.n == 0) return;
    const dim3 grid(t.first_tile[t.n]);
    constexpr int N = decltype(size)::value;
    switch (out) {
      case DType::F32: launch_overlapped(read8_kernel<float, N>, grid, dim3(kThreads), s, t); break;
      case DType::F16: launch_overlapped(read8_kernel<__half, N>, grid, dim3(kThreads), s, t); break;
      case DType::BF16: launch_overlapped(read8_kernel<__nv_bfloat16, N>, grid, dim3(kThreads), s, t); break;
      default: throw BaguaError(ErrorKind::Tensor, std::string("moments are not read into ") + dtype_name(out));
    }
    ++launches;
  };
  constexpr int64_t most = (int64_t)1 << 40;  // elements of a launch: its tiles are counted in 31 bits
  for (int at = 0; at < n;) {
    int count = 0;
    int64_t elements = 0;
    for (; at + count < n && count < kMany && (count == 0 || elements + segs[at + count].n <= most); ++count) elements += segs[at + count].n;
    if (count <= kFew)
      read(std::integral_constant<int, kFew>{}, at, count);
    else if (count <= kSome)
      read(std::integral_constant<int, kSome>{}, at, count);
    else
      read(std::integral_constant<int, kMany>{}, at, count);
    at += count;
  }
  return launches;
}

}  // namespace cuda
}  // namespace adamw
}  // namespace bagua
