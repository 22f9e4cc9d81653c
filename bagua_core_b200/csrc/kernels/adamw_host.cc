// AdamW on host memory, and what host and device share: hyperparameters, which types there are.
#include <algorithm>
#include <cmath>
#include <vector>

#include "adamw.h"
#include "adamw_math.h"
#include "host_float.h"

namespace bagua {
namespace adamw {

Hyper hyper(const GroupValues& g, int64_t step, uint64_t seed) { return make_hyper(g, step, seed); }

bool supported(const Types& t) {
  auto real = [](DType d) { return d == DType::F32 || d == DType::F16 || d == DType::BF16; };
  return real(t.p) && real(t.g) && (t.p == DType::F32 || t.g == t.p || t.g == DType::F32);
}

namespace host {

namespace {
// One block of elements with its scales.
template <typename P, typename G>
void step8(const Segment& a, const Hyper& h, int64_t block) {
  const int64_t lo = block * kMoment8Block, hi = lo + kMoment8Block < a.n ? lo + kMoment8Block : a.n;
  auto* p = (typename P::T*)a.p;
  auto* g = (const typename G::T*)a.g;
  auto *m = (uint8_t*)a.m, *v = (uint8_t*)a.v;
  float mv[kMoment8Block], vv[kMoment8Block];
  uint8_t mc[kMoment8Block], vc[kMoment8Block];
  uint32_t top_m = 0, top_v = 0;
  for (int64_t i = lo; i < hi; ++i) {
    float pv = P::ld(p + i), &mi = mv[i - lo], &vi = vv[i - lo];
    moments(h, G::ld(g + i), code1_bits(m[i]) * kUp * product(h.b1, a.m_scale[block]), code2_bits(v[i]) * kUp * product(h.b2, a.v_scale[block]),
            mi, vi);
    pv = parameter(h, pv, mi, vi);
    P::st(p + i, pv);
    if (a.copy) kernels::Elem<DType::BF16>::st((uint16_t*)a.copy + i, pv);
    const uint32_t mb = float_bits(mi) & 0x7fffffffu, vb = float_bits(vi) & 0x7fffffffu;
    top_m = mb > top_m ? mb : top_m;
    top_v = vb > top_v ? vb : top_v;
  }
  float per_m, per_v;
  float ms = block_scale(top_m, kLargest1, &per_m), vs = block_scale(top_v, kLargest2, &per_v);
  const uint32_t key = segment_key(h.random, a.index);
  bool near = false;
  for (int64_t i = lo; i < hi; ++i) {
    const uint32_t random = random_bits(key, i);
    const uint32_t s1 = sum1(scaled(std::fabs(mv[i - lo]), per_m, ms < kPlainScale), random);
    const uint32_t s2 = sum2(scaled(vv[i - lo], per_v, vs < kPlainScale), random);
    mc[i - lo] = (uint8_t)cut1(s1, mv[i - lo]);
    vc[i - lo] = (uint8_t)cut2(s2, vv[i - lo]);
    near |= above1(s1) < kNear1 || above2(s2) < kNear2;
  }
  if (near && ms < INFINITY && vs < INFINITY) {
    double per1, per2;
    float top1 = 0, top2 = 0;
    for (int64_t i = lo; i < hi; ++i) {
      top1 = std::max(top1, (float)std::fabs(first64(h, G::ld(g + i), m[i], a.m_scale[block])));
      top2 = std::max(top2, (float)second64(h, G::ld(g + i), v[i], a.v_scale[block]));
    }
    ms = scale64(top1, kLargest1, &per1);
    vs = scale64(top2, kLargest2, &per2);
    for (int64_t i = lo; i < hi; ++i) {
      const uint32_t random = random_bits(key, i);
      mc[i - lo] = (uint8_t)first_code64(first64(h, G::ld(g + i), m[i], a.m_scale[block]), per1, random);
      vc[i - lo] = (uint8_t)second_code64(second64(h, G::ld(g + i), v[i], a.v_scale[block]), per2, random);
    }
  }
  std::copy(mc, mc + (hi - lo), m + lo);
  std::copy(vc, vc + (hi - lo), v + lo);
  a.m_scale[block] = ms;
  a.v_scale[block] = vs;
}

template <typename P, typename G>
void step_segment(const Segment& a, const Hyper& h, bool moments8) {
  if (moments8) {
    for (int64_t b = 0; b < moment8_blocks(a.n); ++b) step8<P, G>(a, h, b);
    return;
  }
  auto* p = (typename P::T*)a.p;
  auto* g = (const typename G::T*)a.g;
  auto *m = (float*)a.m, *v = (float*)a.v;
  for (int64_t i = 0; i < a.n; ++i) {
    float pv = P::ld(p + i);
    update(h, pv, G::ld(g + i), m[i], v[i]);
    P::st(p + i, pv);
    if (a.copy) kernels::Elem<DType::BF16>::st((uint16_t*)a.copy + i, pv);
  }
}
}  // namespace

void step(const Types& t, const Segment* segs, int n, const Hyper* hypers) {
  BAGUA_CHECK(supported(t), Tensor, "AdamW: unsupported types " << dtype_name(t.p) << " and " << dtype_name(t.g));
  kernels::dispatch_float(t.p, [&](auto p) {
    kernels::dispatch_float(t.g, [&](auto g) {
      for (int k = 0; k < n; ++k) step_segment<decltype(p), decltype(g)>(segs[k], hypers[segs[k].group], t.moments8);
    });
  });
}

void read8(const cuda::Read8* segs, int n, DType out) {
  kernels::dispatch_float(out, [&](auto e) {
    using E = decltype(e);
    for (int k = 0; k < n; ++k) {
      const cuda::Read8& a = segs[k];
      for (int64_t i = 0; i < a.n; ++i) {
        E::st((typename E::T*)a.m_out + i, decode1(a.m[i], a.m_scale[i / kMoment8Block]));
        E::st((typename E::T*)a.v_out + i, decode2(a.v[i], a.v_scale[i / kMoment8Block]));
      }
    }
  });
}

}  // namespace host
}  // namespace adamw
}  // namespace bagua
