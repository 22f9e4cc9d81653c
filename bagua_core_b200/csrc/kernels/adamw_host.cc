// AdamW on host memory, and what host and device share: hyperparameters, which types there are.
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
  const float ms = a.m_scale[block] = block_scale(top_m, kLargest1, &per_m);
  const float vs = a.v_scale[block] = block_scale(top_v, kLargest2, &per_v);
  const uint32_t key = segment_key(h.random, a.index);
  for (int64_t i = lo; i < hi; ++i) {
    const uint32_t random = random_bits(key, i);
    m[i] = (uint8_t)encode1(scaled(std::fabs(mv[i - lo]), per_m, ms < kPlainScale), mv[i - lo], random);
    v[i] = (uint8_t)encode2(scaled(vv[i - lo], per_v, vs < kPlainScale), vv[i - lo], random);
  }
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
