// Indices that a kernel meets outside their table: it goes on without them and leaves the last one in host memory, where the
// next call's host side finds it (check_indices() in encoder_ops.h).
#pragma once

#include <cstdint>

namespace bagua {
namespace encoder_ops {

enum { kTokenId = 0, kSpanTarget = 1, kTarget = 2, kIndexKinds = 3 };
struct IndexReport {
  long long value[kIndexKinds];  // the value is written first, then that there is one
  unsigned int seen[kIndexKinds];
};
// One per device, never given back: a captured graph keeps its address.
IndexReport* index_report();

#ifdef __CUDACC__
static __device__ __noinline__ void report_index(IndexReport* r, int kind, int64_t value) {
  *(volatile long long*)&r->value[kind] = value;
  __threadfence_system();
  *(volatile unsigned int*)&r->seen[kind] = 1u;
}
#endif

}  // namespace encoder_ops
}  // namespace bagua
