// Rows of a table looked up by token and scaled, and the table's gradient, for any number of tokens (sm_100a).
//
//   out[t] = s W[id_t]            dW[v] = s * sum of dout[t] over the tokens t with id_t = v
//
// The gradient goes by sorted tokens: a stable sort of the ids brings the rows that belong to one row of the table together, and
// each row of the table is then written once, by one unit of work, in the tokens' order.  No atomics: the same call gives the same
// bits.  No counterpart in the reference, which has no model code.
#pragma once

#include <cuda_runtime_api.h>

#include <cstddef>
#include <cstdint>

#include "../common.h"

namespace bagua {
namespace embedding {

struct Ids {
  const void* data;
  bool wide;  // int64, or int32
  int64_t n;
};
constexpr int64_t kMaxTokens = (1ll << 31) - 4096, kMaxRows = (1ll << 31) - 64;

// out [n, H] of type `out_type`, contiguous, from rows of W [rows, H] that lie `row_stride` elements apart.  An id outside the table
// gives a row of NaN (check_indices() in encoder_ops.h tells).
void lookup(const Ids& ids, const void* table, DType table_type, int64_t rows, int64_t row_stride, int64_t H, float scale, void* out,
            DType out_type, cudaStream_t s);

// dtable [rows, H] from dout [n, H], both contiguous: all of its rows are written, or, with `accumulate` (dtable in F32), those that occur are
// added to.  Ids outside the table and `padding` (-1: none) have no part in it.  Scratch: backward_scratch_bytes() of it, 16-byte aligned.
// dtable starts on 16 bytes unless it is added to.  Returns the number of kernels launched.
size_t backward_scratch_bytes(int64_t n, int64_t H);
int backward(const Ids& ids, const void* dout, DType dout_type, int64_t rows, int64_t H, float scale, int64_t padding, void* dtable,
             DType table_type, bool accumulate, void* scratch, cudaStream_t s);

}  // namespace embedding
}  // namespace bagua
