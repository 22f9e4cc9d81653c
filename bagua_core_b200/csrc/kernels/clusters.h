// How many blocks of a kernel may form a cluster on a stream.
#pragma once

#include <cuda_runtime_api.h>

#include <cstddef>

namespace bagua {
namespace kernels {

// The largest power of two up to `wanted` for which the stream's context has room for a cluster of that many blocks of `threads` threads with
// `shared` bytes of dynamic shared memory each; 1 at least.  Not every context can run every cluster: the whole GPU runs 16 blocks, a green
// context of few SMs may not run 8.  Asked once per kernel, size and stream, by an id that no other stream of the process gets.  The kernel
// has its attributes (shared memory, clusters of more than 8 blocks) before.
int fitting_cluster(const void* kernel, int wanted, int threads, size_t shared, cudaStream_t s);

}  // namespace kernels
}  // namespace bagua
