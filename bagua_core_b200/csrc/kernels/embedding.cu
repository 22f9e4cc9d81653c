// See embedding.h.
//
// Bound by memory where tables and batches are large: 65536 rows of 2048 looked up in bf16 in 66 us (6.1 TB/s of output and rows, of which the
// L2 cache holds many), the gradient of 131072 x 2048 in 158 us (its floor is 123: rows that occur are written twice, and reads of
// rows all over memory reach three quarters of a stream's rate); the gradient of 30522 x 1024 from 12288 tokens in 39 us (floor 23).  Small
// ones are bound by the launches and the latency of sorting, 12 us for 256 tokens.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "clusters.h"
#include "embedding.h"
#include "index_report.cuh"
#include "launch.cuh"
#include "typed_vec.cuh"

namespace bagua {
namespace embedding {

namespace {

namespace cg = cooperative_groups;
using namespace kernels;
using encoder_ops::IndexReport;
using encoder_ops::report_index;

constexpr int kThreads = 256;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---- lookup -------------------------------------------------------------------------------------
// A thread takes eight columns of a row, or of four rows, whose loads wait for their ids together, where enough threads are left (65536
// rows of 2048 in bf16: 66 us, 84 with one row each).  Rows that do not lie on 16 bytes go the other way: a warp takes a row, its
// lanes pairs of columns or single ones, eight of them under way together (40001 rows of 333 in fp16: 13 us, 73 with a thread for
// each element).
constexpr int kRowsAhead = 4;
constexpr int64_t kManyElements = 148ll * 2048 * 8 * kRowsAhead;
template <typename Id, typename W, typename O, int kRows>
__global__ void __launch_bounds__(kThreads)
    lookup_kernel(const Id* __restrict__ ids, const W* __restrict__ table, int64_t rows, int64_t row_stride, O* __restrict__ out, int64_t n,
                  int64_t H, int shift, float scale, IndexReport* report) {
  wait_for_predecessor();
  const int columns = 1 << shift;  // threads of a row
  const int per = kThreads >> shift;
  const int64_t t0 = (int64_t)blockIdx.x * per * kRows + (threadIdx.x >> shift);
  const int64_t c = ((int64_t)blockIdx.y * columns + (threadIdx.x & (columns - 1))) * 8;
  if (c >= H) return;
  int64_t id[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) id[k] = t0 + k * per < n ? (int64_t)ids[t0 + k * per] : 0;
  Raw8<W> raw[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k)
    if (t0 + k * per < n && id[k] >= 0 && id[k] < rows) raw[k] = load8(table + id[k] * row_stride + c);
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const int64_t t = t0 + k * per;
    if (t >= n) break;
    const bool known = id[k] >= 0 && id[k] < rows;
    if (!known && c == 0) report_index(report, encoder_ops::kTokenId, id[k]);
    float f[8];
    widen8(raw[k], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = known ? f[e] * scale : nanf("");
    store8(out + t * H + c, narrow8<O>(f));
  }
}
template <typename T, int N>
struct alignas(N * sizeof(T)) Few {
  T x[N];
};
template <typename Id, typename W, typename O, int kFew>
__global__ void __launch_bounds__(kThreads)
    lookup_any_kernel(const Id* __restrict__ ids, const W* __restrict__ table, int64_t rows, int64_t row_stride, O* __restrict__ out, int64_t n,
                      int64_t H, float scale, IndexReport* report) {
  wait_for_predecessor();
  const int lane = (int)threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (t >= n) return;
  const int64_t id = (int64_t)ids[t];
  const bool known = id >= 0 && id < rows;
  if (!known && lane == 0) report_index(report, encoder_ops::kTokenId, id);
  const W* row = table + (known ? id : 0) * row_stride;
  constexpr int kAhead = 8;
  for (int64_t c0 = lane * kFew; c0 < H; c0 += kAhead * 32 * kFew) {
    Few<W, kFew> w[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t c = c0 + k * 32 * kFew;
      if (known && c < H) w[k] = *reinterpret_cast<const Few<W, kFew>*>(row + c);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t c = c0 + k * 32 * kFew;
      if (c >= H) break;
      Few<O, kFew> o;
#pragma unroll
      for (int e = 0; e < kFew; ++e) o.x[e] = from_float<O>(known ? to_float(w[k].x[e]) * scale : nanf(""));
      *reinterpret_cast<Few<O, kFew>*>(out + t * H + c) = o;
    }
  }
}

// ---- clearing -----------------------------------------------------------------------------------
// The gradient's rows that no token names are zero.  Sorting keeps few blocks busy: its kernel lets this one start at once, which clears the
// whole gradient meanwhile, and the rows that do occur are written again later.  Nothing is read here, and what was queued before the
// sort has finished when it lets go, so that no block waits but the first, at its end: by that this kernel ends behind the sort, and what
// follows it may rely on both.  (Cleared by the launch that writes the sums instead, and of rows that do not occur alone, 12288 tokens of
// 30522 x 1024 took 67 us, now 39.)
constexpr int kClearVecs = 4;
constexpr int64_t kClearBytes = (int64_t)kThreads * kClearVecs * 16;  // of a block
__global__ void __launch_bounds__(kThreads) clear_kernel(char* __restrict__ at, int64_t bytes) {  // `at` lies on 16 bytes
  const int64_t base = (int64_t)blockIdx.x * kClearBytes;
#pragma unroll
  for (int k = 0; k < kClearVecs; ++k) {
    const int64_t i = base + ((int64_t)k * kThreads + threadIdx.x) * 16;
    if (i + 16 <= bytes) *reinterpret_cast<uint4*>(at + i) = make_uint4(0, 0, 0, 0);
  }
  if (blockIdx.x > 0) return;
  const int64_t tail = bytes / 16 * 16;
  if (threadIdx.x < bytes - tail) at[tail + threadIdx.x] = 0;
  wait_for_predecessor();
}
void clear(void* at, int64_t bytes, cudaStream_t s) {
  launch_overlapped(clear_kernel, dim3((unsigned)((bytes + kClearBytes - 1) / kClearBytes)), dim3(kThreads), s, (char*)at, bytes);
}

// ---- sorting ------------------------------------------------------------------------------------
// A token's key is its row, or `rows` for those without a part in the gradient, which so come last.  Stable, least significant digit
// first: a pass puts the tokens in the order of 8 bits and leaves equal ones as they were.
constexpr int kDigits = 256;
struct Keys {
  int64_t rows, padding;
  template <typename Id>
  __device__ __forceinline__ uint32_t operator()(Id id) const {
    const int64_t v = (int64_t)id;
    return (uint32_t)(v >= 0 && v < rows && v != padding ? v : rows);
  }
};

// Number of a lane's key among the equal digits of its warp's keys so far, which `seen` counts.  All lanes of the warp come here.
// (Equal digits are found bit by bit: the instruction that matches values takes a turn for each different one, 15,700 cycles for
// 8192 keys in 512 digits where this takes 9,600.)
template <int kBits>
__device__ __forceinline__ uint32_t rank_in_warp(uint32_t* seen, uint32_t digit, bool valid) {
  uint32_t peers = __ballot_sync(0xffffffffu, valid);
#pragma unroll
  for (int b = 0; b < kBits; ++b) {
    const uint32_t set = __ballot_sync(0xffffffffu, digit >> b & 1u);
    peers &= digit >> b & 1u ? set : ~set;
  }
  const int lane = (int)threadIdx.x & 31;
  const uint32_t before = valid ? seen[digit] : 0u;
  __syncwarp();
  if (valid && (peers >> lane) == 1u) seen[digit] = before + __popc(peers);  // the last of them
  __syncwarp();
  return before + __popc(peers & ((1u << lane) - 1u));
}

// Sorting in blocks that hand tiles to each other through memory.
constexpr int kRounds = 8, kTile = kThreads * kRounds, kWarps = kThreads / 32;
// counts[digit][tile]: how many of a tile's keys have a digit.
template <typename Id>
__global__ void __launch_bounds__(kThreads)
    histogram_kernel(const Id* __restrict__ ids, const uint32_t* __restrict__ keys, Keys key, int64_t n, int shift, uint32_t* __restrict__ counts,
                     int tiles) {
  __shared__ uint32_t s_count[kDigits];
  wait_for_predecessor();
  s_count[threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kTile;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = base + r * kThreads + threadIdx.x;
    if (i >= n) break;
    const uint32_t k = keys ? keys[i] : key(ids[i]);
    atomicAdd(&s_count[(k >> shift) & (kDigits - 1)], 1u);
  }
  __syncthreads();
  counts[(int64_t)threadIdx.x * tiles + blockIdx.x] = s_count[threadIdx.x];
}
constexpr int kScanThreads = 1024, kScanEach = 16;
// Exclusive sums of n counts, a multiple of 4 of them on a 16-byte border, in one block.  Lets its successor start at once, and sets
// `zero` to 0.
__global__ void __launch_bounds__(kScanThreads) scan_kernel(uint32_t* __restrict__ counts, int64_t n, uint32_t* __restrict__ zero) {
  __shared__ uint32_t s_warp[32];
  __shared__ uint32_t s_total;
  wait_for_predecessor();
  let_successor_start();
  if (threadIdx.x == 0) *zero = 0;
  const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
  uint32_t carry = 0;
  for (int64_t base = 0; base < n; base += kScanThreads * kScanEach) {
    uint4* at = reinterpret_cast<uint4*>(counts + base + (int64_t)threadIdx.x * kScanEach);
    const int64_t left = (n - base) / 4 - (int64_t)threadIdx.x * (kScanEach / 4);  // vectors
    uint32_t v[kScanEach], sum = 0;
#pragma unroll
    for (int k = 0; k < kScanEach / 4; ++k) {
      const uint4 x = k < left ? at[k] : make_uint4(0, 0, 0, 0);
      v[4 * k] = x.x;
      v[4 * k + 1] = x.y;
      v[4 * k + 2] = x.z;
      v[4 * k + 3] = x.w;
    }
#pragma unroll
    for (int k = 0; k < kScanEach; ++k) sum += v[k];
    uint32_t up = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += x;
    }
    if (lane == 31) s_warp[warp] = up;
    __syncthreads();
    if (warp == 0) {
      uint32_t w = s_warp[lane], wu = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, wu, o);
        if (lane >= o) wu += x;
      }
      s_warp[lane] = wu - w;
      if (lane == 31) s_total = wu;
    }
    __syncthreads();
    uint32_t before = carry + s_warp[warp] + up - sum;
#pragma unroll
    for (int k = 0; k < kScanEach; ++k) {
      const uint32_t c = v[k];
      v[k] = before;
      before += c;
    }
#pragma unroll
    for (int k = 0; k < kScanEach / 4; ++k)
      if (k < left) at[k] = make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    carry += s_total;
    __syncthreads();
  }
}
template <typename Id>
__global__ void __launch_bounds__(kThreads)
    scatter_kernel(const Id* __restrict__ ids, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ places, Keys key, int64_t n,
                   int shift, const uint32_t* __restrict__ offsets, int tiles, uint32_t* __restrict__ keys_out,
                   uint32_t* __restrict__ places_out) {
  __shared__ uint32_t s_seen[kWarps][kDigits];
  wait_for_predecessor();
  const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
  for (int k = (int)threadIdx.x; k < kWarps * kDigits; k += kThreads) s_seen[0][k] = 0;
  __syncthreads();
  // a warp's keys are neighbours
  const int64_t base = (int64_t)blockIdx.x * kTile + warp * (kTile / kWarps) + lane;
  uint32_t k[kRounds], p[kRounds], rank[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = base + r * 32;
    const bool valid = i < n;
    k[r] = !valid ? 0u : keys ? keys[i] : key(ids[i]);
    p[r] = !valid ? 0u : places ? places[i] : (uint32_t)i;
    rank[r] = rank_in_warp<8>(s_seen[warp], (k[r] >> shift) & (kDigits - 1), valid);
  }
  __syncthreads();
  {
    uint32_t at = offsets[(int64_t)threadIdx.x * tiles + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const uint32_t c = s_seen[w][threadIdx.x];
      s_seen[w][threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if (base + r * 32 >= n) break;
    const uint32_t to = s_seen[warp][(k[r] >> shift) & (kDigits - 1)] + rank[r];
    keys_out[to] = k[r];
    places_out[to] = p[r];
  }
}

// Sorting in one launch, which lets its successor start at once: the blocks of a cluster hold all tokens in their shared memory and hand
// them to each other there.  A pass counts its digits by warp, makes the counts into places by sums over warps, blocks and digits, puts
// the block's tokens in their order, and copies them, now neighbours for the most part, to where they belong.  (Stored one by one from
// where they were, 8192 tokens a block took 20,600 cycles to get there, 3,400 so.)  12288 tokens: 13 us, 65536: 32, hidden behind the
// clearing of a large gradient; through memory 200,000 take 52.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortRounds = 8;
// Blocks of a cluster at most: 8, or 16 where so many tokens are left for each that it pays (us of 65536 tokens' whole gradient, 1000 x 64:
// 46.7, 53.5 with 8; but 13.3 for 256 tokens, and 16.0 by a kernel that may form clusters of 16).  More tokens than they hold go through memory.
constexpr int kSortBlocks = 8, kSortBlocksMany = 16;
constexpr int64_t kSortMany = 32768, kSortTokens = (int64_t)kSortBlocksMany * kSortThreads * kSortRounds;
// A block of it clears so many bytes itself, in about a microsecond; a launch of its own for that would cost two.
constexpr int64_t kSmallClear = 128 << 10;
constexpr int kSortBits = 9, kSortDigits = 1 << kSortBits;  // of a pass at most: two for up to 2^18 - 1 rows
struct SortShared {
  uint32_t seen[kSortWarps][kSortDigits];
  uint32_t count[kSortDigits], offset[kSortDigits], warp[2][kSortDigits / 32];
  // of a digit: where the block's tokens begin in the block's order, and how much further they go in everybody's
  uint32_t own[kSortDigits];
};
size_t sort_shared_bytes(int rounds) { return sizeof(SortShared) + (size_t)rounds * kSortThreads * 2 * sizeof(uint2); }
template <typename Id, int kMaxBlocks>
__global__ void __launch_bounds__(kSortThreads)
    sort_kernel(const Id* __restrict__ ids, Keys key, int n, int bits, int digit_bits, int rounds, uint32_t* __restrict__ keys_out,
                uint32_t* __restrict__ places_out, uint32_t* __restrict__ zero, uint4* __restrict__ clear_at, int64_t clear_bytes) {
  extern __shared__ __align__(16) char s_memory[];
  SortShared& s = *reinterpret_cast<SortShared*>(s_memory);
  const int room = rounds * kSortThreads;  // tokens of a block
  uint2* s_tokens = reinterpret_cast<uint2*>(s_memory + sizeof(SortShared));  // keys and places, of this pass and of the next
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), blocks = (int)cluster.num_blocks();
  const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = warp * rounds * 32 + lane;  // a warp's tokens are neighbours
  const int held = min(room, n - rank * room);  // may be negative
  wait_for_predecessor();
  let_successor_start();
  if (rank == 0 && tid == 0) *zero = 0;
  if (clear_at) {
    for (int64_t i = rank * kSortThreads + tid; i < clear_bytes / 16; i += blocks * kSortThreads) clear_at[i] = make_uint4(0, 0, 0, 0);
    if (rank == 0 && tid < clear_bytes % 16) reinterpret_cast<char*>(clear_at)[clear_bytes / 16 * 16 + tid] = 0;
  }
  const int digits = 1 << digit_bits;
  for (int shift = 0, from = 0; shift < bits; shift += digit_bits, from ^= 1) {
    uint2* in = s_tokens + from * room;
    for (int k = tid; k < kSortWarps * digits; k += kSortThreads) s.seen[k >> digit_bits][k & (digits - 1)] = 0;
    __syncthreads();
    uint2 token[kSortRounds];
    uint32_t at[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      if (r >= rounds) break;
      const int slot = first + r * 32, i = rank * room + slot;
      token[r] = slot >= held ? make_uint2(0, 0) : shift == 0 ? make_uint2(key(ids[i]), (uint32_t)i) : in[slot];
    }
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      if (r >= rounds) break;
      at[r] = rank_in_warp<kSortBits>(s.seen[warp], (token[r].x >> shift) & (digits - 1), first + r * 32 < held);
    }
    __syncthreads();
    if (tid < digits) {
      uint32_t sum = 0;
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = s.seen[w][tid];
        s.seen[w][tid] = sum;
        sum += c;
      }
      s.count[tid] = sum;
    }
    cluster.sync();
    uint32_t before = 0, all = 0, mine = 0, up = 0, own_up = 0;
    if (tid < digits) {
#pragma unroll
      for (int b = 0; b < kMaxBlocks; ++b) {
        const uint32_t c = b < blocks ? cluster.map_shared_rank(s.count, b)[tid] : 0u;
        before += b < rank ? c : 0u;
        mine = b == rank ? c : mine;
        all += c;
      }
      up = all;
      own_up = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, up, o), y = __shfl_up_sync(0xffffffffu, own_up, o);
        if (lane >= o) {
          up += x;
          own_up += y;
        }
      }
      if (lane == 31) {
        s.warp[0][warp] = up;
        s.warp[1][warp] = own_up;
      }
    }
    __syncthreads();
    if (tid < digits) {
      uint32_t sum = before + up - all, own = own_up - mine;
#pragma unroll
      for (int w = 0; w < kSortDigits / 32; ++w) {
        sum += w < warp ? s.warp[0][w] : 0u;
        own += w < warp ? s.warp[1][w] : 0u;
      }
      s.own[tid] = own;
      s.offset[tid] = sum - own;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      if (r >= rounds || first + r * 32 >= held) break;
      const uint32_t digit = (token[r].x >> shift) & (digits - 1);
      in[s.own[digit] + s.seen[warp][digit] + at[r]] = token[r];
    }
    __syncthreads();
    const bool last = shift + digit_bits >= bits;
    for (int slot = tid; slot < held; slot += kSortThreads) {
      const uint2 t = in[slot];
      const uint32_t to = (uint32_t)slot + s.offset[(t.x >> shift) & (digits - 1)];
      if (last) {
        keys_out[to] = t.x;
        places_out[to] = t.y;
      } else {
        const uint32_t block = to / (uint32_t)room;
        cluster.map_shared_rank(s_tokens, block)[(from ^ 1) * room + to - block * room] = t;
      }
    }
    cluster.sync();
  }
}

// ---- sums ---------------------------------------------------------------------------------------
// The sorted tokens are cut into chunks of equal length.  A group of lanes takes a chunk and 8 columns a lane, adds up the rows of
// equal tokens in their order and writes each sum to its row of the table.  Sums over a border between chunks go to scratch, two rows
// a chunk (of the run that comes in, of the run that goes out), and join_kernel adds those up in the chunks' order.
struct SumArgs {
  const uint32_t *keys, *places;
  uint32_t *runs, *run_count;  // first chunks of the runs that go over a border
  float* partial;
  int64_t n, rows, H, chunks;
  int length;   // of a chunk: 8, 16 or a multiple of 32
  int slices;   // of a row's columns
  float scale;
  bool accumulate;  // sums are added to what the rows hold
};

// The column of element k of a lane that stands at `lane` in a slice of `width` lanes.
template <bool kVec>
__device__ __forceinline__ int64_t column(int slice, int lane, int width, int k) {
  return (int64_t)slice * width * 8 + (kVec ? lane * 8 + k : k * width + lane);
}
template <typename T, bool kVec>
__device__ __forceinline__ Raw8<T> load_row(const T* row, int slice, int lane, int width, int64_t H) {
  if constexpr (kVec) {
    const int64_t c = column<true>(slice, lane, width, 0);
    if (c < H) return load8(row + c);
    return Raw8<T>{};
  } else {
    Raw8<T> r{};
    T* x = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t c = column<false>(slice, lane, width, k);
      if (c < H) x[k] = row[c];
    }
    return r;
  }
}
template <typename T, bool kVec>
__device__ __forceinline__ void store_row(T* row, const float (&f)[8], int slice, int lane, int width, int64_t H) {
  if constexpr (kVec) {
    const int64_t c = column<true>(slice, lane, width, 0);
    if (c < H) store8(row + c, narrow8<T>(f));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t c = column<false>(slice, lane, width, k);
      if (c < H) row[c] = from_float<T>(f[k]);
    }
  }
}
template <typename T, bool kVec>
__device__ __forceinline__ void finish_row(T* row, float (&f)[8], float scale, bool accumulate, int slice, int lane, int width, int64_t H) {
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] *= scale;
  if (accumulate) {
    float old[8];
    widen8(load_row<T, kVec>(row, slice, lane, width, H), old);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] += old[k];
  }
  store_row<T, kVec>(row, f, slice, lane, width, H);
}

constexpr int kSumBlocks = 3;  // resident on an SM
template <typename D, typename W, bool kVec, int kWidth>
__global__ void __launch_bounds__(kThreads, kSumBlocks)
    sum_kernel(const __grid_constant__ SumArgs a, const D* __restrict__ dout, W* __restrict__ dtable) {
  wait_for_predecessor();
  const int warp_lane = (int)threadIdx.x & 31;
  const int64_t unit = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / kWidth;
  const int lane = warp_lane % kWidth;
  const int64_t chunk = unit / a.slices;
  const int slice = (int)(unit % a.slices);
  const bool on = chunk < a.chunks;
  const int64_t lo = on ? chunk * a.length : 0, hi = on ? min(lo + a.length, a.n) : 0;
  const uint32_t none = (uint32_t)a.rows;
  // what lies on the two borders
  const uint32_t before = lo > 0 ? a.keys[lo - 1] : none, behind = hi < a.n ? a.keys[hi] : none;
  float acc[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] = 0.f;
  uint32_t run = none;  // whose sum `acc` is
  bool first = true;    // it is the chunk's first run
  auto flush = [&](bool last) {
    if (run == none) return;
    const bool in = first && run == before, out = last && run == behind;
    if (in || out) {
      store_row<float, kVec>(a.partial + (2 * chunk + (in ? 0 : 1)) * a.H, acc, slice, lane, kWidth, a.H);
      if (!in && slice == 0 && lane == 0) a.runs[atomicAdd(a.run_count, 1u)] = (uint32_t)chunk;
    } else
      finish_row<W, kVec>(dtable + (int64_t)run * a.H, acc, a.scale, a.accumulate, slice, lane, kWidth, a.H);
  };
  constexpr int kAhead = 4;  // rows that are added while as many are on their way
  const int turn = min(kWidth, a.length);
  uint32_t next_key = lo + lane < hi ? a.keys[lo + lane] : none, next_place = lo + lane < hi ? a.places[lo + lane] : 0u;
  for (int64_t base = lo; __any_sync(0xffffffffu, base < hi); base += kWidth) {
    // tokens of this turn, one a lane, and of the next
    const uint32_t key = next_key, place = next_place;
    if (!__any_sync(0xffffffffu, key != none)) break;  // the rest has no part
    const int64_t mine = base + kWidth + lane;
    next_key = mine < hi ? a.keys[mine] : none;
    next_place = mine < hi ? a.places[mine] : 0u;
    Raw8<D> next[kAhead];
    uint32_t next_id[kAhead];
    auto load = [&](int j0) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        next_id[j] = __shfl_sync(0xffffffffu, key, j0 + j, kWidth);
        const uint32_t p = __shfl_sync(0xffffffffu, place, j0 + j, kWidth);
        if (next_id[j] != none) next[j] = load_row<D, kVec>(dout + (int64_t)p * a.H, slice, lane, kWidth, a.H);
      }
    };
    load(0);
#pragma unroll 1
    for (int j0 = 0; j0 < turn; j0 += kAhead) {
      Raw8<D> row[kAhead];
      uint32_t id[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        row[j] = next[j];
        id[j] = next_id[j];
      }
      if (j0 + kAhead < turn) load(j0 + kAhead);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (id[j] == none) continue;
        if (id[j] != run) {
          if (run != none) {
            flush(false);
            first = false;
          }
          run = id[j];
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] = 0.f;
        }
        float f[8];
        widen8(row[j], f);
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] += f[k];
      }
      __syncwarp();
    }
  }
  flush(true);
}

// Sums over borders: a block takes a run that leaves its first chunk, and 128 columns; its 8 rows of threads add up every eighth chunk's
// part each.  The runs are listed in any order, each is added up in the chunks' order.
constexpr int kJoinColumns = 32, kJoinRows = kThreads / kJoinColumns;
template <typename W>
__global__ void __launch_bounds__(kThreads) join_kernel(const __grid_constant__ SumArgs a, W* __restrict__ dtable) {
  __shared__ float s_acc[kJoinRows][kJoinColumns * 4];
  wait_for_predecessor();
  const int64_t slices = (a.H + kJoinColumns * 4 - 1) / (kJoinColumns * 4), items = *a.run_count * slices;
  const int tx = (int)threadIdx.x % kJoinColumns, ty = (int)threadIdx.x / kJoinColumns;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t chunk = a.runs[item / slices], slice = item % slices;
    const uint32_t run = a.keys[chunk * a.length + a.length - 1];
    // the run's last chunk: the last that begins with it
    int64_t last = chunk;
    for (int more = kThreads; more == kThreads;) {
      const int64_t k = last + 1 + threadIdx.x;
      more = __syncthreads_count(k < a.chunks && a.keys[k * a.length] == run);
      last += more;
    }
    const int64_t c0 = slice * kJoinColumns * 4 + tx;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int64_t k = chunk + ty; k <= last; k += kJoinRows) {
      const float* row = a.partial + (2 * k + (k == chunk ? 1 : 0)) * a.H;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c0 + e * kJoinColumns < a.H) acc[e] += row[c0 + e * kJoinColumns];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s_acc[ty][e * kJoinColumns + tx] = acc[e];
    __syncthreads();
    const int64_t c = slice * kJoinColumns * 4 + threadIdx.x;
    if (threadIdx.x < kJoinColumns * 4 && c < a.H) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < kJoinRows; ++r) s += s_acc[r][threadIdx.x];
      W* out = dtable + (int64_t)run * a.H + c;
      s *= a.scale;
      *out = from_float<W>(a.accumulate ? s + to_float(*out) : s);
    }
    __syncthreads();
  }
}

// ---- plans --------------------------------------------------------------------------------------
struct Plan {
  int64_t tiles, chunks, sum_blocks;
  int length, slices, width;
  size_t keys, counts, runs, partial, bytes;  // offsets into the scratch
};
Plan plan(int64_t n, int64_t H) {
  Plan p{};
  auto take = [&p](size_t bytes) {
    const size_t at = p.bytes;
    p.bytes += align_up(bytes, 256);
    return at;
  };
  p.tiles = ceil_div(n, kTile);
  p.width = H > 128 ? 32 : H > 64 ? 16 : 8;
  p.slices = (int)ceil_div(H, p.width * 8);
  // As many chunks as the SMs hold at once: with more of them a second wave comes, and more runs go over borders.
  const int64_t lanes = (int64_t)148 * kSumBlocks * kThreads, units = std::max<int64_t>(1, lanes / p.width / p.slices);
  const int64_t each = ceil_div(n, units);
  p.length = each <= 8 ? 8 : each <= 16 ? 16 : (int)std::min<int64_t>(1024, ceil_div(each, 32) * 32);
  p.chunks = ceil_div(n, p.length);
  p.sum_blocks = ceil_div(p.chunks * p.slices * p.width, kThreads);
  p.keys = take((size_t)n * 4 * 4);
  p.counts = take((size_t)p.tiles * kDigits * 4);
  p.runs = take((size_t)(p.chunks + 1) * 4);
  p.partial = take((size_t)p.chunks * 2 * H * 4);
  return p;
}

// Lets a kernel have more shared memory, and with `large` form larger clusters, than any may; once for each device.
template <typename K>
void allow_large(K kernel, size_t bytes, bool large, std::atomic<bool> (&allowed)[64]) {
  int device = 0;
  BAGUA_CUDA_CHECK(cudaGetDevice(&device));
  if (device < 64 && allowed[device].load(std::memory_order_acquire)) return;
  BAGUA_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  if (large) BAGUA_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  if (device < 64) allowed[device].store(true, std::memory_order_release);
}

template <typename Id>
int sort(const Ids& ids, Keys key, const Plan& p, uint32_t* buffers, uint32_t* counts, uint32_t* zero, void* clear_at, int64_t clear_bytes,
         const uint32_t** keys, const uint32_t** places, cudaStream_t s) {
  const int64_t n = ids.n;
  int bits = 1;
  while (bits < 32 && (key.rows >> bits) != 0) ++bits;
  const int passes = (bits + kSortBits - 1) / kSortBits;
  const int digit_bits = std::max(5, (bits + passes - 1) / passes);  // whole warps of digits
  // In one launch, by as many blocks as there is work for and the stream's context has room for; -1: not by this kernel.
  auto in_cluster = [&](auto most) {
    auto* kernel = sort_kernel<Id, decltype(most)::value>;
    static std::atomic<bool> allowed[64];
    allow_large(kernel, sort_shared_bytes(kSortRounds), most > 8, allowed);
    int blocks = 1;
    while (blocks < most && (int64_t)blocks * kSortThreads < n) blocks *= 2;
    for (; blocks >= 1; blocks /= 2) {
      const int64_t rounds = ceil_div(n, (int64_t)blocks * kSortThreads);
      if (rounds > kSortRounds) return -1;
      const size_t shared = sort_shared_bytes((int)rounds);
      if (fitting_cluster((const void*)kernel, blocks, kSortThreads, shared, s) != blocks) continue;
      const bool small = clear_bytes <= kSmallClear * blocks;
      launch_clusters_shared(kernel, 1, blocks, dim3(kSortThreads), shared, s, (const Id*)ids.data, key, (int)n, bits, digit_bits, (int)rounds,
                             buffers, buffers + n, zero, (uint4*)(small ? clear_at : nullptr), clear_bytes);
      if (clear_at && !small) clear(clear_at, clear_bytes, s);
      *keys = buffers;
      *places = buffers + n;
      return clear_at && !small ? 2 : 1;
    }
    return -1;
  };
  if (n > kSortMany && n <= kSortTokens)
    if (const int launches = in_cluster(std::integral_constant<int, kSortBlocksMany>{}); launches > 0) return launches;
  if (n <= (int64_t)kSortBlocks * kSortThreads * kSortRounds)
    if (const int launches = in_cluster(std::integral_constant<int, kSortBlocks>{}); launches > 0) return launches;
  uint32_t* k[2] = {buffers, buffers + 2 * n};
  const uint32_t *in_k = nullptr, *in_p = nullptr;
  int launches = 0, to = 0;
  for (int shift = 0; shift < bits; shift += 8, to ^= 1) {
    launch_overlapped(histogram_kernel<Id>, dim3((unsigned)p.tiles), dim3(kThreads), s, (const Id*)ids.data, in_k, key, n, shift, counts,
                      (int)p.tiles);
    launch_overlapped(scan_kernel, dim3(1), dim3(kScanThreads), s, counts, p.tiles * kDigits, zero);
    if (clear_at && shift == 0) clear(clear_at, clear_bytes, s);
    launch_overlapped(scatter_kernel<Id>, dim3((unsigned)p.tiles), dim3(kThreads), s, (const Id*)ids.data, in_k, in_p, key, n, shift, counts,
                      (int)p.tiles, k[to], k[to] + n);
    in_k = k[to];
    in_p = k[to] + n;
    launches += 3;
  }
  *keys = in_k;
  *places = in_p;
  return launches + (clear_at != nullptr);
}

template <typename D, typename W>
void sums(const SumArgs& a, const Plan& p, const void* dout, void* dtable, cudaStream_t s) {
  const bool vec = a.H % 8 == 0 && ((uintptr_t)dout | (uintptr_t)dtable) % 16 == 0;
  const dim3 grid((unsigned)p.sum_blocks);
  auto go = [&](auto kernel) { launch_overlapped(kernel, grid, dim3(kThreads), s, a, (const D*)dout, (W*)dtable); };
  if (vec)
    p.width == 32 ? go(sum_kernel<D, W, true, 32>) : p.width == 16 ? go(sum_kernel<D, W, true, 16>) : go(sum_kernel<D, W, true, 8>);
  else
    p.width == 32 ? go(sum_kernel<D, W, false, 32>) : p.width == 16 ? go(sum_kernel<D, W, false, 16>) : go(sum_kernel<D, W, false, 8>);
  if (a.chunks > 1) {
    const int64_t items = (a.chunks - 1) * ceil_div(a.H, kJoinColumns * 4);  // at most
    launch_overlapped(join_kernel<W>, dim3((unsigned)std::min<int64_t>(items, 8 * 148)), dim3(kThreads), s, a, (W*)dtable);
  }
}

template <typename F>
void typed(DType t, F&& f) {
  switch (t) {
    case DType::F32: f((float*)nullptr); return;
    case DType::F16: f((__half*)nullptr); return;
    case DType::BF16: f((__nv_bfloat16*)nullptr); return;
    default: throw BaguaError(ErrorKind::Tensor, std::string("embedding: unsupported type ") + dtype_name(t));
  }
}

}  // namespace

void lookup(const Ids& ids, const void* table, DType table_type, int64_t rows, int64_t row_stride, int64_t H, float scale, void* out,
            DType out_type, cudaStream_t s) {
  BAGUA_CHECK(ids.n > 0 && ids.n <= kMaxTokens && H > 0, Tensor, "embedding: " << ids.n << " tokens of " << H << " columns");
  typed(table_type, [&](auto* w) {
    using W = std::remove_pointer_t<decltype(w)>;
    typed(out_type, [&](auto* o) {
      using O = std::remove_pointer_t<decltype(o)>;
      auto go = [&](auto* id) {
        using Id = std::remove_pointer_t<decltype(id)>;
        // whether runs of so many elements start on multiples of their size, up to 16 bytes, in every row
        auto fits = [&](int64_t e) {
          const int64_t w = std::min<int64_t>(16, e * (int64_t)sizeof(W)), o = std::min<int64_t>(16, e * (int64_t)sizeof(O));
          return H % e == 0 && (int64_t)((uintptr_t)table % w) == 0 && row_stride * (int64_t)sizeof(W) % w == 0 &&
                 (int64_t)((uintptr_t)out % o) == 0;
        };
        if (fits(8)) {
          int shift = 0;
          while ((1 << shift) < kThreads && (1 << shift) < H / 8) ++shift;
          const int64_t slices = ceil_div(H / 8, 1 << shift);
          BAGUA_CHECK(slices < 65536, Tensor, "embedding: " << H << " columns");
          const bool many = ids.n * H >= kManyElements;
          const dim3 grid((unsigned)ceil_div(ids.n, (int64_t)(kThreads >> shift) * (many ? kRowsAhead : 1)), (unsigned)slices);
          launch_overlapped(many ? lookup_kernel<Id, W, O, kRowsAhead> : lookup_kernel<Id, W, O, 1>, grid, dim3(kThreads), s,
                            (const Id*)ids.data, (const W*)table, rows, row_stride, (O*)out, ids.n, H, shift, scale, encoder_ops::index_report());
        } else {
          launch_overlapped(fits(2) ? lookup_any_kernel<Id, W, O, 2> : lookup_any_kernel<Id, W, O, 1>, dim3((unsigned)ceil_div(ids.n, kThreads / 32)),
                            dim3(kThreads), s, (const Id*)ids.data, (const W*)table, rows, row_stride, (O*)out, ids.n, H, scale,
                            encoder_ops::index_report());
        }
      };
      ids.wide ? go((int64_t*)nullptr) : go((int32_t*)nullptr);
    });
  });
}

size_t backward_scratch_bytes(int64_t n, int64_t H) { return plan(n, H).bytes; }

int backward(const Ids& ids, const void* dout, DType dout_type, int64_t rows, int64_t H, float scale, int64_t padding, void* dtable,
             DType table_type, bool accumulate, void* scratch, cudaStream_t s) {
  BAGUA_CHECK(ids.n > 0 && ids.n <= kMaxTokens && rows > 0 && rows <= kMaxRows && H > 0, Tensor,
              "embedding backward: " << ids.n << " tokens, " << rows << " rows of " << H << " columns");
  BAGUA_CHECK(!accumulate || table_type == DType::F32, Tensor, "embedding gradients are added to in float32");
  const Plan p = plan(ids.n, H);
  auto at = [&](size_t offset) { return (uint32_t*)((char*)scratch + offset); };
  void* clear_at = accumulate ? nullptr : dtable;
  const int64_t clear_bytes = rows * H * (int64_t)dtype_bytes(table_type);
  BAGUA_CHECK(p.sum_blocks < (1ll << 31) && ceil_div(clear_bytes, kClearBytes) < (1ll << 31), Tensor,
              "embedding backward: " << rows << " rows of " << H << " columns");
  BAGUA_CHECK((uintptr_t)dtable % 16 == 0 || accumulate, Tensor, "embedding backward: the gradient does not start on 16 bytes");
  SumArgs a{};
  const Keys key{rows, padding};
  int launches = ids.wide ? sort<int64_t>(ids, key, p, at(p.keys), at(p.counts), at(p.runs), clear_at, clear_bytes, &a.keys, &a.places, s)
                          : sort<int32_t>(ids, key, p, at(p.keys), at(p.counts), at(p.runs), clear_at, clear_bytes, &a.keys, &a.places, s);
  a.accumulate = accumulate;
  a.run_count = at(p.runs);
  a.runs = a.run_count + 1;
  a.partial = (float*)at(p.partial);
  a.n = ids.n;
  a.rows = rows;
  a.H = H;
  a.chunks = p.chunks;
  a.length = p.length;
  a.slices = p.slices;
  a.scale = scale;
  typed(dout_type, [&](auto* d) {
    typed(table_type, [&](auto* w) { sums<std::remove_pointer_t<decltype(d)>, std::remove_pointer_t<decltype(w)>>(a, p, dout, dtable, s); });
  });
  return launches + 1 + (p.chunks > 1);
}

}  // namespace embedding
}  // namespace bagua
