// Sums of gradient rows by sorted token: every table row's terms added up in
// the order of their positions and handed, finished, to an epilogue (a store,
// or Adam). No float atomics: the order of the additions depends on the sizes
// alone.
//
// The sorted list is cut into blocks of equal length and these into groups of
// lanes; a group walks its tokens with the running sum of the current row in
// registers (each lane a vector of columns) and hands on a row when the next
// one begins. Rows that cross a border leave the part behind the border (the
// group's "head"): borders between groups are joined in shared memory, borders
// between blocks through partial sums in the workspace by a second kernel.
//
// Bound by reading the gradient rows, which lie anywhere: every lane keeps
// kStages - 1 asynchronous copies of 16 bytes in flight into slots of its own
// (about 60 KB an SM, twice what covers the latency of memory), so the loop
// over tokens is rolled and the epilogue is compiled once.
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "counter_mask.cuh"
#include "element_types.cuh"
#include "gaussian_math.cuh"

namespace clad3dgs {
namespace sums {

constexpr int kThreads = 256;
constexpr int kStages = 6;
constexpr int kSms = 148, kBlocksPerSm = 4;
constexpr int kMostTokens = 2048;  // of a block: their order entries lie in shared memory
constexpr uint32_t kNoRow = ~0u;

// How [n][width] gradients are cut: `lanes` vectors side by side in a group,
// `slices` groups a row, `tokens` of one group, `block` of one block.
struct Cut {
  int lanes, tokens, block;
  int64_t slices, blocks;
};

inline Cut cut_of(int64_t n, int64_t width, int vec) {
  const int64_t vectors = (width + vec - 1) / vec;
  Cut c{};
  if (vectors < 8) {
    c.lanes = 1;
    while (c.lanes < vectors) c.lanes *= 2;
  } else {
    // The group width that leaves the fewest lanes without a column.
    int64_t least = INT64_MAX;
    for (int lanes = 32; lanes >= 8; lanes /= 2) {
      const int64_t padded = (vectors + lanes - 1) / lanes * lanes;
      if (padded < least) least = padded, c.lanes = lanes;
    }
  }
  c.slices = (vectors + c.lanes - 1) / c.lanes;
  // Tokens of a group: what fills the GPU once, within bounds that keep the
  // partial sums few (8) and the order entries in shared memory.
  const int groups = kThreads / c.lanes;
  const int64_t resident =
      std::max<int64_t>(1, int64_t(kSms) * kBlocksPerSm * groups / c.slices);
  const int most = std::min(128, kMostTokens / groups);
  c.tokens = int(std::min<int64_t>(most, std::max<int64_t>(8, (n + resident - 1) / resident)));
  c.block = groups * c.tokens;
  c.blocks = (n + c.block - 1) / c.block;
  return c;
}

template <class T>
struct Args {
  int64_t n, rows, width;
  Cut cut;
  const T* grad;
  int64_t stride;
  const uint2* order;
  float factor;
  CounterMask mask;
  float* partial;  // [2 * blocks][width]: a block's head, and the end of its last row
};

// ---- epilogues: element `at` of the table and V finished sums ----

template <class T>
struct Store {
  T* out;

  template <int V>
  __device__ __forceinline__ void operator()(int64_t at, const float (&sum)[V]) const {
    Vec<T, V> v;
#pragma unroll
    for (int j = 0; j < V; ++j) v.v[j] = from_float<T>(sum[j]);
    *reinterpret_cast<Vec<T, V>*>(out + at) = v;
  }
};

struct Adam {
  float *table, *first, *second;
  float step;
  double inv_bias2;

  template <int V>
  __device__ __forceinline__ void operator()(int64_t at, const float (&sum)[V]) const {
    constexpr int W = V < 4 ? V : 4;
#pragma unroll
    for (int h = 0; h < V; h += W) {
      auto* p = reinterpret_cast<Vec<float, W>*>(table + at + h);
      auto* m = reinterpret_cast<Vec<float, W>*>(first + at + h);
      auto* v = reinterpret_cast<Vec<float, W>*>(second + at + h);
      Vec<float, W> pv = *p, mv = *m, vv = *v;
#pragma unroll
      for (int j = 0; j < W; ++j)
        torch_adam(pv.v[j], mv.v[j], vv.v[j], sum[h + j], step, inv_bias2);
      *p = pv;
      *m = mv;
      *v = vv;
    }
  }
};

// ---- vectors of sums in memory ----

template <int V>
__device__ __forceinline__ void put(float* to, const float (&sum)[V]) {
  constexpr int W = V < 4 ? V : 4;
#pragma unroll
  for (int h = 0; h < V; h += W) {
    Vec<float, W> v;
#pragma unroll
    for (int j = 0; j < W; ++j) v.v[j] = sum[h + j];
    *reinterpret_cast<Vec<float, W>*>(to + h) = v;
  }
}

template <int V>
__device__ __forceinline__ void add(const float* from, float (&sum)[V]) {
  constexpr int W = V < 4 ? V : 4;
#pragma unroll
  for (int h = 0; h < V; h += W) {
    const Vec<float, W> v = *reinterpret_cast<const Vec<float, W>*>(from + h);
#pragma unroll
    for (int j = 0; j < W; ++j) sum[h + j] += v.v[j];
  }
}

template <int V>
__device__ __forceinline__ void clear(float (&sum)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = 0.f;
}

template <int V, class End>
__device__ __forceinline__ void finish(const End& end, int64_t at, float (&sum)[V],
                                       float factor) {
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] *= factor;
  end.template operator()<V>(at, sum);
}

template <int kBytes>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to));
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(kBytes)
                 : "memory");
}

// Shared memory of sum_kernel, in bytes.
inline size_t order_bytes(const Cut& c) { return (size_t(c.block + 2) * sizeof(uint2) + 15) / 16 * 16; }

template <class T, int V>
size_t shared_bytes(const Cut& c) {
  return order_bytes(c) + size_t(kThreads) * (V * sizeof(float) + kStages * V * sizeof(T)) +
         kThreads;
}

// A group's head: none, ended within the group, or open at its end.
enum Head : unsigned char { kNone = 0, kEnded = 1, kOpen = 2 };

template <class T, int V, bool kDrop, class End>
__global__ void __launch_bounds__(kThreads)
    sum_kernel(const __grid_constant__ Args<T> a, const End end) {
  constexpr int kBytes = V * sizeof(T);
  extern __shared__ __align__(16) char shared[];
  const size_t order_size = (size_t(a.cut.block + 2) * sizeof(uint2) + 15) / 16 * 16;
  uint2* entries = reinterpret_cast<uint2*>(shared);
  float* heads = reinterpret_cast<float*>(shared + order_size);
  char* slots = shared + order_size + size_t(kThreads) * V * sizeof(float);
  unsigned char* kinds = reinterpret_cast<unsigned char*>(slots + kThreads * kStages * kBytes);

  const unsigned long long offset = kDrop ? mask_offset(a.mask) : 0;
  const int64_t block = blockIdx.x / a.cut.slices;
  const int lane = threadIdx.x % a.cut.lanes, group = threadIdx.x / a.cut.lanes;
  const int groups = kThreads / a.cut.lanes;
  const int64_t column = ((blockIdx.x - block * a.cut.slices) * a.cut.lanes + lane) * V;
  const bool live = column < a.width;
  const int64_t first = block * a.cut.block;
  const int count = int(a.n - first < a.cut.block ? a.n - first : a.cut.block);
  // Entries of the block and one on each side (kNoRow past the list's ends).
  for (int i = threadIdx.x; i < count + 2; i += kThreads) {
    const int64_t at = first + i - 1;
    entries[i] = at >= 0 && at < a.n ? a.order[at] : make_uint2(kNoRow, 0);
  }
  __syncthreads();
  const uint2* entry = entries + 1;

  const int begin = group * a.cut.tokens;
  const int stop = begin + a.cut.tokens < count ? begin + a.cut.tokens : count;
  float sum[V];
  clear<V>(sum);
  uint32_t row = begin < stop ? entry[begin].x : kNoRow;
  bool before = row < a.rows && entry[begin - 1].x == row;
  Head kind = kNone;

  // One token's terms; hands the row before on when a new one begins.
  auto take = [&](const uint2& token, const Vec<T, V>& g) {
    if (token.x != row) {
      if (before) {
        put<V>(heads + threadIdx.x * V, sum);
        kind = kEnded;
      } else if (live) {
        finish<V>(end, row * a.width + column, sum, a.factor);
      }
      before = false;
      row = token.x;
      clear<V>(sum);
    }
    if (row >= a.rows) return;
    if constexpr (kDrop) {
      bool keep[V];
      mask_vector<V>(a.mask, offset, token.y * a.width + column, keep);
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += keep[j] ? to_float(g.v[j]) : 0.f;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += to_float(g.v[j]);
    }
  };

  if constexpr (kBytes >= 4) {
    char* mine = slots + threadIdx.x * kBytes;
    auto fetch = [&](int i) {
      if (i < stop && live && entry[i].x < a.rows)
        copy_async<kBytes>(mine + (i - begin) % kStages * (kThreads * kBytes),
                           a.grad + entry[i].y * a.stride + column);
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int s = 0; s < kStages - 1; ++s) fetch(begin + s);
    for (int i = begin; i < stop && row < a.rows; ++i) {
      fetch(i + kStages - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      take(entry[i],
           *reinterpret_cast<const Vec<T, V>*>(mine + (i - begin) % kStages * (kThreads * kBytes)));
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // Single 16-bit elements, which no asynchronous copy takes: loads in batches.
    constexpr int kBatch = 8;
    for (int i = begin; i < stop && row < a.rows; i += kBatch) {
      Vec<T, V> g[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (i + u < stop && live && entry[i + u].x < a.rows)
          g[u] = *reinterpret_cast<const Vec<T, V>*>(a.grad + entry[i + u].y * a.stride + column);
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (i + u < stop) take(entry[i + u], g[u]);
    }
  }

  // The group's last row: finished, a head that stays open, or continued by
  // the next group.
  const bool after = row < a.rows && entry[stop].x == row;
  if (row < a.rows) {
    if (before) {
      put<V>(heads + threadIdx.x * V, sum);
      kind = after ? kOpen : kEnded;
    } else if (!after && live) {
      finish<V>(end, row * a.width + column, sum, a.factor);
    }
  }
  if (lane == 0) kinds[group] = kind;
  __syncthreads();
  const bool continued = after && !before;
  auto join = [&](int from) {  // adds the heads from group `from` on; true if the last is open
    bool open = true;
    for (int h = from; h < groups && open; ++h) {
      add<V>(heads + (h * a.cut.lanes + lane) * V, sum);
      open = kinds[h] == kOpen;
    }
    return open;
  };
  if (continued) {
    if (join(group + 1)) {
      if (live) put<V>(a.partial + (2 * block + 1) * a.width + column, sum);
    } else if (live) {
      finish<V>(end, row * a.width + column, sum, a.factor);
    }
  }
  if (group == 0 && kind != kNone) {
    clear<V>(sum);
    add<V>(heads + lane * V, sum);
    if (kind == kOpen) join(1);
    if (live) put<V>(a.partial + 2 * block * a.width + column, sum);
  }
}

// Rows that cross borders between blocks: the block that a row begins in adds
// the heads of the blocks behind it, each group a share of them, the shares in
// order.
template <class T, int V, class End>
__global__ void __launch_bounds__(kThreads)
    join_kernel(const __grid_constant__ Args<T> a, const End end) {
  __shared__ __align__(16) float shares[kThreads * V];
  const int64_t block = blockIdx.x / a.cut.slices;
  const int64_t first = block * a.cut.block, stop = first + a.cut.block;
  if (stop >= a.n) return;
  const uint32_t row = a.order[stop - 1].x;
  if (row >= a.rows || a.order[stop].x != row) return;
  if (first > 0 && a.order[first - 1].x == row) return;  // began earlier
  const int lane = threadIdx.x % a.cut.lanes, group = threadIdx.x / a.cut.lanes;
  const int groups = kThreads / a.cut.lanes;
  const int64_t column = ((blockIdx.x - block * a.cut.slices) * a.cut.lanes + lane) * V;
  const bool live = column < a.width;
  // How many blocks behind begin with this row (they are the next ones).
  int64_t heads = 0;
  for (int more = kThreads; more == kThreads; heads += more) {
    const int64_t at = stop + (heads + threadIdx.x) * a.cut.block;
    more = __syncthreads_count(at < a.n && a.order[at].x == row);
  }
  float sum[V];
  clear<V>(sum);
  if (live)
    for (int64_t h = heads * group / groups; h < heads * (group + 1) / groups; ++h)
      add<V>(a.partial + 2 * (block + 1 + h) * a.width + column, sum);
  put<V>(shares + threadIdx.x * V, sum);
  __syncthreads();
  if (group > 0 || !live) return;
  clear<V>(sum);
  add<V>(a.partial + (2 * block + 1) * a.width + column, sum);
  for (int g = 0; g < groups; ++g) add<V>(shares + (g * a.cut.lanes + lane) * V, sum);
  finish<V>(end, row * a.width + column, sum, a.factor);
}

// Rows that no token names: a gradient of zero. One warp takes 32 rows, each
// lane looks one of them up in the order.
template <int V, class End>
__global__ void __launch_bounds__(kThreads)
    rest_kernel(int64_t n, int64_t rows, int64_t width, const uint2* __restrict__ order,
                const End end) {
  const int64_t first = (blockIdx.x * int64_t(kThreads) + threadIdx.x) / 32 * 32;
  if (first >= rows) return;
  const int lane = threadIdx.x & 31;
  const int64_t mine = first + lane;
  bool named = true;
  if (mine < rows) {
    int64_t low = 0, high = n;
    while (low < high) {
      const int64_t middle = (low + high) / 2;
      if (order[middle].x < mine) low = middle + 1;
      else high = middle;
    }
    named = low < n && order[low].x == mine;
  }
  unsigned left = __ballot_sync(~0u, !named);
  const float zero[V] = {};
  while (left) {
    const int64_t row = first + __ffs(left) - 1;
    left &= left - 1;
    for (int64_t column = lane * V; column < width; column += 32 * V)
      end.template operator()<V>(row * width + column, zero);
  }
}

// ---- host ----

template <class T, int V, class End>
cudaError_t run_sums(Args<T> a, const End& end, bool drop, cudaStream_t stream) {
  if (a.n == 0) return cudaSuccess;
  a.cut = cut_of(a.n, a.width, V);
  const size_t shared = shared_bytes<T, V>(a.cut);
  const unsigned grid = unsigned(a.cut.blocks * a.cut.slices);
  auto* kernel = drop ? sum_kernel<T, V, true, End> : sum_kernel<T, V, false, End>;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(shared));
  if (e != cudaSuccess) return e;
  kernel<<<grid, kThreads, shared, stream>>>(a, end);
  if (a.cut.blocks > 1) join_kernel<T, V, End><<<grid, kThreads, 0, stream>>>(a, end);
  return cudaGetLastError();
}

template <int V, class End>
cudaError_t run_rest(int64_t n, int64_t rows, int64_t width, const uint2* order, const End& end,
                     cudaStream_t stream) {
  const unsigned grid = unsigned((rows + kThreads - 1) / kThreads);
  rest_kernel<V, End><<<grid, kThreads, 0, stream>>>(n, rows, width, order, end);
  return cudaGetLastError();
}

// `bytes`: what every row of the gradients starts on; `end_bytes`: the same of
// the epilogue's arrays, whose elements are E. Vectors are the longest that
// both allow.
template <class T, class E, class End>
cudaError_t run(const Args<T>& a, const End& end, int bytes, int end_bytes, bool drop,
                cudaStream_t stream) {
  constexpr int kMost = 16 / sizeof(T), kEndMost = 16 / sizeof(E);
  const int end_vec = end_bytes / int(sizeof(E));
  // An epilogue moves 16 bytes at a time, so longer vectors need no more than that.
  const int vec = std::min(bytes / int(sizeof(T)), end_vec >= kEndMost ? kMost : end_vec);
  cudaError_t e;
  if (vec >= 8 && kMost >= 8) e = run_sums<T, (kMost >= 8 ? 8 : 1), End>(a, end, drop, stream);
  else if (vec >= 4) e = run_sums<T, 4, End>(a, end, drop, stream);
  else if (vec >= 2) e = run_sums<T, 2, End>(a, end, drop, stream);
  else e = run_sums<T, 1, End>(a, end, drop, stream);
  if (e != cudaSuccess) return e;
  if (end_vec >= 8 && kEndMost >= 8)
    return run_rest<(kEndMost >= 8 ? 8 : 1)>(a.n, a.rows, a.width, a.order, end, stream);
  if (end_vec >= 4) return run_rest<4>(a.n, a.rows, a.width, a.order, end, stream);
  if (end_vec >= 2) return run_rest<2>(a.n, a.rows, a.width, a.order, end, stream);
  return run_rest<1>(a.n, a.rows, a.width, a.order, end, stream);
}

// Workspace for any vector length (the most blocks any cut of these sizes has).
inline size_t workspace_bytes(int64_t n, int64_t width) {
  int64_t blocks = 0;
  for (int vec = 1; vec <= 8; vec *= 2) blocks = std::max(blocks, cut_of(n, width, vec).blocks);
  return size_t(2 * blocks) * width * sizeof(float);
}

}  // namespace sums
}  // namespace clad3dgs
