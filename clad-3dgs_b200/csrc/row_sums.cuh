// Sums of gradient rows by sorted token: every table row's terms added up in
// the order of their positions and handed, finished, to an epilogue (a store,
// or Adam). No float atomics: the order of the additions depends on the sizes
// alone.
//
// The sorted list is cut into blocks of equal length and these into groups of
// lanes; a group walks its tokens with the running sum of the current row in
// registers and hands on a row when the next one begins. Rows that cross a
// border leave the part behind the border (the group's "head"): borders
// between groups are joined in shared memory, borders between blocks through
// partial sums in the workspace by a second kernel. Rows that no token names
// are written by further blocks of the same launch.
//
// Bound by reading the gradient rows, which lie anywhere: every lane holds up to
// C vectors of 16 bytes of a row and keeps kStages - 1 rows in flight as
// asynchronous copies into slots of its own (60 to 80 KB an SM, twice what covers
// the latency of memory), so the loop over tokens is rolled and the epilogue is
// compiled once. Several vectors a lane share the loop's instructions, which
// else cost as much time as the memory does.
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
constexpr int kSms = 148;
constexpr int kSharedPerSm = 220 * 1024;
constexpr int kMostTokens = 2560;  // of a block: their order entries lie in shared memory
constexpr int kLeastTokens = 8;    // of a group: keeps the joins few
constexpr uint32_t kNoRow = ~0u;

// Rows in flight per lane, and one that is being added.
constexpr int stages_of(int c) { return c == 1 ? 6 : 3; }

// How [n][width] gradients are cut: C vectors of `lanes` lanes in a group,
// `slices` groups a row, `tokens` of one group, `block` of one block.
struct Cut {
  int lanes, tokens, block;
  int64_t slices, blocks;
};

inline size_t order_bytes(int block) { return (size_t(block + 2) * sizeof(uint2) + 15) / 16 * 16; }

// Shared memory of sum_kernel besides the order entries: heads, slots, kinds.
template <class T, int V, int C>
constexpr size_t lane_bytes() {
  return size_t(kThreads) * (C * V * (sizeof(float) + stages_of(C) * sizeof(T)) + 1);
}

// Lanes of a group for rows of `vectors` vectors, C a lane: a short row whole;
// else the width from 4 lanes (which read 64 bytes side by side) to 32 that
// leaves the fewest lanes without a column. `padded` is what it covers.
inline int lanes_of(int64_t vectors, int c, int64_t* padded) {
  int best = 1;
  while (best < 4 && best * c < vectors) best *= 2;
  *padded = (vectors + best * c - 1) / (best * c) * (best * c);
  if (best < 4) return best;
  *padded = INT64_MAX;
  for (int lanes = 32; lanes >= 4; lanes /= 2) {
    const int64_t covered = (vectors + lanes * c - 1) / (lanes * c) * (lanes * c);
    if (covered < *padded) *padded = covered, best = lanes;
  }
  return best;
}

inline Cut cut_of(int64_t n, int64_t width, int vec, int c, size_t per_block) {
  const int64_t vectors = (width + vec - 1) / vec;
  Cut cut{};
  int64_t padded;
  cut.lanes = lanes_of(vectors, c, &padded);
  cut.slices = padded / (cut.lanes * c);
  // Tokens of a group: as many as fill the GPU in whole waves.
  const int groups = kThreads / cut.lanes;
  const int64_t resident = std::max<int64_t>(
      1, int64_t(kSms) * (kSharedPerSm / (per_block + order_bytes(kMostTokens))) * groups /
             cut.slices);
  const int most = std::max(kLeastTokens, kMostTokens / groups);
  const int64_t waves = (n + resident * most - 1) / (resident * most);
  cut.tokens = int(std::max<int64_t>(kLeastTokens, (n + resident * waves - 1) / (resident * waves)));
  cut.block = groups * cut.tokens;
  cut.blocks = (n + cut.block - 1) / cut.block;
  return cut;
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
  int64_t rest;    // blocks in front that write the rows without tokens
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

// Rows that no token names: a gradient of zero. One warp takes 32 rows and one
// slice of columns; each lane looks one of the rows up in the order.
template <int V, class End>
__device__ void write_rest(int64_t n, int64_t rows, int64_t width, const uint2* order,
                           const End& end) {
  const int64_t job = (blockIdx.x * int64_t(kThreads) + threadIdx.x) / 32;
  const int64_t slices = (width + 32 * V - 1) / (32 * V);
  const int64_t first = job / slices * 32;
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
  const int64_t column = (job % slices * 32 + lane) * V;
  if (column >= width) return;
  const float zero[V] = {};
  while (left) {
    end.template operator()<V>((first + __ffs(left) - 1) * width + column, zero);
    left &= left - 1;
  }
}

inline int64_t rest_blocks(int64_t rows, int64_t width, int vec) {
  const int64_t jobs = (rows + 31) / 32 * ((width + 32 * vec - 1) / (32 * vec));
  return (jobs + kThreads / 32 - 1) / (kThreads / 32);
}

// A group's head: none, ended within the group, or open at its end.
enum Head : unsigned char { kNone = 0, kEnded = 1, kOpen = 2 };

// V: elements of a vector of gradients, C: vectors of a lane, R: elements of a
// vector of the rows without tokens.
template <class T, int V, int C, int R, bool kDrop, class End>
__global__ void __launch_bounds__(kThreads)
    sum_kernel(const __grid_constant__ Args<T> a, const End end) {
  if (blockIdx.x < a.rest) {
    write_rest<R, End>(a.n, a.rows, a.width, a.order, end);
    return;
  }
  constexpr int kBytes = V * sizeof(T);
  constexpr int kStages = stages_of(C);
  extern __shared__ __align__(16) char shared[];
  uint2* entries = reinterpret_cast<uint2*>(shared);
  const size_t order_size = (size_t(a.cut.block + 2) * sizeof(uint2) + 15) / 16 * 16;
  float* heads = reinterpret_cast<float*>(shared + order_size);  // [C][kThreads][V]
  char* slots = shared + order_size + size_t(kThreads) * C * V * sizeof(float);
  unsigned char* kinds =
      reinterpret_cast<unsigned char*>(slots + size_t(kThreads) * kStages * C * kBytes);

  const unsigned long long offset = kDrop ? mask_offset(a.mask) : 0;
  const int64_t job = blockIdx.x - a.rest;
  const int64_t block = job / a.cut.slices;
  const int lane = threadIdx.x % a.cut.lanes, group = threadIdx.x / a.cut.lanes;
  const int groups = kThreads / a.cut.lanes;
  // This lane's columns: `column` and C - 1 more, `apart` from each other.
  const int apart = a.cut.lanes * V;
  const int64_t column = (job - block * a.cut.slices) * (apart * C) + lane * V;
  bool live[C];
#pragma unroll
  for (int c = 0; c < C; ++c) live[c] = column + c * apart < a.width;
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
  int stop = begin + a.cut.tokens < count ? begin + a.cut.tokens : count;
  if (begin < stop && entry[stop - 1].x >= a.rows) {
    // Tokens without a row end the list: keep those in front of them.
    int low = begin;
    while (low < stop) {
      const int middle = (low + stop) / 2;
      if (entry[middle].x < a.rows) low = middle + 1;
      else stop = middle;
    }
  }
  float sum[C][V];
  auto reset = [&] {
#pragma unroll
    for (int c = 0; c < C; ++c) clear<V>(sum[c]);
  };
  uint32_t row = begin < stop ? entry[begin].x : kNoRow;
  auto done = [&] {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (live[c]) finish<V>(end, row * a.width + column + c * apart, sum[c], a.factor);
  };
  auto put_head = [&] {
#pragma unroll
    for (int c = 0; c < C; ++c) put<V>(heads + (c * kThreads + threadIdx.x) * V, sum[c]);
  };
  reset();
  bool before = begin < stop && entry[begin - 1].x == row;
  Head kind = kNone;

  // One token's terms; hands the row before on when a new one begins.
  auto take = [&](const uint2& token, const Vec<T, V> (&g)[C]) {
    if (token.x != row) {
      if (before) {
        put_head();
        kind = kEnded;
        before = false;
      } else {
        done();
      }
      row = token.x;
      reset();
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if constexpr (kDrop) {
        bool keep[V];
        mask_vector<V>(a.mask, offset, token.y * a.width + column + c * apart, keep);
#pragma unroll
        for (int j = 0; j < V; ++j) sum[c][j] += keep[j] ? to_float(g[c].v[j]) : 0.f;
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[c][j] += to_float(g[c].v[j]);
      }
    }
  };

  const T* grad = a.grad + column;
  if constexpr (kBytes >= 4) {
    char* mine = slots + threadIdx.x * kBytes;
    constexpr int kStageBytes = kThreads * C * kBytes;
    auto fetch = [&](int i, int slot) {
      if (i < stop) {
        const T* from = grad + entry[i].y * a.stride;
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (live[c])
            copy_async<kBytes>(mine + slot * kStageBytes + c * (kThreads * kBytes),
                               from + c * apart);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) fetch(begin + s, s);
    int slot = 0;
    for (int i = begin; i < stop; ++i) {
      fetch(i + kStages - 1, slot == 0 ? kStages - 1 : slot - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      Vec<T, V> g[C];
#pragma unroll
      for (int c = 0; c < C; ++c)
        g[c] = *reinterpret_cast<const Vec<T, V>*>(mine + slot * kStageBytes +
                                                   c * (kThreads * kBytes));
      take(entry[i], g);
      if (++slot == kStages) slot = 0;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // Single 16-bit elements, which no asynchronous copy takes: loads in batches.
    constexpr int kBatch = 4;
    for (int i = begin; i < stop; i += kBatch) {
      Vec<T, V> g[kBatch][C];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (i + u < stop) {
#pragma unroll
          for (int c = 0; c < C; ++c)
            if (live[c])
              g[u][c] = *reinterpret_cast<const Vec<T, V>*>(grad + entry[i + u].y * a.stride +
                                                            c * apart);
        }
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (i + u < stop) take(entry[i + u], g[u]);
    }
  }

  // The group's last row: finished, a head that stays open, or continued by
  // the next group.
  const bool after = begin < stop && entry[stop].x == row;
  const bool continued = after && !before;
  if (begin < stop) {
    if (before) {
      put_head();
      kind = after ? kOpen : kEnded;
    } else if (!after) {
      done();
    }
  }
  if (lane == 0) kinds[group] = kind;
  __syncthreads();
  auto join = [&](int from) {  // adds the heads from group `from` on; true if the last is open
    bool open = true;
    for (int h = from; h < groups && open; ++h) {
#pragma unroll
      for (int c = 0; c < C; ++c)
        add<V>(heads + (c * kThreads + h * a.cut.lanes + lane) * V, sum[c]);
      open = kinds[h] == kOpen;
    }
    return open;
  };
  auto put_partial = [&](int64_t which) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (live[c]) put<V>(a.partial + which * a.width + column + c * apart, sum[c]);
  };
  if (continued) {
    if (join(group + 1)) put_partial(2 * block + 1);
    else done();
  }
  if (group == 0 && kind != kNone) {
    reset();
#pragma unroll
    for (int c = 0; c < C; ++c) add<V>(heads + (c * kThreads + lane) * V, sum[c]);
    if (kind == kOpen) join(1);
    put_partial(2 * block);
  }
}

// Rows that cross borders between blocks: the block that a row begins in adds
// the heads of the blocks behind it, each group a share of them, the shares in
// order.
template <class T, int V, class End>
__global__ void __launch_bounds__(kThreads)
    join_kernel(const __grid_constant__ Args<T> a, int lanes, int64_t slices, const End end) {
  __shared__ __align__(16) float shares[kThreads * V];
  const int64_t block = blockIdx.x / slices;
  const int64_t first = block * a.cut.block, stop = first + a.cut.block;
  if (stop >= a.n) return;
  const uint32_t row = a.order[stop - 1].x;
  if (row >= a.rows || a.order[stop].x != row) return;
  if (first > 0 && a.order[first - 1].x == row) return;  // began earlier
  const int lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
  const int groups = kThreads / lanes;
  const int64_t column = ((blockIdx.x - block * slices) * lanes + lane) * V;
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
  for (int g = 0; g < groups; ++g) add<V>(shares + (g * lanes + lane) * V, sum);
  finish<V>(end, row * a.width + column, sum, a.factor);
}

// The launch without any token.
template <int R, class End>
__global__ void __launch_bounds__(kThreads)
    rest_kernel(int64_t rows, int64_t width, const End end) {
  write_rest<R, End>(0, rows, width, nullptr, end);
}

// ---- host ----

// Vectors of a lane: one, three or four, whatever covers a row with the fewest
// idle lanes; more of them where that is equal, unless the rows are so few
// that the groups would not fill the GPU.
inline int vectors_of_lane(int64_t n, int64_t width, int vec) {
  const int64_t vectors = (width + vec - 1) / vec;
  int64_t one, three, four;
  lanes_of(vectors, 1, &one);
  lanes_of(vectors, 3, &three);
  lanes_of(vectors, 4, &four);
  const int64_t least = std::min(one, std::min(three, four));
  auto fills = [&](int c, int64_t padded) {
    return padded == least && n * (padded / c) >= int64_t(kSms) * 512 * kLeastTokens;
  };
  if (fills(4, four)) return 4;
  return fills(3, three) ? 3 : 1;
}

template <class T, int V, int C, int R, class End>
cudaError_t run_cut(Args<T> a, const End& end, bool drop, cudaStream_t stream) {
  a.cut = cut_of(a.n, a.width, V, C, lane_bytes<T, V, C>());
  a.rest = rest_blocks(a.rows, a.width, R);
  const size_t shared = order_bytes(a.cut.block) + lane_bytes<T, V, C>();
  const unsigned grid = unsigned(a.rest + a.cut.blocks * a.cut.slices);
  auto* kernel = drop ? sum_kernel<T, V, C, R, true, End> : sum_kernel<T, V, C, R, false, End>;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(shared));
  if (e != cudaSuccess) return e;
  kernel<<<grid, kThreads, shared, stream>>>(a, end);
  if (a.cut.blocks > 1) {
    int64_t padded;
    const int lanes = lanes_of((a.width + V - 1) / V, 1, &padded);
    join_kernel<T, V, End><<<unsigned(a.cut.blocks * (padded / lanes)), kThreads, 0, stream>>>(
        a, lanes, padded / lanes, end);
  }
  return cudaGetLastError();
}

template <class T, int V, int R, class End>
cudaError_t run_sums(const Args<T>& a, const End& end, bool drop, cudaStream_t stream) {
  switch (vectors_of_lane(a.n, a.width, V)) {
    case 4: return run_cut<T, V, 4, R, End>(a, end, drop, stream);
    case 3: return run_cut<T, V, 3, R, End>(a, end, drop, stream);
    default: return run_cut<T, V, 1, R, End>(a, end, drop, stream);
  }
}

// `bytes`: what every row of the gradients starts on; `end_bytes`: the same of
// the epilogue's arrays, whose elements are E. Vectors are 16 bytes where both
// allow it, else single elements.
template <class T, class E, class End>
cudaError_t run(const Args<T>& a, const End& end, int bytes, int end_bytes, bool drop,
                cudaStream_t stream) {
  constexpr int kMost = 16 / sizeof(T), kEndMost = 16 / sizeof(E);
  if (a.n == 0) {
    if (end_bytes >= 16)
      rest_kernel<kEndMost, End><<<unsigned(rest_blocks(a.rows, a.width, kEndMost)), kThreads, 0,
                                   stream>>>(a.rows, a.width, end);
    else
      rest_kernel<1, End><<<unsigned(rest_blocks(a.rows, a.width, 1)), kThreads, 0, stream>>>(
          a.rows, a.width, end);
    return cudaGetLastError();
  }
  if (end_bytes < 16) return run_sums<T, 1, 1, End>(a, end, drop, stream);
  if (bytes < 16) return run_sums<T, 1, kEndMost, End>(a, end, drop, stream);
  return run_sums<T, kMost, kEndMost, End>(a, end, drop, stream);
}

// Workspace for any cut of these sizes: a group has kLeastTokens at least, a
// block at least a group for each 32 lanes.
inline size_t workspace_bytes(int64_t n, int64_t width) {
  const int64_t least = kThreads / 32 * kLeastTokens;
  return size_t(2 * ((n + least - 1) / least)) * width * sizeof(float);
}

}  // namespace sums
}  // namespace clad3dgs
