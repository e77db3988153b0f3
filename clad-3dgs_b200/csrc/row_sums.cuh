// Sums of gradient rows by sorted token: every table row's terms added up in
// the order of their positions. A row's sum is stored as the table's gradient,
// or kept for the Adam pass. No float atomics: the order of the additions
// depends on the sizes alone. Sums are 32 bits within a block and 64 where the
// blocks' parts of a long row meet (a row of 1.1M random terms came out up to
// 1.4e-6 off with 32 bits and one running sum throughout, now 3.4e-7).
//
// The sorted list is cut into blocks of equal length and these into groups of
// lanes; a group walks its tokens with the running sum of the current row in
// registers and hands on a row when the next one begins. Rows that cross a
// border leave the part behind the border (the group's "head"): borders
// between groups are joined in shared memory, borders between blocks through
// partial sums in the workspace by a second kernel. Rows that no token names
// are written by further blocks of the same launch.
//
// Bound by reading the gradient rows, which lie anywhere. Every lane holds C
// vectors of 16 bytes of a row and asks for U rows before it adds the first
// (64 to 128 bytes a thread, 50 to 100 KB an SM in flight). Several vectors a
// lane share the loop's instructions, which else cost as much time as the
// memory does. 1.1M rows of 48 floats over 8192 table rows: 45 us (4.7 TB/s; 38
// with the rows in order, so that random rows cost 7) and 5 us for the second
// kernel, 48 for both in a row. One wave of long blocks is best: 53 us with two
// waves, 63 with four, 56 with four blocks an SM instead of three.
//
// Adam is a pass of its own over the table, because an update inside the walk
// would wait for three loads at the end of every row (a walk over 8192 short
// rows took 77 us instead of 52). Only the sums of rows that tokens name go
// through memory in between, from a compact list.
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "counter_mask.cuh"
#include "element_types.cuh"
#include "gaussian_math.cuh"
#include "launch.cuh"
#include "token_index.cuh"

namespace clad3dgs {
namespace sums {

constexpr int kThreads = 256;
// A number of its own, not the device's: cuts, and with them the order of the
// additions, depend on the sizes alone.
constexpr int kSms = 148;
constexpr int kMostTokens = 3584;  // of a block: their order entries lie in shared memory
constexpr int kLeastTokens = 8;    // of a group: keeps the joins few
constexpr uint32_t kNoRow = ~0u;

// Rows a thread asks for at once (of each it takes `bytes`), and the blocks that
// an SM's registers hold (200000 rows of 256 floats, 64 bytes a thread and row: 47
// us with two blocks, 51 with three; 1M of 48 bf16, 32 bytes: 56 with three, 58 with
// two, although with three the kernels of two 16-bit vectors a lane spill 28 to 38
// bytes a thread).
constexpr int rows_at_once(int bytes, bool loose) {
  return loose ? 2 : bytes <= 8 ? 8 : bytes <= 16 ? 4 : 2;
}
constexpr int blocks_per_sm(int elements, int bytes) {
  return elements <= 4 ? 4 : bytes < 64 ? 3 : 2;
}

// How [n][width] gradients are cut: C vectors of `lanes` lanes in a group,
// `slices` groups a row, `tokens` of one group, `block` of one block.
struct Cut {
  int lanes, tokens, block;
  int64_t slices, blocks;
};

// Whether a cut that covers `padded` columns wastes little beside `least`: an
// eighth. Gradient of 200000 tokens with no slack, an eighth and a quarter: rows
// of 2020 floats 519, 332 and 331 us, of 1764 floats 273, 231 and 285, of 600 bf16
// 112, 68 and 74; the worst found for an eighth, 276 floats, 44, 50 and 44.
inline bool close_to(int64_t padded, int64_t least) { return padded * 8 <= least * 9; }

// Lanes of a group for rows of `vectors` vectors, C a lane: a short row whole;
// else the most, from 32 down to four (which read 64 bytes side by side), that
// leave few lanes without a column. `padded` is what they cover.
inline int lanes_of(int64_t vectors, int c, int64_t* padded) {
  auto covered = [&](int lanes) {
    return (vectors + lanes * c - 1) / (lanes * c) * (lanes * c);
  };
  int lanes = 1;
  while (lanes < 4 && lanes * c < vectors) lanes *= 2;
  if (lanes == 4) {
    const int64_t least = std::min(std::min(covered(4), covered(8)),
                                   std::min(covered(16), covered(32)));
    lanes = 32;
    while (!close_to(covered(lanes), least)) lanes /= 2;
  }
  *padded = covered(lanes);
  return lanes;
}

inline Cut cut_of(int64_t n, int64_t width, int vec, int c, int sm_blocks, int64_t rest) {
  const int64_t vectors = (width + vec - 1) / vec;
  Cut cut{};
  int64_t padded;
  cut.lanes = lanes_of(vectors, c, &padded);
  cut.slices = padded / (cut.lanes * c);
  // Tokens of a group: as many as fill the GPU in whole waves.
  const int groups = kThreads / cut.lanes;
  // (a few blocks in front for the rows without tokens take places of the first).
  // With more slices than places one block a slice, its groups all at work: 448
  // rows of 300000 floats 88 us, 321 with one group of eight.
  const int64_t places = int64_t(kSms) * sm_blocks;
  const int64_t resident =
      std::max<int64_t>(1, (places - (rest < places / 2 ? rest : 0)) / cut.slices) * groups;
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

// ---- what becomes of a finished row: where it goes, and V of its sums ----

template <class T>
struct Store {  // out[rows][width]
  static constexpr bool kRest = true;  // the other rows are zeroed
  T* out;

  __device__ __forceinline__ int64_t place(uint32_t row, int64_t, int64_t) const { return row; }
  template <int V>
  __device__ __forceinline__ void put(int64_t at, const float (&sum)[V]) const {
    Vec<T, V> v;
#pragma unroll
    for (int j = 0; j < V; ++j) v.v[j] = from_float<T>(sum[j]);
    *reinterpret_cast<Vec<T, V>*>(out + at) = v;
  }
};

template <int V>
__device__ __forceinline__ void put(float* to, const float (&sum)[V]);

struct Keep {  // sums[slot][width]; slots[row] = slot + 1
  static constexpr bool kRest = false;
  float* sums;
  int32_t* slots;
  bool by_row;  // a slot for each row, else for each token

  __device__ __forceinline__ int64_t place(uint32_t row, int64_t token, int64_t column) const {
    const int64_t slot = by_row ? int64_t(row) : token;
    if (column == 0) slots[row] = int32_t(slot + 1);
    return slot;
  }
  template <int V>
  __device__ __forceinline__ void put(int64_t at, const float (&sum)[V]) const {
    sums::put<V>(sums + at, sum);
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

template <int V, class S>
__device__ __forceinline__ void add(const float* from, S (&sum)[V]) {
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

template <int V>
__device__ __forceinline__ void scale(float (&sum)[V], float factor) {
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] *= factor;
}

// A vector that is read once.
template <class T, int V>
__device__ __forceinline__ Vec<T, V> read_once(const T* from) {
  Vec<T, V> v;
  constexpr int kBytes = V * sizeof(T);
  static_assert(kBytes == 16 || kBytes == 4 || kBytes == 2, "vectors of 16 bytes, or one element");
  if constexpr (kBytes == 16)
    *reinterpret_cast<uint4*>(&v) = __ldcs(reinterpret_cast<const uint4*>(from));
  else if constexpr (kBytes == 4)
    *reinterpret_cast<unsigned*>(&v) = __ldcs(reinterpret_cast<const unsigned*>(from));
  else
    *reinterpret_cast<unsigned short*>(&v) = __ldcs(reinterpret_cast<const unsigned short*>(from));
  return v;
}

// Which of the rows first to first + 31 the order names (bits). The warp looks
// up where the 32 rows begin and end with 32 probes a step, both at once (four
// steps for a million tokens, where a lane alone takes twenty), and then reads
// what lies between.
__device__ inline unsigned named_rows(int64_t n, const uint2* order, int64_t first) {
  const int lane = threadIdx.x & 31;
  int64_t low[2] = {0, 0}, high[2] = {n, n};
  while (high[0] > low[0] || high[1] > low[1]) {
    int64_t probe[2];
    uint32_t key[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t length = high[e] - low[e];
      probe[e] = length > 32 ? low[e] + length * (lane + 1) / 33 : low[e] + lane;
      key[e] = probe[e] < high[e] ? order[probe[e]].x : kNoRow;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int less = __popc(__ballot_sync(~0u, key[e] < first + 32 * e));
      const int64_t last = __shfl_sync(~0u, probe[e], less > 0 ? less - 1 : 0);
      const int64_t next = __shfl_sync(~0u, probe[e], less < 32 ? less : 31);
      if (high[e] - low[e] > 32) {
        if (less < 32) high[e] = next;
        if (less > 0) low[e] = last + 1;
      } else {
        low[e] = high[e] = low[e] + less;
      }
    }
  }
  unsigned named = 0;
  if (low[1] - low[0] <= 1024) {
    for (int64_t i = low[0] + lane; i < low[1]; i += 32)
      named |= 1u << (unsigned(order[i].x - first) & 31);
  } else {
    int64_t from = low[0], to = low[1];
    while (from < to) {
      const int64_t middle = (from + to) / 2;
      if (order[middle].x < first + lane) from = middle + 1;
      else to = middle;
    }
    if (from < low[1] && order[from].x == first + lane) named = 1u << lane;
  }
  return __reduce_or_sync(~0u, named);
}

// Rows that no token names: a gradient of zero. One warp takes 32 rows and one
// slice of columns.
template <int V, class End>
__device__ void write_rest(int64_t n, int64_t rows, int64_t width, const uint2* order,
                           const End& end) {
  const int64_t job = (blockIdx.x * int64_t(kThreads) + threadIdx.x) / 32;
  const int64_t slices = (width + 32 * V - 1) / (32 * V);
  const int64_t first = job / slices * 32;
  if (first >= rows) return;
  const int lane = threadIdx.x & 31;
  unsigned left = ~named_rows(n, order, first);
  if (rows - first < 32) left &= (1u << (rows - first)) - 1;
  const float zero[V] = {};
  const int64_t vectors = width / V;
  if (vectors <= 16) {  // several rows at once
    int lanes = 1;
    while (lanes < vectors) lanes *= 2;
    const int column = lane % lanes;
    for (int r = lane / lanes; r < 32; r += 32 / lanes)
      if ((left >> r & 1) && column < vectors)
        end.template put<V>((first + r) * width + column * V, zero);
    return;
  }
  const int64_t column = (job % slices * 32 + lane) * V;
  if (column >= width) return;
  while (left) {
    end.template put<V>((first + __ffs(left) - 1) * width + column, zero);
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
// vector of the rows without tokens. kLoose: vectors of four elements that may
// begin anywhere and end behind the row, moved one by one (for dropout on odd
// rows: single elements would draw four words for every one they use).
template <class T, int V, int C, int R, bool kDrop, bool kLoose, class End>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(C * V, C * V * sizeof(T)))
    sum_kernel(const __grid_constant__ Args<T> a, const End end) {
  wait_before();
  if constexpr (End::kRest) {
    if (blockIdx.x < a.rest) {
      write_rest<R, End>(a.n, a.rows, a.width, a.order, end);
      return;
    }
  }
  __shared__ uint2 entries[kMostTokens + 2];
  __shared__ __align__(16) float heads[C * kThreads * V];
  __shared__ unsigned char kinds[kThreads];

  const unsigned long long offset = kDrop ? mask_offset(a.mask) : 0;
  const int64_t job = blockIdx.x - a.rest;
  const int64_t block = job / a.cut.slices;
  const int lane = threadIdx.x % a.cut.lanes, group = threadIdx.x / a.cut.lanes;
  const int groups = kThreads / a.cut.lanes;
  // This lane's columns: `column` and C - 1 more, `apart` from each other.
  const int apart = a.cut.lanes * V;
  const int64_t column = (job - block * a.cut.slices) * (apart * C) + lane * V;
  // How many elements of each vector there are (all or none unless kLoose).
  int live[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int64_t left = a.width - column - c * apart;
    live[c] = left >= V ? V : left > 0 ? int(left) : 0;
  }
  const int64_t first = block * a.cut.block;
  const int count = int(a.n - first < a.cut.block ? a.n - first : a.cut.block);
  // Entries of the block and one on each side (kNoRow past the list's ends). A
  // list that no sort has made must not lead anywhere else: positions are held
  // in range here, rows where sums are handed on.
  for (int i = threadIdx.x; i < count + 2; i += kThreads) {
    const int64_t at = first + i - 1;
    uint2 one = at >= 0 && at < a.n ? a.order[at] : make_uint2(kNoRow, 0);
    if (one.y >= a.n) one.y = 0;
    entries[i] = one;
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
  auto done = [&](int i) {  // i: a token of the row
    if (row >= a.rows) return;
    const int64_t at = end.place(row, first + i, column) * a.width + column;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (live[c]) {
        scale<V>(sum[c], a.factor);
        if constexpr (kLoose) {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (j < live[c]) end.template put<1>(at + c * apart + j, {sum[c][j]});
        } else {
          end.template put<V>(at + c * apart, sum[c]);
        }
      }
  };
  auto put_head = [&] {
#pragma unroll
    for (int c = 0; c < C; ++c) put<V>(heads + (c * kThreads + threadIdx.x) * V, sum[c]);
  };
  reset();
  bool before = begin < stop && entry[begin - 1].x == row;
  Head kind = kNone;

  auto add_terms = [&](uint32_t position, const Vec<T, V> (&g)[C]) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      bool keep[V];
      const uint64_t element = uint64_t(position * a.width + column + c * apart);
      if constexpr (kDrop && kLoose) mask_four(a.mask, offset, element, keep);
      else if constexpr (kDrop) mask_vector<V>(a.mask, offset, element, keep);
#pragma unroll
      for (int j = 0; j < V; ++j)
        sum[c][j] += !kDrop || keep[j] ? to_float(g[c].v[j]) : 0.f;
    }
  };

  const T* grad = a.grad + column;
  constexpr int U = rows_at_once(C * V * sizeof(T), kLoose);
  for (int i = begin; i < stop; i += U) {
    uint2 token[U];
    Vec<T, V> g[U][C];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u < stop) {
        token[u] = entry[i + u];
        const T* from = grad + token[u].y * a.stride;
#pragma unroll
        for (int c = 0; c < C; ++c)
          if constexpr (kLoose) {
#pragma unroll
            for (int j = 0; j < V; ++j)
              if (j < live[c]) g[u][c].v[j] = from[c * apart + j];
          } else if (live[c]) {
            g[u][c] = read_once<T, V>(from + c * apart);
          }
      }
    if (i + U <= stop && token[U - 1].x == row) {  // all of one row, which is the current one
#pragma unroll
      for (int u = 0; u < U; ++u) add_terms(token[u].y, g[u]);
      continue;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u < stop) {
        if (token[u].x != row) {  // hand the row before on
          if (before) {
            put_head();
            kind = kEnded;
            before = false;
          } else {
            done(i + u - 1);
          }
          row = token[u].x;
          reset();
        }
        add_terms(token[u].y, g[u]);
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
      done(stop - 1);
    }
  }
  if (lane == 0) kinds[group] = kind;
  __syncthreads();
  // Adds the heads from group `from` on; true if the last is open. Eight at a
  // time among themselves: of a long row's additions those to the large partial
  // sums lose the most.
  auto join = [&](int from) {
    bool open = true;
    float part[C][V];
    auto pass_on = [&] {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) sum[c][j] += part[c][j], part[c][j] = 0.f;
    };
#pragma unroll
    for (int c = 0; c < C; ++c) clear<V>(part[c]);
    for (int h = from; h < groups && open; ++h) {
#pragma unroll
      for (int c = 0; c < C; ++c)
        add<V>(heads + (c * kThreads + h * a.cut.lanes + lane) * V, part[c]);
      open = kinds[h] == kOpen;
      if ((h - from) % 8 == 7) pass_on();
    }
    pass_on();
    return open;
  };
  auto put_partial = [&](int64_t which) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (live[c]) {
        float* to = a.partial + which * a.width + column + c * apart;
        if constexpr (kLoose) {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (j < live[c]) to[j] = sum[c][j];
        } else {
          put<V>(to, sum[c]);
        }
      }
  };
  if (continued) {
    if (join(group + 1)) put_partial(2 * block + 1);
    else done(stop - 1);
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
// order. Bound by latency: what decides is loaded at once.
template <class T, int V, class End>
__global__ void __launch_bounds__(kThreads)
    join_kernel(const __grid_constant__ Args<T> a, int lanes, int64_t slices, const End end) {
  __shared__ double shares[V][kThreads];
  wait_before();
  const unsigned block = blockIdx.x / unsigned(slices);
  const int64_t first = int64_t(block) * a.cut.block, stop = first + a.cut.block;
  if (stop >= a.n) return;
  // The row that is open behind this block, and the rows that the next blocks
  // begin with.
  int64_t at = stop + int64_t(threadIdx.x) * a.cut.block;
  const uint32_t row = a.order[stop - 1].x;
  const uint32_t earlier = first > 0 ? a.order[first - 1].x : kNoRow;
  uint32_t begins = at < a.n ? a.order[at].x : kNoRow;
  if (row >= a.rows || earlier == row) return;  // none, or begun earlier
  int heads = 0;
  for (;;) {
    const int more = __syncthreads_count(begins == row);
    heads += more;
    if (more < kThreads) break;
    at += int64_t(kThreads) * a.cut.block;
    begins = at < a.n ? a.order[at].x : kNoRow;
  }
  if (heads == 0) return;
  const int lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
  const int groups = kThreads / lanes;
  const int64_t column = (int64_t(blockIdx.x - block * unsigned(slices)) * lanes + lane) * V;
  const bool live = column < a.width;
  const float* partial = a.partial + 2 * int64_t(block) * a.width + column;
  double wide[V] = {};
  const int sharing = heads < groups ? heads : groups;
  if (live && group < sharing) {
    if (group == 0) add<V>(partial + a.width, wide);
    const int each = heads / sharing, more = heads % sharing;  // the first ones take one more
    const int from = group * each + (group < more ? group : more);
    const int to = from + each + (group < more ? 1 : 0);
#pragma unroll 4
    for (int h = from; h < to; ++h) add<V>(partial + 2 * int64_t(1 + h) * a.width, wide);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) shares[j][threadIdx.x] = wide[j];
  __syncthreads();
  if (group > 0 || !live) return;
  for (int g = 1; g < sharing; ++g)
#pragma unroll
    for (int j = 0; j < V; ++j) wide[j] += shares[j][g * lanes + lane];
  float sum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = float(wide[j]);
  scale<V>(sum, a.factor);
  end.template put<V>(end.place(row, stop - 1, column) * a.width + column, sum);
}

// The launch without any token.
template <int R, class End>
__global__ void __launch_bounds__(kThreads)
    rest_kernel(int64_t rows, int64_t width, const End end) {
  wait_before();
  write_rest<R, End>(0, rows, width, nullptr, end);
}

// ---- Adam ----

struct Adam {
  float *table, *first, *second;
  float step;
  double inv_bias2;
};

// Vectors of W elements of the table, U of them a thread, all loaded before the
// first is updated. slots null: no token at all. Bound by memory: six streams
// of the table's size.
template <class Division, int W, int U>
__global__ void __launch_bounds__(kThreads)
    adam_kernel(typename Division::Number total, const Division vectors, int64_t width,
                const int32_t* slots, const float* sums, const Adam a) {
  wait_before();
  using Number = typename Division::Number;
  using F = Vec<float, W>;
  const Number first = Number(blockIdx.x) * (U * kThreads) + threadIdx.x;
  F p[U], m[U], v[U], g[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Number at = first + u * kThreads;
    if (at < total) {
      const Number row = vectors.quotient(at);
      const int32_t slot = slots ? slots[row] : 0;
      p[u] = reinterpret_cast<const F*>(a.table)[at];
      m[u] = reinterpret_cast<const F*>(a.first)[at];
      v[u] = reinterpret_cast<const F*>(a.second)[at];
      g[u] = {};
      if (slot > 0)
        g[u] = *reinterpret_cast<const F*>(sums + int64_t(slot - 1) * width +
                                           int64_t(at - row * vectors.divisor) * W);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Number at = first + u * kThreads;
    if (at >= total) return;
#pragma unroll
    for (int j = 0; j < W; ++j)
      torch_adam(p[u].v[j], m[u].v[j], v[u].v[j], g[u].v[j], a.step, a.inv_bias2);
    reinterpret_cast<F*>(a.table)[at] = p[u];
    reinterpret_cast<F*>(a.first)[at] = m[u];
    reinterpret_cast<F*>(a.second)[at] = v[u];
  }
}

// ---- few tokens, small tables ----

// One launch for all of it: what counts at these sizes is the host's time for
// each launch (2.3 us) and the workspace. Every block ranks the few tokens by
// comparing each with all, then eight lanes share the tokens of a vector of the
// table and add up in a fixed tree, in 32 bits (32 terms a lane at most and three
// joins: 35 roundings). A call on 37 tokens and 1000 x 45 f32 takes
// 11 us instead of 17, Adam of 60 x 48 with 184 tokens 13 instead of 22.
//
// The GPU's time must stay below the host's as well: at 128 tokens 5 us for 1365
// x 48 and 7 for 64 x 1024 (10 and 10 in two launches), at 256 tokens 5 to 8 us for
// 50 x 48 (7 to 8) but 12 for 1365 x 48 (11) and 14 for 64 x 1024 (11), at 512 tokens
// 17 for a single row of 16 (10).
constexpr int kFewTokens = 256;
constexpr int kFewThreads = 256;
constexpr int64_t kSmallTable = int64_t(1) << 16;  // elements
constexpr int64_t kSmallWork = int64_t(1) << 23;   // tokens x elements
constexpr int kSharing = 8;

inline bool few(int64_t n, int64_t rows, int64_t width) {
  return n > 0 && n <= kFewTokens && rows * width <= kSmallTable && n * rows * width <= kSmallWork;
}

// Adam as what becomes of a row's sums.
struct Update {
  Adam adam;

  template <int V>
  __device__ __forceinline__ void put(int64_t at, const float (&sum)[V]) const {
    constexpr int W = V < 4 ? V : 4;
#pragma unroll
    for (int h = 0; h < V; h += W) {
      auto* p = reinterpret_cast<Vec<float, W>*>(adam.table + at + h);
      auto* m = reinterpret_cast<Vec<float, W>*>(adam.first + at + h);
      auto* v = reinterpret_cast<Vec<float, W>*>(adam.second + at + h);
      Vec<float, W> pv = *p, mv = *m, vv = *v;
#pragma unroll
      for (int j = 0; j < W; ++j)
        torch_adam(pv.v[j], mv.v[j], vv.v[j], sum[h + j], adam.step, adam.inv_bias2);
      *p = pv;
      *m = mv;
      *v = vv;
    }
  }
};

// total: vectors of the table. The tokens come from a.order if it is given, else
// from index.
template <class T, int V, bool kDrop, class End>
__global__ void __launch_bounds__(kFewThreads)
    few_kernel(const __grid_constant__ Args<T> a, const tokens::Index index, uint32_t total,
               const Narrow vectors, const End end) {
  wait_before();
  __shared__ uint2 sorted[kFewTokens];
  __shared__ uint32_t keys[kFewTokens];
  const int n = int(a.n), me = threadIdx.x;
  if (a.order) {
    if (me < n) {
      uint2 one = a.order[me];
      if (one.y >= a.n) one.y = 0;  // see sum_kernel
      sorted[me] = one;
    }
  } else {
    bool bad = false;
    const uint32_t key =
        me < n ? tokens::row_of(index, tokens::raw_index(index, me), &bad) : kNoRow;
    tokens::report(index, bad);
    if (me < n) keys[me] = key;
    __syncthreads();
    if (me < n) {
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += keys[j] < key || (keys[j] == key && j < me);
      sorted[rank] = make_uint2(key, uint32_t(me));
    }
  }
  __syncthreads();
  const unsigned long long offset = kDrop ? mask_offset(a.mask) : 0;
  auto before = [&](uint32_t row) {  // tokens in front of a row's
    int low = 0, high = n;
    while (low < high) {
      const int middle = (low + high) / 2;
      if (sorted[middle].x < row) low = middle + 1;
      else high = middle;
    }
    return low;
  };
  const int share = me % kSharing;
  constexpr uint32_t kVectors = kFewThreads / kSharing;  // of a block at once
  for (uint32_t first = blockIdx.x * kVectors; first < total; first += gridDim.x * kVectors) {
    const uint32_t at = first + me / kSharing;
    const uint32_t row = vectors.quotient(at);
    const int64_t column = int64_t(at - row * vectors.divisor) * V;
    const bool real = at < total;
    float sum[V];
    clear<V>(sum);
    const int stop = real ? before(row + 1) : 0;
#pragma unroll 4
    for (int i = (real ? before(row) : 0) + share; i < stop; i += kSharing) {
      const uint32_t position = sorted[i].y;
      const Vec<T, V> g = read_once<T, V>(a.grad + position * a.stride + column);
      bool keep[V];
      if constexpr (kDrop)
        mask_vector<V>(a.mask, offset, uint64_t(position * a.width + column), keep);
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += !kDrop || keep[j] ? to_float(g.v[j]) : 0.f;
    }
#pragma unroll
    for (int o = 1; o < kSharing; o *= 2)
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += __shfl_xor_sync(~0u, sum[j], o);
    if (real && share == 0) {
      scale<V>(sum, a.factor);
      end.template put<V>(row * a.width + column, sum);
    }
  }
}

template <class T, int V, class End>
cudaError_t run_few_vectors(const Args<T>& a, const tokens::Index& index, const End& end,
                            bool drop, cudaStream_t stream) {
  const int64_t vectors = a.width / V, total = a.rows * vectors;
  const int64_t blocks = (total + kFewThreads / kSharing - 1) / (kFewThreads / kSharing);
  auto* kernel = drop ? few_kernel<T, V, true, End> : few_kernel<T, V, false, End>;
  return launch_after(kernel, unsigned(std::min<int64_t>(blocks, kSms * 6)), kFewThreads, 0, stream,
                      a, index, uint32_t(total), Narrow(vectors), end);
}

template <class T>
bool aligned(const Args<T>& a) {
  return common_bytes(uint64_t(a.width * sizeof(T)) | uint64_t(a.stride * sizeof(T)) |
                      uint64_t(a.grad)) == 16;
}

template <class T, class End>
cudaError_t run_few(const Args<T>& a, const tokens::Index& index, const End& end, bool whole,
                    bool drop, cudaStream_t stream) {
  return whole && aligned(a) ? run_few_vectors<T, 16 / sizeof(T)>(a, index, end, drop, stream)
                             : run_few_vectors<T, 1>(a, index, end, drop, stream);
}

// ---- host ----

// Vectors of a lane: one, three or four floats' vectors, one or two of 16-bit
// elements (16 running sums a lane at most): the most that leave few lanes
// idle, unless the rows are so few that the groups would not fill the GPU (kernels
// alone, bf16: 128000 rows of 256 18 us, 20 if four times as many were asked for;
// 128000 rows of 48 9.7, 11.4 if a quarter was enough).
inline int vectors_of_lane(int64_t n, int64_t width, int vec, bool floats) {
  const int64_t vectors = (width + vec - 1) / vec;
  const int more = floats ? 4 : 2, other = floats ? 3 : 1;
  int64_t one, some, most;
  lanes_of(vectors, 1, &one);
  lanes_of(vectors, other, &some);
  lanes_of(vectors, more, &most);
  const int64_t least = std::min(one, std::min(some, most));
  auto fills = [&](int c, int64_t padded) {
    return close_to(padded, least) && n * (padded / c) >= int64_t(kSms) * 512 * kLeastTokens;
  };
  if (fills(more, most)) return more;
  return fills(other, some) ? other : 1;
}

template <class T, int V, int C, int R, bool kDrop, bool kLoose, class End>
cudaError_t run_cut(Args<T> a, const End& end, cudaStream_t stream) {
  a.rest = End::kRest ? rest_blocks(a.rows, a.width, R) : 0;
  a.cut = cut_of(a.n, a.width, V, C, blocks_per_sm(C * V, C * V * sizeof(T)), a.rest);
  const unsigned grid = unsigned(a.rest + a.cut.blocks * a.cut.slices);
  const cudaError_t e = launch_after(sum_kernel<T, V, C, R, kDrop, kLoose, End>, grid, kThreads, 0,
                                     stream, a, end);
  if (e != cudaSuccess || a.cut.blocks == 1) return e;
  constexpr int J = kLoose ? 1 : V;
  int64_t padded;
  const int lanes = lanes_of((a.width + J - 1) / J, 1, &padded);
  return launch_after(join_kernel<T, J, End>, unsigned(a.cut.blocks * (padded / lanes)), kThreads,
                      0, stream, a, lanes, padded / lanes, end);
}

template <class T, int V, int R, bool kDrop, class End>
cudaError_t run_vectors(const Args<T>& a, const End& end, cudaStream_t stream) {
  constexpr bool kFloats = sizeof(T) == 4;
  const int c = vectors_of_lane(a.n, a.width, V, kFloats);
  if (c == 1) return run_cut<T, V, 1, R, kDrop, false, End>(a, end, stream);
  if constexpr (kFloats)
    return c == 3 ? run_cut<T, V, 3, R, kDrop, false, End>(a, end, stream)
                  : run_cut<T, V, 4, R, kDrop, false, End>(a, end, stream);
  else
    return run_cut<T, V, 2, R, kDrop, false, End>(a, end, stream);
}

template <class T, int V, int R, class End>
cudaError_t run_sums(const Args<T>& a, const End& end, bool drop, cudaStream_t stream) {
  if (!drop) return run_vectors<T, V, R, false, End>(a, end, stream);
  if constexpr (V == 1) return run_cut<T, 4, 1, R, true, true, End>(a, end, stream);
  else return run_vectors<T, V, R, true, End>(a, end, stream);
}

// Vectors are 16 bytes where the rows of all arrays begin on 16, else single
// elements.
template <class T>
cudaError_t gradient(const Args<T>& a, const tokens::Index& index, T* out, bool drop,
                     cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const Store<T> end{out};
  const bool whole = common_bytes(uint64_t(a.width * sizeof(T)) | uint64_t(out)) == 16;
  if (few(a.n, a.rows, a.width)) return run_few(a, index, end, whole, drop, stream);
  if (a.n == 0) {
    auto* kernel = whole ? rest_kernel<V, Store<T>> : rest_kernel<1, Store<T>>;
    return launch_after(kernel, unsigned(rest_blocks(a.rows, a.width, whole ? V : 1)), kThreads, 0,
                        stream, a.rows, a.width, end);
  }
  if (!whole) return run_sums<T, 1, 1>(a, end, drop, stream);
  return aligned(a) ? run_sums<T, V, V>(a, end, drop, stream)
                    : run_sums<T, 1, V>(a, end, drop, stream);
}

// Workspace of the partial sums for any cut of these sizes: a group has
// kLeastTokens at least, a block at least a group for each 32 lanes.
inline size_t partial_bytes(int64_t n, int64_t width) {
  const int64_t least = kThreads / 32 * kLeastTokens;
  const size_t bytes = size_t(2 * ((n + least - 1) / least)) * width * sizeof(float);
  return (bytes + 15) / 16 * 16;
}

// ... and of Adam: a slot number for each row, sums for the rows that tokens
// name (no more than rows, nor than tokens).
inline size_t slot_bytes(int64_t rows) { return (size_t(rows) * sizeof(int32_t) + 15) / 16 * 16; }

inline size_t workspace_bytes(int64_t n, int64_t rows, int64_t width, bool consume) {
  if (n == 0 || few(n, rows, width)) return 0;
  if (!consume) return partial_bytes(n, width);
  return partial_bytes(n, width) + slot_bytes(rows) +
         size_t(std::min(n, rows)) * width * sizeof(float);
}

template <class Division, int W>
cudaError_t run_adam(int64_t rows, int64_t width, const int32_t* slots, const float* sums,
                     const Adam& adam, cudaStream_t stream) {
  constexpr int U = 2;
  const int64_t vectors = width / W, total = rows * vectors;
  return launch_after(adam_kernel<Division, W, U>,
                      unsigned((total + U * kThreads - 1) / (U * kThreads)), kThreads, 0, stream,
                      typename Division::Number(total), Division(vectors), width, slots, sums,
                      adam);
}

// Where the Adam pass finds the sums: behind the partial ones in the workspace.
struct Kept {
  int32_t* slots;
  float* sums;

  Kept(float* partial, int64_t n, int64_t rows, int64_t width) {
    char* at = reinterpret_cast<char*>(partial) + partial_bytes(n, width);
    slots = reinterpret_cast<int32_t*>(at);
    sums = reinterpret_cast<float*>(at + slot_bytes(rows));
  }
  // No row has a slot. Comes first of a call's work: in between it would keep
  // the kernels behind it from starting early.
  cudaError_t clear(int64_t rows, cudaStream_t stream) const {
    return cudaMemsetAsync(slots, 0, size_t(rows) * sizeof(int32_t), stream);
  }
};

template <class T>
cudaError_t consume(const Args<T>& a, const tokens::Index& index, const Adam& adam, bool drop,
                    cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool whole = common_bytes(uint64_t(a.width * sizeof(float)) | uint64_t(adam.table) |
                                  uint64_t(adam.first) | uint64_t(adam.second)) == 16;
  if (few(a.n, a.rows, a.width)) return run_few(a, index, Update{adam}, whole, drop, stream);
  const Kept kept(a.partial, a.n, a.rows, a.width);
  if (a.n > 0) {
    const Keep end{kept.sums, kept.slots, a.rows <= a.n};
    const cudaError_t e = aligned(a) ? run_sums<T, V, 1>(a, end, drop, stream)
                                     : run_sums<T, 1, 1>(a, end, drop, stream);
    if (e != cudaSuccess) return e;
  }
  const bool narrow = Narrow::fits(a.rows * a.width + 2 * kThreads);
  auto* run = whole ? (narrow ? run_adam<Narrow, 4> : run_adam<Wide, 4>)
                    : (narrow ? run_adam<Narrow, 1> : run_adam<Wide, 1>);
  return run(a.rows, a.width, a.n > 0 ? kept.slots : nullptr, kept.sums, adam, stream);
}

// The kernels of each element type are compiled in a file of their own.
#define CLAD3DGS_ROW_SUMS(prefix, T)                                                      \
  prefix template cudaError_t gradient<T>(const Args<T>&, const tokens::Index&, T*, bool,  \
                                          cudaStream_t);                                   \
  prefix template cudaError_t consume<T>(const Args<T>&, const tokens::Index&, const Adam&, \
                                         bool, cudaStream_t);

}  // namespace sums
}  // namespace clad3dgs
