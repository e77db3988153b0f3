// Stable order of tokens by the table row they name: (row, position) pairs
// sorted by row, positions ascending within a row. Tokens that name no row
// (padding, or an index outside the table) get the row number `rows` and so
// come last.
//
// Least-significant-digit radix sort. Ranks come from the lanes of a warp that
// hold equal digits, in token order, so the sort is stable and the order the
// same on every run.
//
// Up to kSmall tokens: one cluster of up to eight blocks sorts in shared memory,
// all passes in one launch; blocks read each other's digit counts and scatter
// into each other's tiles. More: two kernels a pass; every block (one an SM at
// most) counts the digits of a contiguous share of the tokens, then adds up
// the other blocks' counts itself (they lie in L2) and scatters its share tile
// by tile. Bound by latency at these sizes: everything a thread reads of a tile
// is asked for before any of it is used. 16384 tokens over 131072 rows: 14 us
// (one block took 37, six kernels over four tiles 66); 1.1M tokens over 4096
// rows, two passes: 33 us, of which counting 5.5 + 4 and scattering 16 + 12,
// half of that the launches, loads and barriers and a quarter each the ranks
// and the scattered stores. With eight tokens a thread scattering spills 32 bytes a
// thread: blocks of 1024 leave 64 registers each.
#pragma once
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "launch.cuh"
#include "token_index.cuh"

namespace clad3dgs {
namespace tokens {

// The tokens at `at(j)`, j < I, where that is below n: from the caller's indices
// in the first pass, else from the pass before.
template <int I, class At>
__device__ __forceinline__ void load_pairs(const Index& index, const uint2* from, int64_t n, At at,
                                           uint2 (&pair)[I]) {
  if (from) {
#pragma unroll
    for (int j = 0; j < I; ++j)
      if (at(j) < n) pair[j] = from[at(j)];
    return;
  }
  int64_t raw[I];
#pragma unroll
  for (int j = 0; j < I; ++j) raw[j] = at(j) < n ? raw_index(index, at(j)) : 0;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < I; ++j)
    if (at(j) < n) pair[j] = make_uint2(row_of(index, raw[j], &bad), uint32_t(at(j)));
  report(index, bad);
}

// Ranks of a tile: thread t of warp w holds the tokens w * 32 * I + 32 * j + lane,
// j < I, the first `count` of the tile being real. bins: [warps][digits], zero
// on entry; afterwards the tokens of each warp and digit. rank: how many tokens
// of the same warp and digit stand before.
template <int I>
__device__ __forceinline__ void rank_tile(const uint2 (&pair)[I], int count, int shift, int bits,
                                          uint16_t* bins, uint32_t (&rank)[I]) {
  const int digits = 1 << bits;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint16_t* mine = bins + warp * digits;
  const int base = warp * 32 * I + lane;
  // Lanes with an equal digit, by one ballot a bit (a match instruction took
  // half as long again: 53 us against 37 for 16384 tokens in one block).
  uint32_t same[I];
#pragma unroll
  for (int j = 0; j < I; ++j) same[j] = __ballot_sync(~0u, base + 32 * j < count);
  for (uint32_t bit = 1u << shift, end = bit << bits; bit != end; bit <<= 1) {
#pragma unroll
    for (int j = 0; j < I; ++j) {
      const bool set = (pair[j].x & bit) != 0;
      const uint32_t lanes = __ballot_sync(~0u, set);
      same[j] &= set ? lanes : ~lanes;
    }
  }
#pragma unroll
  for (int j = 0; j < I; ++j) {
    const uint32_t digit = (pair[j].x >> shift) & (digits - 1);
    const uint32_t below = __popc(same[j] & ((1u << lane) - 1));
    uint32_t before = 0;
    if (base + 32 * j < count) {
      before = mine[digit];
      rank[j] = before + below;
    }
    __syncwarp();
    if (base + 32 * j < count && below == 0) mine[digit] = uint16_t(before + __popc(same[j]));
    __syncwarp();
  }
}

// Exclusive sum over the block's threads of one value each; sums: one a warp.
__device__ __forceinline__ uint32_t exclusive_sum(uint32_t value, uint32_t* sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t inclusive = value;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t below = __shfl_up_sync(~0u, inclusive, o);
    if (lane >= o) inclusive += below;
  }
  if (lane == 31) sums[warp] = inclusive;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < warp; ++w) before += sums[w];
  return before + inclusive - value;
}

inline int key_bits(int64_t rows) {  // of the keys 0 to rows
  int bits = 1;
  while (bits < 32 && (rows >> bits) != 0) ++bits;
  return bits;
}

// A little memory to be zeroed by the way, in vectors of 16 bytes: saves the
// launch (2 us) where a later kernel needs it.
struct Fill {
  uint4* to = nullptr;
  int64_t vectors = 0;

  __device__ __forceinline__ void run() const {
    for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < vectors;
         i += int64_t(gridDim.x) * blockDim.x)
      to[i] = make_uint4(0, 0, 0, 0);
  }
};

// Digits have nine bits at most: with 10 or 11 a pass less is needed for some
// tables, but costs more than it saves (1.1M tokens over 2000 rows 31 us in two
// passes, 41 in one; over a million rows 50 in three, 55 in two).
constexpr int kDigitBits = 9;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;

// Shared memory of the counts by digit (two sums, and one count a warp).
constexpr size_t digit_bytes(int bits) {
  return (size_t(1) << bits) * (kSortWarps * sizeof(uint16_t) + 2 * sizeof(uint32_t));
}

// Lets a kernel have the most that any launch of it asks for. The limit belongs
// to the kernel, not to a launch: one that followed the launch's own digits
// would lower it between another host thread's setting and launch.
template <class Kernel>
cudaError_t allow_shared(Kernel* kernel, size_t most) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(most));
}

// ---- one cluster ----

constexpr int kMostBlocks = 8;  // of a cluster
// Up to here the cluster is as fast as many blocks or faster (32000 tokens over
// 4096 rows 13.6 against 15.6 us, 65000 tokens 21.4 against 16.1) and takes
// fewer launches.
constexpr int kSmall = kMostBlocks * kSortThreads * 4;

// Block r of the cluster holds the tokens [r * tile, (r + 1) * tile) of the list
// as sorted so far, tile = I * kSortThreads.
template <int I>
__global__ void __launch_bounds__(kSortThreads)
    cluster_sort_kernel(int n, Index index, int passes, int bits, uint2* __restrict__ order,
                        const Fill fill) {
  wait_before();
  fill.run();
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = int(cluster.num_blocks()), me = int(cluster.block_rank());
  constexpr int kTile = I * kSortThreads;
  extern __shared__ __align__(16) char shared[];
  const int digits = 1 << bits;
  uint2* pairs = reinterpret_cast<uint2*>(shared);                    // [tile]
  uint32_t* counts = reinterpret_cast<uint32_t*>(pairs + kTile);      // [digits]
  uint32_t* starts = counts + digits;                                 // [digits]
  uint16_t* bins = reinterpret_cast<uint16_t*>(starts + digits);      // [warps][digits]
  __shared__ uint32_t sums[kSortWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int base = warp * 32 * I + lane;
  const int first = me * kTile;
  const int count = n - first < kTile ? n - first : kTile;
  uint2 pair[I];
  uint32_t rank[I];
  load_pairs<I>(index, nullptr, n, [&](int j) { return int64_t(first + base + 32 * j); }, pair);
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    for (int d = threadIdx.x; d < kSortWarps * digits / 2; d += kSortThreads)
      reinterpret_cast<uint32_t*>(bins)[d] = 0;
    __syncthreads();
    rank_tile<I>(pair, count, shift, bits, bins, rank);
    __syncthreads();
    // Each warp's tokens of a digit among the block's.
    const int d = threadIdx.x;
    if (d < digits) {
      uint32_t total = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = bins[w * digits + d];
        bins[w * digits + d] = uint16_t(total);
        total += c;
      }
      counts[d] = total;
    }
    cluster.sync();  // all counts are there, and all tiles are in registers
    uint32_t all = 0, front = 0;
    if (d < digits) {
      for (int r = 0; r < blocks; ++r) {
        const uint32_t c = cluster.map_shared_rank(counts, r)[d];
        all += c;
        if (r < me) front += c;
      }
    }
    const uint32_t start = exclusive_sum(all, sums);
    if (d < digits) starts[d] = start + front;
    __syncthreads();
    const bool last = pass + 1 == passes;
#pragma unroll
    for (int j = 0; j < I; ++j)
      if (base + 32 * j < count) {
        const uint32_t digit = (pair[j].x >> shift) & (digits - 1);
        const uint32_t at = starts[digit] + bins[warp * digits + digit] + rank[j];
        if (last) order[at] = pair[j];
        else cluster.map_shared_rank(pairs, at / kTile)[at % kTile] = pair[j];
      }
    cluster.sync();  // the tiles are complete, and nobody reads a block that is gone
    if (last) break;
#pragma unroll
    for (int j = 0; j < I; ++j)
      if (base + 32 * j < count) pair[j] = pairs[base + 32 * j];
  }
}

// Tokens of a thread, and blocks: as many blocks as give each thread one token,
// then more tokens a thread.
inline int cluster_items(int64_t n) { return n <= kSmall / 4 ? 1 : n <= kSmall / 2 ? 2 : 4; }

inline unsigned cluster_blocks(int64_t n) {
  unsigned blocks = 1;
  while (int64_t(blocks) * cluster_items(n) * kSortThreads < n) blocks *= 2;
  return blocks;
}

template <int I>
cudaError_t cluster_sort(int64_t n, const Index& index, uint2* order, const Fill& fill,
                         cudaStream_t stream) {
  const int all = key_bits(index.rows);
  const int passes = (all + kDigitBits - 1) / kDigitBits, bits = (all + passes - 1) / passes;
  const unsigned blocks = cluster_blocks(n);
  constexpr size_t kTileBytes = size_t(I) * kSortThreads * sizeof(uint2);
  const size_t shared = kTileBytes + digit_bytes(bits);
  cudaError_t e = allow_shared(cluster_sort_kernel<I>, kTileBytes + digit_bytes(kDigitBits));
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attributes[2]{};
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = blocks;
  attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // as in launch_after
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3(kSortThreads);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  config.attrs = attributes;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, cluster_sort_kernel<I>, int(n), index, passes, bits, order,
                            fill);
}

// ---- many blocks ----

constexpr int kSortBlocks = 148;  // a number of its own: it sets the workspace's size

struct SortPlan {
  int items;         // tokens of a thread in a tile
  int passes, bits;  // digit width of every pass
  int blocks, tiles;  // blocks, and tiles of each
  size_t pair_bytes, count_bytes;  // workspace parts

  size_t bytes() const { return pair_bytes + count_bytes; }
};

inline SortPlan sort_plan(int64_t n, int64_t rows) {
  SortPlan p{};
  if (n <= kSmall) return p;
  const int all = key_bits(rows);
  p.passes = (all + kDigitBits - 1) / kDigitBits;
  p.bits = (all + p.passes - 1) / p.passes;
  // The smallest tiles that leave no block more than one (250000 tokens over 4096
  // rows: 20, 21 and 29 us with two, four and eight tokens a thread; 500000: 27, 26
  // and 31; 1.1M: 40, 36 and 33).
  const int64_t threads = int64_t(kSortBlocks) * kSortThreads;
  p.items = n <= threads * 2 ? 2 : n <= threads * 4 ? 4 : 8;
  const int64_t tiles = (n + kSortThreads * p.items - 1) / (kSortThreads * p.items);
  p.tiles = int((tiles + kSortBlocks - 1) / kSortBlocks);
  p.blocks = int((tiles + p.tiles - 1) / p.tiles);
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  p.pair_bytes = p.passes > 1 ? up(size_t(n) * sizeof(uint2)) : 0;
  p.count_bytes = up((size_t(1) << p.bits) * p.blocks * sizeof(uint32_t));
  return p;
}

// counts[block][digit]
template <int I>
__global__ void __launch_bounds__(kSortThreads)
    count_kernel(int64_t n, Index index, const uint2* from, int tiles, int shift,
                 int bits, uint32_t* __restrict__ counts, const Fill fill) {
  wait_before();
  fill.run();
  __shared__ uint32_t bins[1 << kDigitBits];
  const int digits = 1 << bits;
  for (int d = threadIdx.x; d < digits; d += kSortThreads) bins[d] = 0;
  __syncthreads();
  for (int t = 0; t < tiles; ++t) {
    const int64_t base = (int64_t(blockIdx.x) * tiles + t) * (kSortThreads * I) + threadIdx.x;
    uint2 pair[I];
    load_pairs<I>(index, from, n, [&](int j) { return base + j * kSortThreads; }, pair);
#pragma unroll
    for (int j = 0; j < I; ++j)
      if (base + j * kSortThreads < n) atomicAdd(&bins[(pair[j].x >> shift) & (digits - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads)
    counts[int64_t(blockIdx.x) * digits + d] = bins[d];
}

template <int I>
__global__ void __launch_bounds__(kSortThreads)
    scatter_kernel(int64_t n, Index index, const uint2* from, int tiles, int shift,
                   int bits, const uint32_t* counts, uint2* __restrict__ to) {
  wait_before();
  extern __shared__ __align__(16) char shared[];
  const int digits = 1 << bits;
  uint32_t* starts = reinterpret_cast<uint32_t*>(shared);               // [digits]
  uint32_t* earlier = starts + digits;                                  // [digits]
  uint16_t* bins = reinterpret_cast<uint16_t*>(earlier + digits);       // [warps][digits]
  __shared__ uint32_t sums[kSortWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Where this block's tokens of each digit begin: all smaller digits, then
  // this digit's tokens of the blocks in front.
  for (int d = threadIdx.x; d < 2 * digits; d += kSortThreads) starts[d] = 0;
  __syncthreads();
  const int parts = digits < kSortThreads ? kSortThreads / digits : 1;
  for (int d = threadIdx.x % digits; d < digits; d += kSortThreads) {
    uint32_t all = 0, front = 0;
#pragma unroll 8
    for (int b = threadIdx.x / digits % parts; b < int(gridDim.x); b += parts) {
      const uint32_t c = counts[int64_t(b) * digits + d];
      all += c;
      if (b < int(blockIdx.x)) front += c;
    }
    atomicAdd(&starts[d], all);
    atomicAdd(&earlier[d], front);
  }
  __syncthreads();
  const int each = (digits + kSortThreads - 1) / kSortThreads;
  uint32_t mine = 0;
  for (int k = 0; k < each; ++k) {
    const int d = threadIdx.x * each + k;
    if (d < digits) mine += starts[d];
  }
  uint32_t start = exclusive_sum(mine, sums);
  for (int k = 0; k < each; ++k) {
    const int d = threadIdx.x * each + k;
    if (d >= digits) break;
    const uint32_t c = starts[d];
    starts[d] = start + earlier[d];
    start += c;
  }
  for (int t = 0; t < tiles; ++t) {
    const int64_t first = (int64_t(blockIdx.x) * tiles + t) * (kSortThreads * I);
    if (first >= n) break;
    const int count = int(n - first < kSortThreads * I ? n - first : kSortThreads * I);
    const int base = warp * 32 * I + lane;
    uint2 pair[I];
    uint32_t rank[I];
    load_pairs<I>(index, from, n, [&](int j) { return first + base + 32 * j; }, pair);
    for (int d = threadIdx.x; d < kSortWarps * digits / 2; d += kSortThreads)
      reinterpret_cast<uint32_t*>(bins)[d] = 0;
    __syncthreads();
    rank_tile<I>(pair, count, shift, bits, bins, rank);
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kSortThreads) {
      uint32_t total = 0;
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = bins[w * digits + d];
        bins[w * digits + d] = uint16_t(total);
        total += c;
      }
      earlier[d] = total;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < I; ++j)
      if (base + 32 * j < count) {
        const uint32_t digit = (pair[j].x >> shift) & (digits - 1);
        to[starts[digit] + bins[warp * digits + digit] + rank[j]] = pair[j];
      }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kSortThreads) starts[d] += earlier[d];
    // (the next tile's first barrier orders these sums before their use)
  }
}

template <int I>
cudaError_t large_sort(int64_t n, const Index& index, const SortPlan& p, uint2* order,
                       void* workspace, const Fill& fill, cudaStream_t stream) {
  uint2* spare = static_cast<uint2*>(workspace);
  uint32_t* counts =
      reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + p.pair_bytes);
  const size_t shared = digit_bytes(p.bits);
  cudaError_t e = allow_shared(scatter_kernel<I>, digit_bytes(kDigitBits));
  if (e != cudaSuccess) return e;
  const uint2* from = nullptr;
  for (int pass = 0; pass < p.passes; ++pass) {
    // Alternating so that the last pass ends in `order`.
    uint2* to = (p.passes - 1 - pass) % 2 == 0 ? order : spare;
    const int shift = pass * p.bits;
    e = launch_after(count_kernel<I>, p.blocks, kSortThreads, 0, stream, n, index, from, p.tiles,
                     shift, p.bits, counts, pass == 0 ? fill : Fill{});
    if (e != cudaSuccess) return e;
    e = launch_after(scatter_kernel<I>, p.blocks, kSortThreads, shared, stream, n, index, from,
                     p.tiles, shift, p.bits, counts, to);
    if (e != cudaSuccess) return e;
    from = to;
  }
  return cudaSuccess;
}

// Whether the sort should clear `words` of memory by the way (Fill): its blocks
// are few, so up to 32768 words each and as many again (Adam's slots, whole calls:
// 300 tokens and 2^16 rows 22 us against 24 with a launch of its own, 2^18 rows 36
// against 24; 16000 tokens and 2^18 rows 33 against 34, 2^19 rows 38 against 36;
// 150000 tokens and 2^20 rows 54 against 57).
inline bool sort_clears(int64_t n, int64_t rows, int64_t words) {
  const int64_t blocks = n <= kSmall ? cluster_blocks(n) : sort_plan(n, rows).blocks;
  return words <= (blocks + 1) << 15;
}

// Sorts into order[n]; workspace of sort_plan(n, rows).bytes() (none for few
// tokens).
inline cudaError_t sort_tokens(int64_t n, const Index& index, uint2* order, void* workspace,
                               const Fill& fill, cudaStream_t stream) {
  if (n <= kSmall) {
    switch (cluster_items(n)) {
      case 1: return cluster_sort<1>(n, index, order, fill, stream);
      case 2: return cluster_sort<2>(n, index, order, fill, stream);
      default: return cluster_sort<4>(n, index, order, fill, stream);
    }
  }
  const SortPlan p = sort_plan(n, index.rows);
  switch (p.items) {
    case 2: return large_sort<2>(n, index, p, order, workspace, fill, stream);
    case 4: return large_sort<4>(n, index, p, order, workspace, fill, stream);
    default: return large_sort<8>(n, index, p, order, workspace, fill, stream);
  }
}

}  // namespace tokens
}  // namespace clad3dgs
