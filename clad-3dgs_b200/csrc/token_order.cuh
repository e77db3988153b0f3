// Stable order of tokens by the table row they name: (row, position) pairs
// sorted by row, positions ascending within a row. Tokens that name no row
// (padding, or an index outside the table) get the row number `rows` and so
// come last.
//
// Least-significant-digit radix sort, at most ten bits a pass. A pass is three
// kernels: every block counts the digits of its tile; one warp per digit turns
// the blocks' counts into exclusive sums; every block ranks its tile and
// scatters it. Ranks come from ballots of equal digits within a warp, taken in
// token order, so the sort is stable and the order the same on every run.
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

namespace clad3dgs {
namespace tokens {

// Set when a kernel met an index outside its table that is not the padding.
constexpr unsigned kFaultTokenRange = 256u;
__device__ unsigned int g_token_fault = 0;

// The indices a caller gives.
struct Index {
  const void* data;
  bool wide;  // int64, else int32
  bool has_padding;
  int64_t padding;
  int64_t rows;
};

// The row that token i names, or `rows` for none.
__device__ __forceinline__ uint32_t row_of(const Index& x, int64_t i) {
  const int64_t t = x.wide ? static_cast<const int64_t*>(x.data)[i]
                           : int64_t(static_cast<const int32_t*>(x.data)[i]);
  if (x.has_padding && t == x.padding) return uint32_t(x.rows);
  if (t >= 0 && t < x.rows) return uint32_t(t);
  atomicOr(&g_token_fault, kFaultTokenRange);
  return uint32_t(x.rows);
}

constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortItems = 16;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kDigitBits = 10;

struct SortPlan {
  int passes, bits;  // digit width of every pass
  int64_t blocks;
  size_t pair_bytes, count_bytes, total_bytes;  // workspace parts

  size_t bytes() const { return pair_bytes + count_bytes + total_bytes; }
};

inline SortPlan sort_plan(int64_t n, int64_t rows) {
  int key_bits = 1;
  while (key_bits < 32 && (rows >> key_bits) != 0) ++key_bits;  // rows itself is a key
  SortPlan p;
  p.passes = (key_bits + kDigitBits - 1) / kDigitBits;
  p.bits = (key_bits + p.passes - 1) / p.passes;
  p.blocks = (n + kSortTile - 1) / kSortTile;
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  p.pair_bytes = p.passes > 1 ? up(size_t(n) * sizeof(uint2)) : 0;
  p.count_bytes = up((size_t(1) << p.bits) * p.blocks * sizeof(uint32_t));
  p.total_bytes = up((size_t(1) << p.bits) * sizeof(uint32_t));
  return p;
}

// The pair at i: from the caller's indices in the first pass, else from the
// pass before.
__device__ __forceinline__ uint2 pair_at(const Index& index, const uint2* from, int64_t i) {
  return from ? from[i] : make_uint2(row_of(index, i), uint32_t(i));
}

static __global__ void __launch_bounds__(kSortThreads)
    count_kernel(int64_t n, Index index, const uint2* __restrict__ from, int shift, int bits,
                 uint32_t* __restrict__ counts) {
  __shared__ uint32_t bins[1 << kDigitBits];
  const uint32_t mask = (1u << bits) - 1;
  for (uint32_t d = threadIdx.x; d <= mask; d += kSortThreads) bins[d] = 0;
  __syncthreads();
  const int64_t base = int64_t(blockIdx.x) * kSortTile;
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = base + j * kSortThreads + threadIdx.x;
    if (i < n) {
      const uint32_t key = from ? from[i].x : row_of(index, i);
      atomicAdd(&bins[(key >> shift) & mask], 1u);
    }
  }
  __syncthreads();
  for (uint32_t d = threadIdx.x; d <= mask; d += kSortThreads)
    counts[int64_t(d) * gridDim.x + blockIdx.x] = bins[d];
}

// One warp per digit: counts[d][blocks] to exclusive sums, totals[d] their sum.
static __global__ void __launch_bounds__(kSortThreads)
    scan_counts_kernel(int digits, int64_t blocks, uint32_t* __restrict__ counts,
                       uint32_t* __restrict__ totals) {
  const int d = int(blockIdx.x) * kSortWarps + int(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (d >= digits) return;
  uint32_t* row = counts + int64_t(d) * blocks;
  uint32_t sum = 0;
  for (int64_t at = 0; at < blocks; at += 32) {
    const uint32_t mine = at + lane < blocks ? row[at + lane] : 0;
    uint32_t inclusive = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t below = __shfl_up_sync(~0u, inclusive, o);
      if (lane >= o) inclusive += below;
    }
    if (at + lane < blocks) row[at + lane] = sum + inclusive - mine;
    sum += __shfl_sync(~0u, inclusive, 31);
  }
  if (lane == 0) totals[d] = sum;
}

static __global__ void __launch_bounds__(kSortThreads)
    scatter_kernel(int64_t n, Index index, const uint2* __restrict__ from, int shift, int bits,
                   const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals,
                   uint2* __restrict__ to) {
  __shared__ uint32_t warp_bins[kSortWarps][1 << kDigitBits];
  __shared__ uint32_t warp_sums[kSortWarps];
  const int digits = 1 << bits;
  const uint32_t mask = uint32_t(digits) - 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int d = threadIdx.x; d < digits * kSortWarps; d += kSortThreads)
    warp_bins[d / digits][d % digits] = 0;
  __syncthreads();
  // Ranks within the warp's share of the tile, in token order.
  const int64_t base = int64_t(blockIdx.x) * kSortTile + warp * 32 * kSortItems + lane;
  uint2 pair[kSortItems];
  uint32_t rank[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = base + 32 * j;
    const bool real = i < n;
    pair[j] = real ? pair_at(index, from, i) : make_uint2(0, 0);
    const uint32_t digit = real ? (pair[j].x >> shift) & mask : ~0u;
    const uint32_t same = __match_any_sync(~0u, digit);
    const int leader = __ffs(same) - 1;
    uint32_t before = 0;
    if (lane == leader && real) {
      before = warp_bins[warp][digit];
      warp_bins[warp][digit] = before + __popc(same);
    }
    rank[j] = __shfl_sync(~0u, before, leader) + __popc(same & ((1u << lane) - 1));
    __syncwarp();
  }
  __syncthreads();
  // Where each warp's tokens of a digit begin: all smaller digits, then this
  // digit's earlier blocks, then its earlier warps.
  const int each = (digits + kSortThreads - 1) / kSortThreads;
  uint32_t mine = 0;
  for (int k = 0; k < each; ++k) {
    const int d = threadIdx.x * each + k;
    if (d < digits) mine += totals[d];
  }
  uint32_t inclusive = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t below = __shfl_up_sync(~0u, inclusive, o);
    if (lane >= o) inclusive += below;
  }
  if (lane == 31) warp_sums[warp] = inclusive;
  __syncthreads();
  uint32_t start = inclusive - mine;
  for (int w = 0; w < warp; ++w) start += warp_sums[w];
  for (int k = 0; k < each; ++k) {
    const int d = threadIdx.x * each + k;
    if (d >= digits) break;
    uint32_t at = start + counts[int64_t(d) * gridDim.x + blockIdx.x];
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = warp_bins[w][d];
      warp_bins[w][d] = at;
      at += c;
    }
    start += totals[d];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j)
    if (base + 32 * j < n)
      to[warp_bins[warp][(pair[j].x >> shift) & mask] + rank[j]] = pair[j];
}

// Sorts into order[n]; workspace of sort_plan(n, rows).bytes().
inline cudaError_t sort_tokens(int64_t n, const Index& index, uint2* order, void* workspace,
                               cudaStream_t stream) {
  const SortPlan p = sort_plan(n, index.rows);
  char* at = static_cast<char*>(workspace);
  uint2* spare = reinterpret_cast<uint2*>(at);
  uint32_t* counts = reinterpret_cast<uint32_t*>(at + p.pair_bytes);
  uint32_t* totals = reinterpret_cast<uint32_t*>(at + p.pair_bytes + p.count_bytes);
  const unsigned blocks = unsigned(p.blocks);
  const uint2* from = nullptr;
  for (int pass = 0; pass < p.passes; ++pass) {
    // Alternating so that the last pass ends in `order`.
    uint2* to = (p.passes - 1 - pass) % 2 == 0 ? order : spare;
    const int shift = pass * p.bits;
    count_kernel<<<blocks, kSortThreads, 0, stream>>>(n, index, from, shift, p.bits, counts);
    scan_counts_kernel<<<((1 << p.bits) + kSortWarps - 1) / kSortWarps, kSortThreads, 0, stream>>>(
        1 << p.bits, p.blocks, counts, totals);
    scatter_kernel<<<blocks, kSortThreads, 0, stream>>>(n, index, from, shift, p.bits, counts,
                                                        totals, to);
    from = to;
  }
  return cudaGetLastError();
}

}  // namespace tokens
}  // namespace clad3dgs
