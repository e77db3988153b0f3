// The keep/drop decisions of the dropout, drawn from a counter and never stored.
//
// Element e of a call keeps its value iff word e % 4 of Philox4x32-10 at the
// counter (e / 4 low, e / 4 high, offset low, offset high) under the key
// (seed low, seed high) is at least floor(p * 2^32). The generator is the one
// of Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3" (SC'11): ten rounds of two 32 x 32 -> 64 bit products, their high
// halves mixed with the other words and a key that grows by a constant every
// round. One call serves four elements; any kernel that knows an element's
// number finds its decision again, so the backward pass needs no mask.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace clad3dgs {

constexpr int kMaskRounds = 10;

// One dropout as a kernel argument: kept iff word >= limit, for p < 1; `none`
// keeps nothing (p = 1, whose limit does not fit a word). The rounds' keys are
// made on the host, so that a round is two products and two three-way
// exclusive-ors with one operand from the argument.
struct CounterMask {
  uint32_t key0[kMaskRounds], key1[kMaskRounds];
  unsigned long long offset;
  const long long* offset_device;  // nullable: added to offset by the kernel
  uint32_t limit;
  bool none;

  __device__ __forceinline__ bool keeps(uint32_t word) const { return word >= limit && !none; }
};

inline CounterMask counter_mask(double p, uint64_t seed, uint64_t offset,
                                const long long* offset_device) {
  CounterMask m;
  for (int r = 0; r < kMaskRounds; ++r) {
    m.key0[r] = uint32_t(seed) + uint32_t(r) * 0x9E3779B9u;
    m.key1[r] = uint32_t(seed >> 32) + uint32_t(r) * 0xBB67AE85u;
  }
  m.offset = offset;
  m.offset_device = offset_device;
  m.none = p >= 1.0;
  m.limit = m.none ? 0 : uint32_t(p * 4294967296.0);
  return m;
}

__device__ __forceinline__ unsigned long long mask_offset(const CounterMask& m) {
  return m.offset + (m.offset_device ? (unsigned long long)*m.offset_device : 0ull);
}

// The four words of a block of four elements. Number: uint32_t where every block
// number fits one (its high half is then a constant zero).
template <class Number>
__device__ __forceinline__ uint4 mask_words(const CounterMask& m, unsigned long long offset,
                                            Number block) {
  uint32_t c0 = uint32_t(block), c1 = sizeof(Number) > 4 ? uint32_t(uint64_t(block) >> 32) : 0u,
           c2 = uint32_t(offset), c3 = uint32_t(offset >> 32);
#pragma unroll
  for (int r = 0; r < kMaskRounds; ++r) {
    const unsigned long long a = (unsigned long long)0xD2511F53u * c0;
    const unsigned long long b = (unsigned long long)0xCD9E8D57u * c2;
    c0 = uint32_t(b >> 32) ^ c1 ^ m.key0[r];
    c1 = uint32_t(b);
    c2 = uint32_t(a >> 32) ^ c3 ^ m.key1[r];
    c3 = uint32_t(a);
  }
  return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ uint32_t word_of(const uint4& w, unsigned j) {
  return j == 0 ? w.x : j == 1 ? w.y : j == 2 ? w.z : w.w;
}

// The decisions for four elements that begin at any element e.
__device__ __forceinline__ void mask_four(const CounterMask& m, unsigned long long offset,
                                          uint64_t e, bool (&keep)[4]) {
  const unsigned shift = unsigned(e) % 4;
  const uint4 a = mask_words(m, offset, e / 4);
  uint4 b = make_uint4(0, 0, 0, 0);
  if (shift) b = mask_words(m, offset, e / 4 + 1);
  const uint32_t w[7] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    keep[j] = m.keeps(shift == 0 ? w[j] : shift == 1 ? w[j + 1] : shift == 2 ? w[j + 2] : w[j + 3]);
}

// The decisions for V elements that begin at element e, e a multiple of V (a
// multiple of four, or V = 1). Number: uint32_t where every e / 4 fits one.
template <int V, class Number = uint64_t>
__device__ __forceinline__ void mask_vector(const CounterMask& m, unsigned long long offset,
                                            uint64_t e, bool (&keep)[V]) {
  static_assert(V == 1 || V % 4 == 0, "whole blocks, or one element");
#pragma unroll
  for (int j = 0; j < V; j += 4) {
    const uint4 words = mask_words(m, offset, Number((e + j) / 4));
    if constexpr (V == 1) {
      keep[0] = m.keeps(word_of(words, unsigned(e) % 4));
    } else {
      keep[j] = m.keeps(words.x);
      keep[j + 1] = m.keeps(words.y);
      keep[j + 2] = m.keeps(words.z);
      keep[j + 3] = m.keeps(words.w);
    }
  }
}

}  // namespace clad3dgs
