// Counter-based random bits: Philox4x32 of ten rounds (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011), 16 bits an element.
#pragma once
#include "common.h"

namespace ssla {

struct Draw {
  const int64_t *seed;     // on the device
  uint32_t subsequence;
  uint32_t threshold;      // round(p 2^16): an element is kept where its bits reach it; 0: all kept
  float scale;             // 2^16 / (2^16 - threshold), 0 where nothing is kept
};

struct Bits { uint32_t w[4]; };   // element e of eight: half e & 1 of word e >> 1

// The bits of elements 8 i .. 8 i + 7.
__device__ __forceinline__ Bits bits_of(uint64_t i, uint64_t seed, uint32_t subsequence) {
  uint32_t c0 = static_cast<uint32_t>(i), c1 = static_cast<uint32_t>(i >> 32), c2 = subsequence, c3 = 0;
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t x = static_cast<uint64_t>(c0) * 0xD2511F53u, y = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(y >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(y);
    c2 = static_cast<uint32_t>(x >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(x);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// Which of the eight elements of a block are kept, a bit each.
__device__ __forceinline__ uint32_t kept_of(const Draw &d, uint64_t seed, uint64_t block) {
  const Bits b = bits_of(block, seed, d.subsequence);
  uint32_t keep = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) keep |= static_cast<uint32_t>((e & 1 ? b.w[e >> 1] >> 16 : b.w[e >> 1] & 0xffffu) >= d.threshold) << e;
  return keep;
}
// Which of the W elements from `at` on are kept: W of 4 or 8.  FULL: `at` is a multiple of W;
// else they may lie in two blocks.
template <int W, bool FULL>
__device__ __forceinline__ uint32_t kept(const Draw &d, uint64_t seed, uint64_t at) {
  const uint32_t off = static_cast<uint32_t>(at) & 7;
  uint32_t keep = kept_of(d, seed, at >> 3) >> off;
  if (!FULL && off + W > 8) keep |= kept_of(d, seed, (at >> 3) + 1) << (8 - off);
  return keep;
}

}  // namespace ssla
