// Philox4x32-10, the counter-based generator of Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3" (SC 2011).
#pragma once
#include <cstdint>

namespace cfb {

// 128 random bits of counter (block, stream, 0) under the 64-bit key `seed`.  Element e of a
// tensor takes 16 of the bits of block e / 8: bits 16 (e % 8) and up, low word first.
__device__ __forceinline__ uint4 philox_block(uint64_t block, uint32_t stream, uint64_t seed) {
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
  uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32), c2 = stream,
           c3 = 0;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = static_cast<uint64_t>(0xD2511F53u) * c0;
    const uint64_t b = static_cast<uint64_t>(0xCD9E8D57u) * c2;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// The 16 bits of lane j (compile-time after unrolling) of a block.
__device__ __forceinline__ int philox_lane(const uint4& r, int j) {
  const uint32_t w = j < 4 ? (j < 2 ? r.x : r.y) : (j < 6 ? r.z : r.w);
  return static_cast<int>((j & 1) ? w >> 16 : w & 0xffffu);
}

}  // namespace cfb
