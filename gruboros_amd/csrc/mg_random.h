// Counter-based random words for dropout: Philox4x32-10 (Salmon, Moraes, Dror
// and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011).
#pragma once

#include "mg_common.h"

namespace mg {

// The four words of counter (i, offset) under the 64-bit key `seed`. Ten rounds of two 32 x 32 -> 64
// bit products; nothing is kept between calls, so any element's words can be made again anywhere.
__device__ __forceinline__ void philox(uint64_t i, uint64_t offset, uint64_t seed, uint32_t (&w)[4]) {
  uint32_t c0 = static_cast<uint32_t>(i), c1 = static_cast<uint32_t>(i >> 32);
  uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u, p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
    c1 = static_cast<uint32_t>(p1);
    c3 = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0, w[1] = c1, w[2] = c2, w[3] = c3;
}

// What a call drops: element e of its tensor takes word e % 4 of counter e / 4 and is dropped where
// the word is below `threshold` = floor(p 2^32); the others are multiplied by scale = 1 / (1 - p).
struct Drop {
  uint64_t seed, offset;
  const int64_t* seed_p;  // read instead of `seed` when not null (a captured graph's next replay sees a new one)
  uint32_t threshold;
  float scale;
  __device__ __forceinline__ uint64_t key() const { return seed_p ? static_cast<uint64_t>(*seed_p) : seed; }
};

// The words of the four elements from e on
template <bool ALIGNED>
__device__ __forceinline__ void drop_words(uint64_t e, uint64_t offset, uint64_t key, uint32_t (&w)[4]) {
  philox(e >> 2, offset, key, w);
  if constexpr (!ALIGNED) {
    const uint32_t s = static_cast<uint32_t>(e) & 3u;
    if (s) {
      uint32_t n[4];
      philox((e >> 2) + 1, offset, key, n);
      const uint32_t a[8] = {w[0], w[1], w[2], w[3], n[0], n[1], n[2], n[3]};
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = s == 1 ? a[j + 1] : s == 2 ? a[j + 2] : a[j + 3];
    }
  }
}

}  // namespace mg
