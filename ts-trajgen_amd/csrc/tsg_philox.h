// Counter-based random words for dropout: Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as
// 1, 2, 3; SC'11).  key = the 64-bit seed, counter = (element / 4 as two words, site, step); element i takes word i & 3 of
// its block and is kept iff that word >= floor(p 2^32), so P(dropped) is p to 2^-32.  A mask is a function of
// (seed, site, step, element) alone: it is computed where it is needed and stored nowhere.
#pragma once
#include "tsg_common.h"

struct TsgRng {
  unsigned k0, k1, site, step;
  const long long* step_dev;  // when non-null the step is read from device memory (a captured graph then advances it)
  unsigned threshold;         // floor(p 2^32); p == 1 drops everything whatever the words
  int all;                    // p == 1
  float scale;                // 1 / (1 - p), 0 when all
};

static inline TsgRng tsg_make_rng(double p, uint64_t seed, uint32_t site, uint32_t step, const int64_t* step_dev) {
  TsgRng r;
  r.k0 = (unsigned)seed;
  r.k1 = (unsigned)(seed >> 32);
  r.site = site;
  r.step = step;
  r.step_dev = reinterpret_cast<const long long*>(step_dev);
  r.all = p >= 1.0;
  r.threshold = r.all ? 0u : (unsigned)(p * 4294967296.0);
  r.scale = r.all ? 0.0f : (float)(1.0 / (1.0 - p));
  return r;
}

__device__ __forceinline__ unsigned tsg_rng_step(const TsgRng& r) { return r.step_dev ? (unsigned)*r.step_dev : r.step; }

__device__ __forceinline__ uint4 tsg_philox(unsigned long long block, unsigned site, unsigned step, unsigned k0, unsigned k1) {
  unsigned c0 = (unsigned)block, c1 = (unsigned)(block >> 32), c2 = site, c3 = step;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
    c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
    c1 = (unsigned)b;
    c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
    c3 = (unsigned)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// factor of ONE element: 0 or 1 / (1 - p)
__device__ __forceinline__ float tsg_drop_factor(const TsgRng& r, unsigned step, unsigned long long i) {
  const uint4 w = tsg_philox(i >> 2, r.site, step, r.k0, r.k1);
  const unsigned v = (i & 2) ? ((i & 1) ? w.w : w.z) : ((i & 1) ? w.y : w.x);
  return v >= r.threshold ? r.scale : 0.0f;
}
