// Dropout whose mask is never stored: element i of call `site` in step numbers[1] stays where 16 bits of a counter-based generator reach
// the threshold, forward and backward alike.
//
// The generator is Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, 2011): ten rounds of two
// 32 x 32 -> 64 products over the counter (group low, group high, site, step) under the key numbers[0], four words out.  A group is
// eight neighbouring elements, of which element e takes the lower (e even) or upper half of word e / 2: 16 bits an element, so the
// share that is dropped is a multiple of 2^-16 and what stays is scaled by that very share -- 32 bits would double the generator's
// work, which is the larger part of a dropout's instructions, to move the share by less than 1e-5.
#pragma once
#include "l8_common.h"

namespace l8 {

struct Drop {
  const int64_t *numbers;   // {seed, step}, read when the kernel runs; NULL: nothing is dropped
  uint32_t site, threshold;
  float factor;             // 1 / (1 - threshold / 2^16); 0 where everything is dropped
};

struct DropKey {
  uint32_t k0, k1, site, step;
};
L8_DEV DropKey drop_key(const Drop &d) {
  const int64_t seed = d.numbers[0], step = d.numbers[1];
  return DropKey{(uint32_t)seed, (uint32_t)((uint64_t)seed >> 32), d.site, (uint32_t)step};
}

// The four words of a group.
L8_DEV void drop_words(uint32_t (&c)[4], const DropKey &key, uint64_t group) {
  c[0] = (uint32_t)group, c[1] = (uint32_t)(group >> 32), c[2] = key.site, c[3] = key.step;
  uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c[0] * 0xD2511F53u, b = (uint64_t)c[2] * 0xCD9E8D57u;
    const uint32_t n0 = (uint32_t)(b >> 32) ^ c[1] ^ k0, n2 = (uint32_t)(a >> 32) ^ c[3] ^ k1;
    c[1] = (uint32_t)b, c[3] = (uint32_t)a;
    c[0] = n0, c[2] = n2;
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
}
L8_DEV bool drop_keeps(const uint32_t (&c)[4], int e, uint32_t threshold) {
  const uint32_t half = (e & 1) ? c[e >> 1] >> 16 : c[e >> 1] & 0xffffu;
  return half >= threshold;
}
// What is left of v: a dropped element is zero whatever it held.
L8_DEV float drop_one(float v, const uint32_t (&c)[4], int e, const Drop &d) { return drop_keeps(c, e, d.threshold) ? v * d.factor : 0.0f; }

// Checks and the kernel's view of what the C entries are given.
int drop_of(const char *who, const int64_t *numbers, int64_t site, int64_t threshold, Drop *out);

}  // namespace l8
