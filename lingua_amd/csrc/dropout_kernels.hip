// Dropout of a tensor, alone or into a sum: y = residual + drop(x), in fp32, rounded once.  The backward pass is the same kernel on the
// gradient (the residual's gradient is the sum's).  What the generator is: dropout.h.
//
// A thread takes a group of eight elements, one 16-byte load and store and one call of the generator.  Bound by memory where the tensor
// is large, 4 bytes an element and 6 with a residual: [16384,4096] 41 us, 6.6 TB/s (a part of it from the caches), and 70 us, 5.7 TB/s.
// [333,2064] 2.7 us, a launch.
#include "dropout.h"

namespace l8 {

constexpr int kDropBlock = 256;

int drop_of(const char *who, const int64_t *numbers, int64_t site, int64_t threshold, Drop *out) {
  L8_REQUIRE(site >= 0 && site < (1ll << 32), "%s: site %lld is not a number of 32 bits", who, (long long)site);
  L8_REQUIRE(threshold >= 0 && threshold <= 65536, "%s: threshold %lld is not within 0 .. 65536", who, (long long)threshold);
  L8_REQUIRE(((uintptr_t)numbers % 8) == 0, "%s: misaligned seed and step", who);
  *out = Drop{numbers, (uint32_t)site, (uint32_t)threshold, threshold == 65536 ? 0.0f : 65536.0f / (float)(65536 - threshold)};
  return L8_OK;
}

// LINES: the pointers are on 16-byte lines; else every element goes by itself.  (y may be x or residual: an element is read before it is written.)
template <bool ADD, bool LINES>
__global__ __launch_bounds__(kDropBlock) void dropout_kernel(const uint16_t *x, const uint16_t *residual, uint16_t *y, int64_t n, const Drop drop) {
  const int64_t group = (int64_t)blockIdx.x * kDropBlock + threadIdx.x, at = group * 8;
  if (at >= n) return;
  uint32_t words[4];
  if (LINES && at + 8 <= n) {
    const v4i in = *(const v4i *)(x + at);
    [[maybe_unused]] v4i res;
    if constexpr (ADD) res = *(const v4i *)(residual + at);
    drop_words(words, drop_key(drop), (uint64_t)group);
    v4i out;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float lo = drop_one(__uint_as_float((uint32_t)in[k] << 16), words, 2 * k, drop);
      float hi = drop_one(__uint_as_float((uint32_t)in[k] & 0xffff0000u), words, 2 * k + 1, drop);
      if constexpr (ADD) {
        lo = __uint_as_float((uint32_t)res[k] << 16) + lo;
        hi = __uint_as_float((uint32_t)res[k] & 0xffff0000u) + hi;
      }
      out[k] = (int)(bf16_rne_bits(lo) | (bf16_rne_bits(hi) << 16));
    }
    *(v4i *)(y + at) = out;
    return;
  }
  drop_words(words, drop_key(drop), (uint64_t)group);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (at + e >= n) break;
    float v = drop_one(bf16_bits_to_f32(x[at + e]), words, e, drop);
    if constexpr (ADD) v = bf16_bits_to_f32(residual[at + e]) + v;
    y[at + e] = (uint16_t)bf16_rne_bits(v);
  }
}

}  // namespace l8

using namespace l8;

extern "C" int l8_dropout(const void *x, const void *residual, void *y, int64_t n, const int64_t *numbers, int64_t site, int64_t threshold,
                          void *stream) {
  L8_REQUIRE(n >= 0, "l8_dropout: negative size %lld", (long long)n);
  Drop d;
  const int code = drop_of("l8_dropout", numbers, site, threshold, &d);
  if (code != L8_OK) return code;
  if (n == 0) return L8_OK;
  L8_REQUIRE(x && y && numbers, "l8_dropout: null pointer");
  L8_REQUIRE((((uintptr_t)x | (uintptr_t)y | (uintptr_t)residual) % 2) == 0, "l8_dropout: misaligned pointer");
  const int64_t blocks = ((n + 7) / 8 + kDropBlock - 1) / kDropBlock;
  L8_REQUIRE(blocks < (1ll << 24), "l8_dropout: %lld elements, 2^35 or more", (long long)n);
  const bool lines = (((uintptr_t)x | (uintptr_t)y | (uintptr_t)residual) % 16) == 0;
  const dim3 grid((unsigned)blocks), threads(kDropBlock);
  hipStream_t st = (hipStream_t)stream;
  const uint16_t *xp = (const uint16_t *)x, *rp = (const uint16_t *)residual;
  uint16_t *yp = (uint16_t *)y;
  if (residual) {
    if (lines) hipLaunchKernelGGL((dropout_kernel<true, true>), grid, threads, 0, st, xp, rp, yp, n, d);
    else hipLaunchKernelGGL((dropout_kernel<true, false>), grid, threads, 0, st, xp, rp, yp, n, d);
  } else {
    if (lines) hipLaunchKernelGGL((dropout_kernel<false, true>), grid, threads, 0, st, xp, rp, yp, n, d);
    else hipLaunchKernelGGL((dropout_kernel<false, false>), grid, threads, 0, st, xp, rp, yp, n, d);
  }
  L8_HIP(hipGetLastError());
  return L8_OK;
}
