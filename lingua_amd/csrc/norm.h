// What the norm kernels share: sums over a wave, a row in registers, the parameters of a lane's columns, the fold of the
// parameters' gradients.
#pragma once
#include "l8_common.h"

namespace l8 {

constexpr int kNormBlock = 256;
constexpr int kNormWaves = kNormBlock / 64;

// sum over the 64 lanes of a wave, result uniform
L8_DEV float wave_sum_f32(float v) {
  auto step = [&](int moved) { v += __int_as_float(moved); };
  step(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, true));   // quad_perm [1,0,3,2]
  step(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, true));   // quad_perm [2,3,0,1]
  step(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xF, 0xF, true));  // row_ror:4
  step(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, true));  // row_ror:8
  const float a = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 0));
  const float b = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 16));
  const float c = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 32));
  const float d = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 48));
  return (a + b) + (c + d);
}

// The weights of a lane's columns, kept in registers for all rows it sees: packed pairs as they are in memory (bf16),
// or one register each (fp32).  Zero beyond column C.
template <int N, bool W_F32>
struct NormWeights {
  uint32_t reg[N * (W_F32 ? 8 : 4)];
  template <typename ColOf>
  L8_DEV void load(const void *w, int C, ColOf col_of) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = col_of(j);
#pragma unroll
      for (int e = 0; e < (W_F32 ? 8 : 4); ++e) {
        uint32_t v = 0;
        // a bf16 weight may start at any even address: the copy states two-byte alignment
        if (c < C) {
          if (W_F32) v = ((const uint32_t *)w)[c + e];
          else __builtin_memcpy(&v, (const uint16_t *)w + c + 2 * e, 4);
        }
        reg[j * (W_F32 ? 8 : 4) + e] = v;
      }
    }
  }
  L8_DEV float get(int j, int e) const {
    if (W_F32) return __uint_as_float(reg[j * 8 + e]);
    const uint32_t p = reg[j * 4 + (e >> 1)];
    return __uint_as_float((e & 1) ? (p & 0xffff0000u) : (p << 16));
  }
};

#if defined(__HIP_DEVICE_COMPILE__)
// row r of x; zeros beyond column C and for a row at or beyond R (no branch around a load)
template <int N, typename ColOf>
L8_DEV void load_norm_row(v4i (&buf)[N], const uint16_t *x, int64_t r, int64_t R, int64_t ldx, int C, ColOf col_of) {
  const __amdgpu_buffer_rsrc_t rs = make_rsrc(x + (r < R ? r : 0) * ldx, r < R ? (uint32_t)C * 2u : 0u);
#pragma unroll
  for (int j = 0; j < N; ++j) buf[j] = load16_nt(rs, (uint32_t)col_of(j) * 2u, 0);
}
L8_DEV void store16_nt(__amdgpu_buffer_rsrc_t rs, uint32_t voff, v4i data) {
  __builtin_amdgcn_raw_buffer_store_b128(data, rs, (int)voff, 0, 2 /* non-temporal */);
}
L8_DEV void store8_nt(__amdgpu_buffer_rsrc_t rs, uint32_t voff, v2i data) {
  __builtin_amdgcn_raw_buffer_store_b64(data, rs, (int)voff, 0, 2 /* non-temporal */);
}
// Eight bf16 plus eight bf16, each sum rounded to nearest even.
L8_DEV v4i sum_bf16x8(v4i a, v4i b) {
  v4i out;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float lo = __uint_as_float((uint32_t)a[k] << 16) + __uint_as_float((uint32_t)b[k] << 16);
    const float hi = __uint_as_float((uint32_t)a[k] & 0xffff0000u) + __uint_as_float((uint32_t)b[k] & 0xffff0000u);
    out[k] = (int)(bf16_rne_bits(lo) | (bf16_rne_bits(hi) << 16));
  }
  return out;
}
// The row of x becomes the row of h = bf16(x + residual), which is also written: the norm is that of the sum as it is kept.
template <int N, typename ColOf>
L8_DEV void add_residual(v4i (&cur)[N], const v4i (&res)[N], uint16_t *h, int64_t r, int64_t ldh, int C, ColOf col_of) {
  const __amdgpu_buffer_rsrc_t rsH = make_rsrc(h + r * ldh, (uint32_t)C * 2u);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    cur[j] = sum_bf16x8(cur[j], res[j]);
    store16_nt(rsH, (uint32_t)col_of(j) * 2u, cur[j]);
  }
}
#endif

constexpr int64_t kNormMaxC = 4 * kNormWaves * 512;  // 8192: the weights of a thread's columns live in registers

// Workgroups of a kernel with a row each, a row of partial sums each: two per compute unit.
int64_t norm_blocks(int64_t R);

// Where a parameter's gradient goes: n columns in fp32 or rounded to bf16; p NULL: nowhere.
struct GradOut {
  void *p;
  int f32, n;
};
// Adds up the `slots` rows of first.n + second.n partial sums (fp32), column by column in the order of the rows.
int fold_norm_grads(const float *partials, int64_t slots, const GradOut &first, const GradOut &second, hipStream_t st);

}  // namespace l8
