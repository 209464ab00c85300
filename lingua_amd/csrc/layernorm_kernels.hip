// Layer norm, forward and backward, with the fp8 copy of its output and of a residual sum if wanted; and both norms of a sum of which
// one operand is dropped out (dropout.h).  nn.LayerNorm in the place of the model's RMSNorm (lingua/transformer.py:264-292).
//
//   h  = bf16(residual + drop(x))                     (or x itself)
//   m  = mean(h), v = mean((h - m)^2), r = 1 / sqrt(v + eps)
//   y  = bf16(((h - m) * r) * w + b),  q, scale = row-wise cast of y, [column amaxes of y]
//
// RMSNorm (CENTRED false) has m = 0 and no b.  A wave finds mean and sum of squared differences of its own columns, from registers, and
// the waves' pairs are joined: v = sum over waves of (M2 + n * (m_wave - m)^2) / C.  No difference of large sums is taken, and a row
// that a workgroup shares meets at one barrier.  Everything in fp32.
// Two layouts, as in the RMSNorm: a wavefront per row for short rows, a workgroup for the longer ones; both join the same chunks of 512
// columns in the same order up to 2048 columns, so a row's result does not hang on how many rows come with it.
// Bound by memory where there are rows enough: one read and one write of everything, the next row requested while one is worked on.
#include <algorithm>
#include "dropout.h"
#include "norm.h"

namespace l8 {

struct NormFwd {
  const uint16_t *x, *residual;
  const void *w, *b;
  uint16_t *h, *y;
  uint8_t *q;
  float *scale, *mean, *rstd;
  uint16_t *col_partials;
  int64_t R, ldx, ldr, ldh, ldy, ldq;
  int C, w_f32, b_f32, scale_rule;
  float eps;
  Drop drop;
};

// A parameter of a lane's columns in fp32, `none` where there is no parameter; zero beyond column C.
template <int N, typename ColOf>
L8_DEV void load_param(float (&out)[N][8], const void *p, int f32, float none, int C, ColOf col_of) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = col_of(j);
#pragma unroll
    for (int e = 0; e < 8; ++e) out[j][e] = c < C ? none : 0.0f;
    if (c < C && p) {
      if (f32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) out[j][e] = ((const float *)p)[c + e];
      } else {   // a bf16 parameter may start at any even address: the copy states two-byte alignment
        uint32_t v[4];
        __builtin_memcpy(v, (const uint16_t *)p + c, 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) out[j][e] = __uint_as_float((e & 1) ? (v[e >> 1] & 0xffff0000u) : (v[e >> 1] << 16));
      }
    }
  }
}

L8_DEV float lo_of(int p) { return __uint_as_float((uint32_t)p << 16); }
L8_DEV float hi_of(int p) { return __uint_as_float((uint32_t)p & 0xffff0000u); }
L8_DEV int pack2(float lo, float hi) { return (int)(bf16_rne_bits(lo) | (bf16_rne_bits(hi) << 16)); }

// N chunks of 512 columns per wave, WPR waves to a row (1 or the workgroup's four).  As many chunks as the row has: of rows that have a wave
// each, us at [16384,1152] with the cast 27.7 with four chunks, 23.9 with three.
// us at [16384,4096], bytes an element: layer norm 50 (4, 5.4 TB/s), with the cast 67 (5, 5.0), of a sum 91 (8, 5.9), of a sum with a dropped
// operand and the cast 115 (9, 5.3): the generator hides behind memory.  [1,2048] 3.0, a launch.
template <int N, int WPR, bool CENTRED, bool ADD, bool DROP, bool COLMAX>
__global__ __launch_bounds__(kNormBlock, 2) void norm_fwd_kernel(const NormFwd p) {
#if defined(__HIP_DEVICE_COMPILE__)  // buffer descriptors exist in the device pass only
  static_assert(WPR == 1 || WPR == kNormWaves, "a wave or the workgroup per row");
  extern __shared__ __attribute__((aligned(16))) uint8_t dyn_lds[];  // [C] bf16 when COLMAX and WPR is 1
  __shared__ float red_s[2][kNormWaves], red_m[2][kNormWaves];
  __shared__ uint32_t red_mx[2][kNormWaves];
  constexpr int ROWS = kNormWaves / WPR;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int sub = WPR == 1 ? 0 : wave;
  const int C = p.C;
  const int64_t R = p.R;
  auto col_of = [&](int j) { return (j * WPR + sub) * 512 + lane * 8; };
  auto chunk_cols = [&](int j, int s) { const int n = C - (j * WPR + s) * 512; return n < 0 ? 0 : n < 512 ? n : 512; };
  auto wave_cols = [&](int s) {   // columns of wave s
    int n = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) n += chunk_cols(j, s);
    return n;
  };
  [[maybe_unused]] uint32_t cmax[COLMAX ? N * 4 : 1];
  if (COLMAX) {
#pragma unroll
    for (int i = 0; i < N * 4; ++i) cmax[i] = 0;
  }
  float w[N][8], b[CENTRED ? N : 1][8];
  load_param<N>(w, p.w, p.w_f32, 1.0f, C, col_of);
  if constexpr (CENTRED) load_param<N>(b, p.b, p.b_f32, 0.0f, C, col_of);
  const float inv_c = 1.0f / (float)C;
  [[maybe_unused]] DropKey key;
  if constexpr (DROP) key = drop_key(p.drop);
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  int64_t r = (int64_t)blockIdx.x * ROWS + (WPR == 1 ? wave : 0);
  v4i cur[N], nxt[N];
  [[maybe_unused]] v4i rnxt[N];
  load_norm_row<N>(cur, p.x, r, R, p.ldx, C, col_of);
  if constexpr (ADD) load_norm_row<N>(rnxt, p.residual, r, R, p.ldr, C, col_of);
  for (int it = 0; r < R; r += stride, ++it) {
    const int64_t rn = r + stride;
    load_norm_row<N>(nxt, p.x, rn, R, p.ldx, C, col_of);
    if constexpr (ADD) {
      if constexpr (DROP) {
        const __amdgpu_buffer_rsrc_t rsH = make_rsrc(p.h + r * p.ldh, (uint32_t)C * 2u);
        const uint64_t group0 = (uint64_t)r * (uint32_t)(C / 8);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          uint32_t words[4];
          drop_words(words, key, group0 + (uint32_t)(col_of(j) / 8));
#pragma unroll
          for (int k = 0; k < 4; ++k)
            cur[j][k] = pack2(lo_of(rnxt[j][k]) + drop_one(lo_of(cur[j][k]), words, 2 * k, p.drop),
                              hi_of(rnxt[j][k]) + drop_one(hi_of(cur[j][k]), words, 2 * k + 1, p.drop));
          store16_nt(rsH, (uint32_t)col_of(j) * 2u, cur[j]);
        }
      } else {
        add_residual<N>(cur, rnxt, p.h, r, p.ldh, C, col_of);
      }
      load_norm_row<N>(rnxt, p.residual, rn, R, p.ldr, C, col_of);
    }
    float mean = 0.0f, m2 = 0.0f;   // of the row: mean and sum of squared differences (CENTRED) or of squares
    auto squares = [&](int j, float centre) {
      float ss = 0.0f;
      const bool in = col_of(j) < C;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float lo = lo_of(cur[j][k]) - centre, hi = hi_of(cur[j][k]) - centre;
        ss += lo * lo;
        ss += hi * hi;
      }
      return !CENTRED || in ? ss : 0.0f;   // (what is read beyond column C is zero, and no difference)
    };
    auto sum_of = [&](int j) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; ++k) s += lo_of(cur[j][k]) + hi_of(cur[j][k]);
      return s;
    };
    auto inverse = [](int n) { return n ? 1.0f / (float)n : 0.0f; };
    auto apart = [&](float s, int n) {   // n columns of sum s: what their mean's distance adds to the squared differences
      const float d = s * inverse(n) - mean;
      return n ? (float)n * (d * d) : 0.0f;   // (no columns add nothing, also where the square is infinite)
    };
    if constexpr (WPR == 1) {
      float s[N], m[N];
#pragma unroll
      for (int j = 0; j < N; ++j) s[j] = CENTRED ? wave_sum_f32(sum_of(j)) : 0.0f;
#pragma unroll
      for (int j = 0; j < N; ++j) m[j] = wave_sum_f32(squares(j, s[j] * inverse(chunk_cols(j, 0))));
      if constexpr (CENTRED) {
        float tot = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) tot += s[j];
        mean = tot * inv_c;
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        m2 += m[j];
        if constexpr (CENTRED) m2 += apart(s[j], chunk_cols(j, 0));
      }
    } else {
      float s = 0.0f, m = 0.0f;
      if constexpr (CENTRED) {
#pragma unroll
        for (int j = 0; j < N; ++j) s += sum_of(j);
        s = wave_sum_f32(s);
      }
      const float centre = s * inverse(wave_cols(sub));
      if constexpr (CENTRED) {
#pragma unroll
        for (int j = 0; j < N; ++j) m += squares(j, centre);
      } else {   // (added up as the RMSNorm's kernels add it up: the same result for the same sum)
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float lo = lo_of(cur[j][k]), hi = hi_of(cur[j][k]);
            m += lo * lo;
            m += hi * hi;
          }
      }
      m = wave_sum_f32(m);
      if (lane == 0) {
        if constexpr (CENTRED) red_s[it & 1][wave] = s;
        red_m[it & 1][wave] = m;
      }
      __syncthreads();
      if constexpr (CENTRED) {
        float tot = 0.0f;
#pragma unroll
        for (int wv = 0; wv < kNormWaves; ++wv) tot += red_s[it & 1][wv];
        mean = tot * inv_c;
      }
#pragma unroll
      for (int wv = 0; wv < kNormWaves; ++wv) {
        m2 += red_m[it & 1][wv];
        if constexpr (CENTRED) m2 += apart(red_s[it & 1][wv], wave_cols(wv));
      }
    }
    const float rinv = 1.0f / sqrtf(m2 * inv_c + p.eps);
    const bool first = lane == 0 && sub == 0;
    if (first) {
      if (CENTRED && p.mean) p.mean[r] = mean;
      if (p.rstd) p.rstd[r] = rinv;
    }
    const __amdgpu_buffer_rsrc_t rsY = make_rsrc(p.y + r * p.ldy, (uint32_t)C * 2u);
    uint32_t mx = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      v4i yv;
      auto norm = [&](float v, int e) {
        if constexpr (CENTRED) return ((v - mean) * rinv) * w[j][e] + b[j][e];
        else return (v * rinv) * w[j][e];
      };
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        yv[k] = pack2(norm(lo_of(cur[j][k]), 2 * k), norm(hi_of(cur[j][k]), 2 * k + 1));
        // beyond column C there is no output, and no parameter: zero but for a mean that is not finite
        if (col_of(j) < C) mx = pk_absmax_u16(mx, (uint32_t)yv[k]);
        if (COLMAX) cmax[j * 4 + k] = pk_absmax_u16(cmax[j * 4 + k], (uint32_t)yv[k]);
      }
      store16_nt(rsY, (uint32_t)col_of(j) * 2u, yv);
      cur[j] = yv;  // the row of y replaces the row of h in registers
    }
    if (p.q) {   // the same for the whole grid
      uint32_t amax_bits = wave_max_u32(max(mx & 0xffffu, mx >> 16));
      if constexpr (WPR > 1) {
        if (lane == 0) red_mx[it & 1][wave] = amax_bits;
        __syncthreads();
        amax_bits = 0;
#pragma unroll
        for (int wv = 0; wv < kNormWaves; ++wv) amax_bits = max(amax_bits, red_mx[it & 1][wv]);
      }
      const RowScale rs = row_scale(amax_bits, p.scale_rule);
      if (first) p.scale[r] = rs.s;
      const __amdgpu_buffer_rsrc_t rsQ = make_rsrc(p.q + r * p.ldq, (uint32_t)C);
#pragma unroll
      for (int j = 0; j < N; ++j) store8_nt(rsQ, (uint32_t)col_of(j), cvt8(cur[j], rs.recip));
      if (!rs.finite) {  // a non-finite amax: the bytes are redone from this lane's own y with the integer conversion
        asm volatile("" ::: "memory");
#pragma unroll 1
        for (int c = sub * 512 + lane * 8; c < C; c += WPR * 512) *(v2i *)(p.q + r * p.ldq + c) = cvt8_slow(*(const v4i *)(p.y + r * p.ldy + c), rs.recip);
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) cur[j] = nxt[j];
  }
  if constexpr (COLMAX) {
    if constexpr (WPR > 1) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = col_of(j);
        if (c < C)
          *(v4i *)(p.col_partials + (int64_t)blockIdx.x * C + c) = v4i{(int)cmax[j * 4], (int)cmax[j * 4 + 1], (int)cmax[j * 4 + 2], (int)cmax[j * 4 + 3]};
      }
    } else {  // the waves' column maxima meet in LDS, one wave after the other, and leave as this workgroup's row
      v4i *lds4 = (v4i *)dyn_lds;
      for (int wv = 0; wv < kNormWaves; ++wv) {
        if (wave == wv) {
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const int c = col_of(j);
            if (c < C) {
              v4i mine = {(int)cmax[j * 4], (int)cmax[j * 4 + 1], (int)cmax[j * 4 + 2], (int)cmax[j * 4 + 3]};
              if (wv > 0) {
                const v4i old = lds4[c / 8];
#pragma unroll
                for (int k = 0; k < 4; ++k) mine[k] = (int)pk_absmax_u16((uint32_t)old[k], (uint32_t)mine[k]);
              }
              if (wv == kNormWaves - 1) *(v4i *)(p.col_partials + (int64_t)blockIdx.x * C + c) = mine;
              else lds4[c / 8] = mine;
            }
          }
        }
        __syncthreads();
      }
    }
  }
#endif
}

struct NormBwd {
  const uint16_t *gy, *gh, *h;
  const void *w;
  const float *mean, *rstd;
  uint16_t *gx, *gres;
  float *partials;     // [workgroups, C or (CENTRED) 2 C]; NULL: no parameter learns
  int64_t R, ldgy, ldgh, ldh, ldgx, ldgres;
  int C, w_f32;
  Drop drop;
};

// Backward, us at [16384,4096] with both parameter gradients: 79 (6 bytes an element, 5.1 TB/s), with gh 98 (8, 5.5), with gh and a dropped
// operand 119 (10, 5.6); the fold takes 4 to 5 of each.  With xhat = (h - m) * r and t = gy * w,
//   g  = (t - mean(t) - xhat * mean(t * xhat)) * r   [+ gh]        (RMSNorm: without mean(t))
//   gw = sum over rows of gy * xhat, gb = sum over rows of gy      (fp32)
// g is the gradient of x and of the residual alike, rounded once; with DROP that of x is drop(g), from the same bits as forward.
// A workgroup per row; the sums for gw and gb stay in registers over the rows that a workgroup sees and leave as one row of partial sums
// per workgroup, folded in order (rmsnorm_gw_fold_kernel).  Rows are requested AHEAD - 1 rows before they are used.
// Four waves of up to three chunks; longer rows take eight waves of two, one workgroup per compute unit: the parameter, its two sums and
// two rows of four chunks a lane are more than 256 registers.  Rows of up to three chunks, where there are more of them than workgroups, have
// a wave each: no barrier and no idle waves; us at [16384,256] 32.3 -> 15.1, [16384,1024] 37.5 -> 29.0, [16384,1152] 38.4 -> 33.0 (with gh, folds
// included), [2048,1536] 13.7 and 14.6.  (A wave of four chunks would need more than 256 registers.)
constexpr int bwd_waves(int wpr) { return wpr == 1 ? kNormWaves : wpr; }
template <int N, int WPR, int AHEAD, bool CENTRED, bool GH, bool DROP>
__global__ __launch_bounds__(bwd_waves(WPR) * 64, 8 / bwd_waves(WPR)) void norm_bwd_kernel(const NormBwd p) {
#if defined(__HIP_DEVICE_COMPILE__)
  static_assert(AHEAD % 2 == 0, "a buffer meets the same half of `red` every time");
  constexpr int WAVES = bwd_waves(WPR), ROWS = WAVES / WPR;
  __shared__ float red_t[2][WAVES], red_x[2][WAVES];
  __shared__ __attribute__((aligned(16))) float meet[WPR == 1 ? (CENTRED ? 2 : 1) * N * 512 : 4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int C = p.C;
  const int64_t R = p.R, stride = (int64_t)gridDim.x * ROWS;
  auto col_of = [&](int j) { return (j * WPR + (WPR == 1 ? 0 : wave)) * 512 + lane * 8; };
  float w[N][8];
  load_param<N>(w, p.w, p.w_f32, 1.0f, C, col_of);
  float gw[N][8], gb[CENTRED ? N : 1][8];
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      gw[j][e] = 0.0f;
      if constexpr (CENTRED) gb[j][e] = 0.0f;
    }
  const float inv_c = 1.0f / (float)C;
  [[maybe_unused]] DropKey key;
  if constexpr (DROP) key = drop_key(p.drop);
  v4i xb[AHEAD][N], gyb[AHEAD][N];
  [[maybe_unused]] v4i hb[N];
  float rb[AHEAD], mb[AHEAD];
  auto request = [&](int a, int64_t r) {  // a row beyond R: zeros, nothing is read
    rb[a] = p.rstd[r < R ? r : 0];
    mb[a] = CENTRED ? p.mean[r < R ? r : 0] : 0.0f;
    load_norm_row<N>(xb[a], p.h, r, R, p.ldh, C, col_of);
    load_norm_row<N>(gyb[a], p.gy, r, R, p.ldgy, C, col_of);
  };
#pragma unroll
  for (int a = 0; a < AHEAD - 1; ++a) request(a, (int64_t)blockIdx.x * ROWS + (WPR == 1 ? wave : 0) + a * stride);
  for (int64_t r0 = (int64_t)blockIdx.x * ROWS + (WPR == 1 ? wave : 0); r0 < R; r0 += AHEAD * stride) {
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int64_t r = r0 + a * stride;
      if (r >= R) break;  // the same for all waves of a row
      if constexpr (GH) load_norm_row<N>(hb, p.gh, r, R, p.ldgh, C, col_of);
      request((a + AHEAD - 1) % AHEAD, r + (AHEAD - 1) * stride);
      const v4i(&xc)[N] = xb[a], (&gc)[N] = gyb[a];
      const float rinv = rb[a], mean = mb[a];
      auto value = [](const v4i(&v)[N], int j, int e) { return (e & 1) ? hi_of(v[j][e >> 1]) : lo_of(v[j][e >> 1]); };
      auto xhat = [&](int j, int e) { return (value(xc, j, e) - mean) * rinv; };
      float st = 0.0f, sx = 0.0f, tot_x = 0.0f, tot_t = 0.0f;
#pragma unroll
      for (int j = 0; j < N; ++j) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float ge = value(gc, j, e), xh = xhat(j, e);
          gw[j][e] += ge * xh;
          if constexpr (CENTRED) gb[j][e] += ge;
          const float t = ge * w[j][e];
          if constexpr (CENTRED) st += t;
          sx += t * xh;
        }
        if constexpr (WPR == 1) {   // chunk by chunk, as the waves of the other layout meet
          tot_x += wave_sum_f32(sx);
          if constexpr (CENTRED) tot_t += wave_sum_f32(st);
          st = sx = 0.0f;
        }
      }
      if constexpr (WPR > 1) {
        sx = wave_sum_f32(sx);
        if constexpr (CENTRED) st = wave_sum_f32(st);
        if (lane == 0) {
          red_x[a & 1][wave] = sx;
          if constexpr (CENTRED) red_t[a & 1][wave] = st;
        }
        __syncthreads();
#pragma unroll
        for (int wv = 0; wv < WAVES; ++wv) {
          tot_x += red_x[a & 1][wv];
          if constexpr (CENTRED) tot_t += red_t[a & 1][wv];
        }
      }
      const float cx = tot_x * inv_c, ct = tot_t * inv_c;
      const __amdgpu_buffer_rsrc_t rsG = make_rsrc(p.gx + r * p.ldgx, (uint32_t)C * 2u);
      [[maybe_unused]] const __amdgpu_buffer_rsrc_t rsR = make_rsrc(DROP ? p.gres + r * p.ldgres : p.gx, DROP ? (uint32_t)C * 2u : 0u);
      [[maybe_unused]] const uint64_t group0 = (uint64_t)r * (uint32_t)(C / 8);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        [[maybe_unused]] uint32_t words[4];
        if constexpr (DROP) drop_words(words, key, group0 + (uint32_t)(col_of(j) / 8));
        v4i out, dropped;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          auto grad = [&](int e) {
            const float t = value(gc, j, e) * w[j][e];
            float g = ((CENTRED ? t - ct : t) - xhat(j, e) * cx) * rinv;
            if constexpr (GH) g += value(hb, j, e);
            return g;
          };
          const float lo = grad(2 * k), hi = grad(2 * k + 1);
          out[k] = pack2(lo, hi);
          if constexpr (DROP) dropped[k] = pack2(drop_one(lo, words, 2 * k, p.drop), drop_one(hi, words, 2 * k + 1, p.drop));
        }
        if constexpr (DROP) {
          store16_nt(rsR, (uint32_t)col_of(j) * 2u, out);
          store16_nt(rsG, (uint32_t)col_of(j) * 2u, dropped);
        } else {
          store16_nt(rsG, (uint32_t)col_of(j) * 2u, out);
        }
      }
    }
  }
  if (!p.partials) return;
  if constexpr (WPR == 1) {   // the waves' sums meet in LDS, one wave after the other; the last one has them all
    for (int wv = 0; wv < WAVES; ++wv) {
      if (wave == wv) {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
          for (int part = 0; part < (CENTRED ? 2 : 1); ++part) {
            float(&mine)[8] = part ? gb[CENTRED ? j : 0] : gw[j];
            float *at = &meet[(part * N + j) * 512 + lane * 8];
            if (wv > 0) {
#pragma unroll
              for (int e = 0; e < 8; ++e) mine[e] = at[e] + mine[e];
            }
            if (wv < WAVES - 1) {
#pragma unroll
              for (int e = 0; e < 8; ++e) at[e] = mine[e];
            }
          }
      }
      __syncthreads();
    }
    if (wave != WAVES - 1) return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = col_of(j);
    if (c < C) {
      float *dst = p.partials + (int64_t)blockIdx.x * (CENTRED ? 2 * C : C) + c;
      *(v4f *)dst = v4f{gw[j][0], gw[j][1], gw[j][2], gw[j][3]};
      *(v4f *)(dst + 4) = v4f{gw[j][4], gw[j][5], gw[j][6], gw[j][7]};
      if constexpr (CENTRED) {
        *(v4f *)(dst + C) = v4f{gb[j][0], gb[j][1], gb[j][2], gb[j][3]};
        *(v4f *)(dst + C + 4) = v4f{gb[j][4], gb[j][5], gb[j][6], gb[j][7]};
      }
    }
  }
#endif
}

template <int N, int WPR, bool CENTRED, bool ADD, bool DROP>
static int launch_fwd(const NormFwd &p, float *col_amax, hipStream_t st) {
  int64_t blocks = norm_blocks(WPR == 1 ? (p.R + kNormWaves - 1) / kNormWaves : p.R);
  // (three a unit, where no row of partial maxima goes with each and the registers allow it; us at [16384,1152] 23.9 -> 21.6 with the cast,
  // [16384,256] 12.4 -> 10.7; four a unit 21.4 but 31.5 and not 29.2 with a residual)
  if (WPR == 1 && N <= 3 && !col_amax) blocks = std::min<int64_t>((p.R + kNormWaves - 1) / kNormWaves, 3 * (int64_t)num_cus());
  auto go = [&](auto kernel, size_t lds) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kNormBlock), lds, st, p); };
  if (col_amax) go(norm_fwd_kernel<N, WPR, CENTRED, ADD, DROP, true>, WPR == 1 ? (size_t)p.C * 2 : 0);
  else go(norm_fwd_kernel<N, WPR, CENTRED, ADD, DROP, false>, 0);
  L8_HIP(hipGetLastError());
  return col_amax ? fold_colmax(p.col_partials, blocks, p.C, col_amax, st) : L8_OK;
}

template <bool CENTRED, bool ADD, bool DROP>
static int launch_fwd_for(const NormFwd &p, float *col_amax, hipStream_t st) {
  const int nch = (p.C + 511) / 512, n = (nch + kNormWaves - 1) / kNormWaves;
  if (nch <= 4 && p.R > norm_blocks(p.R)) {
    if (nch <= 1) return launch_fwd<1, 1, CENTRED, ADD, DROP>(p, col_amax, st);
    if (nch <= 2) return launch_fwd<2, 1, CENTRED, ADD, DROP>(p, col_amax, st);
    if (nch <= 3) return launch_fwd<3, 1, CENTRED, ADD, DROP>(p, col_amax, st);
    return launch_fwd<4, 1, CENTRED, ADD, DROP>(p, col_amax, st);
  }
  if (n <= 1) return launch_fwd<1, kNormWaves, CENTRED, ADD, DROP>(p, col_amax, st);
  if (n <= 2) return launch_fwd<2, kNormWaves, CENTRED, ADD, DROP>(p, col_amax, st);
  if (n <= 3) return launch_fwd<3, kNormWaves, CENTRED, ADD, DROP>(p, col_amax, st);
  return launch_fwd<4, kNormWaves, CENTRED, ADD, DROP>(p, col_amax, st);
}

template <int N, int WPR, bool CENTRED, bool GH, bool DROP>
static int launch_bwd(const NormBwd &p, const GradOut &gw, const GradOut &gb, hipStream_t st) {
  const int64_t most = norm_blocks(WPR == 1 ? (p.R + kNormWaves - 1) / kNormWaves : p.R), blocks = WPR > kNormWaves && most > num_cus() ? num_cus() : most;
  hipLaunchKernelGGL((norm_bwd_kernel<N, WPR, N == 1 ? 4 : 2, CENTRED, GH, DROP>), dim3((unsigned)blocks), dim3(bwd_waves(WPR) * 64), 0, st, p);
  L8_HIP(hipGetLastError());
  return p.partials ? fold_norm_grads(p.partials, blocks, gw, gb, st) : L8_OK;
}

template <bool CENTRED, bool GH, bool DROP>
static int launch_bwd_for(const NormBwd &p, const GradOut &gw, const GradOut &gb, hipStream_t st) {
  const int nch = (p.C + 511) / 512, n = (nch + kNormWaves - 1) / kNormWaves;
  if (nch <= 3 && p.R > norm_blocks(p.R)) {
    if (nch <= 1) return launch_bwd<1, 1, CENTRED, GH, DROP>(p, gw, gb, st);
    if (nch <= 2) return launch_bwd<2, 1, CENTRED, GH, DROP>(p, gw, gb, st);
    return launch_bwd<3, 1, CENTRED, GH, DROP>(p, gw, gb, st);
  }
  if (n <= 1) return launch_bwd<1, kNormWaves, CENTRED, GH, DROP>(p, gw, gb, st);
  if (n <= 2) return launch_bwd<2, kNormWaves, CENTRED, GH, DROP>(p, gw, gb, st);
  if (n <= 3) return launch_bwd<3, kNormWaves, CENTRED, GH, DROP>(p, gw, gb, st);
  return launch_bwd<2, 2 * kNormWaves, CENTRED, GH, DROP>(p, gw, gb, st);
}

static bool on_lines(const void *p, int64_t ld, int64_t C) { return ((uintptr_t)p % 16) == 0 && ld % 8 == 0 && ld >= C; }

}  // namespace l8

using namespace l8;

extern "C" int l8_norm_fwd(const l8_norm_fwd_args *a) {
  L8_REQUIRE(a, "l8_norm_fwd: null pointer");
  const int64_t R = a->R, C = a->C;
  L8_REQUIRE(R >= 0 && C >= 0, "l8_norm_fwd: negative shape R=%lld C=%lld", (long long)R, (long long)C);
  hipStream_t st = (hipStream_t)a->stream;
  NormFwd p{};
  const int code = drop_of("l8_norm_fwd", a->numbers, a->site, a->threshold, &p.drop);
  if (code != L8_OK) return code;
  if (R == 0 || C == 0) return empty_col_amax(a->col_amax, C, st);
  L8_REQUIRE(a->x && a->y && (!a->residual || a->h), "l8_norm_fwd: null pointer");
  L8_REQUIRE(a->centred || (a->w && !a->b && a->residual && a->numbers), "l8_norm_fwd: an RMSNorm here is that of a sum with a dropped operand, with a weight and no bias");
  L8_REQUIRE(!a->numbers || a->residual, "l8_norm_fwd: a dropped operand needs a residual");
  L8_REQUIRE((a->q == nullptr) == (a->scale == nullptr), "l8_norm_fwd: pass q and scale together");
  L8_REQUIRE(C % 8 == 0 && C <= kNormMaxC, "l8_norm_fwd: C=%lld must be a multiple of 8 up to %lld", (long long)C, (long long)kNormMaxC);
  L8_REQUIRE(on_lines(a->x, a->ldx, C) && on_lines(a->y, a->ldy, C) && (!a->residual || (on_lines(a->residual, a->ldr, C) && on_lines(a->h, a->ldh, C))),
             "l8_norm_fwd: the bf16 operands must be 16-byte aligned, their leading dimensions multiples of 8 and at least C");
  L8_REQUIRE(!a->q || (((uintptr_t)a->q % 8) == 0 && a->ldq % 8 == 0 && a->ldq >= C), "l8_norm_fwd: q must be 8-byte aligned, its leading dimension a multiple of 8 and at least C");
  L8_REQUIRE(((uintptr_t)a->w % (a->w_is_f32 ? 4 : 2)) == 0 && ((uintptr_t)a->b % (a->b_is_f32 ? 4 : 2)) == 0, "l8_norm_fwd: misaligned parameter");
  L8_REQUIRE(!a->col_amax || a->q, "l8_norm_fwd: column amaxes come with the cast");
  if (a->col_amax) {
    const int64_t need = l8_rmsnorm_workspace(R, C);
    L8_REQUIRE(a->workspace && a->workspace_bytes >= need && ((uintptr_t)a->workspace % 16) == 0, "l8_norm_fwd: col_amax needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  }
  p.x = (const uint16_t *)a->x, p.residual = (const uint16_t *)a->residual, p.w = a->w, p.b = a->b;
  p.h = (uint16_t *)a->h, p.y = (uint16_t *)a->y, p.q = (uint8_t *)a->q, p.scale = a->scale;
  p.mean = a->mean, p.rstd = a->rstd, p.col_partials = (uint16_t *)a->workspace;
  p.R = R, p.ldx = a->ldx, p.ldr = a->ldr, p.ldh = a->ldh, p.ldy = a->ldy, p.ldq = a->ldq;
  p.C = (int)C, p.w_f32 = a->w_is_f32 != 0, p.b_f32 = a->b_is_f32 != 0, p.scale_rule = scale_rule(), p.eps = (float)a->eps;
  if (!a->centred) return launch_fwd_for<false, true, true>(p, a->col_amax, st);
  if (a->numbers) return launch_fwd_for<true, true, true>(p, a->col_amax, st);
  if (a->residual) return launch_fwd_for<true, true, false>(p, a->col_amax, st);
  return launch_fwd_for<true, false, false>(p, a->col_amax, st);
}

extern "C" int64_t l8_norm_bwd_workspace(int64_t R, int64_t C, int64_t centred) {
  if (R <= 0 || C <= 0) return 0;
  return norm_blocks(R) * C * (centred ? 2 : 1) * (int64_t)sizeof(float);
}

extern "C" int l8_norm_bwd(const l8_norm_bwd_args *a) {
  L8_REQUIRE(a, "l8_norm_bwd: null pointer");
  const int64_t R = a->R, C = a->C;
  L8_REQUIRE(R >= 0 && C >= 0, "l8_norm_bwd: negative shape R=%lld C=%lld", (long long)R, (long long)C);
  hipStream_t st = (hipStream_t)a->stream;
  NormBwd p{};
  const int code = drop_of("l8_norm_bwd", a->numbers, a->site, a->threshold, &p.drop);
  if (code != L8_OK) return code;
  if (C == 0) return L8_OK;
  L8_REQUIRE(C % 8 == 0 && C <= kNormMaxC, "l8_norm_bwd: C=%lld must be a multiple of 8 up to %lld", (long long)C, (long long)kNormMaxC);
  const GradOut gw{a->gw, a->gw_is_f32 != 0, (int)C}, gb{a->gb, a->gb_is_f32 != 0, a->centred ? (int)C : 0};
  if (R == 0) return gw.p || gb.p ? fold_norm_grads(nullptr, 0, gw, gb, st) : L8_OK;   // no rows: the sums over them are zero
  L8_REQUIRE(a->gy && a->h && a->gx && a->rstd && (!a->centred || a->mean), "l8_norm_bwd: null pointer");
  L8_REQUIRE(a->centred || (a->w && !a->gb && a->numbers), "l8_norm_bwd: an RMSNorm here is that of a sum with a dropped operand, with a weight and no bias");
  L8_REQUIRE((a->numbers == nullptr) == (a->gres == nullptr), "l8_norm_bwd: a dropped operand's sum has a gradient of its own, and only that");
  L8_REQUIRE(on_lines(a->gy, a->ldgy, C) && on_lines(a->h, a->ldh, C) && on_lines(a->gx, a->ldgx, C) && (!a->gh || on_lines(a->gh, a->ldgh, C)) &&
                 (!a->gres || on_lines(a->gres, a->ldgres, C)),
             "l8_norm_bwd: the bf16 operands must be 16-byte aligned, their leading dimensions multiples of 8 and at least C");
  L8_REQUIRE(((uintptr_t)a->w % (a->w_is_f32 ? 4 : 2)) == 0, "l8_norm_bwd: misaligned parameter");
  if (gw.p || gb.p) {
    const int64_t need = l8_norm_bwd_workspace(R, C, a->centred);
    L8_REQUIRE(a->workspace && a->workspace_bytes >= need && ((uintptr_t)a->workspace % 16) == 0, "l8_norm_bwd: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
    p.partials = (float *)a->workspace;
  }
  p.gy = (const uint16_t *)a->gy, p.gh = (const uint16_t *)a->gh, p.h = (const uint16_t *)a->h, p.w = a->w;
  p.mean = a->mean, p.rstd = a->rstd, p.gx = (uint16_t *)a->gx, p.gres = (uint16_t *)a->gres;
  p.R = R, p.ldgy = a->ldgy, p.ldgh = a->ldgh, p.ldh = a->ldh, p.ldgx = a->ldgx, p.ldgres = a->ldgres;
  p.C = (int)C, p.w_f32 = a->w_is_f32 != 0;
#define L8_GO(CENTRED, DROP) return p.gh ? launch_bwd_for<CENTRED, true, DROP>(p, gw, gb, st) : launch_bwd_for<CENTRED, false, DROP>(p, gw, gb, st)
  if (!a->centred) L8_GO(false, true);
  if (a->numbers) L8_GO(true, true);
  L8_GO(true, false);
#undef L8_GO
}
