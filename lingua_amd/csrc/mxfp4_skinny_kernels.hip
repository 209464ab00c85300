// Products of a few tokens with a weight kept in MXFP4: y[M,N] = bf16(x[M,K] . w[N,K]^T + bias), M <= 64.
//
// Every weight byte is used for a handful of tokens, so the bytes per second of the weight are what counts: 17/32 byte per element,
// 9 MiB of a [4096,4096] one.  A workgroup owns 16 weight rows (or 32) and all tokens:
//
//   * its eight waves share K out in windows of 512 columns (256 bytes of codes, 16 scales of a row), each wave a run of neighbours, so
//     a small weight still puts a thousand waves to work and no wave waits for another;
//   * codes are read in whole lines, 16 lanes to a row, and turned into the matrix instruction's layout through 4 KiB of LDS of the
//     wave's own (operations of one wave are served in order: no barrier).  16-byte chunk c of row r lives at chunk c ^ r: the reads
//     of 16 rows cover all banks once;
//   * lane group g of the four takes blocks 4 g .. 4 g + 3 of a window, one per instruction: its four scale bytes are one dword, picked
//     apart by the instruction's op_sel;
//   * a few tokens come in bf16 and are quantised on the way: 64 lanes hold a row's window, four lanes a block, and the codes and
//     scales are written to LDS in the layout that they are read in.  Every workgroup does it over again, so where that is much
//     (quantised_inside below) a launch of their own casts them;
//   * the eight partial tiles meet in LDS and are added in the order of the waves.
#include "mxfp4.h"

namespace l8 {

constexpr int kFewWaves = 8, kFewBlock = kFewWaves * 64;
constexpr int kWindow = 512, kWinBytes = 256;   // columns, bytes of codes
constexpr int kFewTile = 16 * kWinBytes;        // 16 rows of a window
[[maybe_unused]] constexpr uint32_t kBeyondAll = 0x80000000u;

// MT tiles of 16 tokens, NT of 16 weight rows.  QX: x in bf16, one tile of tokens.
template <int MT, int NT, bool QX>
__global__ __launch_bounds__(kFewBlock) void linear_mxfp4_few_kernel(const MxFewArgs p) {
#if defined(__HIP_DEVICE_COMPILE__)
  static_assert(!QX || MT == 1, "x is quantised for one tile of tokens");
  constexpr int kBuf = kFewTile + (QX ? 256 : 0), kRed = MT * NT * 1024;   // (every tile of a wave goes through one buffer)
  __shared__ __attribute__((aligned(16))) uint8_t lds[kFewWaves * (kBuf > kRed ? kBuf : kRed)];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * (16 * NT);
  const int kbytes = p.blocks * 16, windows = (p.blocks + 15) >> 4;
  const int share = (windows + kFewWaves - 1) / kFewWaves;
  const int w_first = wave * share, w_last = w_first + share < windows ? w_first + share : windows;
  uint8_t *const buf = lds + wave * kBuf;
  uint32_t *const xsc = (uint32_t *)(buf + kFewTile);   // QX: scales of 16 tokens, a dword per lane group

  auto range = [](int64_t n) { return n < 0x7fffffff ? (uint32_t)n : 0x7fffffffu; };
  const __amdgpu_buffer_rsrc_t rsW = make_rsrc(p.qw + (int64_t)n0 * p.ldqw, range((int64_t)(p.N - n0 - 1) * p.ldqw + kbytes));
  const __amdgpu_buffer_rsrc_t rsX = QX ? make_rsrc(p.x, range(((int64_t)(p.M - 1) * p.ldx + p.K) * 2)) : make_rsrc(p.x, range((int64_t)(p.M - 1) * p.ldx + kbytes));
  // loads: four rows at a time, 16 lanes to a row
  const int lrow = lane >> 4, lchunk = lane & 15;
  // fragments: lane (g, r) = 16 g + r
  const int fr = lane & 15, fg = lane >> 4;
  auto put = [&](int r, int c) { return r * kWinBytes + ((c ^ r) & 15) * 16; };
  auto load_codes = [&](__amdgpu_buffer_rsrc_t rs, int64_t ld, int row0, int w, v4i (&v)[4], bool once) {
    const int k = w * kWinBytes + lchunk * 16;
    const uint32_t off = (uint32_t)((row0 + lrow) * (int)ld + k) | (k < kbytes ? 0u : kBeyondAll);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = once ? load16_nt(rs, off, (uint32_t)(j * 4 * (int)ld)) : __builtin_amdgcn_raw_buffer_load_b128(rs, (int)off, j * 4 * (int)ld, 0);
  };
  // scales of blocks 4 g .. 4 g + 3 of the window, of row `row` (which may not exist); bytes behind K are zeros
  auto load_scale = [&](const uint8_t *s, int64_t ld, int row, int rows, int w) {
    uint32_t v = 0;
    const int first = w * 16 + fg * 4;
    if (row < rows) {
      const uint8_t *at = s + (int64_t)row * ld + first;
      if (first + 4 <= p.blocks) {
        __builtin_memcpy(&v, at, 4);
      } else {
#pragma unroll
        for (int k = 0; k < 3; ++k)
          if (first + k < p.blocks) v |= (uint32_t)at[k] << (8 * k);
      }
    }
    return v;
  };
  auto turn = [&](const v4i (&v)[4], v4i (&f)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) *(v4i *)(buf + put(j * 4 + lrow, lchunk)) = v[j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int s = 0; s < 4; ++s) f[s] = *(const v4i *)(buf + put(fr, fg * 4 + s));
    __builtin_amdgcn_wave_barrier();
  };

  v4f acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  auto mma = [&](const v4i (&wf)[4], uint32_t ws, const v4i (&xf)[4], uint32_t xs, v4f c) {
    auto wide = [](v4i v) { return v8i{v[0], v[1], v[2], v[3], 0, 0, 0, 0}; };
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(wf[0]), wide(xf[0]), c, 4, 4, 0, (int)ws, 0, (int)xs);
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(wf[1]), wide(xf[1]), c, 4, 4, 1, (int)ws, 1, (int)xs);
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(wf[2]), wide(xf[2]), c, 4, 4, 2, (int)ws, 2, (int)xs);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(wf[3]), wide(xf[3]), c, 4, 4, 3, (int)ws, 3, (int)xs);
  };
  for (int w = w_first; w < w_last; ++w) {
    v4i wv[NT][4];
    uint32_t ws[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      load_codes(rsW, p.ldqw, t * 16, w, wv[t], true);
      ws[t] = load_scale(p.sw, p.ldsw, n0 + t * 16 + fr, p.N, w);
    }
    v4i xf[MT][4];
    uint32_t xs[MT];
    if constexpr (QX) {
      const int c = w * kWindow + lane * 8;
      const uint32_t off = (uint32_t)(c * 2) | (c < p.K ? 0u : kBeyondAll);
      // (rows of tokens that are not there keep whatever LDS holds: it only reaches columns of the accumulators that nobody stores)
      // two rows requested together: 8 tokens, [4096,4096] 6.3 -> 5.8 us, [32000,4096] 21.5 -> 20.2; with four 5.6 and 21.3, their registers
      // cost one token through [32000,4096] 13.2 -> 14.0
      constexpr int AT_ONCE = 2;
      for (int m0 = 0; m0 < p.M; m0 += AT_ONCE) {
        v4i v[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) v[u] = __builtin_amdgcn_raw_buffer_load_b128(rsX, (int)off, (m0 + u) * (int)p.ldx * 2, 0);
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
          if (m0 + u >= p.M) break;
          const uint32_t byte = mx_byte(quad_max(amax8(v[u])));
          const uint32_t codes = byte == 255u ? 0u : mx_codes8((uint32_t)v[u][0], (uint32_t)v[u][1], (uint32_t)v[u][2], (uint32_t)v[u][3], mx_scale(byte));
          const uint32_t four = byte | dpp<0x104>(byte) << 8 | dpp<0x108>(byte) << 16 | dpp<0x10C>(byte) << 24;
          *(uint32_t *)(buf + put(m0 + u, lane >> 2) + (lane & 3) * 4) = codes;
          if (lchunk == 0) xsc[(m0 + u) * 4 + lrow] = four;
        }
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int s = 0; s < 4; ++s) xf[0][s] = *(const v4i *)(buf + put(fr, fg * 4 + s));
      xs[0] = xsc[fr * 4 + fg];
      __builtin_amdgcn_wave_barrier();
    } else {
      v4i v[MT][4];   // all tiles requested, then turned: 64 tokens, [4096,4096] 9.6 -> 9.4 us, [8192,2048] 9.6 -> 9.2
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        load_codes(rsX, p.ldx, i * 16, w, v[i], false);
        xs[i] = load_scale(p.sx, p.ldsx, i * 16 + fr, p.M, w);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) turn(v[i], xf[i]);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      v4i wf[4];
      turn(wv[t], wf);
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i][t] = mma(wf, ws[t], xf[i], xs[i], acc[i][t]);
    }
  }
  __syncthreads();
  v4f *const red = (v4f *)lds;   // [wave][MT * NT][lane]
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) red[(wave * MT * NT + i * NT + t) * 64 + lane] = acc[i][t];
  __syncthreads();
  for (int tile = wave; tile < MT * NT; tile += kFewWaves) {
    v4f sum = red[tile * 64 + lane];
#pragma unroll
    for (int v = 1; v < kFewWaves; ++v) {
      const v4f o = red[(v * MT * NT + tile) * 64 + lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += o[e];
    }
    const int m = tile / NT * 16 + fr, n = n0 + tile % NT * 16 + fg * 4;   // four neighbouring columns
    if (m >= p.M) continue;
    uint16_t out[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = (uint16_t)bf16_rne_bits(sum[e] + (p.bias && n + e < p.N ? bf16_bits_to_f32(p.bias[n + e]) : 0.0f));
    uint16_t *const dst = p.y + (int64_t)m * p.ldy + n;
    if (n + 4 <= p.N && ((uintptr_t)dst & 7) == 0) {
      v2i packed;
      __builtin_memcpy(&packed, out, 8);
      *(v2i *)dst = packed;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.N) dst[e] = out[e];
    }
  }
#endif
}

// Rows of scales onto 16-byte lines, where the product's tiles want them: 16 bytes a thread.
__global__ __launch_bounds__(256) void mxfp4_scales_on_lines_kernel(const uint8_t *__restrict__ s, int64_t lds, int64_t rows, int blocks, uint8_t *__restrict__ t, int pieces) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / pieces;
  if (row >= rows) return;
  const int first = (int)(i - row * pieces) * 16;
  const uint8_t *const at = s + row * lds + first;
  uint32_t v[4] = {0, 0, 0, 0};
  if (first + 16 <= blocks) {
    __builtin_memcpy(v, at, 16);
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (first + k < blocks) v[k >> 2] |= (uint32_t)at[k] << (8 * (k & 3));
  }
  *(v4i *)(t + i * 16) = v4i{(int)v[0], (int)v[1], (int)v[2], (int)v[3]};
#endif
}

template <int MT, int NT, bool QX>
static int launch_few(const MxFewArgs &a, hipStream_t st) {   // (fewer than 2^32 threads: the entry sees to it)
  hipLaunchKernelGGL((linear_mxfp4_few_kernel<MT, NT, QX>), dim3((unsigned)((a.N + 16 * NT - 1) / (16 * NT))), dim3(kFewBlock), 0, st, a);
  L8_HIP(hipGetLastError());
  return L8_OK;
}

// One window in flight per wave: the registers that more would take are worth more as a second workgroup on the unit.  us, four
// windows / one: one token, [11008,4096] 9.7 / 6.9, [4096,4096] 5.1 / 4.4.
static int mxfp4_few_bf16(const MxFewArgs &a, hipStream_t st) { return launch_few<1, 1, true>(a, st); }
// Two tiles of weight rows to a workgroup, which share the tokens' codes, where six in ten units still get one and the tokens are more
// than one tile.  us, one tile / two: 32 tokens, [8192,2048] 8.3 / 7.9, [5504,4096] 9.8 / 9.2, [4096,4096] 8.0 / 8.9; 64 tokens,
// [8192,2048] 11.3 / 9.4, [5504,4096] 13.4 / 10.9, [4096,4096] 9.5 / 10.4; 16 tokens, [11008,4096] 10.5 / 11.0, [8192,2048] 6.8 / 7.2.
static int64_t enough_groups() { return num_cus() * 6 / 10; }
static int mxfp4_few_packed(const MxFewArgs &a, hipStream_t st) {
  if (a.M <= 16) return launch_few<1, 1, false>(a, st);
  const bool two = a.N >= enough_groups() * 32;
  if (a.M <= 32) return two ? launch_few<2, 2, false>(a, st) : launch_few<2, 1, false>(a, st);
  return two ? launch_few<4, 2, false>(a, st) : launch_few<4, 1, false>(a, st);
}

}  // namespace l8

using namespace l8;

// Do the kernels above take the problem?  Beyond one tile of tokens a weight of a row of tiles for six in ten units is the product's.  us,
// here / there: 32 tokens, [8192,8192] 15.5 / 16.9, [11008,4096] 11.4 / 11.1, [22016,8192] 33.4 / 29.6, [32000,4096] 21.6 / 19.5; 64 tokens,
// [4096,11008] 16.3 / 18.7, [8192,8192] 18.4 / 17.9, [11008,4096] 13.5 / 11.3, [32000,4096] 25.8 / 20.3.
static bool few_tokens(int64_t M, int64_t N) { return M <= 16 || (M <= 64 && N < enough_groups() * 64); }

// Are the tokens quantised inside the product?  Every workgroup does it over again, a wave for each of its windows, and that is set
// against a launch and a pass over the tokens; where a unit has several workgroups one after the other it counts as often.  us, inside /
// cast before:
//   one window a wave   [4096,4096]   4 tokens 5.0 / 6.5, 8: 6.1 / 7.0, 12: 6.9 / 7.0   [32000,4096]  4: 15.7 / 15.8, 6: 18.0 / 15.9
//                                                                                       [11008,4096]  4: 7.8 / 8.9, 6: 9.0 / 9.0
//   two                 [4096,8192]   4 tokens 7.7 / 9.1, 6: 8.8 / 8.7, 8: 9.7 / 8.7    [22016,8192]  3: 21.2 / 22.2, 5: 24.1 / 22.5
//   three               [4096,11008]  2 tokens 8.0 / 9.5, 4: 9.6 / 10.0, 5: 10.9 / 10.2 [11008,11008] 3: 16.5 / 17.2, 4: 17.6 / 17.3
//   four                [512,16384]   2 tokens 7.6 / 9.1, 3: 9.7 / 9.1                  [8192,16384]  3: 16.5 / 19.4, 6: 20.5 / 19.7
static bool quantised_inside(int64_t M, int64_t N, int64_t K) {
  const int64_t share = ((K + kWindow - 1) / kWindow + kFewWaves - 1) / kFewWaves;   // windows a wave
  return M == 1 || (M <= (N < enough_groups() * 64 ? 8 : 4) && M * share <= 12);
}

// Codes and scales of the activation in the workspace, then the product's own.
struct MxLinearPlan {
  int64_t ldq, lds, q, s, product, scales, total;   // scales: of the weight, on lines
};
static MxLinearPlan plan_of(int64_t M, int64_t N, int64_t K) {
  const int64_t blocks = (K + 31) / 32;
  MxLinearPlan p;
  p.ldq = (blocks * 16 + 127) / 128 * 128;
  p.lds = (blocks + 15) / 16 * 16;
  p.q = 0;
  p.s = p.q + M * p.ldq;
  p.product = p.s + (M * p.lds + 15) / 16 * 16;
  const bool few = few_tokens(M, N);
  p.scales = p.product + (few ? 0 : (l8_gemm_mxfp4_workspace(M, N, K) + 15) / 16 * 16);
  p.total = quantised_inside(M, N, K) ? 0 : p.scales + (few ? 0 : N * p.lds);
  return p;
}

extern "C" int64_t l8_mxfp4_linear_workspace(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return plan_of(M, N, K).total;
}

extern "C" int l8_mxfp4_linear(const void *x, int64_t M, int64_t K, int64_t ldx, const void *qw, int64_t ldqw, const void *sw, int64_t ldsw, int64_t N,
                               const void *bias, void *y, int64_t ldy, void *workspace, int64_t workspace_bytes, void *stream) {
  L8_REQUIRE(M >= 0 && N >= 0 && K >= 0, "l8_mxfp4_linear: negative shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (M == 0 || N == 0) return L8_OK;
  const int64_t blocks = (K + 31) / 32;
  L8_REQUIRE(y && ldy >= N && ((uintptr_t)y % 2) == 0 && ((uintptr_t)bias % 2) == 0, "l8_mxfp4_linear: null or misaligned y, or ldy < N");
  L8_REQUIRE(K == 0 || (x && qw && sw), "l8_mxfp4_linear: null pointer");
  L8_REQUIRE(K == 0 || (K % 8 == 0 && ldx % 8 == 0 && ldx >= K && ((uintptr_t)x % 16) == 0), "l8_mxfp4_linear: K=%lld and ldx must be multiples of 8, x 16-byte aligned", (long long)K);
  L8_REQUIRE(M < (1 << 20) - 16 && N < (1 << 28) && K < (1 << 24), "l8_mxfp4_linear: M < 2^20 - 16, N < 2^28 and K < 2^24 are served");
  // (a workgroup for 16 weight rows, of 512 threads: fewer than 2^32 of them)
  L8_REQUIRE(!few_tokens(M, N) || N <= (1 << 27) - 16, "l8_mxfp4_linear: N <= 2^27 - 16 is served for up to 16 tokens");
  if (K == 0) ldx = ldqw = ldsw = 0, x = qw = sw = nullptr;
  L8_REQUIRE(ldqw % 16 == 0 && ldqw >= blocks * 16 && ldqw <= (1 << 23) - 16 && ((uintptr_t)qw % 16) == 0 && ldsw >= blocks,
             "l8_mxfp4_linear: rows of codes on 16-byte lines less than 2^23 bytes apart, and a scale per block, are wanted");
  const MxLinearPlan plan = plan_of(M, N, K);
  const bool move_scales = !few_tokens(M, N) && (ldsw % 16 || ldsw > (1 << 23) - 16 || ((uintptr_t)sw % 16));
  const int64_t pieces = plan.lds / 16, move_groups = (N * pieces + 255) / 256;
  L8_REQUIRE(!move_scales || move_groups < (1 << 24), "l8_mxfp4_linear: more scales to copy than a grid has threads");
  L8_REQUIRE(plan.total == 0 || (workspace && workspace_bytes >= plan.total && ((uintptr_t)workspace % 16) == 0),
             "l8_mxfp4_linear: needs a 16-byte aligned workspace of %lld bytes", (long long)plan.total);
  hipStream_t st = (hipStream_t)stream;
  MxFewArgs a = {x, nullptr, (const uint8_t *)qw, (const uint8_t *)sw, ldx, 0, ldqw, ldsw, (const uint16_t *)bias, (uint16_t *)y, ldy, (int)M, (int)N, (int)K, (int)blocks};
  if (quantised_inside(M, N, K)) {
    L8_REQUIRE(ldx <= (1 << 25), "l8_mxfp4_linear: rows of x further apart than 2^25 elements");   // (32-bit offsets)
    return mxfp4_few_bf16(a, st);
  }
  uint8_t *const ws = (uint8_t *)workspace;
  const int rc = l8_cast_mxfp4(x, M, K, ldx, ws + plan.q, plan.ldq, ws + plan.s, plan.lds, nullptr, 0, nullptr, 0, stream);
  if (rc != L8_OK) return rc;
  if (few_tokens(M, N)) {
    a.x = ws + plan.q, a.ldx = plan.ldq, a.sx = ws + plan.s, a.ldsx = plan.lds;
    return mxfp4_few_packed(a, st);
  }
  if (move_scales) {   // a launch of 3 us
    hipLaunchKernelGGL(mxfp4_scales_on_lines_kernel, dim3((unsigned)move_groups), dim3(256), 0, st, (const uint8_t *)sw, ldsw, N, (int)blocks, ws + plan.scales, (int)pieces);
    L8_HIP(hipGetLastError());
    sw = ws + plan.scales, ldsw = plan.lds;
  }
  return l8_gemm_mxfp4_nt(ws + plan.q, ws + plan.s, qw, sw, M, N, K, plan.ldq, plan.lds, ldqw, ldsw, bias, y, ldy, ws + plan.product,
                          plan.scales - plan.product, stream);
}
