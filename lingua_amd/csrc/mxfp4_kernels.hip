// MXFP4 casts: bf16 to e2m1 codes in blocks of 32 with one power-of-two scale (e8m0) each, along the rows of a matrix, along its
// columns (written transposed), or both from one read; and back to bf16.  The format is the OCP Microscaling one (version 1.0):
//
//   byte = max(E - 2, 0)   E the biased exponent of the block's amax: 2^(byte - 127) = 2^(floor(log2 amax) - 2)
//   code = e2m1(x * 2^(127 - byte))   nearest even, saturating at 6, sign kept
//   a block that holds an infinity or a NaN: byte 255 (NaN), codes 0
//
// All of it is integer work on the exponent and one conversion instruction (v_cvt_scalef32_pk_fp4_bf16), exact by definition: no
// rounding but the format's own.
//
// Bound by memory: 2 bytes read and 17/32 written per element and direction.  Both directions in one pass, us (TB/s): [16384,4096]
// 37.9 (5.4), [16384,11008] 121.6 (4.5), [11008,4096] 28.0 (4.9), [4096,4096] 12.5, [2064,2048] 5.2.
//   * rows: a lane takes 8 columns (16 bytes), four neighbours share a block: its amax takes two DPP steps, the four lanes' codes
//     leave as 16 bytes side by side;
//   * columns: a workgroup passes a tile of 256 rows x 128 columns through LDS, so that rows are read in 256-byte pieces and the
//     transposed copy is written in whole 128-byte lines: 8 lanes side by side take the 8 blocks of one column.  The block index
//     shifts a lane's LDS address by 8 banks, so the lanes of a read touch no bank twice.  Where such tiles would
//     leave units without work, tiles of 64 rows: [1021,2048] 7.4 -> 4.5 us.
#include "mxfp4.h"

namespace l8 {

constexpr int kMxTileC = 128;

struct MxCastArgs {
  const uint16_t *x;
  int64_t R, C, ldx;
  uint8_t *q, *s, *qt, *st;                  // row-wise copy and its scales, transposed copy and its scales (NULL: not wanted)
  int64_t ldq, lds, ldqt, ldst;              // bytes
};

// Operands of one launch of the tile kernel: the second's tiles come behind the first's.
struct MxCastTiles {
  MxCastArgs op[2];
  int across[2], first;   // tiles side by side; tiles of the first operand
};

#if defined(__HIP_DEVICE_COMPILE__)
// Eight columns of a row from c on (a lane; zeros beyond C): the block's codes and scale, the four scales of 16 lanes as one
// dword where all four exist.
L8_DEV void cast_row_piece(const MxCastArgs &p, v4i v, int64_t r, int64_t c) {
  const uint32_t byte = mx_byte(quad_max(amax8(v)));
  const uint32_t codes = byte == 255u ? 0u : mx_codes8((uint32_t)v[0], (uint32_t)v[1], (uint32_t)v[2], (uint32_t)v[3], mx_scale(byte));
  const int64_t padded = (p.C + kMxBlock - 1) / kMxBlock * kMxBlock;
  // lanes 0, 4, 8, 12 of a row of 16 hold the four bytes of 128 columns
  const uint32_t four = byte | dpp<0x104>(byte) << 8 | dpp<0x108>(byte) << 16 | dpp<0x10C>(byte) << 24;
  if (r >= p.R || c >= padded) return;
  *(uint32_t *)(p.q + r * p.ldq + c / 2) = codes;
  const int lane16 = threadIdx.x & 15;
  if (c - lane16 * 8 + 128 <= padded) {
    if (lane16 == 0) *(uint32_t *)(p.s + r * p.lds + c / kMxBlock) = four;
  } else if ((lane16 & 3) == 0) {
    p.s[r * p.lds + c / kMxBlock] = (uint8_t)byte;
  }
}
#endif

// Rows alone: a wave takes 512 columns of a row at a time, UNROLL rows requested together.
template <int UNROLL>
__global__ __launch_bounds__(256) void mxfp4_rows_kernel(const MxCastArgs p) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 512 + lane * 8;
  const int64_t r0 = ((int64_t)blockIdx.y * 4 + wave) * UNROLL;
  v4i v[UNROLL];
#pragma unroll
  for (int i = 0; i < UNROLL; ++i) {
    v[i] = v4i{0, 0, 0, 0};
    if (r0 + i < p.R && c < p.C) v[i] = *(const v4i *)(p.x + (r0 + i) * p.ldx + c);
  }
#pragma unroll
  for (int i = 0; i < UNROLL; ++i) cast_row_piece(p, v[i], r0 + i, c);
#endif
}

// Columns, and rows from the same read where ROWS; BANDS blocks of 32 rows to a tile, one block of a column to a
// thread.
template <bool ROWS, int BANDS>
__global__ __launch_bounds__(BANDS * 128) void mxfp4_tile_kernel(const MxCastTiles tiles) {
#if defined(__HIP_DEVICE_COMPILE__)
  // LDS image of a tile: bands of rows of 64 dwords, each band padded so that the bands' first dwords share the banks evenly
  constexpr int kBandDwords = kMxBlock * (kMxTileC / 2) + 64 / BANDS;
  constexpr int kLanes = kMxTileC / 8, kStep = BANDS * 128 / kLanes, kLoads = BANDS * kMxBlock / kStep;   // 16 lanes a row, kStep rows a load
  __shared__ __attribute__((aligned(16))) uint32_t tile[BANDS * kBandDwords];
  const int which = (int)blockIdx.x >= tiles.first ? 1 : 0, id = (int)blockIdx.x - (which ? tiles.first : 0);
  const MxCastArgs &p = tiles.op[which];
  const int64_t r0 = (int64_t)(id / tiles.across[which]) * (BANDS * kMxBlock), c0 = (int64_t)(id % tiles.across[which]) * kMxTileC;
  const int lr = threadIdx.x / kLanes, lc = (threadIdx.x % kLanes) * 8;
  v4i v[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int64_t r = r0 + i * kStep + lr;
    v[i] = v4i{0, 0, 0, 0};
    if (r < p.R && c0 + lc < p.C) v[i] = *(const v4i *)(p.x + r * p.ldx + c0 + lc);
  }
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = i * kStep + lr;
    *(v4i *)(tile + row / kMxBlock * kBandDwords + row % kMxBlock * (kMxTileC / 2) + lc / 2) = v[i];
  }
  if constexpr (ROWS) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) cast_row_piece(p, v[i], r0 + i * kStep + lr, c0 + lc);
  }
  __syncthreads();
  const int64_t bands = (p.R + kMxBlock - 1) / kMxBlock;
  const int band = threadIdx.x % BANDS, half = threadIdx.x / BANDS & 1, pair = threadIdx.x / (2 * BANDS);   // this thread's block of 32 rows, its column
  const int64_t gb = r0 / kMxBlock + band, col = c0 + pair * 2 + half;
  uint32_t w[kMxBlock], m = 0;
#pragma unroll
  for (int i = 0; i < kMxBlock; ++i) {
    w[i] = tile[band * kBandDwords + i * (kMxTileC / 2) + pair];
    m = pk_absmax_u16(m, w[i]);
  }
  const uint32_t byte = mx_byte(half ? m >> 16 : m & 0xffffu);
  const float scale = mx_scale(byte);
  const uint32_t pick = half ? 0x07060302u : 0x05040100u;   // this column of two neighbouring rows
  v4i codes;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t pr[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) pr[j] = __builtin_amdgcn_perm(w[k * 8 + 2 * j + 1], w[k * 8 + 2 * j], pick);
    codes[k] = byte == 255u ? 0 : (int)mx_codes8(pr[0], pr[1], pr[2], pr[3], scale);
  }
  const uint32_t four = byte | dpp<0x101>(byte) << 8 | dpp<0x102>(byte) << 16 | dpp<0x103>(byte) << 24;   // of four bands side by side
  if (col < p.C && gb < bands) {
    *(v4i *)(p.qt + col * p.ldqt + gb * 16) = codes;
    if (BANDS >= 4 && (gb & ~(int64_t)3) + 4 <= bands) {
      if ((band & 3) == 0) *(uint32_t *)(p.st + col * p.ldst + gb) = four;
    } else {
      p.st[col * p.ldst + gb] = (uint8_t)byte;
    }
  }
#endif
}

// Back to bf16: the products of codes and scales are exact but for scales beyond 2^125 (6 * 2^126 and more are infinite).
__global__ __launch_bounds__(256) void mxfp4_to_bf16_kernel(const uint8_t *__restrict__ q, int64_t ldq, const uint8_t *__restrict__ s, int64_t lds,
                                                            int64_t R, int64_t C, uint16_t *__restrict__ y, int64_t ldy) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  const int64_t r = blockIdx.y;
  if (c >= C) return;
  const uint32_t codes = *(const uint32_t *)(q + r * ldq + c / 2);
  const uint32_t byte = s[r * lds + c / kMxBlock];
  const float scale = byte == 255u ? __uint_as_float(0x7fc00000u) : mx_scale(byte);
  uint32_t out[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t lohi[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t code = codes >> (8 * k + 4 * h) & 15u, mag = code & 7u;
      // 0, 0.5, 1, 1.5, 2, 3, 4, 6: the values at twice their size fit a byte each
      const float v = 0.5f * (float)((mag < 4u ? 0x03020100u >> (8u * mag) : 0x0c080604u >> (8u * (mag - 4u))) & 255u);
      lohi[h] = bf16_rne_bits((code & 8u ? -v : v) * scale);
    }
    out[k] = lohi[0] | lohi[1] << 16;
  }
  if (c + 8 <= C && ((uintptr_t)(y + r * ldy + c) % 16) == 0) {
    *(v4i *)(y + r * ldy + c) = v4i{(int)out[0], (int)out[1], (int)out[2], (int)out[3]};
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < C) y[r * ldy + c + k] = (uint16_t)(k & 1 ? out[k / 2] >> 16 : out[k / 2] & 0xffffu);
  }
#endif
}

}  // namespace l8

using namespace l8;

namespace l8 {

static int64_t large_tiles(const l8_mxfp4_cast &o) { return (o.C + kMxTileC - 1) / kMxTileC * ((o.R + 255) / 256); }
constexpr int64_t kMostLargeTiles = (1 << 22) - 1;   // of 1024 threads each: a grid has fewer than 2^32

static int check_cast(const l8_mxfp4_cast &o) {
  L8_REQUIRE(o.R >= 0 && o.C >= 0, "l8_cast_mxfp4: negative shape R=%lld C=%lld", (long long)o.R, (long long)o.C);
  if (o.R == 0 || o.C == 0) return L8_OK;
  L8_REQUIRE((o.q == nullptr) == (o.s == nullptr) && (o.qt == nullptr) == (o.st == nullptr) && (o.q || o.qt), "l8_cast_mxfp4: a copy comes with its scales, and one copy at least");
  const int64_t blocks = (o.C + 31) / 32, bands = (o.R + 31) / 32;
  L8_REQUIRE(o.x && o.C % 8 == 0 && o.ldx % 8 == 0 && o.ldx >= o.C && ((uintptr_t)o.x % 16) == 0,
             "l8_cast_mxfp4: C=%lld and ldx must be multiples of 8 with ldx >= C, x 16-byte aligned", (long long)o.C);
  L8_REQUIRE(!o.q || (o.ldq % 16 == 0 && o.ldq >= blocks * 16 && ((uintptr_t)o.q % 16) == 0 && o.lds % 4 == 0 && o.lds >= blocks && ((uintptr_t)o.s % 4) == 0),
             "l8_cast_mxfp4: rows of 16 bytes per block on 16-byte lines and of a scale per block on 4-byte lines are wanted");
  L8_REQUIRE(!o.qt || (o.ldqt % 16 == 0 && o.ldqt >= bands * 16 && ((uintptr_t)o.qt % 16) == 0 && o.ldst % 4 == 0 && o.ldst >= bands && ((uintptr_t)o.st % 4) == 0),
             "l8_cast_mxfp4: transposed rows of 16 bytes per block on 16-byte lines and of a scale per block on 4-byte lines are wanted");
  L8_REQUIRE(o.R <= (int64_t)65535 * 16 && o.C <= (int64_t)1 << 30, "l8_cast_mxfp4: R=%lld exceeds %d or C=%lld 2^30", (long long)o.R, 65535 * 16, (long long)o.C);
  L8_REQUIRE(!o.qt || large_tiles(o) <= kMostLargeTiles, "l8_cast_mxfp4: R=%lld, C=%lld are more tiles of 256 x %d than a grid has threads for", (long long)o.R,
             (long long)o.C, kMxTileC);
  return L8_OK;
}

// n operands (1 or 2) with columns wanted, and rows of all or none.  Tiles of 256 rows where they give every unit one.
static int launch_tiles(const l8_mxfp4_cast *const *o, int n, hipStream_t st) {
  auto down = [](int64_t R, int rows) { return (R + rows - 1) / rows; };
  auto across = [](int64_t C) { return (C + kMxTileC - 1) / kMxTileC; };
  MxCastTiles t = {};
  int64_t large = 0;
  for (int i = 0; i < n; ++i) {
    const l8_mxfp4_cast &c = *o[i];
    t.op[i] = {(const uint16_t *)c.x, c.R, c.C, c.ldx, (uint8_t *)c.q, (uint8_t *)c.s, (uint8_t *)c.qt, (uint8_t *)c.st, c.ldq, c.lds, c.ldqt, c.ldst};
    t.across[i] = (int)across(c.C);
    large += large_tiles(c);
  }
  const int rows = large >= num_cus() ? 256 : 64;
  t.first = (int)(t.across[0] * down(o[0]->R, rows));
  const int64_t all = t.first + (n > 1 ? t.across[1] * down(o[1]->R, rows) : 0);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)all), dim3((unsigned)rows * 4), 0, st, t); };
  if (rows == 256) {
    if (o[0]->q) go(mxfp4_tile_kernel<true, 8>);
    else go(mxfp4_tile_kernel<false, 8>);
  } else {
    if (o[0]->q) go(mxfp4_tile_kernel<true, 2>);
    else go(mxfp4_tile_kernel<false, 2>);
  }
  L8_HIP(hipGetLastError());
  return L8_OK;
}

}  // namespace l8

extern "C" int l8_cast_mxfp4_two(const l8_mxfp4_cast *two, void *stream) {
  L8_REQUIRE(two, "l8_cast_mxfp4_two: null pointer");
  for (int i = 0; i < 2; ++i) {
    const int rc = check_cast(two[i]);
    if (rc != L8_OK) return rc;
  }
  hipStream_t st = (hipStream_t)stream;
  auto some = [](const l8_mxfp4_cast &o) { return o.R > 0 && o.C > 0; };
  const l8_mxfp4_cast *const both[2] = {two, two + 1};
  // one launch where the same copies are wanted of both and a grid holds them: [1021,2048] and [2064,2048] 9.6 -> 6.4 us, [4096,4096] and [11008,4096]
  // 40.9 -> 36.1
  if (some(two[0]) && some(two[1]) && two[0].qt && two[1].qt && !two[0].q == !two[1].q && large_tiles(two[0]) + large_tiles(two[1]) <= kMostLargeTiles)
    return launch_tiles(both, 2, st);
  for (const l8_mxfp4_cast *o : both) {
    const int rc = l8_cast_mxfp4(o->x, o->R, o->C, o->ldx, o->q, o->ldq, o->s, o->lds, o->qt, o->ldqt, o->st, o->ldst, stream);
    if (rc != L8_OK) return rc;
  }
  return L8_OK;
}

extern "C" int l8_cast_mxfp4(const void *x, int64_t R, int64_t C, int64_t ldx, void *q, int64_t ldq, void *s, int64_t lds, void *qt,
                             int64_t ldqt, void *st, int64_t ldst, void *stream) {
  const l8_mxfp4_cast o = {x, R, C, ldx, q, ldq, s, lds, qt, ldqt, st, ldst}, *const one = &o;
  const int rc = check_cast(o);
  if (rc != L8_OK || R == 0 || C == 0) return rc;
  if (qt) return launch_tiles(&one, 1, (hipStream_t)stream);
  const MxCastArgs a = {(const uint16_t *)x, R, C, ldx, (uint8_t *)q, (uint8_t *)s, nullptr, nullptr, ldq, lds, 0, 0};
  constexpr int U = 4;
  hipLaunchKernelGGL((mxfp4_rows_kernel<U>), dim3((unsigned)((C + 511) / 512), (unsigned)((R + 4 * U - 1) / (4 * U))), dim3(256), 0, (hipStream_t)stream, a);
  L8_HIP(hipGetLastError());
  return L8_OK;
}

extern "C" int l8_mxfp4_to_bf16(const void *q, int64_t ldq, const void *s, int64_t lds, int64_t R, int64_t C, void *y, int64_t ldy, void *stream) {
  L8_REQUIRE(R >= 0 && C >= 0, "l8_mxfp4_to_bf16: negative shape R=%lld C=%lld", (long long)R, (long long)C);
  if (R == 0 || C == 0) return L8_OK;
  const int64_t blocks = (C + 31) / 32;
  L8_REQUIRE(q && s && y, "l8_mxfp4_to_bf16: null pointer");
  L8_REQUIRE(ldq % 4 == 0 && ldq >= blocks * 16 && ((uintptr_t)q % 4) == 0 && lds >= blocks && ldy >= C,
             "l8_mxfp4_to_bf16: rows of 16 bytes and a scale per block of 32 columns are wanted, the codes on 4-byte lines");
  L8_REQUIRE(R <= 65535 * (int64_t)16 && C <= (int64_t)1 << 30, "l8_mxfp4_to_bf16: R=%lld exceeds %d or C=%lld 2^30", (long long)R, 65535 * 16, (long long)C);
  for (int64_t r = 0; r < R; r += 65535) {   // (rows are the grid's second dimension)
    const int64_t n = R - r < 65535 ? R - r : 65535;
    hipLaunchKernelGGL(mxfp4_to_bf16_kernel, dim3((unsigned)((C + 2047) / 2048), (unsigned)n), dim3(256), 0, (hipStream_t)stream,
                       (const uint8_t *)q + r * ldq, ldq, (const uint8_t *)s + r * lds, lds, n, C, (uint16_t *)y + r * ldy, ldy);
  }
  L8_HIP(hipGetLastError());
  return L8_OK;
}
