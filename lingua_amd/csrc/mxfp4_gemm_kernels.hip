// MXFP4 x MXFP4 -> bf16 "NT" product on the gfx950 matrix cores:
//
//   C[m,n] = bf16( sum over blocks b of 2^(sa[m,b] + sb[n,b] - 254) * sum over 32 k of A[m,32 b + k] * B[n,32 b + k]  + bias[n] )
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes both operands' scales: a lane holds 32 consecutive codes of one row -- exactly one block --
// and a byte of scale for it, so the scaling costs no instruction of its own.
//
// Structure
//   * a stage is 128 bytes (256 codes, 8 blocks) of every row of the tile's operands, two matrix instructions deep; lane group g of
//     the four takes blocks 2 g and 2 g + 1 of a stage, so that its two scale bytes lie side by side;
//   * codes go from memory to LDS without passing registers (buffer loads to LDS, whole 128-byte lines), into a ring of NS stages;
//     scales of two stages (16 bytes a row) travel the same way into a ring of their own;
//   * LDS rows are 128 bytes in 16-byte chunks, chunk c of row r at position c ^ f(r), f(r) = (r & 7) ^ ((r >> 3) & 1): the
//     fragment reads of 16 rows cover all banks once.  The permutation is applied on the global side of the loads;
//   * LDS row tn * 16 + j of a wave's share of B holds row TN * j + tn of that share, so that lane j ends up with TN consecutive
//     columns of C and stores them straight from the accumulators;
//   * rows beyond M / N and chunks beyond K lie outside the buffers' ranges: zeros.  Scale bytes beyond K are cleared when they are
//     read (what lies behind a row's end may be a NaN);
//   * workgroups are dealt to the 8 XCDs in contiguous ranges of a grouped tile order, so that an XCD's share panels in its L2.
#include "l8_common.h"

namespace l8 {

typedef __attribute__((address_space(3))) void *lds_void_ptr;
[[maybe_unused]] constexpr uint32_t kBeyond = 0x80000000u;   // an offset that no buffer covers

struct MxGemmArgs {
  const uint8_t *A, *B, *sa, *sb;
  int64_t lda, ldb, ldsa, ldsb;   // bytes
  const uint16_t *bias;
  uint16_t *C;
  int64_t ldc;
  int M, N, blocks;               // blocks of 32 along K
  int tiles_m, tiles_n;
  bool wide;                      // TN columns of C can be stored at once
};

// s_waitcnt vmcnt(n), and lgkmcnt(0), alone
#define MX_WAIT_VM(n) __builtin_amdgcn_s_waitcnt(((n) & 0xF) | (0x7 << 4) | (0xF << 8) | ((((n) >> 4) & 0x3) << 14))
#define MX_WAIT_LGKM0() __builtin_amdgcn_s_waitcnt(0xF | (0x7 << 4) | (0x0 << 8) | (0x3 << 14))

template <int WM, int WN, int TM, int TN, int NS>
__global__ __launch_bounds__(WM *WN * 64) void gemm_mxfp4_kernel(const MxGemmArgs p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int BM = WM * TM * 16, BN = WN * TN * 16, NW = WM * WN, GROUP = 8;
  constexpr int NLA = BM / 8 / NW, NLB = BN / 8 / NW;           // wave loads (8 rows) of a stage
  constexpr int STAGE = (BM + BN) * 128, SROWS = BM + BN, SLOADS = SROWS / 64, NSW = NS / 2 + 1;
  static_assert(NS % 2 == 0 && BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && SROWS % 64 == 0 && BM % 64 == 0, "");
  static_assert((NS - 1) * (NLA + NLB) <= 63, "vmcnt is a 6-bit counter");
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];   // NS stages, NSW windows of scales
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;

  int m0, n0;
  {
    const int nb = p.tiles_m * p.tiles_n, q = nb >> 3, rem = nb & 7;
    const int xcd = blockIdx.x & 7, loc = blockIdx.x >> 3;
    const int lin = (xcd < rem) ? xcd * (q + 1) + loc : rem * (q + 1) + (xcd - rem) * q + loc;
    const int per_group = GROUP * p.tiles_n, grp = lin / per_group, in_grp = lin - grp * per_group;
    const int size = p.tiles_m - grp * GROUP < GROUP ? p.tiles_m - grp * GROUP : GROUP;
    m0 = (grp * GROUP + in_grp % size) * BM;
    n0 = (in_grp / size) * BN;
  }

  const int kbytes = p.blocks * 16;
  auto range = [](int64_t n) { return n < 0x7fffffff ? (uint32_t)n : 0x7fffffffu; };
  const __amdgpu_buffer_rsrc_t rsA = make_rsrc(p.A + (int64_t)m0 * p.lda, range((int64_t)(p.M - m0 - 1) * p.lda + kbytes));
  const __amdgpu_buffer_rsrc_t rsB = make_rsrc(p.B + (int64_t)n0 * p.ldb, range((int64_t)(p.N - n0 - 1) * p.ldb + kbytes));
  // (up to the end of the dword that the last scale lies in)
  const __amdgpu_buffer_rsrc_t rsSa = make_rsrc(p.sa + (int64_t)m0 * p.ldsa, range((int64_t)(p.M - m0 - 1) * p.ldsa + (p.blocks + 3) / 4 * 4));
  const __amdgpu_buffer_rsrc_t rsSb = make_rsrc(p.sb + (int64_t)n0 * p.ldsb, range((int64_t)(p.N - n0 - 1) * p.ldsb + (p.blocks + 3) / 4 * 4));

  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_ptr)smem;
  const int lrow = lane >> 3, lpos = lane & 7;
  const int chunk[2] = {(lpos ^ lrow) * 16, (lpos ^ lrow ^ 1) * 16};   // of even and odd groups of 8 rows
  const int a_row = lrow * (int)p.lda, b_row = lrow * TN * (int)p.ldb;
  // row of B (in the tile) that LDS row r of its panel holds
  auto b_of = [](int r) { return r / (TN * 16) * (TN * 16) + TN * (r % 16) + r % (TN * 16) / 16; };
  auto load_stage = [&](int j, int slot) {
    const int k0 = j * 128;
    const uint32_t off[2] = {(k0 + chunk[0] < kbytes) ? 0u : kBeyond, (k0 + chunk[1] < kbytes) ? 0u : kBeyond};
    const uint32_t dst = lds0 + slot * STAGE;
#pragma unroll
    for (int i = 0; i < NLA; ++i) {
      const int g = wave * NLA + i;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsA, reinterpret_cast<lds_void_ptr>(dst + g * 1024), 16, (uint32_t)(a_row + chunk[g & 1]) | off[g & 1],
                                               k0 + g * 8 * (int)p.lda, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < NLB; ++i) {
      const int g = wave * NLB + i;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsB, reinterpret_cast<lds_void_ptr>(dst + BM * 128 + g * 1024), 16, (uint32_t)(b_row + chunk[g & 1]) | off[g & 1],
                                               k0 + b_of(g * 8) * (int)p.ldb, 0, 0);
    }
  };
  auto load_scales = [&](int w) {
    const uint32_t dst = lds0 + NS * STAGE + (w % NSW) * (SROWS * 16);
    const uint32_t off = w * 16 < p.blocks ? 0u : kBeyond;
    for (int i = wave; i < SLOADS; i += NW) {
      const int r = i * 64 + lane;
      if (i < BM / 64)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsSa, reinterpret_cast<lds_void_ptr>(dst + i * 1024), 16, (uint32_t)(r * (int)p.ldsa) | off, w * 16, 0, 0);
      else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsSb, reinterpret_cast<lds_void_ptr>(dst + i * 1024), 16, (uint32_t)(b_of(r - BM) * (int)p.ldsb) | off, w * 16, 0, 0);
    }
  };

  v4f acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  const int stages = (p.blocks + 7) / 8;
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    if (j % 2 == 0) load_scales(j / 2);
    load_stage(j, j);
  }
  const int frow = lane & 15, fg = lane >> 4;
  const int fr = (frow & 7) ^ (frow >> 3);
  const uint32_t foff[2] = {(uint32_t)(frow * 128 + (((fg * 2) ^ fr) * 16)), (uint32_t)(frow * 128 + (((fg * 2 + 1) ^ fr) * 16))};
  typedef const __attribute__((address_space(3))) v4i *lds_v4i;
  typedef const __attribute__((address_space(3))) uint16_t *lds_u16;

  for (int j = 0; j < stages; ++j) {
    const int slot = j % NS;
    MX_WAIT_VM((NS - 1) * (NLA + NLB));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    uint32_t base = lds0 + slot * STAGE, sbase = lds0 + NS * STAGE + ((j >> 1) % NSW) * (SROWS * 16) + frow * 16 + (j & 1) * 8 + fg * 2;
    asm volatile("" : "+v"(base), "+v"(sbase));
    const int left = p.blocks - (j * 8 + fg * 2);
    const uint32_t smask = left >= 2 ? 0xffffu : (left == 1 ? 0xffu : 0u);
    v4i a[TM][2], b[TN][2];
    uint32_t as[TM], bs[TN];
#pragma unroll
    for (int t = 0; t < TN; ++t) {
#pragma unroll
      for (int h = 0; h < 2; ++h) b[t][h] = *reinterpret_cast<lds_v4i>(base + BM * 128 + (wn * TN + t) * 2048 + foff[h]);
      bs[t] = *reinterpret_cast<lds_u16>(sbase + (BM + (wn * TN + t) * 16) * 16) & smask;
    }
#pragma unroll
    for (int t = 0; t < TM; ++t) {
#pragma unroll
      for (int h = 0; h < 2; ++h) a[t][h] = *reinterpret_cast<lds_v4i>(base + (wm * TM + t) * 2048 + foff[h]);
      as[t] = *reinterpret_cast<lds_u16>(sbase + (wm * TM + t) * 256) & smask;
    }
    MX_WAIT_LGKM0();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if ((j & 1) == 0) load_scales((j + NS) / 2);
    load_stage(j + NS, slot);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int t = 0; t < TN; ++t) {
          const v8i af = {a[i][h][0], a[i][h][1], a[i][h][2], a[i][h][3], 0, 0, 0, 0};
          const v8i bf = {b[t][h][0], b[t][h][1], b[t][h][2], b[t][h][3], 0, 0, 0, 0};
          if (h == 0) acc[i][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(af, bf, acc[i][t], 4, 4, 0, (int)as[i], 0, (int)bs[t]);
          else acc[i][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(af, bf, acc[i][t], 4, 4, 1, (int)as[i], 1, (int)bs[t]);
        }
  }
  // what was requested beyond the last stage (zeros) must have landed before the workgroup's LDS is released
  MX_WAIT_VM(0);

  const int col = n0 + wn * (TN * 16) + TN * frow;
  float bv[TN];
#pragma unroll
  for (int t = 0; t < TN; ++t) bv[t] = p.bias && col + t < p.N ? bf16_bits_to_f32(p.bias[col + t]) : 0.0f;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = m0 + (wm * TM + i) * 16 + fg * 4 + e;
      uint32_t out[TN / 2];
#pragma unroll
      for (int t = 0; t < TN / 2; ++t)
        out[t] = bf16_rne_bits(acc[i][2 * t][e] + bv[2 * t]) | (bf16_rne_bits(acc[i][2 * t + 1][e] + bv[2 * t + 1]) << 16);
      if (row >= p.M) continue;
      uint16_t *dst = p.C + (int64_t)row * p.ldc + col;
      if (p.wide) {
        if (col < p.N) {
          if constexpr (TN == 8) *(v4i *)dst = v4i{(int)out[0], (int)out[1], (int)out[2], (int)out[3]};
          else if constexpr (TN == 4) *(v2i *)dst = v2i{(int)out[0], (int)out[1]};
          else *(uint32_t *)dst = out[0];
        }
      } else {
#pragma unroll
        for (int t = 0; t < TN; ++t)
          if (col + t < p.N) dst[t] = (uint16_t)(t & 1 ? out[t / 2] >> 16 : out[t / 2] & 0xffffu);
      }
    }
#endif
}

template <int WM, int WN, int TM, int TN, int NS>
static int launch_gemm_mxfp4(MxGemmArgs a, hipStream_t st) {
  constexpr int BM = WM * TM * 16, BN = WN * TN * 16;
  constexpr int lds = NS * (BM + BN) * 128 + (NS / 2 + 1) * (BM + BN) * 16;
  a.tiles_m = (a.M + BM - 1) / BM, a.tiles_n = (a.N + BN - 1) / BN;
  a.wide = a.N % TN == 0 && a.ldc % TN == 0 && ((uintptr_t)a.C % (TN * 2)) == 0;
  static bool ready[kMaxDev];   // benign race: every thread sets the same attribute
  const int slot = device_slot();
  if (slot < 0 || !ready[slot]) {
    L8_HIP(hipFuncSetAttribute((const void *)gemm_mxfp4_kernel<WM, WN, TM, TN, NS>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    if (slot >= 0) ready[slot] = true;
  }
  hipLaunchKernelGGL((gemm_mxfp4_kernel<WM, WN, TM, TN, NS>), dim3((unsigned)(a.tiles_m * a.tiles_n)), dim3(WM * WN * 64), lds, st, a);
  L8_HIP(hipGetLastError());
  return L8_OK;
}

}  // namespace l8

using namespace l8;

extern "C" int l8_gemm_mxfp4_nt(const void *A, const void *sa, const void *B, const void *sb, int64_t M, int64_t N, int64_t K, int64_t lda,
                                int64_t ldsa, int64_t ldb, int64_t ldsb, const void *bias, void *C, int64_t ldc, void *stream) {
  L8_REQUIRE(M >= 0 && N >= 0 && K >= 0, "l8_gemm_mxfp4_nt: negative shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (M == 0 || N == 0) return L8_OK;
  const int64_t blocks = (K + 31) / 32;
  L8_REQUIRE(C && ldc >= N, "l8_gemm_mxfp4_nt: null C or ldc < N");
  L8_REQUIRE(blocks == 0 || (A && B && sa && sb), "l8_gemm_mxfp4_nt: null pointer");
  L8_REQUIRE(M < (1 << 28) && N < (1 << 28) && K < (1 << 24), "l8_gemm_mxfp4_nt: M, N < 2^28 and K < 2^24 are served");
  L8_REQUIRE(lda % 16 == 0 && ldb % 16 == 0 && lda >= blocks * 16 && ldb >= blocks * 16 && lda <= (1 << 23) - 16 && ldb <= (1 << 23) - 16 &&
                 ((uintptr_t)A % 16) == 0 && ((uintptr_t)B % 16) == 0,
             "l8_gemm_mxfp4_nt: rows of codes, 16 bytes per block, on 16-byte lines less than 2^23 bytes apart are wanted");
  L8_REQUIRE(ldsa % 16 == 0 && ldsb % 16 == 0 && ldsa >= blocks && ldsb >= blocks && ldsa <= (1 << 23) - 16 && ldsb <= (1 << 23) - 16 &&
                 ((uintptr_t)sa % 16) == 0 && ((uintptr_t)sb % 16) == 0,
             "l8_gemm_mxfp4_nt: rows of scales, a byte per block, on 16-byte lines less than 2^23 bytes apart are wanted");
  L8_REQUIRE(((uintptr_t)C % 2) == 0 && ((uintptr_t)bias % 2) == 0, "l8_gemm_mxfp4_nt: misaligned C or bias");
  const MxGemmArgs a = {(const uint8_t *)A, (const uint8_t *)B, (const uint8_t *)sa, (const uint8_t *)sb, lda, ldb, ldsa, ldsb,
                        (const uint16_t *)bias, (uint16_t *)C, ldc, (int)M, (int)N, (int)blocks, 0, 0, false};
  hipStream_t st = (hipStream_t)stream;
  L8_REQUIRE(((M + 255) / 256) * ((N + 255) / 256) < (1 << 24), "l8_gemm_mxfp4_nt: more tiles than a grid has");
  const int64_t big = ((M + 255) / 256) * ((N + 255) / 256), mid = ((M + 127) / 128) * ((N + 127) / 128);
  if (big >= num_cus() / 2) return launch_gemm_mxfp4<2, 2, 8, 8, 2>(a, st);
  if (mid >= num_cus() / 2) return launch_gemm_mxfp4<2, 2, 4, 4, 4>(a, st);
  return launch_gemm_mxfp4<2, 2, 2, 2, 8>(a, st);
}
