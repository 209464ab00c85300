// MXFP4 x MXFP4 -> bf16 "NT" product on the gfx950 matrix cores:
//
//   C[m,n] = bf16( sum over blocks b of 2^(sa[m,b] + sb[n,b] - 254) * sum over 32 k of A[m,32 b + k] * B[n,32 b + k]  + bias[n] )
//
// v_mfma_scale_f32_32x32x64_f8f6f4 and its 16x16x128 form take both operands' scales: a lane holds 32 consecutive codes of one row --
// exactly one block -- and a byte of scale for it, so the scaling costs no instruction of its own.
//
// Structure
//   * a stage is 128 bytes (256 codes, 8 blocks) of every row of the tile's operands, four matrix instructions (32 x 32 x 64) deep; the
//     lower half of a wave takes blocks 0 .. 3 of a stage, the upper 4 .. 7, so that a lane's four scale bytes are one dword, picked
//     apart by the instruction's op_sel.  Half of a stage is multiplied while the next half's fragments are read;
//   * codes go from memory to LDS without passing registers (buffer loads to LDS, whole 128-byte lines), into a ring of NS stages;
//     scales of two stages (16 bytes a row) travel the same way into a ring of their own;
//   * LDS rows are 128 bytes in 16-byte chunks, chunk c of row r at position c ^ f(r), f(r) = (r & 7) ^ ((r >> 3) & 1): the
//     fragment reads of 16 rows cover all banks once.  The permutation is applied on the global side of the loads;
//   * LDS row tn * 32 + j of a wave's share of B holds row TN * j + tn of that share, so that lane j ends up with TN neighbouring
//     columns of C and stores them straight from the accumulators;
//   * rows beyond M / N and chunks beyond K lie outside the buffers' ranges: zeros.  Scale bytes beyond K are cleared when they are
//     read (what lies behind a row's end may be a NaN);
//   * workgroups are dealt to the 8 XCDs in contiguous ranges of a grouped tile order, so that an XCD's share panels in its L2.
// Bound by what a stage costs beside its matrix instructions (512 of some 1200 cycles for a 128 x 128 tile): scales, 16 bytes from every
// row, fragment reads, the loads' way through the L2, the barrier.
#include <type_traits>
#include <utility>

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

// s_waitcnt vmcnt(n) alone, and with lgkmcnt(0).  In front of a barrier that hands a ring slot back to the loads it is the second: the
// wave's fragment reads of that slot must have returned, or a load to LDS overtakes them.
#define MX_WAIT_VM(n) __builtin_amdgcn_s_waitcnt(((n) & 0xF) | (0x7 << 4) | (0xF << 8) | ((((n) >> 4) & 0x3) << 14))
#define MX_WAIT_VM_LGKM0(n) __builtin_amdgcn_s_waitcnt(((n) & 0xF) | (0x7 << 4) | ((((n) >> 4) & 0x3) << 14))

// f(0), f(1), .. as straight code, each with its number as a constant
template <typename F, int... I>
L8_DEV void in_turn(std::integer_sequence<int, I...>, F &&f) {
  (f(std::integral_constant<int, I>{}), ...);
}

template <int WM, int WN, int TM, int TN, int NS>
__global__ __launch_bounds__(WM *WN * 64) void gemm_mxfp4_kernel(const MxGemmArgs p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int BM = WM * TM * 32, BN = WN * TN * 32, NW = WM * WN, GROUP = 8;
  constexpr int NLA = BM / 8 / NW, NLB = BN / 8 / NW;           // wave loads (8 rows) of a stage
  constexpr int STAGE = (BM + BN) * 128, SROWS = BM + BN, SLOADS = SROWS / 64, NSW = NS / 2 + 1;
  static_assert((TN == 1 || TN == 2) && NS % 2 == 0 && BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && SROWS % 64 == 0 && BM % 64 == 0, "");
  static_assert((NS - 2) * (NLA + NLB) <= 63 && (NS - 1) * (NLA + NLB) + NS <= 63, "vmcnt is a 6-bit counter");
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
  auto b_of = [](int r) { return r / (TN * 32) * (TN * 32) + TN * (r % 32) + r % (TN * 32) / 32; };
  // i-th wave load of stage j's panels into ring slot `slot`
  auto load_one = [&](int j, int slot, int i) __attribute__((always_inline)) {
    const int k0 = j * 128;
    const uint32_t dst = lds0 + slot * STAGE;
    const int g = i < NLA ? wave * NLA + i : wave * NLB + i - NLA;
    const uint32_t off = (k0 + chunk[g & 1] < kbytes) ? 0u : kBeyond;
    if (i < NLA)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsA, reinterpret_cast<lds_void_ptr>(dst + g * 1024), 16, (uint32_t)(a_row + chunk[g & 1]) | off,
                                               k0 + g * 8 * (int)p.lda, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsB, reinterpret_cast<lds_void_ptr>(dst + BM * 128 + g * 1024), 16, (uint32_t)(b_row + chunk[g & 1]) | off,
                                               k0 + b_of(g * 8) * (int)p.ldb, 0, 0);
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

  v16f acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

  const int stages = (p.blocks + 7) / 8;
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    if (j % 2 == 0) load_scales(j / 2);
#pragma unroll
    for (int i = 0; i < NLA + NLB; ++i) load_one(j, j, i);
  }
  const int frow = lane & 31, fg = lane >> 5;
  const int fr = (frow & 7) ^ (frow >> 3 & 1);
  uint32_t foff[4];   // block 4 g + s of a stage
#pragma unroll
  for (int s = 0; s < 4; ++s) foff[s] = (uint32_t)(frow * 128 + (((fg * 4 + s) ^ fr) * 16));
  typedef const __attribute__((address_space(3))) v4i *lds_v4i;
  typedef const __attribute__((address_space(3))) uint32_t *lds_u32;

  // Fragments of a stage's four steps of 64 codes (s: blocks 4 g + s), and scales of two stages, a byte for each step.
  v4i fa[4][TM], fb[4][TN];
  uint32_t sa[2][TM], sb[2][TN];
  uint32_t at, sat, smask;   // of the stage that is read next
  auto open = [&](int j) __attribute__((always_inline)) {
    at = lds0 + (j % NS) * STAGE;
    sat = lds0 + NS * STAGE + ((j >> 1) % NSW) * (SROWS * 16) + frow * 16 + (j & 1) * 8 + fg * 4;
    asm volatile("" : "+v"(at), "+v"(sat));
    const int left = p.blocks - (j * 8 + fg * 4);
    smask = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
  };
  auto read_frag = [&](int h, int r) __attribute__((always_inline)) {   // r-th read of half h: two steps of TM + TN
    const int s = 2 * h + r / (TM + TN), q = r % (TM + TN);
    auto of_b = [&](int t) __attribute__((always_inline)) { fb[s][t] = *reinterpret_cast<lds_v4i>(at + BM * 128 + (wn * TN + t) * 4096 + foff[s]); };
    auto of_a = [&](int t) __attribute__((always_inline)) { fa[s][t] = *reinterpret_cast<lds_v4i>(at + (wm * TM + t) * 4096 + foff[s]); };
    if (q == 0) of_b(0);
    else if (q == 1) of_a(0);
    else if (q <= TN) of_b(q - 1);
    else of_a(q - TN);
  };
  auto read_scale = [&](int to, int r) __attribute__((always_inline)) {
    if (r < TN) sb[to][r] = *reinterpret_cast<lds_u32>(sat + (BM + (wn * TN + r) * 32) * 16);
    else sa[to][r - TN] = *reinterpret_cast<lds_u32>(sat + (wm * TM + r - TN) * 512);
  };
  auto mask_scales = [&](int to) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < TM; ++t) sa[to][t] &= smask;
#pragma unroll
    for (int t = 0; t < TN; ++t) sb[to][t] &= smask;
  };
  constexpr int N_MMA = 2 * TM * TN, N_RD = 2 * (TM + TN), N_SC = TM + TN;
  auto mma_one = [&](auto half, int cur, auto number) __attribute__((always_inline)) {
    constexpr int i = decltype(number)::value, s = 2 * decltype(half)::value + i / (TM * TN), tm = i % (TM * TN) / TN, tn = i % TN;
    const v4i x = fa[s][tm], y = fb[s][tn];
    const v8i a = {x[0], x[1], x[2], x[3], 0, 0, 0, 0}, b = {y[0], y[1], y[2], y[3], 0, 0, 0, 0};
    acc[tm][tn] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, acc[tm][tn], 4, 4, s, (int)sa[cur][tm], s, (int)sb[cur][tn]);
  };
  constexpr std::integral_constant<int, 0> lower{};
  constexpr std::integral_constant<int, 1> upper{};
  // One stage.  Its lower half is multiplied while its upper half is read; at the barrier every wave has read all of it and the next
  // stage has landed; its upper half is multiplied while the next stage's lower half and scales are read and the stage NS further on
  // is requested into the slot that has become free.
  auto trip = [&](int j, auto parity) __attribute__((always_inline)) {
    constexpr int cur = decltype(parity)::value;
    in_turn(std::make_integer_sequence<int, N_MMA>{}, [&](auto number) __attribute__((always_inline)) {
      constexpr int i = decltype(number)::value;
      mma_one(lower, cur, number);
#pragma unroll
      for (int r = (N_RD * i) / N_MMA; r < (N_RD * (i + 1)) / N_MMA; ++r) read_frag(1, r);
      __builtin_amdgcn_sched_barrier(0);
    });
    MX_WAIT_VM_LGKM0((NS - 2) * (NLA + NLB));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    open(j + 1);
    if (cur == 0) load_scales((j + NS) / 2);
    in_turn(std::make_integer_sequence<int, N_MMA>{}, [&](auto number) __attribute__((always_inline)) {
      constexpr int i = decltype(number)::value;
      mma_one(upper, cur, number);
#pragma unroll
      for (int r = ((N_RD + N_SC) * i) / N_MMA; r < ((N_RD + N_SC) * (i + 1)) / N_MMA; ++r) {
        if (r < N_RD) read_frag(0, r);
        else read_scale(1 - cur, r - N_RD);
      }
#pragma unroll
      for (int l = ((NLA + NLB) * i) / N_MMA; l < ((NLA + NLB) * (i + 1)) / N_MMA; ++l) load_one(j + NS, j % NS, l);
      __builtin_amdgcn_sched_barrier(0);
    });
    mask_scales(1 - cur);
  };
  MX_WAIT_VM((NS - 1) * (NLA + NLB));
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  open(0);
#pragma unroll
  for (int r = 0; r < N_RD; ++r) read_frag(0, r);
#pragma unroll
  for (int r = 0; r < N_SC; ++r) read_scale(0, r);
  mask_scales(0);
  // (a last stage that stands alone is a trip of its own: with a branch around the second of a pair the accumulators were copied in every trip)
  int j = 0;
#pragma unroll 1
  for (; j + 2 <= stages; j += 2) {
    trip(j, lower);
    trip(j + 1, upper);
  }
  if (j < stages) trip(j, lower);
  // what was requested beyond the last stage (zeros) must have landed before the workgroup's LDS is released
  MX_WAIT_VM(0);

  const int col = n0 + wn * (TN * 32) + TN * frow;
  float bv[TN];
#pragma unroll
  for (int t = 0; t < TN; ++t) bv[t] = p.bias && col + t < p.N ? bf16_bits_to_f32(p.bias[col + t]) : 0.0f;
  if (p.wide) {   // through a buffer: rows beyond M lie outside it
    const __amdgpu_buffer_rsrc_t rsC = make_rsrc(p.C + (int64_t)m0 * p.ldc + n0, range(((int64_t)(p.M - m0 - 1) * p.ldc + (p.N - n0)) * 2));
    const int ldc2 = (int)p.ldc * 2;
    const uint32_t voff = col < p.N ? (uint32_t)((wm * TM * 32 + fg * 4) * ldc2 + (col - n0) * 2) : kBeyond;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int soff = (i * 32 + e / 4 * 8 + e % 4) * ldc2;
        if constexpr (TN == 1) {
          __builtin_amdgcn_raw_buffer_store_b16((short)bf16_rne_bits(acc[i][0][e] + bv[0]), rsC, (int)voff, soff, 0);
        } else {
          const uint32_t two = bf16_rne_bits(acc[i][0][e] + bv[0]) | (bf16_rne_bits(acc[i][1][e] + bv[1]) << 16);
          __builtin_amdgcn_raw_buffer_store_b32((int)two, rsC, (int)voff, soff, 0);
        }
      }
    return;
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int row = m0 + (wm * TM + i) * 32 + fg * 4 + e / 4 * 8 + e % 4;
      if (row >= p.M) continue;
      uint16_t *dst = p.C + (int64_t)row * p.ldc + col;
#pragma unroll
      for (int t = 0; t < TN; ++t)
        if (col + t < p.N) dst[t] = (uint16_t)bf16_rne_bits(acc[i][t][e] + bv[t]);
    }
#endif
}

// ---------------------------------------------------------------------------
// Large products: one workgroup per compute unit walks a list of 256 x 256 tiles, and the stream of panels (one operand's 256 rows of
// a stage, 32 KiB) runs on from the last stage of a tile into the first of the next, so that only a workgroup's first tile waits for
// its operands.  Four waves, 128 x 128 each: the least LDS traffic per flop.
//
//   * LDS is a ring of five panels, 2.5 stages; a trip (one stage, 128 matrix instructions of 16 cycles) requests one panel in front of
//     its barrier, into the slot that the barrier before released, and one behind it, into the slot that this stage's A panel left;
//   * the barrier stands between a stage's two halves of 128 codes.  While a half is multiplied, the eight A and eight B fragments of
//     the next one are read: 16 KiB of LDS to 64 matrix instructions, and never more than two sets in registers.  Each group of two
//     matrix instructions carries at most one LDS read and one load, and fences keep it so: the matrix cores want an instruction
//     every 16 cycles, four issue slots;
//   * the LDS is full, so scales go straight to registers, in the layout that the instruction wants (lane group g: the bytes of
//     blocks 2 g and 2 g + 1 of both stages of a window, picked by its op_sel).  A kernel of its own lays them out so beforehand, 1 KiB
//     of consecutive bytes per load: it moves 1/16 of the operands' bytes.  (Loaded as they lie, 16 bytes of each of 64 rows, and
//     turned in registers, they took 40 of 340 us.)
//   * C leaves straight from the accumulators, 16 bytes a lane, under the next tile's first panels.
// ---------------------------------------------------------------------------
#if defined(__HIP_DEVICE_COMPILE__)
// A 16-byte buffer store with a register offset, and two wait states: a write to its data registers right behind it may overtake it.
L8_DEV void store16_streaming(v4i data, __amdgpu_buffer_rsrc_t rs, uint32_t voff, int soff) {
  __builtin_amdgcn_raw_buffer_store_b128(data, rs, (int)voff, soff, 2);
  asm volatile("s_nop 1" : : "v"(data));
}
#endif

// Scales as the kernel below loads them: for every 64 LDS rows of a panel and window of 16 blocks 64 lanes' 16 bytes, lane (g, r) = 16 g +
// r holding, for q = 0 .. 3, the bytes of blocks 2 g, 2 g + 1, 8 + 2 g and 9 + 2 g of row 16 q + r.  Zeros for rows beyond the last and
// blocks beyond K (the codes there are zeros and must not meet a NaN).  LDS row l of B is row 8 (l % 16) + l / 16 of its 128.
struct MxScaleArgs {
  const uint8_t *s[2];
  uint8_t *t[2];
  int64_t ld[2];
  int rows[2], chunks[2];   // rows; groups of 64 of them, up to whole tiles
  int blocks, windows;
};
__global__ __launch_bounds__(256) void mxfp4_lay_scales_kernel(const MxScaleArgs p) {
#if defined(__HIP_DEVICE_COMPILE__)
  // a workgroup: 64 rows, 4 windows (64 bytes a row), in LDS as rows of 17 dwords
  __shared__ uint32_t rows[64 * 17];
  const bool is_b = (int)blockIdx.y >= p.chunks[0];
  const int o = is_b ? 1 : 0, chunk = blockIdx.y - (is_b ? p.chunks[0] : 0), w0 = blockIdx.x * 4;
  const int row = threadIdx.x >> 2, part = threadIdx.x & 3;   // this thread's row and window
  const int l = (chunk & 1) * 64 + row;
  const int src = (chunk >> 1) * 128 + (is_b ? 8 * (l & 15) + (l >> 4) : l);
  const int first = (w0 + part) * 16;
  uint32_t v[4] = {0, 0, 0, 0};
  if (src < p.rows[o]) {
    const uint8_t *at = p.s[o] + (int64_t)src * p.ld[o] + first;
    if (first + 16 <= p.blocks) {
      __builtin_memcpy(v, at, 16);
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (first + k < p.blocks) v[k >> 2] |= (uint32_t)at[k] << (8 * (k & 3));
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) rows[row * 17 + part * 4 + k] = v[k];
  __syncthreads();
  const int win = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  if (w0 + win >= p.windows) return;
  v4i out;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t lo = rows[(16 * q + r) * 17 + win * 4 + (g >> 1)], hi = rows[(16 * q + r) * 17 + win * 4 + 2 + (g >> 1)];
    out[q] = (int)__builtin_amdgcn_perm(hi, lo, g & 1 ? 0x07060302u : 0x05040100u);
  }
  *(v4i *)(p.t[o] + ((int64_t)chunk * p.windows + w0 + win) * 1024 + lane * 16) = out;
#endif
}

template <bool HAS_BIAS>
__global__ __launch_bounds__(256) void gemm_mxfp4_stream_kernel(const MxGemmArgs p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int BM = 256, BN = 256, TM = 8, TN = 8, GROUP = 4, R = 5, UNIT = 256 * 128;
  constexpr int NL = 8;                 // wave loads (8 rows) of a panel per wave
  constexpr int NSC = 4;                // scale loads of a window per wave
  constexpr int N_STORES = TM * 4;      // of a C tile per wave
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;

  // ---- this workgroup's tiles: first + loc, + W, + 2 W, ... of the grouped order ----
  const int nb = p.tiles_m * p.tiles_n;
  const int xcd = blockIdx.x & 7, loc = blockIdx.x >> 3, W = gridDim.x >> 3;
  const int q = nb >> 3, rem = nb & 7;
  const int first = (xcd < rem) ? xcd * (q + 1) : rem * (q + 1) + (xcd - rem) * q;
  const int cnt = q + (xcd < rem ? 1 : 0);
  const int KT = (p.blocks + 7) / 8;    // at least 2 (the host sees to it)
  const int n_seg = loc < cnt ? (cnt - loc + W - 1) / W : 0;
  if (n_seg == 0) return;
  const int per_group = GROUP * p.tiles_n;
  struct Cursor { int grp, in_grp; };   // one for the loader, one for the multiplying side: a tile's origin without a division
  Cursor cur_mul, cur_ld;
  cur_mul.grp = (first + loc) / per_group;
  cur_mul.in_grp = first + loc - cur_mul.grp * per_group;
  cur_ld = cur_mul;
  auto origin = [&](const Cursor &c, int &m0, int &n0) {
    const int first_m = c.grp * GROUP, left = p.tiles_m - first_m;
    if (left >= GROUP) {
      m0 = (first_m + (c.in_grp & (GROUP - 1))) * BM;
      n0 = (c.in_grp / GROUP) * BN;
    } else {
      m0 = (first_m + c.in_grp % left) * BM;
      n0 = (c.in_grp / left) * BN;
    }
  };
  auto step = [&](Cursor &c) {
    c.in_grp += W;
    while (c.in_grp >= per_group) {
      c.in_grp -= per_group;
      ++c.grp;
    }
  };

  // ---- loads ----
  const int kbytes = p.blocks * 16;
  const int lrow = lane >> 3, lpos = lane & 7;
  const int chunk[2] = {(lpos ^ lrow) * 16, (lpos ^ lrow ^ 1) * 16};
  const uint32_t a_voff[2] = {(uint32_t)(lrow * (int)p.lda + chunk[0]), (uint32_t)(lrow * (int)p.lda + chunk[1])};
  const uint32_t b_voff[2] = {(uint32_t)(lrow * 8 * (int)p.ldb + chunk[0]), (uint32_t)(lrow * 8 * (int)p.ldb + chunk[1])};
  const int windows = (KT + 1) >> 1;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_ptr)smem;
  auto wrap = [](int slot) { return slot >= R ? slot - R : slot; };
  auto range = [](int64_t n) { return n < 0x7fffffff ? (uint32_t)n : 0x7fffffffu; };
  int ld_seg = 0, ld_kt = 0;
  __amdgpu_buffer_rsrc_t ld_rsA, ld_rsB, ld_rsSa, ld_rsSb;
  auto ld_open = [&](int seg) {
    if (seg < n_seg) {
      int m0, n0;
      origin(cur_ld, m0, n0);
      step(cur_ld);
      ld_rsA = make_rsrc(p.A + (int64_t)m0 * p.lda, range((int64_t)(p.M - m0 - 1) * p.lda + kbytes));
      ld_rsB = make_rsrc(p.B + (int64_t)n0 * p.ldb, range((int64_t)(p.N - n0 - 1) * p.ldb + kbytes));
      ld_rsSa = make_rsrc(p.sa + (int64_t)(m0 / 64 + wm * 2) * windows * 1024, windows * 2048);
      ld_rsSb = make_rsrc(p.sb + (int64_t)(n0 / 64 + wn * 2) * windows * 1024, windows * 2048);
    } else {   // past the last tile: zeros
      ld_rsA = make_rsrc(p.A, 0);
      ld_rsB = make_rsrc(p.B, 0);
      ld_rsSa = make_rsrc(p.sa, 0);
      ld_rsSb = make_rsrc(p.sb, 0);
    }
  };
  auto ld_advance = [&]() {
    if (++ld_kt == KT) {
      ld_kt = 0;
      ld_open(++ld_seg);
    }
  };
  // i-th wave load of the loader's A or B panel into the panel at LDS offset `at`.  A load's row offset is formed from the one before
  // (kept in scalar registers, all sixteen would spill).
  int ld_off = 0, step_a = 8 * (int)p.lda, step_b = 64 * (int)p.ldb, back_b = -63 * (int)p.ldb;
  int a0_off = wave * NL * 8 * (int)p.lda, b0_off = ((wave >> 1) * 128 + (wave & 1) * 4) * (int)p.ldb;
  asm volatile("" : "+s"(step_a), "+s"(step_b), "+s"(back_b), "+s"(a0_off), "+s"(b0_off));
  auto load_one = [&](bool is_b, int at, int i) __attribute__((always_inline)) {
    const int k0 = ld_kt * 128;
    const uint32_t off = (k0 + chunk[i & 1] < kbytes) ? 0u : kBeyond;
    const uint32_t dst = lds0 + at + (wave * NL + i) * 1024;
    if (!is_b) {
      ld_off = i == 0 ? k0 + a0_off : ld_off + step_a;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ld_rsA, reinterpret_cast<lds_void_ptr>(dst), 16, a_voff[i & 1] | off, ld_off, 0, 0);
    } else {   // LDS rows 8 g .. 8 g + 7 of a span of 128: rows g / 2 + 64 (g % 2) + 0, 8, .. 56 of it
      ld_off = i == 0 ? k0 + b0_off : ld_off + (i & 1 ? step_b : back_b);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ld_rsB, reinterpret_cast<lds_void_ptr>(dst), 16, b_voff[i & 1] | off, ld_off, 0, 0);
    }
  };
  // scales of the window that the loader's stage lies in, of the wave's 128 rows of A and of B
  v4i sc_in[NSC], sc[NSC];
  auto load_scales = [&]() __attribute__((always_inline)) {
    const int at = (ld_kt >> 1) * 1024;
    sc_in[0] = __builtin_amdgcn_raw_buffer_load_b128(ld_rsSa, lane * 16, at, 0);
    sc_in[1] = __builtin_amdgcn_raw_buffer_load_b128(ld_rsSa, lane * 16, at + windows * 1024, 0);
    sc_in[2] = __builtin_amdgcn_raw_buffer_load_b128(ld_rsSb, lane * 16, at, 0);
    sc_in[3] = __builtin_amdgcn_raw_buffer_load_b128(ld_rsSb, lane * 16, at + windows * 1024, 0);
  };
  auto next_scales = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NSC; ++i) sc[i] = sc_in[i];
  };

  // ---- fragments ----
  const int frow = lane & 15, fg = lane >> 4;
  const int fr = (frow & 7) ^ (frow >> 3);
  const uint32_t foff[2] = {(uint32_t)(frow * 128 + (((fg * 2) ^ fr) * 16)), (uint32_t)(frow * 128 + (((fg * 2 + 1) ^ fr) * 16))};
  typedef const __attribute__((address_space(3))) v4i *lds_v4i;
  auto frag_addrs = [&](int panel_a, int panel_b, uint32_t (&ad)[4]) {
    const uint32_t a = lds0 + panel_a + wm * (128 * 128), b = lds0 + panel_b + wn * (128 * 128);
    asm volatile("v_add_u32 %0, %1, %2" : "=v"(ad[0]) : "s"(a), "v"(foff[0]));
    asm volatile("v_add_u32 %0, %1, %2" : "=v"(ad[1]) : "s"(a), "v"(foff[1]));
    asm volatile("v_add_u32 %0, %1, %2" : "=v"(ad[2]) : "s"(b), "v"(foff[0]));
    asm volatile("v_add_u32 %0, %1, %2" : "=v"(ad[3]) : "s"(b), "v"(foff[1]));
  };
  auto read_frag = [&](uint32_t at, int t) { return *reinterpret_cast<lds_v4i>(at + t * 2048); };
  v4i fa[2][TM], fb[2][TN];   // of the stage's two halves
  uint32_t ad[4];
  // r-th read of half h: B0, A0, B1, .. in the order of their use (row by row of the wave's tiles)
  auto read_next = [&](auto half, int r) __attribute__((always_inline)) {
    constexpr int h = decltype(half)::value;
    if (r == 0) fb[h][0] = read_frag(ad[2 + h], 0);
    else if (r == 1) fa[h][0] = read_frag(ad[h], 0);
    else if (r <= TN) fb[h][r - 1] = read_frag(ad[2 + h], r - 1);
    else fa[h][r - TN] = read_frag(ad[h], r - TN);
  };

  v4f acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM * TN * 4; ++i) asm volatile("v_accvgpr_write_b32 %0, 0" : "=a"(acc[i / (4 * TN)][i / 4 % TN][i % 4]));
  // One element, and zero in its place for the next tile: the 256 instructions pass under the stores, and every trip is the same code
  // (one of its own for a tile's first stage, starting from constant zeros, spilled accumulators).
  auto acc_take = [&](int tm, int tn, int e) -> float {
    float x;
    asm volatile("v_accvgpr_read_b32 %0, %1\n\tv_accvgpr_write_b32 %1, 0" : "=v"(x), "+a"(acc[tm][tn][e]));
    return x;
  };
  [[maybe_unused]] v4i seg_bias = {0, 0, 0, 0};
  [[maybe_unused]] const __amdgpu_buffer_rsrc_t rsBias = make_rsrc(HAS_BIAS ? (const void *)p.bias : (const void *)p.A, HAS_BIAS ? (uint32_t)p.N * 2u : 0u);
  auto store_tile = [&](int m0, int n0) {
    int ldc2 = (int)p.ldc * 2;
    asm volatile("" : "+s"(ldc2));
    int l = lane;
    asm volatile("" : "+v"(l));
    const int col = wn * 128 + 8 * (l & 15);
    const __amdgpu_buffer_rsrc_t rsC = make_rsrc(p.C + (int64_t)m0 * p.ldc + n0, range(((int64_t)(p.M - m0 - 1) * p.ldc + (p.N - n0)) * 2));
    const uint32_t voff = (n0 + col < p.N) ? (uint32_t)(4 * (l >> 4) * ldc2 + col * 2) : kBeyond;
#pragma unroll
    for (int tm = 0; tm < TM; ++tm)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v4i out;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float lo = acc_take(tm, 2 * k, e), hi = acc_take(tm, 2 * k + 1, e);
          if constexpr (HAS_BIAS) {
            lo += __uint_as_float((uint32_t)seg_bias[k] << 16);
            hi += __uint_as_float((uint32_t)seg_bias[k] & 0xffff0000u);
          }
          typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
          const bf2 b = {(__bf16)lo, (__bf16)hi};
          out[k] = __builtin_bit_cast(int, b);
        }
        store16_streaming(out, rsC, voff, (wm * 128 + tm * 16 + e) * ldc2);
        __builtin_amdgcn_sched_barrier(0);
      }
  };

  // ---- prologue: two stages and the first window of scales requested, stage 0 published, its first fragments read ----
  ld_open(0);
  load_scales();
#pragma unroll
  for (int u = 0; u < 4; ++u) {
#pragma unroll
    for (int i = 0; i < NL; ++i) load_one(u & 1, u * UNIT, i);
    if (u & 1) ld_advance();
  }
  MX_WAIT_VM(2 * NL);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  frag_addrs(0, UNIT, ad);
  constexpr std::integral_constant<int, 0> lower{};
  constexpr std::integral_constant<int, 1> upper{};
#pragma unroll
  for (int r = 0; r < TM + TN; ++r) read_next(lower, r);
  next_scales();
  int s0 = 0;   // ring slot of this stage's A panel

  constexpr int N_MMA = TM * TN;        // of a half
  constexpr int SPREAD0 = 56, SPREAD1 = 60;   // instructions of the lower and the upper half over which the reads are spread
  // `stores`: those of the tile before were issued since the panels that this trip's barrier waits for were requested.  They are
  // younger than the panels and the counter retires in order, so the count allows for them.  ODD: the second stage of a window.
  // The first stage of a window requests the scales of the next: the loader is two stages ahead, in that window already.
  auto trip = [&](auto odd_tag, bool stores) __attribute__((always_inline)) {
    constexpr int ODD = decltype(odd_tag)::value ? 1 : 0;
    const int at1 = wrap(s0 + 4) * UNIT, at2 = s0 * UNIT;
    if constexpr (!ODD) load_scales();
    auto mma_one = [&](auto half, int i) __attribute__((always_inline)) {
      constexpr int h = decltype(half)::value;
      const int tm = i / TN, tn = i % TN;
      const v4i x = fa[h][tm], y = fb[h][tn];
      // fragments belong in ordinary registers: one among the accumulators' pushes an accumulator out to memory
      if (tn == 0) asm volatile("" : : "v"(x));
      if (tm == 0) asm volatile("" : : "v"(y));
      const v8i a = {x[0], x[1], x[2], x[3], 0, 0, 0, 0}, b = {y[0], y[1], y[2], y[3], 0, 0, 0, 0};
      acc[tm][tn] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc[tm][tn], 4, 4, 2 * ODD + h, sc[tm / 4][tm % 4], 2 * ODD + h, sc[2 + tn / 4][tn % 4]);
    };
    in_turn(std::make_integer_sequence<int, N_MMA>{}, [&](auto number) __attribute__((always_inline)) {
      constexpr int i = decltype(number)::value;
      mma_one(lower, i);
#pragma unroll
      for (int r = ((TM + TN) * i) / SPREAD0; i < SPREAD0 && r < ((TM + TN) * (i + 1)) / SPREAD0; ++r) read_next(upper, r);
#pragma unroll
      for (int j = (NL * i) / N_MMA; j < (NL * (i + 1)) / N_MMA; ++j) load_one(false, at1, j);
      if (i & 1) __builtin_amdgcn_sched_barrier(0);
    });
    frag_addrs(wrap(s0 + 2) * UNIT, wrap(s0 + 3) * UNIT, ad);
    constexpr int PEND = NL + (ODD ? 0 : NSC);
    if (!ODD && stores) MX_WAIT_VM_LGKM0(N_STORES + PEND);
    else MX_WAIT_VM_LGKM0(PEND);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    in_turn(std::make_integer_sequence<int, N_MMA>{}, [&](auto number) __attribute__((always_inline)) {
      constexpr int i = decltype(number)::value;
      mma_one(upper, i);
#pragma unroll
      for (int r = ((TM + TN) * i) / SPREAD1; i < SPREAD1 && r < ((TM + TN) * (i + 1)) / SPREAD1; ++r) read_next(lower, r);
#pragma unroll
      for (int j = (NL * i) / N_MMA; j < (NL * (i + 1)) / N_MMA; ++j) load_one(true, at2, j);
      if (i & 1) __builtin_amdgcn_sched_barrier(0);
    });
    ld_advance();
    s0 = wrap(s0 + 2);
  };
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
#pragma unroll 1
  for (int seg = 0; seg < n_seg; ++seg) {
    int m0, n0;
    origin(cur_mul, m0, n0);
    step(cur_mul);
    if constexpr (HAS_BIAS) {
      int l = lane;
      asm volatile("" : "+v"(l));
      seg_bias = __builtin_amdgcn_raw_buffer_load_b128(rsBias, (wn * 128 + 8 * (l & 15)) * 2, n0 * 2, 0);
    }
#pragma unroll 1
    for (int kt = 0; kt < KT; kt += 2) {
      trip(no, kt == 0 && seg > 0);
      if (kt + 1 < KT) trip(yes, false);
      next_scales();
    }
    if constexpr (HAS_BIAS) asm volatile("" : : "v"(seg_bias));
    store_tile(m0, n0);
  }
  // what was requested beyond the last tile (zeros) must have landed before the workgroup's LDS is released
  MX_WAIT_VM(0);
#else
  (void)p;
#endif
}

template <int WM, int WN, int TM, int TN, int NS>
static int launch_gemm_mxfp4(MxGemmArgs a, hipStream_t st) {
  constexpr int BM = WM * TM * 32, BN = WN * TN * 32;
  constexpr int lds = NS * (BM + BN) * 128 + (NS / 2 + 1) * (BM + BN) * 16;
  a.tiles_m = (a.M + BM - 1) / BM, a.tiles_n = (a.N + BN - 1) / BN;
  L8_REQUIRE((int64_t)a.tiles_m * a.tiles_n * (WM * WN * 64) < (1LL << 32), "l8_gemm_mxfp4_nt: more tiles than a grid has");
  a.wide = a.N % TN == 0 && a.ldc % TN == 0 && ((uintptr_t)a.C % (TN * 2)) == 0 && a.ldc < (1 << 22);
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

// Do the large kernel's tiles fill more than half of the units?  Its stream runs two stages ahead.  us, stream / tiles of 128 x 128, K
// 4096: [2048,4096], half of them, 32.2 / 30.3; [2304,4096] 31.6 / 36.5, [4096,4096] 40.2 / 50.0, [4000,11008] 95.6 / 122.4.
static bool takes_stream(int64_t M, int64_t N, int64_t blocks) {
  return ((M + 255) / 256) * ((N + 255) / 256) > num_cus() / 2 && blocks > 8 && num_cus() >= 8;
}
// bytes of one operand's laid-out scales: whole tiles of 256 rows, whole windows of 16 blocks
static int64_t laid_bytes(int64_t rows, int64_t blocks) { return (rows + 255) / 256 * 4 * ((blocks + 15) / 16) * 1024; }

// one workgroup per compute unit, a multiple of 8 of them (the hardware deals workgroups to the 8 XCDs in turn)
template <bool HAS_BIAS>
static int launch_gemm_mxfp4_stream(MxGemmArgs a, uint8_t *workspace, hipStream_t st) {
  constexpr int lds = 5 * 256 * 128;
  a.tiles_m = (a.M + 255) / 256, a.tiles_n = (a.N + 255) / 256;
  static bool ready[kMaxDev];
  const int slot = device_slot();
  if (slot < 0 || !ready[slot]) {
    L8_HIP(hipFuncSetAttribute((const void *)gemm_mxfp4_stream_kernel<HAS_BIAS>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    if (slot >= 0) ready[slot] = true;
  }
  const int windows = (a.blocks + 15) / 16;
  uint8_t *const tb = workspace + laid_bytes(a.M, a.blocks);
  const MxScaleArgs sc = {{a.sa, a.sb}, {workspace, tb}, {a.ldsa, a.ldsb}, {a.M, a.N}, {a.tiles_m * 4, a.tiles_n * 4}, a.blocks, windows};
  hipLaunchKernelGGL(mxfp4_lay_scales_kernel, dim3((unsigned)((windows + 3) / 4), (unsigned)(sc.chunks[0] + sc.chunks[1])), dim3(256), 0, st, sc);
  L8_HIP(hipGetLastError());
  a.sa = workspace, a.sb = tb;
  const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n, cus8 = (num_cus() / 8) * 8, want = (tiles + 7) / 8 * 8;
  hipLaunchKernelGGL((gemm_mxfp4_stream_kernel<HAS_BIAS>), dim3((unsigned)(want < cus8 ? want : cus8)), dim3(256), lds, st, a);
  L8_HIP(hipGetLastError());
  return L8_OK;
}

}  // namespace l8

using namespace l8;

extern "C" int64_t l8_gemm_mxfp4_workspace(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || M >= (1 << 28) || N >= (1 << 28) || K >= (1 << 24)) return 0;
  const int64_t blocks = (K + 31) / 32;
  return takes_stream(M, N, blocks) ? laid_bytes(M, blocks) + laid_bytes(N, blocks) : 0;
}

extern "C" int l8_gemm_mxfp4_nt(const void *A, const void *sa, const void *B, const void *sb, int64_t M, int64_t N, int64_t K, int64_t lda,
                                int64_t ldsa, int64_t ldb, int64_t ldsb, const void *bias, void *C, int64_t ldc, void *workspace,
                                int64_t workspace_bytes, void *stream) {
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
  L8_REQUIRE(((M + 255) / 256) * ((N + 255) / 256) < (1 << 24), "l8_gemm_mxfp4_nt: more tiles than a grid has");   // (tiles are counted in 32 bits)
  if (takes_stream(M, N, blocks)) {
    const int64_t need = l8_gemm_mxfp4_workspace(M, N, K);
    L8_REQUIRE(workspace && workspace_bytes >= need && ((uintptr_t)workspace % 16) == 0, "l8_gemm_mxfp4_nt: needs a 16-byte aligned workspace of %lld bytes",
               (long long)need);
    // (its stores take eight columns at once, and the groups of rows of its scales are a grid's second dimension)
    if (N % 8 == 0 && ldc % 8 == 0 && ((uintptr_t)C % 16) == 0 && ldc < (1 << 22) && ((uintptr_t)bias % 4) == 0 && (M + 255) / 256 + (N + 255) / 256 < 16384)
      return bias ? launch_gemm_mxfp4_stream<true>(a, (uint8_t *)workspace, st) : launch_gemm_mxfp4_stream<false>(a, (uint8_t *)workspace, st);
  }
  // Otherwise the smallest tile that gives no compute unit a second workgroup, with a ring of four stages; beyond, 128 x 128 ones with
  // two stages, two workgroups a unit.  us, weights that no cache holds, [M,N] K: 64 x 64 / 128 x 64 / 64 x 128 / 128 x 128 / the last:
  //   [65,4096] 4096 8.3 / 9.7 / 10.1 / 12.0 / 13.9, [333,2048] 8192 13.0 / 15.6 / 15.9 / 19.5 / 24.5, [300,4096] 4096 11.0 / 10.4 / 10.5 /
  //   12.4 / 14.2, [128,11008] 4096 16.3 / 13.6 / 14.0 / 16.8 / 20.1, [256,11008] 4096 22.1 / 23.2 / 24.4 / 16.9 / 20.3, from the cache
  //   [2064,2048] 1024 11.9 / 14.9 / 14.9 / 11.9 / 9.3
  // Other rings: 64 x 64 with two stages 11.0 and with eight 8.9 on the first, 128 x 64 with six 11.1 on the third.
  auto tiles = [&](int64_t bm, int64_t bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
  const int64_t cus = num_cus();
  if (tiles(64, 64) <= cus) return launch_gemm_mxfp4<2, 2, 1, 1, 4>(a, st);
  if (tiles(128, 64) <= cus) return launch_gemm_mxfp4<2, 2, 2, 1, 4>(a, st);
  if (tiles(64, 128) <= cus) return launch_gemm_mxfp4<2, 2, 1, 2, 4>(a, st);
  if (tiles(128, 128) <= cus) return launch_gemm_mxfp4<4, 2, 1, 2, 4>(a, st);
  return launch_gemm_mxfp4<4, 2, 1, 2, 2>(a, st);
}
