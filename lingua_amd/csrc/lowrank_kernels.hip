// Low-rank adapters of many requests at once, beside a projection that they share: token t of adapter i gets
//
//   out_t = y_t + s_i (x_t A_i^T) B_i            A [n, r, K], B [n, r, N] bf16, i = index[t]
//
// and the backward pass
//
//   gh_t = s_i gy_t B_i^T,  gx_t = gh_t A_i,  gA_i = sum over its tokens of gh_t (x) x_t,  gB_i = sum of s_i h_t (x) gy_t.
//
// Both factors lie with the rank in front, so that three kernels serve both passes: `shrink` (rows times a factor along its long side),
// `expand` (h times a factor across it, added to y or not) and `outer` (the factors' gradients).  All of it is bound by memory: r is
// far below the 300 flop per byte at which the matrix cores would be, so tokens' rows go from memory to the matrix instruction's
// registers as they lie, in whole lines, and factors, of which there are few, come from the L2.
//
// Tokens are grouped by adapter first (`route`: a stable order, so every sum has one order), and a workgroup's tile holds tokens of one
// adapter: tile s of B tokens belongs to the group g with the largest starts[g] / B + g <= s, since a group of c tokens that begins at
// starts[g] takes at most ceil(c / B) of the starts[g + 1] / B + g + 1 - (starts[g] / B + g) numbers between its own first and the next
// one's.  That leaves at most one number a group unused and needs no table of tiles.  Groups n and n + 1 are the tokens without an adapter
// (out = y) and those whose index is no adapter's (out = NaN: the index is on the GPU, where nothing can be refused).
//
// h is held in 32 bits, [splits, T, r]: K is shared out over `splits` workgroups where there are few tokens, and whoever reads h adds the
// parts up in order.  Where h is an operand of a matrix instruction it goes in as two bf16 numbers, hi + lo, 16 bits of it: the second
// product costs nothing beside memory (with r <= 16 the two halves even share one instruction), and the result is rounded once, at the end.
// (An infinity on the other side of such a product makes infinity or NaN: hi and lo may have different signs.)
#include "l8_common.h"

#include <algorithm>

namespace l8 {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

L8_DEV v4f mfma(v4i a, v4i b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0); }

// ---- tokens by adapter ----

constexpr int kRouteBlock = 1024, kRouteWaves = kRouteBlock / 64, kRouteTimes = 16;

// A workgroup per group: how many tokens stand in front of its own, then its own tokens in their order.  Sixteen tokens a thread are
// requested together and stay in registers between the two counts.  Every workgroup reads the whole index, so that none waits for another:
// 16384 tokens and 8 adapters 6.5 us, 2055 and 12 5.0 (a launch that does nothing: 2 to 3), one launch in place of a count, a sum and a scatter.
template <typename Index>
__global__ __launch_bounds__(kRouteBlock) void lowrank_route_kernel(const Index *__restrict__ index, int T, int n, int *__restrict__ order, int *__restrict__ starts) {
  constexpr int SPAN = kRouteBlock * kRouteTimes, PLACES = kRouteTimes * kRouteWaves;
  static_assert(PLACES == 256, "four places a lane of one wave");
  __shared__ int sums[kRouteWaves], place[PLACES + 1];
  const int mine = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int group[kRouteTimes];
  auto load = [&](int t0) {
    int64_t i[kRouteTimes];
#pragma unroll
    for (int k = 0; k < kRouteTimes; ++k) {
      const int t = t0 + k * kRouteBlock + (int)threadIdx.x;
      i[k] = (int64_t)index[min(t, T - 1)];
    }
#pragma unroll
    for (int k = 0; k < kRouteTimes; ++k)
      group[k] = t0 + k * kRouteBlock + (int)threadIdx.x >= T ? n + 2 : i[k] >= 0 && i[k] < n ? (int)i[k] : i[k] == -1 ? n : n + 1;
  };
  int less = 0;
  for (int t0 = 0; t0 < T; t0 += SPAN) {
    load(t0);
#pragma unroll
    for (int k = 0; k < kRouteTimes; ++k) less += group[k] < mine;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) less += __shfl_xor(less, d);
  if (lane == 0) sums[wave] = less;
  __syncthreads();
  int at = 0;
#pragma unroll
  for (int w = 0; w < kRouteWaves; ++w) at += sums[w];
  if (threadIdx.x == 0) {
    starts[mine] = at;
    if (mine == n + 1) starts[n + 2] = T;
  }
  for (int t0 = 0; t0 < T; t0 += SPAN) {
    if (T > SPAN) load(t0);
#pragma unroll
    for (int k = 0; k < kRouteTimes; ++k) {
      const uint64_t votes = __ballot(group[k] == mine);
      if (lane == 0) place[k * kRouteWaves + wave] = __popcll(votes);
    }
    __syncthreads();
    if (wave == 0) {   // counts -> how many stand in front
      int c[4], sum = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) sum += c[k] = place[lane * 4 + k];
      int upto = sum;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int other = __shfl_up(upto, d);
        if (lane >= d) upto += other;
      }
      int before = upto - sum;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        place[lane * 4 + k] = before;
        before += c[k];
      }
      if (lane == 63) place[PLACES] = upto;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kRouteTimes; ++k) {
      const bool own = group[k] == mine;
      const uint64_t votes = __ballot(own);
      if (own) order[at + place[k * kRouteWaves + wave] + __popcll(votes & ((1ull << lane) - 1))] = t0 + k * kRouteBlock + (int)threadIdx.x;
    }
    at += place[PLACES];
    __syncthreads();
  }
}

// The tokens by adapter: `route`'s answer, or the index itself where there are few enough tokens for a wave to look at all of them.
struct Tokens {
  const int *order, *starts;   // NULL: the index
  const void *index;
  int index_i64;
};
constexpr int kFewTokens = 64;

struct Tile {
  int group, count;            // count 0: a number that no tile has
  int first, piece, tokens;    // (of `route`) where its tokens begin in the order, which of its group's tiles it is, and the group's tokens
  int mine;                    // lane m has token m
  L8_DEV int token(int m) const { return __shfl(mine, min(m, count - 1)); }
};
// What is read of `order` and `starts` is held to their range, so that memory that `route` has not written yet (it was captured and not replayed,
// or runs on another stream) makes wrong results and no access out of bounds.
L8_DEV int within(int v, int top) { return (int)min((unsigned)v, (unsigned)top); }
// Tile `slot` of at most `size` tokens.  The same for the whole workgroup.
L8_DEV Tile tile_of(const int *__restrict__ starts, int T, int n, int size, int slot) {
  const int lane = threadIdx.x & 63;
  Tile t{};
  int before = 0;
  for (int i0 = 0;; i0 += 64) {   // the groups whose first number is at most `slot` come first
    const int i = i0 + lane, from = within(starts[min(i, n + 1)], T), to = within(starts[min(i, n + 1) + 1], T);
    const int have = __popcll(__ballot(i < n + 2 && from / size + i <= slot));
    if (have) {
      const int at = have - 1;
      t.group = i0 + at;
      before = __builtin_amdgcn_readlane(from, at);
      t.tokens = __builtin_amdgcn_readlane(to, at) - before;
    }
    if (have < 64 || i0 + 64 >= n + 2) break;
  }
  t.piece = slot - (before / size + t.group);
  t.first = before + t.piece * size;
  t.count = min(size, max(0, t.tokens - t.piece * size));
  if (t.piece < 0) t.count = 0, t.piece = 1;   // (starts that do not ascend)
  return t;
}
// The same with its tokens: up to 64.
L8_DEV Tile tile_with_tokens(const Tokens &tk, int T, int n, int size, int slot) {
  const int lane = threadIdx.x & 63;
  if (tk.order) {
    Tile t = tile_of(tk.starts, T, n, size, slot);
    t.mine = t.count ? within(tk.order[t.first + min(lane, t.count - 1)], T - 1) : 0;
    return t;
  }
  // few tokens: every lane finds the tokens of its own group, bit by bit of the group's number; every sixteenth of a group begins a tile
  const int64_t i = lane >= T ? -1 : tk.index_i64 ? ((const int64_t *)tk.index)[lane] : (int64_t)((const int32_t *)tk.index)[lane];
  const int group = i >= 0 && i < n ? (int)i : i == -1 ? n : n + 1;
  uint64_t same = __ballot(lane < T);
  for (int bit = 0; (n + 1) >> bit; ++bit) {
    const bool set = group >> bit & 1;
    const uint64_t votes = __ballot(set);
    same &= set ? votes : ~votes;
  }
  const uint64_t below = (1ull << lane) - 1;
  const int place = __popcll(same & below);
  const uint64_t firsts = __ballot(lane < T && place % size == 0);
  Tile t{};
  const uint64_t mine = __ballot((firsts >> lane & 1) && __popcll(firsts & below) == slot);
  if (!mine) return t;
  const int lead = __builtin_ctzll(mine);
  t.group = __builtin_amdgcn_readlane(group, lead);
  const int from = __builtin_amdgcn_readlane(place, lead);
  const bool in = lane < T && group == t.group && place >= from && place < from + size;
  t.count = __popcll(__ballot(in));
  // every token goes to the lane of its place; the others go where no token of the tile is (a tile of 16: the last lane)
  t.mine = __builtin_amdgcn_ds_permute((in ? place - from : 63) * 4, lane);
  return t;
}

// ---- rows times a factor along its long side ----

struct ShrinkArgs {
  const uint16_t *x, *f;
  Tokens tokens;
  float *h;
  int64_t ldx;
  int T, K, n, r, splits;
};

// MT tiles of 16 tokens by RT of 16 ranks; the W waves share K.  A wave takes 64 columns a step, the waves side by side.  Eight neighbouring
// lanes read a row's 128 bytes: the matrix instruction wants neighbouring rows in neighbouring lanes, and read like that every 16 bytes are a
// line of their own to the cache, 64 of them an instruction.  So what was read goes through LDS of the wave's own, chunk c of a row at place c
// ^ (row % 8), where neither side meets a bank twice.  Which column meets which place of the instruction does not matter as long as it is the
// same for both operands.  blockIdx.z: which 16 RT of more than 64 ranks.
// us, rank 16: [16384,4096] 29.8 (134 MB, 4.5 TB/s), [16384,11008] 78 (4.6 TB/s), [1500,4096] in four parts 8.6 (10.3 without the turn through LDS);
// rank 64: [16384,4096] 36.7, [2055,4096] in three parts 14.2.  A unit takes in no more than some 45 bytes a ns (all of them twice the memory's
// rate): few tiles are bound by that, hence the parts, many by memory.
template <int MT, int RT, int W>
__global__ __launch_bounds__(W * 64) void lowrank_shrink_kernel(const ShrinkArgs p) {
  constexpr int BOTH = MT > RT ? MT : RT, RED = MT * RT * 64;
  constexpr int ROOM = W * BOTH * 128 > W / 2 * RED ? W * BOTH * 128 : W / 2 * RED;
  __shared__ v4i room[ROOM];   // of a wave: one operand's tiles, 16 rows of eight chunks each; at the end: sums
  const Tile tile = tile_with_tokens(p.tokens, p.T, p.n, MT * 16, blockIdx.x);
  if (tile.group >= p.n || tile.count == 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
  const int K = p.K, steps = (K + 63) / 64, rank0 = blockIdx.z * RT * 16;
  const int lo = (int)((int64_t)steps * blockIdx.y / p.splits), hi = (int)((int64_t)steps * (blockIdx.y + 1) / p.splits);
  v4i *mine = room + wave * BOTH * 128;
  const int r8 = lane >> 3, chunk = ((lane & 7) ^ r8) * 8;   // this lane reads rows r8 and r8 + 8 of a tile, from column `chunk` of a step on
  const uint16_t *xr[MT][2], *fr[RT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 2; ++i) xr[m][i] = p.x + (int64_t)tile.token(m * 16 + i * 8 + r8) * p.ldx;
#pragma unroll
  for (int j = 0; j < RT; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) fr[j][i] = p.f + ((int64_t)tile.group * p.r + min(rank0 + j * 16 + i * 8 + r8, p.r - 1)) * K;
  v4f acc[MT][RT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[m][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  v4i a[2][MT][2], b[2][RT][2];
  auto request = [&](int s, int step) {
    // the last step may pass the row's end: columns beyond it are read from within the row and zeroed before they are used
    const int k = min(step * 64 + chunk, K - 8);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int j = 0; j < RT; ++j) b[s][j][i] = *(const v4i *)(fr[j][i] + k);
#pragma unroll
      for (int m = 0; m < MT; ++m) a[s][m][i] = *(const v4i *)(xr[m][i] + k);
    }
  };
  auto fragment = [&](int t, int c) { return mine[t * 128 + row * 8 + ((c * 4 + g) ^ (row & 7))]; };
  auto multiply = [&](int s, int step) {
    if (step * 64 + chunk >= K) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int m = 0; m < MT; ++m) a[s][m][i] = v4i{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < RT; ++j) b[s][j][i] = v4i{0, 0, 0, 0};
      }
    }
    v4i f[RT][2];
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) mine[(j * 2 + i) * 64 + lane] = b[s][j][i];
    __builtin_amdgcn_wave_barrier();   // one wave's own LDS: it keeps the order of what it issues
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) f[j][c] = fragment(j, c);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i) mine[(m * 2 + i) * 64 + lane] = a[s][m][i];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const v4i x = fragment(m, c);
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[m][j] = mfma(x, f[j][c], acc[m][j]);
      }
    __builtin_amdgcn_wave_barrier();
  };
  int step = lo + wave;
  if (step < hi) request(0, step);
  while (step < hi) {
    request(1, min(step + W, hi - 1));
    multiply(0, step);
    step += W;
    if (step >= hi) break;
    request(0, min(step + W, hi - 1));
    multiply(1, step);
    step += W;
  }
  // the upper half of the waves hands its sums to the lower half, until one has them all
  __syncthreads();   // (they take the tiles' place)
#pragma unroll
  for (int half = W / 2; half; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < RT; ++j) *(v4f *)&room[(wave - half) * RED + (m * RT + j) * 64 + lane] = acc[m][j];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < RT; ++j) {
          const v4f other = *(const v4f *)&room[wave * RED + (m * RT + j) * 64 + lane];
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][j][i] += other[i];
        }
    }
    __syncthreads();
  }
  if (wave) return;
  // a lane has rank `row` of each sixteen, tokens 4 g .. 4 g + 3
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = m * 16 + g * 4 + i, token = tile.token(at);
      if (at >= tile.count) continue;
      float *out = p.h + ((int64_t)blockIdx.y * p.T + token) * p.r;
#pragma unroll
      for (int j = 0; j < RT; ++j)
        if (rank0 + j * 16 + row < p.r) out[rank0 + j * 16 + row] = acc[m][j][i];
    }
}

// ---- h times a factor across its long side ----

// Eight values of h, `splits` parts added up in order, times the adapter's scale.
L8_DEV void load_h(float (&v)[8], const float *__restrict__ h, int64_t part, int splits, float scale) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.0f;
  for (int s = 0; s < splits; ++s) {
    const v4f u = *(const v4f *)(h + s * part), w = *(const v4f *)(h + s * part + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += u[e], v[e + 4] += w[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= scale;
}
// hi + lo = v to 16 bits, both bf16; a v that is not finite is hi alone.
L8_DEV uint32_t hi_bits(float v) { return bf16_rne_bits(v); }
L8_DEV uint32_t lo_bits(float v) {
  const uint32_t hi = bf16_rne_bits(v);
  return (hi & 0x7f80u) == 0x7f80u ? 0u : bf16_rne_bits(v - bf16_bits_to_f32(hi));
}
L8_DEV v4i pack8(const float (&v)[8], bool low) {
  v4i out;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t a = low ? lo_bits(v[2 * k]) : hi_bits(v[2 * k]), b = low ? lo_bits(v[2 * k + 1]) : hi_bits(v[2 * k + 1]);
    out[k] = (int)(a | (b << 16));
  }
  return out;
}
// Eight rows of eight columns -> for each column the eight rows' values, one v_perm per two values.
L8_DEV void transpose8(v4i (&out)[8], const v4i (&rows)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      out[j][k] = (int)__builtin_amdgcn_perm((uint32_t)rows[2 * k + 1][j >> 1], (uint32_t)rows[2 * k][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
}

struct ExpandArgs {
  const uint16_t *y, *f;
  const float *h, *scale;
  Tokens tokens;
  uint16_t *out;
  int64_t ldy, ldo;
  int T, N, n, r, splits, chunks, per;   // (of 128 columns in a row: a workgroup's)
};

constexpr int kExpandWaves = 4;

// 16 tokens by 128 columns a wave and step; the workgroup's four waves are PARTS parts of a tile's tokens by 4 / PARTS stretches of columns.
// Column 8 c + j of a wave's 128 is column c of matrix instruction j: a lane then reads eight neighbouring columns of eight rows of the
// factor, turns the block round in registers, and ends up with eight neighbouring columns of four tokens: 16-byte loads and stores, 256 bytes
// of a row at once.
// KS steps of 32 ranks, each with the upper and the lower bits of h; KS 0: up to 16 ranks, where one instruction takes both.
// Waves of the same columns and more than 16 ranks share the factor's turned blocks through LDS, each making a part of them, and go on to the
// next 128 columns `per` times: h, 4 r bytes a token and more in parts, is then read once for all of them.  The next step's y and factor are
// requested before the present one is multiplied.
// A tile waits for memory three times: for its place, for its tokens, for everything else.
// us at [16384,4096] with y, 402 MB: up to 16 ranks with five waves a SIMD 52 (7.7 TB/s, a part of it from the caches), with four 61, with six 57;
// 64 ranks 67, up to two steps a workgroup 75, and of h in three parts 91 for up to two and 77 for up to eight.  [16384,11008] of rank 16: 131,
// 5.5 TB/s.
template <int PARTS, int KS>
__global__ __launch_bounds__(kExpandWaves * 64, KS == 0 ? 5 : PARTS == 1 ? 1 : 2) void lowrank_expand_kernel(const ExpandArgs p) {
  constexpr int STEPS = KS ? KS : 1;
  constexpr bool SHARED = PARTS == kExpandWaves && KS > 0;
  __shared__ v4i turned[2][SHARED ? STEPS * 8 * 64 : 1];
  const int slot = blockIdx.x / p.chunks, chunk = blockIdx.x - slot * p.chunks;
  const Tile tile = tile_with_tokens(p.tokens, p.T, p.n, PARTS * 16, slot);
  if (tile.count == 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
  const int part0 = wave % PARTS * 16;
  const int N = p.N, r = p.r, per = SHARED ? p.per : 1;
  const int col0 = SHARED ? chunk * per * 128 + row * 8 : (chunk * (kExpandWaves / PARTS) + wave / PARTS) * 128 + row * 8;
  int64_t t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = tile.token(part0 + g * 4 + i);
  v4i y[SHARED ? 2 : 1][4];
  auto request_y = [&](int s, int col) {   // (beyond the last column: the first ones, which nobody stores)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[s][i] = v4i{0, 0, 0, 0};
      if (p.y) y[s][i] = __builtin_nontemporal_load((const v4i *)(p.y + t[i] * p.ldy + (col < N ? col : 0)));
    }
  };
  auto store = [&](int i, int col, v4i v) {
    if (col < N && part0 + g * 4 + i < tile.count) __builtin_nontemporal_store(v, (v4i *)(p.out + t[i] * p.ldo + col));
  };
  request_y(0, col0);
  if (tile.group >= p.n) {   // no adapter: y as it is; no known adapter: NaN
    for (int c = 0; c < per; ++c) {
      if (c) request_y(0, col0 + c * 128);
#pragma unroll
      for (int i = 0; i < 4; ++i) store(i, col0 + c * 128, tile.group > p.n ? v4i{0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0} : y[0][i]);
    }
    return;
  }
  auto rank_of = [&](int s) { return KS ? s * 32 + g * 8 : (g & 1) * 8; };
  const float *h = p.h + (int64_t)tile.token(part0 + row) * r;
  v4f hp[STEPS][2];   // of h: the first of its parts
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int k0 = min(rank_of(s), r - 8);
    hp[s][0] = *(const v4f *)(h + k0), hp[s][1] = *(const v4f *)(h + k0 + 4);
  }
  const float scale = p.scale ? p.scale[tile.group] : 1.0f;
  auto request_f = [&](v4i (&rows)[8], int s, int col) {
    const uint16_t *f = p.f + ((int64_t)tile.group * r + min(rank_of(s), r - 8)) * N + (col < N ? col : 0);
#pragma unroll
    for (int e = 0; e < 8; ++e) rows[e] = *(const v4i *)(f + (int64_t)e * N);
  };
  auto turn = [&](v4i (&b)[8], v4i (&rows)[8], int s) {
    if (rank_of(s) >= r) {
#pragma unroll
      for (int e = 0; e < 8; ++e) rows[e] = v4i{0, 0, 0, 0};   // (ranks beyond r: zero, whatever the row that was read holds)
    }
    transpose8(b, rows);
  };
  constexpr int MINE = SHARED ? (STEPS + kExpandWaves - 1) / kExpandWaves : STEPS;   // blocks of the factor that a wave reads
  static_assert(!SHARED || MINE == 1, "a wave turns one block");
  v4i rows[MINE][8];
  if constexpr (SHARED) {
    if (wave < STEPS) request_f(rows[0], wave, col0);
  } else {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) request_f(rows[s], s, col0);
  }
  v4i hi[STEPS], lo[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int k0 = rank_of(s);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = hp[s][e >> 2][e & 3];
    for (int q0 = 1; q0 < p.splits; q0 += 3) {   // three parts at a time: what stands in for one that is not there is not added
      v4f u[3], w[3];
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        const float *more = h + (int64_t)min(q0 + q, p.splits - 1) * p.T * r + min(k0, r - 8);
        u[q] = *(const v4f *)more, w[q] = *(const v4f *)(more + 4);
      }
#pragma unroll
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (q0 + q < p.splits) v[e] += u[q][e], v[e + 4] += w[q][e];
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k0 < r ? v[e] * scale : 0.0f;
    if constexpr (KS) {
      hi[s] = pack8(v, false), lo[s] = pack8(v, true);
    } else {
      hi[s] = g < 2 ? pack8(v, false) : pack8(v, true);
    }
  }
  auto step = [&](int s, int c) {   // step c of the columns, with y in y[s]
    const int col = col0 + c * 128;
    v4f acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    v4i own[8];
    if constexpr (SHARED) {
      if (wave < STEPS) {
        turn(own, rows[0], wave);
#pragma unroll
        for (int j = 0; j < 8; ++j) turned[s][(wave * 8 + j) * 64 + lane] = own[j];
      }
      __syncthreads();   // (the other buffer: whoever reads it has not passed the next barrier)
      if (c + 1 < per) {
        request_y(SHARED ? s ^ 1 : 0, col + 128);
        if (wave < STEPS) request_f(rows[0], wave, col + 128);
      }
    }
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      v4i b[8];
      if constexpr (SHARED) {
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] = turned[s][(k * 8 + j) * 64 + lane];
      } else {
        turn(b, rows[k], k);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = mfma(hi[k], b[j], acc[j]);
      if constexpr (KS > 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = mfma(lo[k], b[j], acc[j]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v4i out;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float u = __uint_as_float((uint32_t)y[s][i][k] << 16) + acc[2 * k][i], v = __uint_as_float((uint32_t)y[s][i][k] & 0xffff0000u) + acc[2 * k + 1][i];
        out[k] = (int)(bf16_rne_bits(u) | (bf16_rne_bits(v) << 16));
      }
      store(i, col, out);
    }
  };
  if constexpr (!SHARED) {
    step(0, 0);
  } else {
#pragma unroll 1
    for (int c = 0; c < per; c += 2) {
      step(0, c);
      if (c + 1 < per) step(1, c + 1);
    }
  }
}

// ---- gradients of the factors ----

struct OuterSide {           // grad_i [r, D] = sum over the tokens of i of h_t (x) z_t
  const float *h;
  const uint16_t *z;
  uint16_t *grad;
  float *partials;           // [2 (T / size + 1), r, D]: groups of more than one tile
  int64_t ldz;
  int D, splits, chunks;     // chunks of 512 columns
};
struct OuterArgs {
  OuterSide side[2];
  const float *scale;
  const int *order, *starts;
  int T, n, r, size;
  const uint16_t *f;         // with ALSO_H: the factor that z is multiplied with, [n, r, D]
  float *also;               //              and where that goes, [chunks, T, r], a part for each 512 columns
};

constexpr int kOuterWaves = 4;

// Where a tile of a group that has several leaves its sums: the first of a group and the others apart, since a group's last tile and the
// next group's first may begin within one `size` tokens.
L8_DEV int64_t outer_part(int first, int size, int piece) { return 2 * (int64_t)(first / size) + (piece > 0); }

// RT tiles of 16 ranks by 128 columns a wave, over a tile's tokens.  z is read as `expand` reads the factor: eight neighbouring columns of
// eight tokens' rows a lane, turned round in registers, 32 tokens requested ahead; h is laid out by rank in LDS, TOKENS at a time, both
// halves of its bits.  Two waves a SIMD: 64 ranks of [16384,4096] and [16384,4096] 130 us where the compiler made room for one, 107.
//
// With ALSO_H the kernel also does `shrink`'s work on z, which both read whole: 32 tokens by a wave's 128 columns go through LDS of the wave's
// own, whose rows are what the matrix instruction wants them to be, and meet the factor's 128 columns, which stay in registers; every 64
// tokens (32 with more than 16 ranks) the waves' sums are added up.  Up to 32 ranks, whose registers leave room for that.
// A tile's columns are neighbouring workgroups, so that its rows are read as whole lines of memory at one time: [16384,8192] 72 us, the tiles being
// neighbours 94; the gradients alone do better with neighbouring tiles (both sides of [16384,4096] to [16384,4096] a whole pass of 127 and 134).
// us: [16384,4096] of rank 16 36 (134 MB, 3.7 TB/s), of rank 64 two such sides 90 (3.0; and 67 MB of sums of tiles, written and read); with
// ALSO_H [16384,11008] 97 (361 MB, 3.7 TB/s) where both by themselves take 177.
template <int RT, int TOKENS, bool ALSO_H>
__global__ __launch_bounds__(kOuterWaves * 64, 2) void lowrank_outer_kernel(const OuterArgs p) {
  constexpr int PITCH = TOKENS + 8, ZPITCH = 128 + 8;
  __shared__ __attribute__((aligned(16))) uint16_t zs[ALSO_H ? kOuterWaves : 1][ALSO_H ? 32 : 1][ZPITCH];
  constexpr int HELD = RT == 1 ? 2 : 1;   // times 32 tokens whose sums a wave keeps until the waves' are added up
  static_assert(!ALSO_H || HELD * 32 * RT * 16 * 4 <= 32 * ZPITCH * 2, "these sums take the place of its z");
  __shared__ __attribute__((aligned(16))) uint16_t hs[2][RT * 16][PITCH];
  __shared__ __attribute__((aligned(16))) int toks[TOKENS];
  const int chunks = p.side[1].chunks;
  const int slot = ALSO_H ? (int)blockIdx.x / chunks : (int)blockIdx.x, place = ALSO_H ? (int)blockIdx.x - slot * chunks : (int)blockIdx.y;
  const Tile tile = tile_of(p.starts, p.T, p.n, p.size, slot);
  if (tile.group >= p.n || (tile.count == 0 && tile.piece > 0)) return;
  const int which = place >= p.side[0].chunks;
  const OuterSide &sd = p.side[which];
  const int chunk = place - (which ? p.side[0].chunks : 0);
  const int rank0 = blockIdx.z * RT * 16, r = p.r, D = sd.D;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
  const int col = (chunk * kOuterWaves + wave) * 128 + row * 8;
  const bool in = col < D;
  const uint16_t *z = sd.z + (in ? col : 0);
  const int64_t ldz = sd.ldz;
  const float scale = p.scale ? p.scale[tile.group] : 1.0f;
  v4f acc[RT][8];
#pragma unroll
  for (int m = 0; m < RT; ++m)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[m][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  [[maybe_unused]] v4i f[ALSO_H ? 4 : 1][RT];
  [[maybe_unused]] v4f sums[HELD][ALSO_H ? 2 : 1][RT];   // by 32 tokens, by 16
  if constexpr (ALSO_H) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int at = (chunk * kOuterWaves + wave) * 128 + k * 32 + g * 8;
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        f[k][j] = *(const v4i *)(p.f + ((int64_t)tile.group * r + min(j * 16 + row, r - 1)) * D + (at < D ? at : 0));
        if (at >= D) f[k][j] = v4i{0, 0, 0, 0};
      }
    }
  }
#pragma unroll 1
  for (int p0 = 0; p0 < tile.count; p0 += TOKENS) {
    const int here = min(TOKENS, tile.count - p0), subs = (here + 31) / 32;
    __syncthreads();
    for (int i = threadIdx.x; i < TOKENS * RT * 2; i += kOuterWaves * 64) {   // eight ranks of a token; neighbouring lanes write neighbouring tokens
      const int at = i % TOKENS, k = i / TOKENS * 8;
      const int token = within(p.order[tile.first + p0 + min(at, here - 1)], p.T - 1);
      if (k == 0) toks[at] = token;
      float v[8];
      if (at < here && rank0 + k < r) {
        load_h(v, sd.h + (int64_t)token * r + rank0 + k, (int64_t)p.T * r, sd.splits, scale);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) hs[0][k + e][at] = (uint16_t)hi_bits(v[e]), hs[1][k + e][at] = (uint16_t)lo_bits(v[e]);
    }
    __syncthreads();
    v4i rows[2][8];
    auto request = [&](int s, int sub) {
      const v4i t0 = *(const v4i *)&toks[sub * 32 + g * 8], t1 = *(const v4i *)&toks[sub * 32 + g * 8 + 4];
#pragma unroll
      for (int e = 0; e < 8; ++e) rows[s][e] = *(const v4i *)(z + (int64_t)(e < 4 ? t0[e & 3] : t1[e & 3]) * ldz);
    };
    auto multiply = [&](int s, int sub) {
      v4i(&z8)[8] = rows[s];
      if (sub * 32 + 32 > here) {   // behind the last token stands the last one again: not a number times zero is no zero
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (sub * 32 + g * 8 + e >= here) z8[e] = v4i{0, 0, 0, 0};
      }
      if constexpr (ALSO_H) {
#pragma unroll
        for (int e = 0; e < 8; ++e) *(v4i *)&zs[wave][g * 8 + e][row * 8] = in ? z8[e] : v4i{0, 0, 0, 0};   // (columns that are not there: both factors zero)
        __builtin_amdgcn_wave_barrier();   // one wave's own LDS: it keeps the order of what it issues
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
          for (int j = 0; j < RT; ++j) sums[s % HELD][m][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const v4i a = *(const v4i *)&zs[wave][m * 16 + row][k * 32 + g * 8];
#pragma unroll
            for (int j = 0; j < RT; ++j) sums[s % HELD][m][j] = mfma(a, f[k][j], sums[s % HELD][m][j]);
          }
        }
        __builtin_amdgcn_wave_barrier();
      }
      v4i b[8];
      transpose8(b, z8);
#pragma unroll
      for (int m = 0; m < RT; ++m)
#pragma unroll
        for (int low = 0; low < 2; ++low) {
          const v4i a = *(const v4i *)&hs[low][m * 16 + row][sub * 32 + g * 8];
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[m][j] = mfma(a, b[j], acc[m][j]);
        }
    };
    [[maybe_unused]] auto hand_over = [&](int sub, int count) {   // the sums of `count` times 32 tokens from 32 sub on
      if constexpr (ALSO_H) {
        float *mine = (float *)&zs[wave][0][0];
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
          if (h >= count) break;
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i) mine[(h * 32 + m * 16 + g * 4 + i) * (RT * 16) + j * 16 + row] = sums[h][m][j][i];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < count * 32 * RT * 16; i += kOuterWaves * 64) {
          const int at = sub * 32 + i / (RT * 16), rank = i % (RT * 16);
          float v = 0.0f;
#pragma unroll
          for (int w = 0; w < kOuterWaves; ++w) v += ((const float *)&zs[w][0][0])[i];
          if (at < here && rank < r) p.also[((int64_t)chunk * p.T + toks[at]) * r + rank] = v;
        }
        __syncthreads();
      }
    };
    request(0, 0);
#pragma unroll 1
    for (int sub = 0; sub < subs; sub += 2) {
      request(1, min(sub + 1, subs - 1));
      multiply(0, sub);
      if (HELD == 1 || sub + 1 >= subs) hand_over(sub, 1);
      if (sub + 1 >= subs) break;
      request(0, min(sub + 2, subs - 1));
      multiply(1, sub + 1);
      hand_over(HELD == 1 ? sub + 1 : sub, HELD);
    }
  }
  if (!in) return;
  // a lane has columns col .. col + 7 of ranks 4 g .. 4 g + 3 of each sixteen
  const bool alone = tile.tokens <= p.size;
#pragma unroll
  for (int m = 0; m < RT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rank = rank0 + m * 16 + g * 4 + i;
      if (rank >= r) continue;
      if (alone) {
        v4i out;
#pragma unroll
        for (int k = 0; k < 4; ++k) out[k] = (int)(bf16_rne_bits(acc[m][2 * k][i]) | (bf16_rne_bits(acc[m][2 * k + 1][i]) << 16));
        *(v4i *)(sd.grad + ((int64_t)tile.group * r + rank) * D + col) = out;
      } else {
        float *out = sd.partials + (outer_part(tile.first, p.size, tile.piece) * r + rank) * D + col;
        *(v4f *)out = v4f{acc[m][0][i], acc[m][1][i], acc[m][2][i], acc[m][3][i]};
        *(v4f *)(out + 4) = v4f{acc[m][4][i], acc[m][5][i], acc[m][6][i], acc[m][7][i]};
      }
    }
}

// h = the sum of its parts, in their order: the workgroups of `fold`'s grid from row `row0` on.
L8_DEV void sum_parts(const float *__restrict__ parts, int count, int64_t n, float *__restrict__ h, int row0) {
  const int64_t mine = (int64_t)((int)blockIdx.y - row0) * gridDim.x + blockIdx.x, all = (int64_t)((int)gridDim.y - row0) * gridDim.x;
  for (int64_t at = (mine * 256 + threadIdx.x) * 4; at < n; at += all * 1024) {
    v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int i = 0; i < count; ++i) {
      const v4f u = *(const v4f *)(parts + i * n + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += u[e];
    }
    *(v4f *)(h + at) = v;
  }
}

// The sums of a group's tiles, in their order, rounded: groups of more than one tile, a row of the grid each.  (And with `h`, in the rows behind
// them: the sum of its parts.)
__global__ __launch_bounds__(256) void lowrank_fold_kernel(const OuterArgs p, int groups, int64_t blocks0, int64_t blocks, float *__restrict__ h) {
  if ((int)blockIdx.y >= groups) return sum_parts(p.also, p.side[1].chunks, (int64_t)p.T * p.r, h, groups);
  const int from = within(p.starts[blockIdx.y], p.T), tokens = within(p.starts[blockIdx.y + 1], p.T) - from;
  if (tokens <= p.size) return;
  const int pieces = (tokens + p.size - 1) / p.size;
  const int64_t part0 = outer_part(from, p.size, 0);   // and piece i > 0 at part0 + 2 i + 1
#pragma unroll 1
  for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
    const int which = block >= blocks0;
    const OuterSide &sd = p.side[which];
    const int64_t at = (block - (which ? blocks0 : 0)) * 2048 + threadIdx.x * 8, all = (int64_t)p.r * sd.D;
    if (at >= all) continue;
    v4f lo = {0.0f, 0.0f, 0.0f, 0.0f}, hi = lo;
#pragma unroll 8
    for (int i = 0; i < pieces; ++i) {
      const float *part = sd.partials + (part0 + 2 * i + (i > 0)) * all + at;
      const v4f a = *(const v4f *)part, b = *(const v4f *)(part + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) lo[e] += a[e], hi[e] += b[e];
    }
    v4i out;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float u = k < 2 ? lo[2 * k] : hi[2 * k - 4], w = k < 2 ? lo[2 * k + 1] : hi[2 * k - 3];
      out[k] = (int)(bf16_rne_bits(u) | (bf16_rne_bits(w) << 16));
    }
    *(v4i *)(sd.grad + (int64_t)blockIdx.y * all + at) = out;
  }
}

// ---- host ----

constexpr int64_t kMaxRank = 128, kMaxTokens = 1 << 24, kMaxAdapters = 65534, kMaxCols = 1 << 24;

// Tokens of a tile: 64, which read a factor a quarter as often, where the adapters have that many on average.
static int tile_tokens(int64_t T, int64_t n) { return T >= 64 * (n + 1) ? 64 : 16; }
// The same of `shrink`: with more than 32 ranks, where four tiles of 16 tokens fill a SIMD's registers with one wave, tiles of 32 tokens on twice
// the waves up to one a unit; us, rank 64, 32 tokens and 64: [2055,4096] in three parts 13.5 and 16.0, [8192,4096] 23.3 and 28.8, [12000,4096]
// 40.6 and 31.7.
static int shrink_tokens(int64_t T, int64_t n, int64_t r) {
  const int size = tile_tokens(T, n);
  return size == 64 && r > 32 && T <= 32 * (int64_t)num_cus() ? 32 : size;
}
static int64_t tile_slots(int64_t T, int64_t n, int64_t size) { return T / size + n + 2; }

// Tokens of a tile of the factors' gradients: so many tiles that two workgroups a unit have work.
static int outer_size(int64_t T, int64_t K, int64_t N) {
  const int64_t chunks = (K + 511) / 512 + (N + 511) / 512, wanted = (2 * (int64_t)num_cus() + chunks - 1) / chunks;
  int size = 128;
  while (size < 2048 && size * wanted < T) size *= 2;
  return size;
}

static bool rows_fit(const void *p, int64_t ld, int64_t cols) { return p && ((uintptr_t)p % 16) == 0 && ld % 8 == 0 && ld >= cols; }
static int check_sizes(const char *who, int64_t T, int64_t n, int64_t r, int64_t D) {
  L8_REQUIRE(T >= 0 && T < kMaxTokens, "%s: %lld tokens, fewer than 2^24 are wanted", who, (long long)T);
  L8_REQUIRE(n >= 1 && n <= kMaxAdapters, "%s: %lld adapters, 1 to 65534 are wanted", who, (long long)n);
  L8_REQUIRE(r >= 8 && r <= kMaxRank && r % 8 == 0, "%s: rank %lld is not a multiple of 8 up to %lld", who, (long long)r, (long long)kMaxRank);
  L8_REQUIRE(D >= 8 && D % 8 == 0 && D < kMaxCols, "%s: %lld columns, a multiple of 8 below 2^24 is wanted", who, (long long)D);
  return L8_OK;
}
static int check_grid(const char *who, int64_t x, int64_t y, int64_t z, int64_t threads) {
  L8_REQUIRE(y <= 65535 && x * y * z * threads < (1ll << 32), "%s: 2^32 threads or more", who);
  return L8_OK;
}
static int check_plan(const char *who, int64_t T, const void *order, const void *starts) {
  L8_REQUIRE((order || T == 0) && starts && ((uintptr_t)order % 4) == 0 && ((uintptr_t)starts % 4) == 0, "%s: null or misaligned order of tokens", who);
  return L8_OK;
}
// The fold of a launch of `outer`: with `groups` those of several tiles, with h and `sums` workgroups of elements the sum of its parts.  Each does
// as many blocks as it takes to stay within a launch's 2^32 threads: whatever `outer` takes has a fold.
static int fold(const OuterArgs &p, int groups, float *h, int64_t sums, hipStream_t st) {
  const int64_t blocks0 = ((int64_t)p.r * p.side[0].D + 2047) / 2048, blocks = blocks0 + ((int64_t)p.r * p.side[1].D + 2047) / 2048;
  const int64_t rows = !h ? 0 : groups ? std::min<int64_t>((sums + blocks - 1) / blocks, 65535 - groups) : 1, y = groups + rows;
  const int64_t x = std::min<int64_t>(groups ? blocks : sums, ((1 << 24) - 1) / y);
  hipLaunchKernelGGL(lowrank_fold_kernel, dim3((unsigned)x, (unsigned)y), dim3(256), 0, st, p, groups, blocks0, blocks, h);
  L8_HIP(hipGetLastError());
  return L8_OK;
}
#define L8_CALL(expr)              \
  do {                             \
    const int code_ = (expr);      \
    if (code_ != L8_OK) return code_; \
  } while (0)

}  // namespace l8

using namespace l8;

extern "C" int l8_lowrank_route(const void *index, int index_is_i64, int64_t T, int64_t n, int *order, int *starts, void *stream) {
  const char *who = "l8_lowrank_route";
  L8_CALL(check_sizes(who, T, n, 8, 8));
  L8_CALL(check_plan(who, T, order, starts));
  L8_REQUIRE(T == 0 || (index && ((uintptr_t)index % (index_is_i64 ? 8 : 4)) == 0), "%s: null or misaligned index", who);
  L8_REQUIRE((n + 2) * T < (1ll << 36), "%s: %lld tokens and %lld adapters: each group's workgroup reads the whole index, 2^36 times or more in all", who, (long long)T, (long long)n);
  const dim3 grid((unsigned)(n + 2)), block(kRouteBlock);
  hipStream_t st = (hipStream_t)stream;
  if (index_is_i64) hipLaunchKernelGGL(lowrank_route_kernel<int64_t>, grid, block, 0, st, (const int64_t *)index, (int)T, (int)n, order, starts);
  else hipLaunchKernelGGL(lowrank_route_kernel<int32_t>, grid, block, 0, st, (const int32_t *)index, (int)T, (int)n, order, starts);
  L8_HIP(hipGetLastError());
  return L8_OK;
}

// Workgroups that share K: as many as give every unit one, with at least two steps left for each wave.
extern "C" int64_t l8_lowrank_splits(int64_t T, int64_t n, int64_t r, int64_t K) {
  if (T <= 0 || n <= 0 || K <= 0) return 1;
  const int64_t size = shrink_tokens(T, n, r), tiles = std::min(T, tile_slots(T, n, size)), waves = size == 64 && r > 32 ? 4 : 8;
  return std::max<int64_t>(1, std::min<int64_t>({num_cus() / tiles, (K + 63) / 64 / (2 * waves), 16}));
}

namespace l8 {

// Tiles that a launch has numbers for.  (Of few tokens each may be a tile of its own, and there are no unused numbers.)
static int64_t tiles_of(const Tokens &tk, int64_t T, int64_t n, int64_t size) {
  const int64_t slots = tile_slots(T, n, size);
  return tk.order ? slots : std::min(T, slots);
}

static int shrink_impl(const char *who, const void *x, int64_t T, int64_t K, int64_t ldx, const void *f, int64_t n, int64_t r, const Tokens &tk, float *h, int64_t splits,
                       hipStream_t st) {
  L8_REQUIRE(splits >= 1 && splits <= 64, "%s: 1 to 64 parts, got %lld", who, (long long)splits);
  L8_REQUIRE(rows_fit(x, ldx, K) && rows_fit(f, K, K) && h && ((uintptr_t)h % 16) == 0, "%s: null or misaligned operand, or rows off 16-byte lines", who);
  const int64_t size = shrink_tokens(T, n, r), slots = tiles_of(tk, T, n, size);
  const ShrinkArgs p{(const uint16_t *)x, (const uint16_t *)f, tk, h, ldx, (int)T, (int)K, (int)n, (int)r, (int)splits};
  const unsigned ranks = r <= 64 ? 1 : 2;
#define L8_SHRINK(MT, RT, W)                                                                                             \
  do {                                                                                                                   \
    L8_CALL(check_grid(who, slots, splits, ranks, W * 64));                                                              \
    hipLaunchKernelGGL((lowrank_shrink_kernel<MT, RT, W>), dim3((unsigned)slots, (unsigned)splits, ranks), dim3(W * 64), 0, st, p); \
  } while (0)
  if (size == 16) {
    if (r <= 16) L8_SHRINK(1, 1, 8);
    else if (r <= 32) L8_SHRINK(1, 2, 8);
    else L8_SHRINK(1, 4, 8);
  } else {
    if (r <= 16) L8_SHRINK(4, 1, 8);
    else if (r <= 32) L8_SHRINK(4, 2, 8);
    else if (size == 32) L8_SHRINK(2, 4, 8);
    else L8_SHRINK(4, 4, 4);
  }
#undef L8_SHRINK
  L8_HIP(hipGetLastError());
  return L8_OK;
}

static int expand_impl(const char *who, const void *y, int64_t ldy, const float *h, int64_t splits, const float *scale, const void *f, int64_t T, int64_t N, int64_t n, int64_t r,
                       const Tokens &tk, void *out, int64_t ldo, hipStream_t st) {
  L8_REQUIRE(splits >= 1 && splits <= 64, "%s: 1 to 64 parts, got %lld", who, (long long)splits);
  L8_REQUIRE((!y || rows_fit(y, ldy, N)) && rows_fit(f, N, N) && rows_fit(out, ldo, N) && h && ((uintptr_t)h % 16) == 0 && ((uintptr_t)scale % 4) == 0,
             "%s: null or misaligned operand, or rows off 16-byte lines", who);
  const int64_t size = tile_tokens(T, n), slots = tiles_of(tk, T, n, size);
  // waves that share the factor take as many steps as leave two workgroups a unit ([2055,11008] rank 64, h in three parts, us: 30.7, four a
  // unit 35.5), of an h that is whole up to four, since long ones end unevenly: rank 64, up to four and up to eight, [4096,11008] 46.7 and 55.8,
  // [6000,4096] 27.4 and 35.5, [8192,4096] 35.4 and 41.4, [16384,4096] 69.0 and 70.4
  const int64_t most = splits == 1 ? 4 : 8;
  const int64_t per = size == 16 || r <= 16 ? 1 : std::max<int64_t>(1, std::min<int64_t>(most, slots * ((N + 127) / 128) / (2 * num_cus())));
  const int64_t cols = size == 16 ? kExpandWaves * 128 : per * 128, chunks = (N + cols - 1) / cols;
  L8_CALL(check_grid(who, slots * chunks, 1, 1, kExpandWaves * 64));
  const ExpandArgs p{(const uint16_t *)y, (const uint16_t *)f, h, scale, tk, (uint16_t *)out, ldy, ldo, (int)T, (int)N, (int)n, (int)r, (int)splits, (int)chunks, (int)per};
  const dim3 grid((unsigned)(slots * chunks)), block(kExpandWaves * 64);
#define L8_EXPAND(PARTS)                                                                                          \
  do {                                                                                                       \
    if (r <= 16) hipLaunchKernelGGL((lowrank_expand_kernel<PARTS, 0>), grid, block, 0, st, p);                  \
    else if (r <= 32) hipLaunchKernelGGL((lowrank_expand_kernel<PARTS, 1>), grid, block, 0, st, p);             \
    else if (r <= 64) hipLaunchKernelGGL((lowrank_expand_kernel<PARTS, 2>), grid, block, 0, st, p);             \
    else hipLaunchKernelGGL((lowrank_expand_kernel<PARTS, 4>), grid, block, 0, st, p);                          \
  } while (0)
  if (size == 16) L8_EXPAND(1);
  else L8_EXPAND(4);
#undef L8_EXPAND
  L8_HIP(hipGetLastError());
  return L8_OK;
}

}  // namespace l8

extern "C" int l8_lowrank_shrink(const void *x, int64_t T, int64_t K, int64_t ldx, const void *f, int64_t n, int64_t r, const int *order, const int *starts,
                                 float *h, int64_t splits, void *stream) {
  const char *who = "l8_lowrank_shrink";
  L8_CALL(check_sizes(who, T, n, r, K));
  if (T == 0) return L8_OK;
  L8_CALL(check_plan(who, T, order, starts));
  return shrink_impl(who, x, T, K, ldx, f, n, r, Tokens{order, starts, nullptr, 0}, h, splits, (hipStream_t)stream);
}

extern "C" int l8_lowrank_expand(const void *y, int64_t ldy, const float *h, int64_t splits, const float *scale, const void *f, int64_t T, int64_t N, int64_t n,
                                 int64_t r, const int *order, const int *starts, void *out, int64_t ldo, void *stream) {
  const char *who = "l8_lowrank_expand";
  L8_CALL(check_sizes(who, T, n, r, N));
  if (T == 0) return L8_OK;
  L8_CALL(check_plan(who, T, order, starts));
  return expand_impl(who, y, ldy, h, splits, scale, f, T, N, n, r, Tokens{order, starts, nullptr, 0}, out, ldo, (hipStream_t)stream);
}

extern "C" int64_t l8_lowrank_add_workspace(int64_t T, int64_t K, int64_t n, int64_t r) {
  if (T <= 0 || K <= 0 || n <= 0 || r <= 0) return 0;
  const int64_t plan = T <= kFewTokens ? 0 : (T + n + 3 + 3) / 4 * 16;
  return plan + l8_lowrank_splits(T, n, r, K) * T * r * (int64_t)sizeof(float);
}

extern "C" int l8_lowrank_add(const void *y, int64_t ldy, const void *x, int64_t ldx, const void *a, const void *b, const float *scale, const void *index, int index_is_i64,
                              int64_t T, int64_t K, int64_t N, int64_t n, int64_t r, void *out, int64_t ldo, void *workspace, int64_t workspace_bytes, void *stream) {
  const char *who = "l8_lowrank_add";
  L8_CALL(check_sizes(who, T, n, r, K));
  L8_CALL(check_sizes(who, T, n, r, N));
  if (T == 0) return L8_OK;
  const int64_t need = l8_lowrank_add_workspace(T, K, n, r), splits = l8_lowrank_splits(T, n, r, K);
  L8_REQUIRE(workspace && workspace_bytes >= need && ((uintptr_t)workspace % 16) == 0, "%s: needs a 16-byte aligned workspace of %lld bytes", who, (long long)need);
  L8_REQUIRE(index && ((uintptr_t)index % (index_is_i64 ? 8 : 4)) == 0, "%s: null or misaligned index", who);
  L8_REQUIRE(rows_fit(b, N, N) && rows_fit(out, ldo, N) && rows_fit(y, ldy, N), "%s: null or misaligned operand, or rows off 16-byte lines", who);
  float *h = (float *)workspace;
  Tokens tk{nullptr, nullptr, index, index_is_i64};
  if (T > kFewTokens) {
    int *starts = (int *)workspace, *order = starts + n + 3;
    h = (float *)workspace + (T + n + 3 + 3) / 4 * 4;
    L8_CALL(l8_lowrank_route(index, index_is_i64, T, n, order, starts, stream));
    tk = Tokens{order, starts, nullptr, 0};
  }
  L8_CALL(shrink_impl(who, x, T, K, ldx, a, n, r, tk, h, splits, (hipStream_t)stream));
  return expand_impl(who, y, ldy, h, splits, scale, b, T, N, n, r, tk, out, ldo, (hipStream_t)stream);
}

extern "C" int64_t l8_lowrank_outer_workspace(int64_t T, int64_t r, int64_t K, int64_t N) {
  if (T <= 0 || r <= 0 || K < 0 || N < 0) return 0;
  const int64_t size = outer_size(T, K, N);
  return T <= size ? 0 : 2 * (T / size + 1) * r * (K + N) * (int64_t)sizeof(float);
}

extern "C" int l8_lowrank_outer(const l8_lowrank_side *two, const float *scale, int64_t T, int64_t n, int64_t r, const int *order, const int *starts,
                                void *workspace, int64_t workspace_bytes, void *stream) {
  const char *who = "l8_lowrank_outer";
  L8_REQUIRE(two, "%s: null pointer", who);
  OuterArgs p{};
  int64_t D[2];
  for (int i = 0; i < 2; ++i) {   // a side without a gradient has no columns
    D[i] = two[i].grad ? two[i].D : 0;
    L8_CALL(check_sizes(who, T, n, r, two[i].grad ? D[i] : 8));
    if (!two[i].grad) continue;
    L8_REQUIRE(((uintptr_t)two[i].grad % 16) == 0 && two[i].splits >= 1 && two[i].splits <= 64, "%s: a misaligned gradient, or parts of h that are not 1 to 64", who);
    L8_REQUIRE(T == 0 || (rows_fit(two[i].z, two[i].ldz, D[i]) && two[i].h && ((uintptr_t)two[i].h % 16) == 0), "%s: null or misaligned operand, or rows off 16-byte lines", who);
  }
  if (D[0] + D[1] == 0) return L8_OK;
  L8_CALL(check_plan(who, T, order, starts));
  L8_REQUIRE(((uintptr_t)scale % 4) == 0, "%s: misaligned scale", who);
  const int size = outer_size(T, D[0], D[1]);
  const int64_t need = l8_lowrank_outer_workspace(T, r, D[0], D[1]);
  L8_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace % 16) == 0), "%s: needs a 16-byte aligned workspace of %lld bytes", who, (long long)need);
  const int64_t parts = T <= size ? 0 : 2 * (T / size + 1);
  for (int i = 0; i < 2; ++i) {
    p.side[i] = OuterSide{two[i].h, (const uint16_t *)two[i].z, (uint16_t *)two[i].grad, (float *)workspace + (i ? parts * r * D[0] : 0), two[i].ldz, (int)D[i], (int)two[i].splits,
                          (int)((D[i] + 511) / 512)};
  }
  p.scale = scale, p.order = order, p.starts = starts, p.T = (int)T, p.n = (int)n, p.r = (int)r, p.size = size;
  const int64_t slots = tile_slots(T, n, size), chunks = p.side[0].chunks + p.side[1].chunks, ranks = r <= 64 ? 1 : 2;
  L8_CALL(check_grid(who, slots, chunks, ranks, kOuterWaves * 64));
  const dim3 grid((unsigned)slots, (unsigned)chunks, (unsigned)ranks), block(kOuterWaves * 64);
  hipStream_t st = (hipStream_t)stream;
  if (r <= 16) hipLaunchKernelGGL((lowrank_outer_kernel<1, 256, false>), grid, block, 0, st, p);
  else if (r <= 32) hipLaunchKernelGGL((lowrank_outer_kernel<2, 256, false>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((lowrank_outer_kernel<4, 128, false>), grid, block, 0, st, p);
  L8_HIP(hipGetLastError());
  return parts ? fold(p, (int)n, nullptr, 0, st) : L8_OK;
}

// Does one reading of z for both pay?  It costs two launches more in a backward pass, which else has both factors' gradients in one, so it
// does where z is large, above all where the caches do not hold it for the second reading.  us of the whole backward pass, one reading and two:
// rank 16, [16384,4096] to [16384,11008] 184 and 227, [2055,4096] to [2055,11008] 42.5 and 47.2, [8192,2048] to [8192,8192] 77 and 88, but
// [16384,4096] to [16384,4096] 136 and 126, [6000,2048] to [6000,5632] 58 and 52, [2048,2048] to [2048,2048] 29 and 25; rank 32, [16384,4096] to
// [16384,8192] 191 and 201, [8192,4096] to [8192,11008] 133 and 156, [16384,4096] to [16384,4096] 173 and 160.
extern "C" int l8_lowrank_outer_shrink_pays(int64_t T, int64_t r, int64_t D) { return T >= 2048 && D >= 8192 && r <= 32; }

extern "C" int64_t l8_lowrank_outer_shrink_workspace(int64_t T, int64_t r, int64_t D) {
  if (T <= 0 || r <= 0 || D <= 0) return 0;
  return (D + 511) / 512 * T * r * (int64_t)sizeof(float) + l8_lowrank_outer_workspace(T, r, 0, D);
}

extern "C" int l8_lowrank_outer_shrink(const l8_lowrank_side *one, const float *scale, const void *f, float *also, int64_t T, int64_t n, int64_t r, const int *order, const int *starts,
                                       void *workspace, int64_t workspace_bytes, void *stream) {
  const char *who = "l8_lowrank_outer_shrink";
  L8_REQUIRE(one && one->grad && ((uintptr_t)one->grad % 16) == 0, "%s: null or misaligned gradient", who);
  const int64_t D = one->D;
  L8_CALL(check_sizes(who, T, n, r, D));
  L8_REQUIRE(r <= 32, "%s: rank %lld, up to 32 are wanted", who, (long long)r);
  L8_REQUIRE(T >= 1, "%s: no tokens", who);
  L8_CALL(check_plan(who, T, order, starts));
  L8_REQUIRE(one->splits >= 1 && one->splits <= 64, "%s: 1 to 64 parts, got %lld", who, (long long)one->splits);
  L8_REQUIRE(rows_fit(one->z, one->ldz, D) && rows_fit(f, D, D) && one->h && ((uintptr_t)one->h % 16) == 0 && also && ((uintptr_t)also % 16) == 0 && ((uintptr_t)scale % 4) == 0,
             "%s: null or misaligned operand, or rows off 16-byte lines", who);
  const int64_t need = l8_lowrank_outer_shrink_workspace(T, r, D);
  L8_REQUIRE(workspace && workspace_bytes >= need && ((uintptr_t)workspace % 16) == 0, "%s: needs a 16-byte aligned workspace of %lld bytes", who, (long long)need);
  OuterArgs p{};
  const int size = outer_size(T, 0, D);
  const int64_t chunks = (D + 511) / 512, parts = T <= size ? 0 : 2 * (T / size + 1), slots = tile_slots(T, n, size);
  p.side[1] = OuterSide{one->h, (const uint16_t *)one->z, (uint16_t *)one->grad, (float *)workspace + chunks * T * r, one->ldz, (int)D, (int)one->splits, (int)chunks};
  p.scale = scale, p.order = order, p.starts = starts, p.T = (int)T, p.n = (int)n, p.r = (int)r, p.size = size;
  p.f = (const uint16_t *)f, p.also = (float *)workspace;
  L8_CALL(check_grid(who, slots * chunks, 1, 1, kOuterWaves * 64));
  const dim3 grid((unsigned)(slots * chunks)), block(kOuterWaves * 64);
  hipStream_t st = (hipStream_t)stream;
  if (r <= 16) hipLaunchKernelGGL((lowrank_outer_kernel<1, 128, true>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((lowrank_outer_kernel<2, 128, true>), grid, block, 0, st, p);
  L8_HIP(hipGetLastError());
  // one launch for both sums
  return fold(p, parts ? (int)n : 0, also, std::min<int64_t>((T * r + 1023) / 1024, 4 * num_cus()), st);
}
