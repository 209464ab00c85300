// Rotary positions on the queries and keys of an attention (apply_rotary_emb of lingua/transformer.py, between the
// projections and the product of queries and keys).
//
// A pair (a, b) of a head's columns at position p turns by the angle that the tables hold:
//
//   a' = a * cos[p][i] - b * sin[p][i],   b' = a * sin[p][i] + b * cos[p][i]
//
// in fp32 (products and sums rounded one by one, as the eager chain rounds them: the results are its bits), rounded to bf16
// once.  Pair i is columns (2 i, 2 i + 1) of the interleaved layout or (i, i + rot / 2) of the layout in halves; columns from
// rot on are copied.  The backward pass is the transposed rotation: the same kernel with the sine negated.
//
// Bound by memory: 4 bytes of traffic per element and nothing else of size (the tables are read once per token, from the L2).
// 16384 tokens, q and k of 32 heads of 128: 105 us, 5.1 TB/s, the rate of a large copy.
// A workgroup takes a token: a thread keeps one place in the head -- its cosines and sines stay in registers -- and steps
// through the heads of q, then of k.  q and k come in any strides with a dense head (column slices of one product, heads in
// front of tokens), so nothing is copied on the way in.
//
// With AXES a token stands at a place of several axes (time, height, width of a patch), and each pair turns by the one that its entry
// of a map names: row positions[axis] of the same tables, column i.  A thread looks its pairs up once per token; the map is an argument of
// the launch, two bits a pair.  The same 16384 tokens on three axes: 108 us, 5.0 TB/s.
#include "l8_common.h"

#include <type_traits>

namespace l8 {

struct RotaryArgs {
  l8_rotary_operand op[2];
  const float *cos, *sin;
  int64_t table_row, table_col, length;   // strides of the tables, in elements; positions they hold
  const void *positions;                  // NULL: token s stands at position s
  int64_t pos_b, pos_s;
  int S, D, rot;
  int items, heads_at_once;               // places per head; heads that a workgroup's threads cover in one step
  bool pos_i32, inverse;
};

// Which axis each pair turns by, two bits a pair, and where an axis's positions lie (AXES; else empty).
constexpr int kRotAxes = 4, kRotBlock = 256;
struct RotaryAxes {
  int64_t pos_axis;
  int axes;
  uint32_t map[kRotBlock / 16];
};
struct NoAxes {};

template <int N> struct Bf16Vec;
template <> struct Bf16Vec<1> { typedef uint16_t t; };
template <> struct Bf16Vec<2> { typedef uint32_t t; };
template <> struct Bf16Vec<4> { typedef v2i t; };
template <> struct Bf16Vec<8> { typedef v4i t; };

template <int N>
struct Elems {   // N bf16 values in one register group
  typedef typename Bf16Vec<N>::t T;
  T v;
  L8_DEV float get(int i) const {
    uint32_t w;
    if constexpr (N == 1) w = v;
    else if constexpr (N == 2) w = v;
    else w = (uint32_t)v[i >> 1];
    return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
  }
};
template <int N>
L8_DEV typename Bf16Vec<N>::t packed(const float (&f)[N]) {
  if constexpr (N == 1) return (uint16_t)bf16_rne_bits(f[0]);
  else if constexpr (N == 2) return bf16_rne_bits(f[0]) | (bf16_rne_bits(f[1]) << 16);
  else {
    typename Bf16Vec<N>::t r;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) r[i] = (int)(bf16_rne_bits(f[2 * i]) | (bf16_rne_bits(f[2 * i + 1]) << 16));
    return r;
  }
}

// V pairs per thread and step.  HALF: two vectors of V columns, rot / 2 apart; else one vector of 2 V columns.
template <int V, bool HALF, bool AXES = false>
__global__ __launch_bounds__(kRotBlock) void rotary_kernel(const RotaryArgs p, const std::conditional_t<AXES, RotaryAxes, NoAxes> ax) {
  constexpr int N = HALF ? V : 2 * V;     // columns of a vector
  const int64_t token = blockIdx.x;
  const int64_t b = token / p.S, s = token - b * p.S;
  const int place = threadIdx.x % p.items, sub = threadIdx.x / p.items;
  if (sub >= p.heads_at_once) return;
  auto position = [&](int64_t at) { return p.pos_i32 ? (int64_t)((const int32_t *)p.positions)[at] : ((const int64_t *)p.positions)[at]; };
  int64_t pos = s;
  [[maybe_unused]] int64_t places[kRotAxes];
  bool known = true;   // elsewhere there is no angle: the token's results are NaN
  if constexpr (AXES) {
#pragma unroll
    for (int a = 0; a < kRotAxes; ++a) {
      places[a] = a < ax.axes ? position(a * ax.pos_axis + b * p.pos_b + s * p.pos_s) : 0;
      known = known && (a >= ax.axes || (places[a] >= 0 && places[a] < p.length));
    }
  } else {
    if (p.positions) pos = position(b * p.pos_b + s * p.pos_s);
    known = pos >= 0 && pos < p.length;
  }
  const int turned = p.rot / (2 * V);              // places that turn; the others copy 2 V columns each
  const bool turn = place < turned;
  float c[V], sn[V];
  if (AXES && turn && known) {
    if constexpr (AXES) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int pair = place * V + i;
        const uint32_t a = ax.map[pair >> 4] >> (2 * (pair & 15)) & 3;
        const int64_t lo = a & 1 ? places[1] : places[0], hi = a & 1 ? places[3] : places[2];
        const int64_t at = (a & 2 ? hi : lo) * p.table_row + pair * p.table_col;
        c[i] = p.cos[at];
        sn[i] = p.inverse ? -p.sin[at] : p.sin[at];
      }
    }
  } else if (turn && known) {
    const float *ct = p.cos + pos * p.table_row + (int64_t)place * V * p.table_col;
    const float *st = p.sin + pos * p.table_row + (int64_t)place * V * p.table_col;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      c[i] = ct[i * p.table_col];
      sn[i] = p.inverse ? -st[i * p.table_col] : st[i * p.table_col];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = 1.0f, sn[i] = 0.0f;
  }
  // the thread's two vectors (HALF: of a pair's two columns; a copying place: neighbours), or its only one
  const int first = HALF ? (turn ? place * V : p.rot + (place - turned) * 2 * V) : place * 2 * V;
  const int second = HALF ? (turn ? first + p.rot / 2 : first + V) : 0;
  typedef typename Bf16Vec<N>::t Vec;
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    const l8_rotary_operand &t = p.op[o];
    const uint16_t *in = (const uint16_t *)t.x + b * t.ldb + s * t.lds;
    uint16_t *out = (uint16_t *)t.y + token * t.heads * p.D;
    for (int64_t h = sub; h < t.heads; h += p.heads_at_once) {
      Elems<N> u, w;
      u.v = *(const Vec *)(in + h * t.ldh + first);
      if constexpr (HALF) w.v = *(const Vec *)(in + h * t.ldh + second);
      Vec ru = u.v, rw;
      if constexpr (HALF) rw = w.v;
      if (turn || !known) {
        float a1[N], b1[N];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float a = HALF ? u.get(i) : u.get(2 * i), e = HALF ? w.get(i) : u.get(2 * i + 1);
          float ra = a * c[i] - e * sn[i], re = a * sn[i] + e * c[i];
          if (!known) ra = re = __uint_as_float(0x7fc00000u);
          if constexpr (HALF) a1[i] = ra, b1[i] = re;
          else a1[2 * i] = ra, a1[2 * i + 1] = re;
        }
        ru = packed<N>(a1);
        if constexpr (HALF) rw = packed<N>(b1);
      }
      *(Vec *)(out + h * p.D + first) = ru;
      if constexpr (HALF) *(Vec *)(out + h * p.D + second) = rw;
    }
  }
}

}  // namespace l8

using namespace l8;

namespace l8 {

// Both entries; ax NULL: one position a token.
static int rotary_impl(const char *who, const l8_rotary_operand *given, int64_t B, int64_t S, int64_t D, int64_t rot, int in_halves, int inverse,
                       const float *cos, const float *sin, int64_t table_row, int64_t table_col, int64_t length,
                       const void *positions, int positions_i32, int64_t pos_b, int64_t pos_s, const RotaryAxes *ax, void *stream) {
  L8_REQUIRE(given && B >= 0 && S >= 0 && D >= 0 && given[0].heads >= 0 && given[1].heads >= 0, "%s: null pointer or negative shape", who);
  l8_rotary_operand two[2] = {given[0], given[1]};
  for (auto &t : two) {   // the stride of a single one is never used
    if (B <= 1) t.ldb = 0;
    if (S <= 1) t.lds = 0;
    if (t.heads <= 1) t.ldh = 0;
  }
  if (B == 0 || S == 0 || D == 0 || (two[0].heads == 0 && two[1].heads == 0)) return L8_OK;
  L8_REQUIRE(D <= 2 * kRotBlock && D % 2 == 0, "%s: heads of an even number of columns up to %d, got %lld", who, 2 * kRotBlock, (long long)D);
  L8_REQUIRE(rot >= 2 && rot % 2 == 0 && rot <= D, "%s: an even number of columns up to the head's %lld turns, got %lld", who, (long long)D, (long long)rot);
  L8_REQUIRE(cos && sin && ((uintptr_t)cos % 4) == 0 && ((uintptr_t)sin % 4) == 0, "%s: null or misaligned table", who);
  L8_REQUIRE(length >= 0 && (positions || S <= length), "%s: %lld tokens, the tables hold %lld positions", who, (long long)S, (long long)length);
  L8_REQUIRE(B < (1 << 24) && S < (1 << 24) && B * S < (1 << 24) && two[0].heads < (1 << 24) && two[1].heads < (1 << 24),
             "%s: 2^24 tokens or heads or more", who);
  RotaryArgs a;
  // the widest vectors that the head's parts, the strides and the pointers allow
  int v = in_halves ? 8 : 4;
  auto fits = [&](int n) {
    if (in_halves ? ((rot / 2) % n || (D - rot) % (2 * n)) : (rot % (2 * n) || (D - rot) % (2 * n))) return false;
    const int64_t cols = in_halves ? n : 2 * n;
    for (int o = 0; o < 2; ++o)
      if (two[o].heads && (((uintptr_t)two[o].x | (uintptr_t)two[o].y) % (cols * 2) || two[o].ldb % cols || two[o].lds % cols || two[o].ldh % cols || D % cols))
        return false;
    return true;
  };
  while (v > 1 && !fits(v)) v = v == 8 ? 4 : 1;
  for (int o = 0; o < 2; ++o) {
    a.op[o] = two[o];
    L8_REQUIRE(two[o].heads == 0 || (two[o].x && two[o].y), "%s: null pointer", who);
    L8_REQUIRE(two[o].heads == 0 || fits(v), "%s: operands must be aligned to %d bytes", who, in_halves ? 2 * v : 4 * v);
  }
  a.cos = cos, a.sin = sin, a.table_row = table_row, a.table_col = table_col, a.length = length;
  a.positions = positions, a.pos_i32 = positions_i32 != 0, a.pos_b = pos_b, a.pos_s = pos_s;
  a.S = (int)S, a.D = (int)D, a.rot = (int)rot, a.inverse = inverse != 0;
  a.items = (int)(D / (2 * v));   // at most a workgroup's threads
  const int64_t most_heads = two[0].heads > two[1].heads ? two[0].heads : two[1].heads;
  int64_t block = (int64_t)a.items * most_heads;
  block = block < kRotBlock ? (block + 63) / 64 * 64 : kRotBlock;
  a.heads_at_once = (int)(block / a.items);
  const dim3 grid((unsigned)(B * S)), threads((unsigned)block);
  hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto one, auto several) {
    if (ax) hipLaunchKernelGGL(several, grid, threads, 0, st, a, *ax);
    else hipLaunchKernelGGL(one, grid, threads, 0, st, a, NoAxes{});
  };
  if (in_halves) {
    if (v == 8) launch(rotary_kernel<8, true>, rotary_kernel<8, true, true>);
    else if (v == 4) launch(rotary_kernel<4, true>, rotary_kernel<4, true, true>);
    else launch(rotary_kernel<1, true>, rotary_kernel<1, true, true>);
  } else {
    if (v == 4) launch(rotary_kernel<4, false>, rotary_kernel<4, false, true>);
    else launch(rotary_kernel<1, false>, rotary_kernel<1, false, true>);
  }
  L8_HIP(hipGetLastError());
  return L8_OK;
}

}  // namespace l8

extern "C" int l8_rotary(const l8_rotary_operand *given, int64_t B, int64_t S, int64_t D, int64_t rot, int in_halves, int inverse,
                         const float *cos, const float *sin, int64_t table_row, int64_t table_col, int64_t length,
                         const void *positions, int positions_i32, int64_t pos_b, int64_t pos_s, void *stream) {
  return rotary_impl("l8_rotary", given, B, S, D, rot, in_halves, inverse, cos, sin, table_row, table_col, length, positions, positions_i32,
                     pos_b, pos_s, nullptr, stream);
}

extern "C" int l8_rotary_axes(const l8_rotary_operand *given, int64_t B, int64_t S, int64_t D, const int64_t *sections, int64_t axes, int in_rounds,
                              int in_halves, int inverse, const float *cos, const float *sin, int64_t table_row, int64_t table_col, int64_t length,
                              const void *positions, int positions_i32, int64_t pos_axis, int64_t pos_b, int64_t pos_s, void *stream) {
  const char *who = "l8_rotary_axes";
  L8_REQUIRE(axes >= 1 && axes <= kRotAxes && sections, "%s: 1 to %d axes, got %lld", who, kRotAxes, (long long)axes);
  int64_t left[kRotAxes], pairs = 0;
  for (int a = 0; a < axes; ++a) {
    L8_REQUIRE(sections[a] >= 0 && sections[a] <= kRotBlock, "%s: an axis of %lld pairs", who, (long long)sections[a]);
    pairs += left[a] = sections[a];
  }
  L8_REQUIRE(pairs >= 1 && pairs <= kRotBlock, "%s: %lld pairs turn, 1 to %d are wanted", who, (long long)pairs, kRotBlock);
  L8_REQUIRE(positions || B <= 0 || S <= 0, "%s: null positions", who);
  L8_REQUIRE(((uintptr_t)positions % (positions_i32 ? 4 : 8)) == 0, "%s: misaligned positions", who);
  RotaryAxes ax{};
  ax.axes = (int)axes, ax.pos_axis = axes > 1 ? pos_axis : 0;
  // side by side, or dealt out one to an axis in turn: an axis that has its share is passed over
  for (int64_t pair = 0, a = 0; pair < pairs; a = in_rounds ? (a + 1) % axes : a) {
    while (left[a] == 0) a = (a + 1) % axes;
    --left[a];
    ax.map[pair >> 4] |= (uint32_t)a << (2 * (pair & 15));
    ++pair;
  }
  return rotary_impl(who, given, B, S, D, 2 * pairs, in_halves, inverse, cos, sin, table_row, table_col, length, positions, positions_i32, pos_b, pos_s, &ax, stream);
}
