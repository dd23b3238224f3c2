// Attention of a ragged step's tokens over a paged cache in 4 bits (cache_4bit.h), bfloat16 queries.
//
//   p_j = exp(scale q . k_j) over the keys j that the token sees,  out = sum p_j v_j / sum p_j
//
// Rows are the query heads of one key head, for one or several tokens. A block takes a tile of rows and a part of their keys, which a plan of the
// step lists (row_plan.cpp); waves work on steps of 32 keys. Codes come in one 16-byte load a tile of 16 tokens, become bfloat16 by the
// conversion that takes two codes and their scale, exactly, and feed
//   S^T = K Q^T (A = tokens of keys, B = rows of queries: a row is a lane's column, a lane has the scores of some of the step's tokens),
//   O^T = V^T P^T (A = channels of values, B = the weights where they were born: the tokens of a lane are the same in both products).
// One pass over the keys with a running reference and sum a row; a row's weights may pass its reference by 2^8 before sums are scaled anew.
// For the product a weight is two bfloat16 pieces, 16 of its 24 bits, in every form, so that a token's result does not depend on which one it is given
// (one piece leaves 2^-8 of each term, which shows where terms cancel: portions took 205 us for 268); their sum is that of the float32 ones.
// What no row sees is taken out of the values too: its scale's byte is set to 0, the smallest and finite, so that a weight of 0 hides whatever lies
// behind a sequence's end.
//
// Three forms, by the rows that a sequence's new tokens make:
//   up to 16, or 17 to 95: a wave works alone, from memory to registers, and a block's waves take its steps in turn; their states meet in
//     LDS. Bound by memory: 16 sequences of up to 32768 tokens, 32/8 heads of 128, 66 to 75 us of parts (4.7 to 5.3 TB/s) and 5 to join
//     them; 61 sequences, a window of 4096, 28/4 heads, 28 us (4.5 TB/s). Three waves a SIMD at 128 channels: with accumulators in registers
//     apart, two, the first took 105 us for 96. A fixed number of parts for every sequence took 96 for 82.
//   96 and more (at 256 channels 48): a block's waves have rows of their own and share the conversions, see there. Bound by the products.
#include "cache_4bit.h"

#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <cmath>

namespace cai {
namespace serving {
namespace {

constexpr int STEP = 2 * TILE, WAVES4 = 4;
constexpr float LOG2E4 = 1.4426950408889634f, SLACK = 8.0f;   // a weight may be up to 2^SLACK

struct Attend {
  const bf16s* q;
  long q_stride, pages, page_stride;
  const unsigned char *kpool, *vpool;
  const int *tables, *items, *joins, *positions;
  bf16s* out;
  float* parts;
  int width, H, G, head_bytes, page_shift, window, group, subs;
  float scale;      // of the scores in base 2: positive
  bool negative;    // so that the queries take the sign
};

// A step's codes and scales as they come.
template <int D>
struct Raw {
  static constexpr int W = D / 32;   // 32-bit words of a lane's channels of a tile, keys or values
  unsigned int k[2][W], v[2][W], ks[2], vs[2];
  bool bad[2];
};

template <int W>
DEV_INLINE void load_words(unsigned int (&w)[W], const unsigned char* p) {
  if constexpr (W == 2) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    w[0] = t.x; w[1] = t.y;
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const uint4 t = *reinterpret_cast<const uint4*>(p + 4 * i);
      w[i] = t.x; w[i + 1] = t.y; w[i + 2] = t.z; w[i + 3] = t.w;
    }
  }
}

typedef unsigned int uint4v __attribute__((ext_vector_type(4)));
DEV_INLINE bf16x8_v frag(unsigned int a, unsigned int b, unsigned int c, unsigned int d) {
  return __builtin_bit_cast(bf16x8_v, uint4v{a, b, c, d});
}
DEV_INLINE unsigned int two_bf16(float a, float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned int, __builtin_convertvector((f2{a, b}), bf16x2));
}
// Eight weights as a bfloat16 each, and what that leaves of them as another: 16 of their 24 bits.
DEV_INLINE void two_pieces(float (&e)[8], bf16x8_v& p, bf16x8_v& rest) {
  const uint4v w = {two_bf16(e[0], e[1]), two_bf16(e[2], e[3]), two_bf16(e[4], e[5]), two_bf16(e[6], e[7])};
  p = __builtin_bit_cast(bf16x8_v, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] -= __builtin_bit_cast(float, i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  rest = frag(two_bf16(e[0], e[1]), two_bf16(e[2], e[3]), two_bf16(e[4], e[5]), two_bf16(e[6], e[7]));
}
template <int B>
DEV_INLINE unsigned int number_pair(const unsigned int* words, float scale) { return two_numbers<B & 3>(words[B >> 2], scale); }

// numbers of byte B of four tokens' values as fragments' words: tokens (0, 1) and (2, 3) of the byte's lower and upper channel
template <int D, int B>
DEV_INLINE void value_words(const unsigned int* w, const float* scale, unsigned int (&lo)[2], unsigned int (&hi)[2]) {
  constexpr int S = D / 32;   // bytes of a token
  const unsigned int t0 = number_pair<B>(w, scale[0]), t1 = number_pair<S + B>(w, scale[1]), t2 = number_pair<2 * S + B>(w, scale[2]),
                     t3 = number_pair<3 * S + B>(w, scale[3]);
  lo[0] = __builtin_amdgcn_perm(t1, t0, 0x05040100u);
  hi[0] = __builtin_amdgcn_perm(t1, t0, 0x07060302u);
  lo[1] = __builtin_amdgcn_perm(t3, t2, 0x05040100u);
  hi[1] = __builtin_amdgcn_perm(t3, t2, 0x07060302u);
}

template <int N, typename F>
DEV_INLINE void unrolled(F f) {
  [&]<int... I>(std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>()), ...); }(std::make_integer_sequence<int, N>());
}

// A wave's rows: 16 RT of its tile, from `row0` on. A lane has a row of each 16 as its column.
template <int D, int RT>
struct Rows {
  static constexpr int KF = D / 32, VF = D / 16;   // products of a tile's scores, tiles of channels
  bf16x8_v q[RT][KF];
  int pos[RT], tok[RT], head[RT];
  f32x4 o[RT][VF];
  float2v state[RT];   // the reference, and the sum of the weights

  // R: rows of the tile; p_last: the position of its last token
  DEV_INLINE void start(const Attend& a, int R, int row0, int g, int sub, int t0, int t1, int p_last, int n, int kg) {
    const int per_token = min(a.group, R);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = row0 + rt * 16 + n, in = sub * R + r % per_token;
      tok[rt] = t0 + r / per_token;
      const bool real = tok[rt] < t1 && in < a.group;
      head[rt] = real ? g * a.group + in : -1;
      pos[rt] = real ? a.positions[tok[rt]] : p_last;
      const bf16s* from = a.q + (real ? tok[rt] : t0) * a.q_stride + (long)(real ? head[rt] : g * a.group) * D + kg * (D / 4);
#pragma unroll
      for (int f = 0; f < KF; ++f) {
        q[rt][f] = *reinterpret_cast<const bf16x8_v*>(from + f * 8);
        if (a.negative) q[rt][f] = __builtin_bit_cast(bf16x8_v, __builtin_bit_cast(uint4v, q[rt][f]) ^ 0x80008000u);
      }
      state[rt] = float2v{-INFINITY, 0.0f};
#pragma unroll
      for (int f = 0; f < VF; ++f) o[rt][f] = f32x4{0, 0, 0, 0};
    }
  }

  DEV_INLINE bool sees(const Attend& a, int rt, int key) const { return key <= pos[rt] && (a.window <= 0 || pos[rt] - key < a.window); }

  // A new reference where scores times `scale` (positive; base 2) of S steps would pass the old one by too much.
  template <int S>
  DEV_INLINE void refer(const f32x4 (&s)[RT][2 * S], float scale) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float top = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2 * S; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[rt][h][i]);
      if (__any(top * scale > state[rt][0] + SLACK)) {   // -INFINITY + SLACK is -INFINITY: the first keys that a row sees come here
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32)) * scale;
        // a row's reference is its own affair: what the others need does not show in it
        const float m = state[rt][0], next = top > m + SLACK ? top : m, fall = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - next);
        state[rt] = float2v{next, state[rt][1] * fall};
#pragma unroll
        for (int f = 0; f < VF; ++f) o[rt][f] *= fall;
      }
    }
  }

  // Weights of row rt's scores of a step as the product's operand, and what bfloat16 leaves of them.
  DEV_INLINE void weigh(int rt, const f32x4& s0, const f32x4& s1, float scale, bf16x8_v& p, bf16x8_v& rest) {
    const float ref = state[rt][0] == -INFINITY ? 0.0f : state[rt][0];
    float e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      e[i] = __builtin_amdgcn_exp2f(fmaf(i < 4 ? s0[i & 3] : s1[i & 3], scale, -ref));
      state[rt][1] += e[i];
    }
    two_pieces(e, p, rest);
  }

  // sums of the lanes that share a row
  DEV_INLINE void sum_lanes() {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      state[rt][1] += __shfl_xor(state[rt][1], 16);
      state[rt][1] += __shfl_xor(state[rt][1], 32);
    }
  }

  DEV_INLINE void store(const Attend& a, int kg) const {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (head[rt] < 0) continue;
      const float inv = 1.0f / state[rt][1];
      bf16s* to_row = a.out + ((long)tok[rt] * a.H + head[rt]) * D;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        unsigned int w[VF / 2];
#pragma unroll
        for (int f = 0; f < VF; f += 2) w[f / 2] = two_bf16(o[rt][f][i] * inv, o[rt][f + 1][i] * inv);
        unsigned int* to_ch = reinterpret_cast<unsigned int*>(to_row + (kg * 4 + i) * VF);
#pragma unroll
        for (int f = 0; f < VF / 2; f += 2) *reinterpret_cast<uint2*>(to_ch + f) = make_uint2(w[f], w[f + 1]);
      }
    }
  }

  // into a part of R rows: rows' sums, then their references and weights
  DEV_INLINE void store_part(float* part, int R, int row0, int n, int kg) const {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (head[rt] < 0) continue;
      const int r = row0 + rt * 16 + n;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int f = 0; f < VF; f += 4)
          *reinterpret_cast<float4v*>(part + (long)r * D + (kg * 4 + i) * VF + f) = float4v{o[rt][f][i], o[rt][f + 1][i], o[rt][f + 2][i], o[rt][f + 3][i]};
      if (kg == 0) *reinterpret_cast<float2v*>(part + (long)R * D + r * 2) = state[rt];
    }
  }
};

// Where a step's codes come from: the pages of a sequence, for one key head.
template <int D>
struct Source {
  const int* table;
  int p_last, g;
  // a tile behind the end is its last one again: hidden by its places
  DEV_INLINE void look(const Attend& a, int (&pages)[2], int step) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) pages[h] = table[min(step * STEP + h * TILE, p_last) >> a.page_shift];
  }
  DEV_INLINE void load(const Attend& a, Raw<D>& w, int step, const int (&pages)[2], int n, int kg) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = min(step * STEP + h * TILE, p_last), page = pages[h];
      w.bad[h] = (unsigned)page >= (unsigned long)a.pages;
      const long base = (long)(w.bad[h] ? 0 : page) * a.page_stride + (long)g * a.head_bytes +
                        (long)((at & ((1 << a.page_shift) - 1)) / TILE) * Tile4<D>::BYTES;
      const unsigned char *kt = a.kpool + base, *vt = a.vpool + base;
      load_words(w.k[h], kt + n * (D / 2) + kg * (D / 8));
      if constexpr (D == 256) w.ks[h] = *reinterpret_cast<const unsigned short*>(kt + Tile4<D>::key_scale(n, 2 * kg));
      else w.ks[h] = kt[Tile4<D>::key_scale(n, D == 128 ? kg : kg >> 1)];
      load_words(w.v[h], vt + (kg * 16 + n) * (D / 8));
      w.vs[h] = *reinterpret_cast<const unsigned int*>(vt + Tile4<D>::value_scale(kg * 4, n * (D / 16) / 32));
    }
  }
};

// Fragment f of a tile's keys, and the two of byte B of a step's values.
template <int D>
DEV_INLINE bf16x8_v key_frag(const Raw<D>& w, int h, int f) {
  const float u = scale_of(D == 256 && f >= 4 ? w.ks[h] >> 8 : w.ks[h] & 255u);
  const unsigned int x = w.k[h][f];
  return frag(two_numbers<0>(x, u), two_numbers<1>(x, u), two_numbers<2>(x, u), two_numbers<3>(x, u));
}
template <int D, int B>
DEV_INLINE void value_frags(const Raw<D>& w, const float (&su)[2][4], bf16x8_v& lo, bf16x8_v& hi) {
  unsigned int lo0[2], hi0[2], lo1[2], hi1[2];
  value_words<D, B>(w.v[0], su[0], lo0, hi0);
  value_words<D, B>(w.v[1], su[1], lo1, hi1);
  lo = frag(lo0[0], lo0[1], lo1[0], lo1[1]);
  hi = frag(hi0[0], hi0[1], hi1[0], hi1[1]);
}

// Whether the lane's channels of token i (0 .. 3) of a tile's values, at that scale byte, have a number that is not finite: NaN at 255; infinite from
// 2^128 on, codes of 4 and 6 at 253 and of 2 and more at 254.
template <int D, int I>
DEV_INLINE bool not_finite(const unsigned int (&w)[D / 32], unsigned int byte) {
  constexpr int S = D / 32;   // bytes of a token
  unsigned int codes = 0;     // by their two upper bits: 4 and 6 have both, 2 and more the first
#pragma unroll
  for (int b = 0; b < S; b += 4) {
    const unsigned int x = w[(I * S + b) / 4] >> (I * S % 4 * 8) & (S < 4 ? (1u << (8 * S % 32)) - 1 : ~0u);
    codes |= byte == 253 ? x & x << 1 : x;
  }
  return byte == 255 || (byte >= 253 && (codes & 0x44444444u) != 0);
}

// What a step's values are to be taken at: 0 for keys that no row from position p_first to p_last sees. `odd`: of the lane's keys
// (4 h + i) those that show NaN to the rows that see them, as their page is none or their value has a number that is not finite: a weight of 0 would
// not hide such a value, so that it is taken at 0 too and goes to the rows through their scores.
template <int D>
DEV_INLINE unsigned int value_scales(const Attend& a, const Raw<D>& w, float (&su)[2][4], int step, int p_first, int p_last, int kg, bool look) {
  unsigned int odd = 0, vs[2] = {w.vs[0], w.vs[1]};
  if (look) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = step * STEP + h * TILE + kg * 4 + i;
        if (key > p_last || (a.window > 0 && p_first - key >= a.window)) vs[h] &= ~(255u << (8 * i));
      }
    auto high = [](unsigned int v) { return ((v & 0x7f7f7f7fu) + 0x03030303u) & v & 0x80808080u; };   // the bytes from 253 on
    if (__any((high(vs[0]) | high(vs[1])) != 0) || w.bad[0] || w.bad[1]) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        unrolled<4>([&](auto token) {
          constexpr int I = decltype(token)::value;
          const unsigned long long lanes = __ballot(not_finite<D, I>(w.v[h], (vs[h] >> (8 * I)) & 255u));
          if (!w.bad[h] && ((lanes >> (16 * kg)) & 0xffffu) == 0) return;
          odd |= 1u << (4 * h + I);   // where it is not seen at all, it does not show either
          vs[h] &= ~(255u << (8 * I));
        });
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) su[h][i] = scale_of((vs[h] >> (8 * i)) & 255u);
  return odd;
}

// Few rows: a block has a tile of 16 RT rows and its waves take its steps in turn.
template <int D, int RT>
__global__ __launch_bounds__(64 * WAVES4, D == 64 ? 5 - RT : D == 128 ? 4 - RT : 2) void attention_4bit_kernel(Attend a) {
  constexpr int R = 16 * RT, KF = D / 32, VF = D / 16;
  __shared__ float4v lds[WAVES4 / 2][RT * VF][64];   // at first the waves' states
  float2v(&states)[WAVES4][R] = reinterpret_cast<float2v(&)[WAVES4][R]>(lds);
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;
  const int g = (int)(blockIdx.x % a.G), sub = (int)(blockIdx.x / a.G % a.subs);
  const int* item = a.items + (long)(blockIdx.x / a.G / a.subs) * 6;
  const int seq = item[0], t0 = item[1], t1 = item[2], from = item[3], to = item[4], slot = item[5];
  const int p0 = a.positions[t0], p1 = a.positions[t1 - 1];
  Rows<D, RT> rows;
  rows.start(a, R, 0, g, sub, t0, t1, p1, n, kg);
  const Source<D> source = {a.tables + (long)seq * a.width, p1, g};

  auto compute = [&](const Raw<D>& w, int step) {
    const int j = step * STEP;
    // whether some row does not see some key of the step
    const bool edge = j + STEP - 1 > p0 || (a.window > 0 && p1 - j >= a.window) || w.bad[0] || w.bad[1];
    f32x4 s[RT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][h] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int f = 0; f < KF; ++f) {
        const bf16x8_v k = key_frag(w, h, f);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, rows.q[rt][f], s[rt][h], 0, 0, 0);
      }
    }
    float su[2][4];
    const unsigned int odd = value_scales(a, w, su, step, p0, p1, kg, edge);
    if (edge) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[rt][h][i] = !rows.sees(a, rt, j + h * TILE + kg * 4 + i) ? -INFINITY : odd >> (4 * h + i) & 1 ? __builtin_nanf("") : s[rt][h][i];
    }
    rows.template refer<1>(s, a.scale);
    bf16x8_v p[RT], rest[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) rows.weigh(rt, s[rt][0], s[rt][1], a.scale, p[rt], rest[rt]);
    unrolled<D / 32>([&](auto byte) {
      constexpr int B = decltype(byte)::value;
      bf16x8_v lo, hi;
      value_frags<D, B>(w, su, lo, hi);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        rows.o[rt][2 * B] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, p[rt], rows.o[rt][2 * B], 0, 0, 0);
        rows.o[rt][2 * B + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, p[rt], rows.o[rt][2 * B + 1], 0, 0, 0);
        rows.o[rt][2 * B] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, rest[rt], rows.o[rt][2 * B], 0, 0, 0);
        rows.o[rt][2 * B + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, rest[rt], rows.o[rt][2 * B + 1], 0, 0, 0);
      }
    });
  };

  // the next step's codes are on their way while a step is worked on, and the page numbers of the one after it
  int step = from + wid;
  if (step < to) {
    Raw<D> even, odd;
    int pages[2];
    source.look(a, pages, step);
    source.load(a, even, step, pages, n, kg);
    source.look(a, pages, step + WAVES4);
    while (true) {
      if (step + WAVES4 < to) {
        source.load(a, odd, step + WAVES4, pages, n, kg);
        source.look(a, pages, step + 2 * WAVES4);
      }
      compute(even, step);
      if ((step += WAVES4) >= to) break;
      if (step + WAVES4 < to) {
        source.load(a, even, step + WAVES4, pages, n, kg);
        source.look(a, pages, step + 2 * WAVES4);
      }
      compute(odd, step);
      if ((step += WAVES4) >= to) break;
    }
  }

  // the waves' states meet: a common reference, then sums in pairs
  rows.sum_lanes();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
    if (kg == 0) states[wid][rt * 16 + n] = rows.state[rt];
  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES4; ++w) top = fmaxf(top, states[w][rt * 16 + n][0]);
#pragma unroll
    for (int w = 0; w < WAVES4; ++w) {
      const float2v x = states[w][rt * 16 + n];   // without a reference the sum is 0, or NaN, which stays
      sum += x[0] == -INFINITY ? x[1] : x[1] * __builtin_amdgcn_exp2f(x[0] - top);
    }
    const float mine = rows.state[rt][0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(rows.state[rt][0] - top);
#pragma unroll
    for (int f = 0; f < VF; ++f) rows.o[rt][f] *= mine;
    rows.state[rt] = float2v{top, sum};
  }
  __syncthreads();
#pragma unroll
  for (int live = WAVES4 / 2; live > 0; live >>= 1) {
    if (wid >= live && wid < 2 * live) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int f = 0; f < VF; ++f) lds[wid - live][rt * VF + f][lane] = rows.o[rt][f];
    }
    __syncthreads();
    if (wid < live) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int f = 0; f < VF; ++f) rows.o[rt][f] += lds[wid][rt * VF + f][lane];
    }
    __syncthreads();
  }
  if (wid != 0) return;
  if (slot < 0) rows.store(a, kg);   // the only part
  else rows.store_part(a.parts + (((long)slot * a.subs + sub) * a.G + g) * (R * (D + 2L)), R, 0, n, kg);
}

// Rows of a wave of the kernel below: 32, a lane and its half-wave twin have one as their column of products of 32 x 32 x 16. Of a step's 32 keys a
// lane has those at key_of(i), in the order that the second product takes them.
template <int D>
struct WideRows {
  static constexpr int KQ = D / 16, VB = D / 32;   // products of a step's scores; pairs of a lane's channels, 32 channels each
  bf16x8_v q[KQ];
  int pos, tok, head;
  f32x16 o[VB];
  float2v state;   // the reference, and the sum of the weights
  static DEV_INLINE int key_of(int i, int hf) { return (i & 3) + 8 * (i >> 2) + 4 * hf; }

  DEV_INLINE void start(const Attend& a, int R, int row0, int g, int sub, int t0, int t1, int p_last, int lane) {
    const int per_token = min(a.group, R), hf = lane >> 5, r = row0 + (lane & 31), in = sub * R + r % per_token;
    tok = t0 + r / per_token;
    const bool real = tok < t1 && in < a.group;
    head = real ? g * a.group + in : -1;
    pos = real ? a.positions[tok] : p_last;
    const bf16s* from = a.q + (real ? tok : t0) * a.q_stride + (long)(real ? head : g * a.group) * D;
#pragma unroll
    for (int j = 0; j < KQ; ++j) {   // quarter 2 (j / VB) + hf of the channels, 8 from word j % VB on
      q[j] = *reinterpret_cast<const bf16x8_v*>(from + (2 * (j / VB) + hf) * (D / 4) + j % VB * 8);
      if (a.negative) q[j] = __builtin_bit_cast(bf16x8_v, __builtin_bit_cast(uint4v, q[j]) ^ 0x80008000u);
    }
    state = float2v{-INFINITY, 0.0f};
#pragma unroll
    for (int b = 0; b < VB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;
  }

  DEV_INLINE bool sees(const Attend& a, int key) const { return key <= pos && (a.window <= 0 || pos - key < a.window); }

  template <int S>
  DEV_INLINE void refer(const f32x16 (&s)[S], float scale) {
    float top = -INFINITY;
#pragma unroll
    for (int h = 0; h < S; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[h][i]);
    if (__any(top * scale > state[0] + SLACK)) {
      top = fmaxf(top, __shfl_xor(top, 32)) * scale;
      const float m = state[0], next = top > m + SLACK ? top : m, fall = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - next);
      state = float2v{next, state[1] * fall};
#pragma unroll
      for (int b = 0; b < VB; ++b) o[b] *= fall;
    }
  }

  DEV_INLINE void weigh(const f32x16& s, float scale, bf16x8_v (&p)[2], bf16x8_v (&rest)[2]) {
    const float ref = state[0] == -INFINITY ? 0.0f : state[0];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(fmaf(s[8 * h + i], scale, -ref));
        state[1] += e[i];
      }
      two_pieces(e, p[h], rest[h]);
    }
  }

  // channels of n = key_of(i), i < 8: n * (D / 16) + 2 b + (0 or 1)
  DEV_INLINE void store(const Attend& a, int hf) const {
    if (head < 0) return;
    const float inv = 1.0f / state[1];
    bf16s* to = a.out + ((long)tok * a.H + head) * D;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      unsigned int w[VB];
#pragma unroll
      for (int b = 0; b < VB; ++b) w[b] = two_bf16(o[b][i] * inv, o[b][i + 8] * inv);
      unsigned int* at = reinterpret_cast<unsigned int*>(to + key_of(i, hf) * (D / 16));
#pragma unroll
      for (int b = 0; b < VB; b += 2) *reinterpret_cast<uint2*>(at + b) = make_uint2(w[b], w[b + 1]);
    }
  }
  DEV_INLINE void store_part(float* part, int R, int r, int hf) const {
    if (head < 0) return;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int b = 0; b < VB; b += 2)
        *reinterpret_cast<float4v*>(part + (long)r * D + key_of(i, hf) * (D / 16) + 2 * b) = float4v{o[b][i], o[b][i + 8], o[b + 1][i], o[b + 1][i + 8]};
    if (hf == 0) *reinterpret_cast<float2v*>(part + (long)R * D + r * 2) = state;
  }
};

// Many rows: a block has 32 a wave, and all its waves take the same steps. Each makes one of four steps' codes into fragments in LDS, which all of them
// read: the conversions, half of what a wave of the other form issues, are then done once for the block. Two steps' scores are weighed
// together: the chain from scores to products is what a wave waits for. Portions of 1000 over 4000 tokens, four sequences, 32/8 heads of 128: with
// weights of one piece 276 us by products of 16 x 16 x 32 and a step at a time, 227 with two, 205 by products of 32 x 32 x 16, half the instructions;
// with both pieces 268 (744 TFLOP/s, 1116 of the three products that they are).
template <int D>
__global__ __launch_bounds__(64 * WAVES4, 2) void attention_4bit_wide_kernel(Attend a) {
  constexpr int R = 32 * WAVES4, KF = D / 32, KQ = D / 16, VB = D / 32;
  __shared__ uint4v keys[WAVES4][KQ][64], values[WAVES4][2][VB][64];   // of four steps
  __shared__ unsigned int odds[WAVES4][4];
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4, hf = lane >> 5;
  const int g = (int)(blockIdx.x % a.G), sub = (int)(blockIdx.x / a.G % a.subs);
  const int* item = a.items + (long)(blockIdx.x / a.G / a.subs) * 6;
  const int seq = item[0], t0 = item[1], t1 = item[2], from = item[3], to = item[4], slot = item[5];
  const int p0 = a.positions[t0], p1 = a.positions[t1 - 1], per_token = min(a.group, R), row0 = wid * 32;
  WideRows<D> rows;
  rows.start(a, R, row0, g, sub, t0, t1, p1, lane);
  // of the wave's own rows; without any it works for the others
  const int mine0 = p0 + row0 / per_token, mine1 = min(p1, p0 + (row0 + 31) / per_token);
  const Source<D> source = {a.tables + (long)seq * a.width, p1, g};
  Raw<D> w;
  int pages[2];
  source.look(a, pages, from + wid);
  source.load(a, w, from + wid, pages, n, kg);
  for (int base = from; base < to; base += WAVES4) {
    __syncthreads();   // the fragments before have been used
    if (base + wid < to) {
      const int step = base + wid, j = step * STEP;
      const bool edge = j + STEP - 1 > p0 || (a.window > 0 && p1 - j >= a.window) || w.bad[0] || w.bad[1];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int f = 0; f < KF; ++f)
          keys[wid][(kg >> 1) * KF + f][(kg & 1) * 32 + h * 16 + n] = __builtin_bit_cast(uint4v, key_frag(w, h, f));
      float su[2][4];
      const unsigned int odd = value_scales(a, w, su, step, p0, p1, kg, edge);
      if (n == 0) odds[wid][kg] = odd;
      unrolled<VB>([&](auto byte) {
        constexpr int B = decltype(byte)::value;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          unsigned int lo[2], hi[2];
          value_words<D, B>(w.v[h], su[h], lo, hi);
          uint2* at = reinterpret_cast<uint2*>(&values[wid][h][B][(kg & 1) * 32 + n]) + (kg >> 1);
          at[0] = make_uint2(lo[0], lo[1]);
          at[32] = make_uint2(hi[0], hi[1]);   // 16 lanes on
        }
      });
      if (step + WAVES4 < to) {
        source.look(a, pages, step + WAVES4);
        source.load(a, w, step + WAVES4, pages, n, kg);
      }
    }
    __syncthreads();
    const int ready = min(WAVES4, to - base);
    // S of the steps that lie ready, from the first-th on
    auto compute = [&](auto steps, int first) {
      constexpr int S = decltype(steps)::value;
      const int j = (base + first) * STEP, end = j + S * STEP - 1;
      if (mine0 > mine1 || j > mine1 || (a.window > 0 && mine0 - end >= a.window)) return;   // nothing to see
      f32x16 s[S];
      unsigned int odd = 0;
#pragma unroll
      for (int h = 0; h < S; ++h) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[h][i] = 0.0f;
#pragma unroll
        for (int f = 0; f < KQ; ++f)
          s[h] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_v, keys[first + h][f][lane]), rows.q[f], s[h], 0, 0, 0);
        // bits of the lane's keys: quads hf and 2 + hf of both tiles
        const unsigned int x = odds[first + h][hf], y = odds[first + h][2 + hf];
        odd |= ((x & 15u) | (y & 15u) << 4 | (x >> 4) << 8 | (y >> 4) << 12) << (16 * h);
      }
      if (end > mine0 || (a.window > 0 && mine1 - j >= a.window) || __any(odd != 0)) {
#pragma unroll
        for (int h = 0; h < S; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[h][i] = !rows.sees(a, j + h * STEP + rows.key_of(i, hf)) ? -INFINITY : odd >> (16 * h + i) & 1 ? __builtin_nanf("") : s[h][i];
      }
      rows.refer(s, a.scale);
      bf16x8_v p[S][2], rest[S][2];
#pragma unroll
      for (int h = 0; h < S; ++h) rows.weigh(s[h], a.scale, p[h], rest[h]);
#pragma unroll
      for (int h = 0; h < S; ++h)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int b = 0; b < VB; ++b) {
            const bf16x8_v v = __builtin_bit_cast(bf16x8_v, values[first + h][t][b][lane]);
            rows.o[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, p[h][t], rows.o[b], 0, 0, 0);
            rows.o[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, rest[h][t], rows.o[b], 0, 0, 0);
          }
    };
    int i = 0;
    for (; i + 2 <= ready; i += 2) compute(std::integral_constant<int, 2>(), i);
    if (i < ready) compute(std::integral_constant<int, 1>(), i);
  }
  rows.state[1] += __shfl_xor(rows.state[1], 32);
  if (slot < 0) rows.store(a, hf);
  else rows.store_part(a.parts + (((long)slot * a.subs + sub) * a.G + g) * (R * (D + 2L)), R, row0 + (lane & 31), hf);
}

// The same at 256 channels, where registers are few: 16 rows a wave, products of 16 x 16 x 32, two steps in LDS, which two waves make each.
template <int D>
__global__ __launch_bounds__(64 * WAVES4, 2) void attention_4bit_shared_kernel(Attend a) {
  constexpr int RT = 1, R = 16 * RT * WAVES4, KF = D / 32, VF = D / 16;
  constexpr int READY = 2, SHARES = WAVES4 / READY;   // steps in LDS, waves that make one
  __shared__ uint4v frags[READY][2 * KF + VF][64];
  __shared__ unsigned int odds[READY][4];
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;
  const int g = (int)(blockIdx.x % a.G), sub = (int)(blockIdx.x / a.G % a.subs);
  const int* item = a.items + (long)(blockIdx.x / a.G / a.subs) * 6;
  const int seq = item[0], t0 = item[1], t1 = item[2], from = item[3], to = item[4], slot = item[5];
  const int p0 = a.positions[t0], p1 = a.positions[t1 - 1], per_token = min(a.group, R), row0 = wid * 16 * RT;
  const int made = wid / SHARES, mine = wid % SHARES;   // the step and the share of it that the wave makes
  Rows<D, RT> rows;
  rows.start(a, R, row0, g, sub, t0, t1, p1, n, kg);
  // of the wave's own rows; without any it works for the others
  const int mine0 = p0 + row0 / per_token, mine1 = min(p1, p0 + (row0 + 16 * RT - 1) / per_token);
  const Source<D> source = {a.tables + (long)seq * a.width, p1, g};
  Raw<D> w;
  int pages[2];
  source.look(a, pages, from + made);
  source.load(a, w, from + made, pages, n, kg);
  for (int base = from; base < to; base += READY) {
    __syncthreads();   // the fragments before have been used
    if (base + made < to) {
      const int step = base + made, j = step * STEP;
      const bool edge = j + STEP - 1 > p0 || (a.window > 0 && p1 - j >= a.window) || w.bad[0] || w.bad[1];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h != mine) continue;
#pragma unroll
        for (int f = 0; f < KF; ++f) frags[made][h * KF + f][lane] = __builtin_bit_cast(uint4v, key_frag(w, h, f));
      }
      float su[2][4];
      const unsigned int odd = value_scales(a, w, su, step, p0, p1, kg, edge);
      if (n == 0) odds[made][kg] = odd;
      unrolled<D / 32>([&](auto byte) {
        constexpr int B = decltype(byte)::value;
        if (B / (D / 64) != mine) return;
        bf16x8_v lo, hi;
        value_frags<D, B>(w, su, lo, hi);
        frags[made][2 * KF + 2 * B][lane] = __builtin_bit_cast(uint4v, lo);
        frags[made][2 * KF + 2 * B + 1][lane] = __builtin_bit_cast(uint4v, hi);
      });
      if (step + READY < to) {
        source.look(a, pages, step + READY);
        source.load(a, w, step + READY, pages, n, kg);
      }
    }
    __syncthreads();
    const int ready = min(READY, to - base);
    // S of the steps that lie ready, from the i-th on
    auto compute = [&](auto steps, int i) {
      constexpr int S = decltype(steps)::value;
      const int j = (base + i) * STEP, end = j + S * STEP - 1;
      if (mine0 > mine1 || j > mine1 || (a.window > 0 && mine0 - end >= a.window)) return;   // nothing to see
      f32x4 s[RT][2 * S];
#pragma unroll
      for (int h = 0; h < 2 * S; ++h) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][h] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int f = 0; f < KF; ++f) {
          const bf16x8_v k = __builtin_bit_cast(bf16x8_v, frags[i + h / 2][h % 2 * KF + f][lane]);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[rt][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, rows.q[rt][f], s[rt][h], 0, 0, 0);
        }
      }
      unsigned int odd = 0;
#pragma unroll
      for (int h = 0; h < S; ++h) odd |= odds[i + h][kg] << (8 * h);
      if (end > mine0 || (a.window > 0 && mine1 - j >= a.window) || __any(odd != 0)) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int h = 0; h < 2 * S; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[rt][h][e] = !rows.sees(a, rt, j + h * TILE + kg * 4 + e) ? -INFINITY : odd >> (4 * h + e) & 1 ? __builtin_nanf("") : s[rt][h][e];
      }
      rows.template refer<S>(s, a.scale);
      bf16x8_v p[RT][S], rest[RT][S];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int h = 0; h < S; ++h) rows.weigh(rt, s[rt][2 * h], s[rt][2 * h + 1], a.scale, p[rt][h], rest[rt][h]);
#pragma unroll
      for (int h = 0; h < S; ++h)
#pragma unroll
        for (int f = 0; f < VF; ++f) {
          const bf16x8_v v = __builtin_bit_cast(bf16x8_v, frags[i + h][2 * KF + f][lane]);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            rows.o[rt][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[rt][h], rows.o[rt][f], 0, 0, 0);
            rows.o[rt][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, rest[rt][h], rows.o[rt][f], 0, 0, 0);
          }
        }
    };
    int i = 0;
    for (; i + 2 <= ready; i += 2) compute(std::integral_constant<int, 2>(), i);
    if (i < ready) compute(std::integral_constant<int, 1>(), i);
  }
  rows.sum_lanes();
  if (slot < 0) rows.store(a, kg);
  else rows.store_part(a.parts + (((long)slot * a.subs + sub) * a.G + g) * (R * (D + 2L)), R, row0, n, kg);
}

// Puts the parts of a tile's rows together: a block takes 512 / D rows, eight channels a lane; its waves take eight parts each at a time, so that
// few round trips to memory follow each other, and meet in LDS.
constexpr int JOIN_WAVES = 8, AT_ONCE = 8;

template <int D, int R>
__global__ __launch_bounds__(64 * JOIN_WAVES) void attention_4bit_join_kernel(Attend a) {
  constexpr int LANES = D / 8;
  __shared__ float lds[JOIN_WAVES][10][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, c = lane % LANES * 8, r = blockIdx.y * (64 / LANES) + lane / LANES;
  const int g = (int)(blockIdx.x % a.G), sub = (int)(blockIdx.x / a.G % a.subs);
  const int* join = a.joins + (long)(blockIdx.x / a.G / a.subs) * 4;
  const int t0 = join[0], t1 = join[1], count = join[3];
  const int per_token = min(a.group, R), tok = t0 + r / per_token, in = sub * R + r % per_token;
  if (blockIdx.y * (64 / LANES) >= (t1 - t0) * per_token) return;   // the whole block
  const bool real = tok < t1 && in < a.group;
  const float* part = a.parts + (((long)join[2] * a.subs + sub) * a.G + g) * (R * (D + 2L));
  const long next = (long)a.subs * a.G * (R * (D + 2L));
  float m = -INFINITY, sum = 0.0f, o[8] = {};
  // the sums fall to a new reference; without an old one all is 0, or NaN, which stays
  auto fall = [](float from, float to) { return from == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(from - to); };
  for (int first = wid * AT_ONCE; real && first < count; first += JOIN_WAVES * AT_ONCE) {
    float2v state[AT_ONCE];
    float x[AT_ONCE][8];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const float* p = part + min(first + i, count - 1) * next;
      state[i] = *reinterpret_cast<const float2v*>(p + (long)R * D + r * 2);
      load8(p + r * D + c, x[i]);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) top = fmaxf(top, state[i][0]);
    const float w = fall(m, top);
    sum *= w;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= w;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      if (first + i >= count) break;
      const float u = fall(state[i][0], top);
      sum += u * state[i][1];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] += u * x[i][e];
    }
    m = top;
  }
  if (count > AT_ONCE) {   // other waves had parts
    lds[wid][8][lane] = m;
    lds[wid][9][lane] = sum;
#pragma unroll
    for (int e = 0; e < 8; ++e) lds[wid][e][lane] = o[e];
    __syncthreads();
    if (wid != 0) return;
    float top = m;
#pragma unroll
    for (int w = 1; w < JOIN_WAVES; ++w) top = fmaxf(top, lds[w][8][lane]);
    sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < JOIN_WAVES; ++w) {
      const float u = fall(lds[w][8][lane], top);
      sum += u * lds[w][9][lane];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] += u * lds[w][e][lane];
    }
  }
  if (wid != 0 || !real) return;
  const float inv = 1.0f / sum;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] *= inv;
  store8(a.out + ((long)tok * a.H + g * a.group + in) * D + c, o);
}

// R: rows of a tile, 16 or 32 for one wave's, else the block's
template <int D, int R>
void launch(Attend a, long items, long slots, long joins, const at::Tensor& like) {
  a.subs = (a.group + R - 1) / R;
  const long heads = (long)a.G * a.subs;
  at::Tensor parts;
  if (joins > 0) {
    parts = at::empty({slots * heads * R * (D + 2)}, like.options().dtype(at::kFloat));
    a.parts = parts.data_ptr<float>();
  }
  const dim3 grid((unsigned)(items * heads)), block(64 * WAVES4);
  if constexpr (R == 32 * WAVES4) hipLaunchKernelGGL((attention_4bit_wide_kernel<D>), grid, block, 0, stream(), a);
  else if constexpr (R > 32) hipLaunchKernelGGL((attention_4bit_shared_kernel<D>), grid, block, 0, stream(), a);
  else hipLaunchKernelGGL((attention_4bit_kernel<D, R / 16>), grid, block, 0, stream(), a);
  HIP_CHECK_LAST();
  if (joins > 0) {
    hipLaunchKernelGGL((attention_4bit_join_kernel<D, R>), dim3((unsigned)(joins * heads), R * D / 512), dim3(64 * JOIN_WAVES), 0, stream(), a);
    HIP_CHECK_LAST();
  }
}

}  // namespace

// `plan`: of the tiles with at most 16 rows, then of those with at most 32, then of those with at most 128 (heads of 256 channels: 16, 64), what a block does, (sequence, first token, end token, first step,
// end step, part or -1) for each, then the tiles that have parts, (first token, end token, first part, parts). `sizes`: of each kind the numbers of
// both, and of parts; then the number of sequences, and the longest's tokens.
at::Tensor paged_attention_4bit(at::Tensor q_in, at::Tensor kpool, at::Tensor vpool, at::Tensor block_tables, at::Tensor positions,
                                at::Tensor plan, std::vector<int64_t> sizes, double scale, int64_t window, int64_t page_size) {
  const char* who = "paged_attention_4bit: ";
  TORCH_CHECK_VALUE(q_in.is_cuda() && q_in.dim() == 3 && is_bf16(q_in), who, "q must be bfloat16 [N, H, D]");
  const c10::DeviceGuard guard(q_in.device());
  const int64_t N = q_in.size(0), H = q_in.size(1), D = q_in.size(2);
  TORCH_CHECK_VALUE(D == 64 || D == 128 || D == 256, who, "heads of 64, 128 or 256 channels, got ", D);
  TORCH_CHECK_VALUE(page_size_of(kpool, D) == page_size && page_size_of(vpool, D) == page_size && kpool.sizes() == vpool.sizes() && kpool.size(0) > 0, who,
              "pools must be contiguous uint8 [pages, heads, page size * 17 * D / 32] of the batch's page size ", page_size);
  const int64_t G = kpool.size(1);
  TORCH_CHECK_VALUE(G > 0 && H % G == 0, who, H, " query heads cannot share ", G, " key heads");
  check_i32(block_tables, "block_tables");
  check_i32(plan, "plan");
  check_i32(positions, "positions");
  TORCH_CHECK_VALUE(block_tables.dim() == 2 && positions.numel() == N && sizes.size() == 11 && block_tables.size(0) >= sizes[9] && block_tables.size(1) * page_size >= sizes[10] &&
              plan.numel() == 6 * (sizes[0] + sizes[3] + sizes[6]) + 4 * (sizes[1] + sizes[4] + sizes[7]), who, "batch of other tokens");
  for (const at::Tensor& t : {kpool, vpool, block_tables, positions, plan})
    TORCH_CHECK_VALUE(t.device() == q_in.device(), who, "tensors on ", q_in.device(), " and ", t.device());
  const bool fits = q_in.stride(2) == 1 && q_in.stride(1) == D && q_in.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(q_in.data_ptr()) % 16 == 0;
  const at::Tensor q = fits ? q_in : q_in.clone(at::MemoryFormat::Contiguous), out = at::empty({N, H, D}, q.options());
  if (N == 0) return out;
  Attend a;
  a.q = ptr<bf16s>(q);
  a.q_stride = q.stride(0);
  a.pages = kpool.size(0);
  a.page_stride = kpool.size(1) * kpool.size(2);
  a.head_bytes = (int)kpool.size(2);
  a.kpool = kpool.data_ptr<uint8_t>();
  a.vpool = vpool.data_ptr<uint8_t>();
  a.tables = block_tables.data_ptr<int>();
  a.positions = positions.data_ptr<int>();
  a.out = ptr<bf16s>(out);
  a.width = (int)block_tables.size(1);
  a.H = (int)H;
  a.G = (int)G;
  a.group = (int)(H / G);
  a.page_shift = 0;
  while ((1L << a.page_shift) < page_size) ++a.page_shift;
  a.window = (int)std::min<int64_t>(window, 1L << 30);
  // with a scale of 0 every key has the same weight: the product with a hidden one's -infinity is to stay it
  a.scale = std::max(std::fabs((float)scale) * LOG2E4, 1e-30f);
  a.negative = scale < 0;
  auto run = [&](auto size) {
    constexpr int DD = decltype(size)::value;
    const int* at = plan.data_ptr<int>();
    for (int kind = 0; kind < 3; ++kind) {
      const long items = sizes[3 * kind], joins = sizes[3 * kind + 1], slots = sizes[3 * kind + 2];
      a.items = at;
      a.joins = at + 6 * items;
      at = a.joins + 4 * joins;
      if (items == 0) continue;
      if (kind == 0) launch<DD, 16>(a, items, slots, joins, q);
      else if (kind == 1) launch<DD, DD == 256 ? 16 : 32>(a, items, slots, joins, q);
      else launch<DD, (DD == 256 ? 16 : 32) * WAVES4>(a, items, slots, joins, q);
    }
  };
  if (D == 64) run(std::integral_constant<int, 64>());
  else if (D == 128) run(std::integral_constant<int, 128>());
  else run(std::integral_constant<int, 256>());
  return out;
}

}  // namespace serving
}  // namespace cai
