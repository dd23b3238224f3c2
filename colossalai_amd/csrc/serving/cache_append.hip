// Queries, keys and values of new tokens on their way into a paged cache: query and key heads are normed (if there are weights),
// rotated by their positions, keys and values go to their pool rows, in the activations' type or in 4 bits (cache_4bit.h).
//
//   y = R_p (w * x / sqrt(mean(x^2) + eps))
//
// A code is that of the exact y: keys that become codes are normed and rotated in float64, so that no rounding ahead of it decides between two
// numbers (it goes on in float32 with an odd last bit where bits were lost, which stands to every border as y does); everything else is
// float32, rounded once. A group with a value that is not finite has the scale byte 255. Codes are formed two at a time by the conversion
// instruction, nearest with ties to even.
//
// Bound by memory for prompts and by latency for single tokens. A wave takes a token, or with few tokens a share of its heads: D / 16 lanes a head
// with 8 channels of each half, 64 / lanes heads of one kind at a time; the angles stay in registers. 8192 tokens, 32/8 heads of 128 into a 4-bit
// cache: 43 us, 4.1 TB/s (codes by comparisons in float64 from 180 registers: 109; shares of a token's heads: 44 to 54). 4099 tokens, 28/4
// heads of 128 into a bfloat16 one: 13.4. In float32 8192 tokens of 32/8 heads of 128: 72 us into 4 bits, 82 into float32 (4.8, 4.9 TB/s).
#include "cache_4bit.h"

#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <climits>

namespace cai {
namespace serving {
namespace {

constexpr int CA_BLOCK = 256, CA_WAVES = CA_BLOCK / WAVE;

struct Append {
  long tokens;
  int parts, Hq, G, D, table_rows, page_shift;
  long q_stride, k_stride, v_stride, pool_rows;
  const float* table;
  const int *positions, *rows;
  const void *wq, *wk;
  bool narrow_weights;
  double eps;
};

template <int L, typename F>
DEV_INLINE F lanes_sum(F v) {
#pragma unroll
  for (int off = L / 2; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// y of 16 channels, 8 of each half
template <typename F>
DEV_INLINE void norm_and_turn(F (&y)[16], const float (&x)[16], const float (&w)[16], F r, bool weights, const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    F a = x[i], b = x[8 + i];
    if (weights) {
      a *= r * F(w[i]);
      b *= r * F(w[8 + i]);
    }
    y[i] = a * F(c[i]) - b * F(s[i]);
    y[8 + i] = b * F(c[i]) + a * F(s[i]);
  }
}

// y in float32 with an odd last bit where bits were lost: it stands to every number of fewer bits as y does.
DEV_INLINE float to_odd(double y) {
  const float f = (float)y;
  const double back = (double)f;
  unsigned int bits = __builtin_bit_cast(unsigned int, f);
  if (fabs(back) > fabs(y)) --bits;
  if (back != y) bits |= 1u;
  return fabsf(f) <= 3.4028234663852886e38f ? __builtin_bit_cast(float, bits) : f;
}

// Eight codes of y / 2^e, nearest, ties to the even mantissa, and the group's scale byte from its largest magnitude (4 lanes of 8 channels are
// a group).
DEV_INLINE unsigned int eight_codes(const float* y, unsigned int& byte) {
  float most = 0;
  int odd = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    odd |= !(fabsf(y[i]) <= 3.4028234663852886e38f);
    most = fmaxf(most, fabsf(y[i]));
  }
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    most = fmaxf(most, __shfl_xor(most, off));
    odd |= __shfl_xor(odd, off);
  }
  // the smallest e with most <= 6 * 2^e: most = f * 2^E, 1 <= f < 2, and 6 = 1.5 * 4
  const unsigned int bits = __builtin_bit_cast(unsigned int, most);
  const int e = max((int)(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x400000u ? 2 : 1), -126);
  byte = odd ? 255u : (unsigned)(e + 127);
  const float unit = __builtin_bit_cast(float, (unsigned)(e + 127) << 23);
  unsigned int word = 0;
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[0], y[1], unit, 0);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[2], y[3], unit, 1);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[4], y[5], unit, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[6], y[7], unit, 3);
}

// L: lanes of a head. FOUR: pools of codes, heads of 16 L channels.
template <typename T, int L, bool FOUR>
__global__ __launch_bounds__(CA_BLOCK, 4) void append_kernel(T* __restrict__ out, void* __restrict__ kpool, void* __restrict__ vpool,
                                                             const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, Append a) {
  constexpr int SIDE = WAVE / L, DF = 16 * L;
  const int lane = threadIdx.x & 63, l = lane & (L - 1), side = lane / L, D = FOUR ? DF : a.D, half = D / 2, at = l * 8;
  const bool on = at < half;
  const long wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * CA_WAVES + (threadIdx.x >> 6)));
  const long token = wave / a.parts;
  if (token >= a.tokens) return;
  const long row = a.rows[token];
  const bool kept = row >= 0 && row < a.pool_rows;
  const int p = a.positions[token];
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = s[i] = __builtin_nanf("");   // of a position that the table does not have
  if (on && p >= 0 && p < a.table_rows) {
    load8(a.table + (long)p * D + at, c);
    load8(a.table + (long)p * D + half + at, s);
  }
  const bool weights = a.wq != nullptr;
  // where the token's rows of codes are, from a head's first tile on
  const long head_bytes = FOUR ? ((1L << a.page_shift) / TILE) * Tile4<DF>::BYTES : 0;
  const int off = FOUR ? (int)(row & ((1L << a.page_shift) - 1)) : 0, t = off & (TILE - 1);
  const long base = FOUR ? (row >> a.page_shift) * a.G * head_bytes + (long)(off / TILE) * Tile4<DF>::BYTES : 0;
  const int tq = (a.Hq + SIDE - 1) / SIDE, tk = (a.G + SIDE - 1) / SIDE;
  for (int turn = (int)(wave % a.parts); turn < tq + 2 * tk; turn += a.parts) {
    const bool is_q = turn < tq, is_k = !is_q && turn < tq + tk;
    const int h = (turn - (is_q ? 0 : is_k ? tq : tq + tk)) * SIDE + side;
    const bool here = on && h < (is_q ? a.Hq : a.G);
    if (!is_q && !kept) continue;
    const T* from = (is_q ? q + token * a.q_stride : is_k ? k + token * a.k_stride : v + token * a.v_stride) + (long)h * D + at;
    float x[16], w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.0f;
    if (here) {
      load8(from, x);
      load8(from + half, x + 8);
    }
    if (is_q || is_k) {
      if (weights && on) {
        const void* ws = is_q ? a.wq : a.wk;
        if (a.narrow_weights) {
          load8((const T*)ws + at, w);
          load8((const T*)ws + half + at, w + 8);
        } else {
          load8((const float*)ws + at, w);
          load8((const float*)ws + half + at, w + 8);
        }
      }
      if (FOUR && is_k) {
        double sum = 0, y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += (double)x[i] * x[i];
        if (weights) sum = lanes_sum<L>(sum);
        norm_and_turn(y, x, w, weights ? 1.0 / sqrt(sum * (1.0 / DF) + a.eps) : 1.0, weights, c, s);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = to_odd(y[i]);
      } else {
        float sum = 0.0f, y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += x[i] * x[i];
        if (weights) sum = lanes_sum<L>(sum);
        norm_and_turn(y, x, w, weights ? 1.0f / sqrtf(sum * (1.0f / (float)D) + (float)a.eps) : 1.0f, weights, c, s);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = y[i];
      }
    }
    if (!FOUR || is_q) {
      if (!here) continue;
      T* to = (is_q ? out + (token * a.Hq + h) * D : (T*)(is_k ? kpool : vpool) + (row * a.G + h) * D) + at;
      store8(to, x);
      store8(to + half, x + 8);
      continue;
    }
    unsigned int lo_byte, hi_byte;
    const unsigned int lo = eight_codes(x, lo_byte), hi = eight_codes(x + 8, hi_byte);
    if (!here) continue;
    unsigned char* tile = (unsigned char*)(is_k ? kpool : vpool) + base + h * head_bytes;
    if (is_k) {
      *reinterpret_cast<unsigned int*>(tile + Tile4<DF>::key_codes(t) + at / 2) = lo;
      *reinterpret_cast<unsigned int*>(tile + Tile4<DF>::key_codes(t) + (half + at) / 2) = hi;
    } else if constexpr (DF == 64) {   // a lane's channels are four
      *reinterpret_cast<unsigned short*>(tile + Tile4<DF>::value_codes(t, at)) = (unsigned short)lo;
      *reinterpret_cast<unsigned short*>(tile + Tile4<DF>::value_codes(t, at + 4)) = (unsigned short)(lo >> 16);
      *reinterpret_cast<unsigned short*>(tile + Tile4<DF>::value_codes(t, half + at)) = (unsigned short)hi;
      *reinterpret_cast<unsigned short*>(tile + Tile4<DF>::value_codes(t, half + at + 4)) = (unsigned short)(hi >> 16);
    } else {
      *reinterpret_cast<unsigned int*>(tile + Tile4<DF>::value_codes(t, at)) = lo;
      *reinterpret_cast<unsigned int*>(tile + Tile4<DF>::value_codes(t, half + at)) = hi;
    }
    if ((l & 3) == 0) {
      tile[is_k ? Tile4<DF>::key_scale(t, at / 32) : Tile4<DF>::value_scale(t, at / 32)] = (unsigned char)lo_byte;
      tile[is_k ? Tile4<DF>::key_scale(t, (half + at) / 32) : Tile4<DF>::value_scale(t, (half + at) / 32)] = (unsigned char)hi_byte;
    }
  }
}

// The numbers of pool rows, [N, G, D] in bfloat16; NaN for a row that the pool does not have, and for a group that was not finite.
template <int D>
__global__ __launch_bounds__(CA_BLOCK) void read_kernel(bf16s* __restrict__ k, bf16s* __restrict__ v, const unsigned char* __restrict__ kpool,
                                                        const unsigned char* __restrict__ vpool, const int* __restrict__ rows, long N, int G,
                                                        int page_shift, long pool_rows) {
  const long total = N * G * (D / 8);
  for (long i = (long)blockIdx.x * CA_BLOCK + threadIdx.x; i < 2 * total; i += (long)gridDim.x * CA_BLOCK) {
    const bool is_k = i < total;
    const long u = is_k ? i : i - total;
    const int c0 = (int)(u % (D / 8)) * 8, g = (int)(u / (D / 8) % G);
    const long n = u / (D / 8) / G, row = rows[n];
    unsigned int word = 0, byte = 255;
    if (row >= 0 && row < pool_rows) {
      const int off = (int)(row & ((1L << page_shift) - 1)), t = off & (TILE - 1);
      const unsigned char* tile = (is_k ? kpool : vpool) + ((row >> page_shift) * G + g) * (((1L << page_shift) / TILE) * Tile4<D>::BYTES) +
                                  off / TILE * Tile4<D>::BYTES;
      if (is_k) word = *reinterpret_cast<const unsigned int*>(tile + Tile4<D>::key_codes(t) + c0 / 2);
      else if constexpr (D == 64)
        word = *reinterpret_cast<const unsigned short*>(tile + Tile4<D>::value_codes(t, c0)) |
               (unsigned int)*reinterpret_cast<const unsigned short*>(tile + Tile4<D>::value_codes(t, c0 + 4)) << 16;
      else word = *reinterpret_cast<const unsigned int*>(tile + Tile4<D>::value_codes(t, c0));
      byte = tile[is_k ? Tile4<D>::key_scale(t, c0 / 32) : Tile4<D>::value_scale(t, c0 / 32)];
    }
    const float scale = scale_of(byte);
    uint4 o = make_uint4(two_numbers<0>(word, scale), two_numbers<1>(word, scale), two_numbers<2>(word, scale), two_numbers<3>(word, scale));
    if (byte == 255) o = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
    *reinterpret_cast<uint4*>((is_k ? k : v) + u * 8) = o;
  }
}

// rows of heads that lie together, with 16-byte loads
at::Tensor head_rows(const at::Tensor& t) {
  const int64_t per = 16 / t.element_size();
  if (t.stride(2) == 1 && t.stride(1) == t.size(2) && t.stride(0) % per == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

int log2_of(int64_t v) {
  int s = 0;
  while ((1L << s) < v) ++s;
  return s;
}

}  // namespace

at::Tensor paged_kv_append(at::Tensor q_in, at::Tensor k_in, at::Tensor v_in, at::Tensor kpool, at::Tensor vpool, at::Tensor rows,
                           at::Tensor positions, at::Tensor table, c10::optional<at::Tensor> wq, c10::optional<at::Tensor> wk, double eps) {
  const char* who = "paged_kv_append: ";
  TORCH_CHECK_VALUE(q_in.is_cuda() && q_in.dim() == 3 && k_in.dim() == 3 && v_in.dim() == 3, who, "q, k and v must be [N, heads, D] on a GPU");
  TORCH_CHECK_VALUE((is_bf16(q_in) || is_f32(q_in)) && k_in.scalar_type() == q_in.scalar_type() && v_in.scalar_type() == q_in.scalar_type(), who,
                    "q, k and v must be bfloat16 or float32 and of one type");
  TORCH_CHECK_VALUE(k_in.sizes() == v_in.sizes() && k_in.size(0) == q_in.size(0) && k_in.size(2) == q_in.size(2), who,
                    "keys and values must be as many as the queries, of one size");
  for (const at::Tensor& t : {k_in, v_in, kpool, vpool, rows, positions, table, wq.value_or(q_in), wk.value_or(q_in)})
    TORCH_CHECK_VALUE(t.device() == q_in.device(), who, "tensors on ", q_in.device(), " and ", t.device());
  TORCH_CHECK_VALUE(q_in.size(0) < (1L << 32) / WAVE && q_in.size(1) > 0 && k_in.size(1) > 0, who, "up to 2^26 tokens, one head at least");   // a launch's threads
  const c10::DeviceGuard guard(q_in.device());
  const at::Tensor q = head_rows(q_in), k = head_rows(k_in), v = head_rows(v_in);
  const int64_t N = q.size(0), Hq = q.size(1), D = q.size(2), G = k.size(1);
  TORCH_CHECK_VALUE(rows.scalar_type() == at::kInt && positions.scalar_type() == at::kInt && rows.numel() == N && positions.numel() == N, who,
                    "rows and positions must be int32, one a token");
  rows = rows.contiguous();
  positions = positions.contiguous();
  TORCH_CHECK_VALUE(table.dim() == 2 && is_f32(table) && table.size(1) == D, who, "table must be float32 [positions, D]");
  table = table.contiguous();
  if (reinterpret_cast<uintptr_t>(table.data_ptr()) % 16 != 0) table = table.clone();
  TORCH_CHECK_VALUE(wq.has_value() == wk.has_value(), who, "both weights or none");
  if (wq.has_value()) {
    TORCH_CHECK_VALUE(wq->dim() == 1 && wk->dim() == 1 && wq->numel() == D && wk->numel() == D && wq->scalar_type() == wk->scalar_type() && (is_f32(*wq) || wq->scalar_type() == q.scalar_type()), who, "weights must be [D], of the queries' type or float32");
  }
  for (auto* w : {&wq, &wk})   // 16-byte loads
    if (w->has_value()) *w = reinterpret_cast<uintptr_t>((*w)->data_ptr()) % 16 == 0 ? (*w)->contiguous() : (*w)->clone(at::MemoryFormat::Contiguous);
  const bool four = kpool.scalar_type() == at::kByte;
  Append a;
  if (four) {
    TORCH_CHECK_VALUE(D == 64 || D == 128 || D == 256, who, "4-bit pools take heads of 64, 128 or 256 channels, got ", D);
    const int64_t ps = page_size_of(kpool, D);
    TORCH_CHECK_VALUE(ps > 0 && kpool.size(1) == G && vpool.sizes() == kpool.sizes() && page_size_of(vpool, D) == ps, who,
                "4-bit pools must be contiguous uint8 [pages, ", G, ", page size * 17 * ", D, " / 32] at 16-byte addresses, page sizes powers of two from "
                "16 on");
    a.page_shift = log2_of(ps);
    a.pool_rows = kpool.size(0) * ps;
  } else {
    TORCH_CHECK_VALUE(kpool.dim() == 4 && kpool.is_contiguous() && vpool.is_contiguous() && kpool.sizes() == vpool.sizes() &&
                kpool.size(2) == G && kpool.size(3) == D && kpool.scalar_type() == q.scalar_type() && vpool.scalar_type() == q.scalar_type(),
                who, "pools must be contiguous [pages, page size, ", G, ", ", D, "] of the keys' type, or uint8");
    TORCH_CHECK_VALUE(D % 16 == 0 && D <= 512, who, "head sizes are multiples of 16 up to 512, got ", D);
    TORCH_CHECK_VALUE(reinterpret_cast<uintptr_t>(kpool.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(vpool.data_ptr()) % 16 == 0, who,
                "pools must start at 16-byte addresses");
    a.page_shift = 0;
    a.pool_rows = kpool.size(0) * kpool.size(1);
  }
  const at::Tensor out = at::empty({N, Hq, D}, q.options());
  if (N == 0) return out;
  a.tokens = N;
  a.Hq = (int)Hq;
  a.G = (int)G;
  a.D = (int)D;
  a.table_rows = (int)std::min<int64_t>(table.size(0), INT_MAX);
  a.q_stride = q.stride(0);
  a.k_stride = k.stride(0);
  a.v_stride = v.stride(0);
  a.table = table.data_ptr<float>();
  a.positions = positions.data_ptr<int>();
  a.rows = rows.data_ptr<int>();
  a.wq = wq.has_value() ? wq->data_ptr() : nullptr;
  a.wk = wk.has_value() ? wk->data_ptr() : nullptr;
  a.narrow_weights = wq.has_value() && !is_f32(*wq);
  a.eps = eps;
  auto launch = [&](auto type, auto lanes, auto codes) {
    using T = decltype(type);
    constexpr int L = decltype(lanes)::value;
    const int64_t side = WAVE / L, turns = (Hq + side - 1) / side + 2 * ((G + side - 1) / side);
    a.parts = (int)std::max<int64_t>(1, std::min(turns, 4096 / N));   // 16 waves a CU, while a token's heads give them
    const long blocks = (N * a.parts + CA_WAVES - 1) / CA_WAVES;
    hipLaunchKernelGGL((append_kernel<T, L, decltype(codes)::value>), dim3((unsigned)blocks), dim3(CA_BLOCK), 0, stream(), ptr<T>(out),
                       kpool.data_ptr(), vpool.data_ptr(), ptr<T>(q), ptr<T>(k), ptr<T>(v), a);
  };
  using std::integral_constant;
  auto sized = [&](auto type) {
    if (four) {
      if (D == 64) launch(type, integral_constant<int, 4>(), std::true_type());
      else if (D == 128) launch(type, integral_constant<int, 8>(), std::true_type());
      else launch(type, integral_constant<int, 16>(), std::true_type());
    } else if (D <= 64) launch(type, integral_constant<int, 4>(), std::false_type());
    else if (D <= 128) launch(type, integral_constant<int, 8>(), std::false_type());
    else if (D <= 256) launch(type, integral_constant<int, 16>(), std::false_type());
    else launch(type, integral_constant<int, 32>(), std::false_type());
  };
  if (is_bf16(q)) sized(bf16s());
  else sized(float());
  HIP_CHECK_LAST();
  return out;
}

std::vector<at::Tensor> kv4_read(at::Tensor kpool, at::Tensor vpool, at::Tensor rows, int64_t D) {
  TORCH_CHECK_VALUE(D == 64 || D == 128 || D == 256, "kv4_read: 4-bit pools hold heads of 64, 128 or 256 channels, got ", D);
  const int64_t ps = page_size_of(kpool, D);
  TORCH_CHECK_VALUE(kpool.is_cuda() && ps > 0 && vpool.sizes() == kpool.sizes() && page_size_of(vpool, D) == ps,
              "kv4_read: pools must be contiguous uint8 [pages, heads, page size * 17 * D / 32]");
  const c10::DeviceGuard guard(kpool.device());
  TORCH_CHECK_VALUE(rows.scalar_type() == at::kInt && rows.dim() == 1, "kv4_read: rows must be int32 [N]");
  rows = rows.contiguous();
  TORCH_CHECK_VALUE(vpool.device() == kpool.device() && rows.device() == kpool.device(), "kv4_read: tensors on several devices");
  const int64_t N = rows.numel(), G = kpool.size(1);
  const auto k = at::empty({N, G, D}, kpool.options().dtype(at::kBFloat16)), v = at::empty_like(k);
  if (N == 0) return {k, v};
  const int grid = capped_grid((2 * N * G * (D / 8) + CA_BLOCK - 1) / CA_BLOCK, 8192);
  auto run = [&](auto size) {
    hipLaunchKernelGGL((read_kernel<decltype(size)::value>), dim3(grid), dim3(CA_BLOCK), 0, stream(), ptr<bf16s>(k), ptr<bf16s>(v),
                       kpool.data_ptr<uint8_t>(), vpool.data_ptr<uint8_t>(), rows.data_ptr<int>(), (long)N, (int)G, log2_of(ps),
                       (long)(kpool.size(0) * ps));
  };
  if (D == 64) run(std::integral_constant<int, 64>());
  else if (D == 128) run(std::integral_constant<int, 128>());
  else run(std::integral_constant<int, 256>());
  HIP_CHECK_LAST();
  return {k, v};
}

}  // namespace serving
}  // namespace cai
