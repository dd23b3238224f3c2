// Queries, keys and values of new tokens on their way into a paged cache: query and key heads are normed (if there are weights),
// rotated by their positions, keys and values go to their pool rows, in the activations' type or in 4 bits (cache_4bit.h).
//
//   y = R_p (w * x / sqrt(mean(x^2) + eps))
//
// A code is that of the exact y: keys that become codes are normed and rotated in float64, so that no rounding ahead of it decides between two
// numbers; everything else is float32, rounded once. A group with a value that is not finite has the scale byte 255.
//
// Bound by memory for prompts and by latency for single tokens. A wave takes a token, or with few tokens a share of its heads: D / 16 lanes a head
// with 8 channels of each half, 64 / lanes heads at a time; the angles stay in registers.
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

template <typename F>
DEV_INLINE F larger(F a, F b) { return a > b ? a : b; }

// 1 / sqrt(v)
DEV_INLINE float inverse_root(float v) { return 1.0f / sqrtf(v); }
DEV_INLINE double inverse_root(double v) { return 1.0 / sqrt(v); }

template <typename T, typename F>
DEV_INLINE void norm_and_turn(F (&y)[16], const T* w, bool weights, bool narrow, const float* wide, F eps, F inv_d, const float (&c)[8],
                              const float (&s)[8], int at, int half, int L, bool on, F sum) {
  if (!on) return;
  const F r = weights ? inverse_root(sum * inv_d + eps) : F(1);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    F a = y[i], b = y[8 + i];
    if (weights) {
      a *= r * F(narrow ? ldf(w + at + i) : wide[at + i]);
      b *= r * F(narrow ? ldf(w + half + at + i) : wide[half + at + i]);
    }
    y[i] = a * F(c[i]) - b * F(s[i]);
    y[8 + i] = b * F(c[i]) + a * F(s[i]);
  }
}

// Eight codes of y / 2^e, and the group's scale byte from its largest magnitude (4 lanes of 8 channels are a group).
template <typename F>
DEV_INLINE unsigned int eight_codes(const F* y, unsigned int& byte) {
  F most = 0;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const F a = y[i] < 0 ? -y[i] : y[i];
    odd |= !(a <= F(3.4028234663852886e38));
    most = larger(most, a);
  }
  most = larger(most, __shfl_xor(most, 1));
  most = larger(most, __shfl_xor(most, 2));
  int odds = odd;
  odds |= __shfl_xor(odds, 1);
  odds |= __shfl_xor(odds, 2);
  // the smallest e with most <= 6 * 2^e: most = f * 2^E, 1 <= f < 2, and 6 = 1.5 * 4
  const double m = (double)most;
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, m);
  int e = (int)(bits >> 52) - 1023 - ((bits & 0xfffffffffffffULL) <= 0x8000000000000ULL ? 2 : 1);
  e = max(e, -126);
  byte = odds ? 255u : (unsigned)(e + 127);
  const F unit = (F)__builtin_bit_cast(double, (unsigned long long)(1023 - e) << 52);   // 2^-e: a power of two from 2^-126 to 2^126
  unsigned int word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const F a = (y[i] < 0 ? -y[i] : y[i]) * unit;
    // nearest, ties to the even mantissa
    unsigned int code = (a > F(0.25)) + (a >= F(0.75)) + (a > F(1.25)) + (a >= F(1.75)) + (a > F(2.5)) + (a >= F(3.5)) + (a > F(5));
    code = odds ? 7u : code;
    word |= (code | (y[i] < 0 ? 8u : 0u)) << (4 * i);
  }
  return word;
}

// L: lanes of a head. FOUR: pools of codes, heads of 16 L channels.
template <typename T, int L, bool FOUR>
__global__ __launch_bounds__(CA_BLOCK) void append_kernel(T* __restrict__ out, void* __restrict__ kpool, void* __restrict__ vpool,
                                                          const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, Append a) {
  constexpr int SIDE = WAVE / L, DF = 16 * L;
  const int lane = threadIdx.x & 63, l = lane & (L - 1), side = lane / L, D = FOUR ? DF : a.D, half = D / 2, at = l * 8;
  const bool on = at < half;
  const long wave = (long)blockIdx.x * CA_WAVES + (threadIdx.x >> 6);
  const long token = wave / a.parts;
  if (token >= a.tokens) return;
  const int all = a.Hq + 2 * a.G;
  const long row = a.rows[token];
  const bool kept = row >= 0 && row < a.pool_rows;
  const int p = a.positions[token];
  float c[8], s[8];
  if (on) {
    if (p >= 0 && p < a.table_rows) {
      load8(a.table + (long)p * D + at, c);
      load8(a.table + (long)p * D + half + at, s);
    } else {   // not in the table
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = s[i] = __builtin_nanf("");
    }
  }
  const bool weights = a.wq != nullptr;
  for (int head = (int)(wave % a.parts) * SIDE + side; head < (all + SIDE - 1) / SIDE * SIDE; head += a.parts * SIDE) {
    const bool is_q = head < a.Hq, is_k = !is_q && head < a.Hq + a.G, here = on && head < all;
    const int h = is_q ? head : is_k ? head - a.Hq : head - a.Hq - a.G;
    const T* from = is_q ? q + token * a.q_stride : is_k ? k + token * a.k_stride : v + token * a.v_stride;
    float x[16];
    if (here) {
      load8(from + (long)h * D + at, x);
      load8(from + (long)h * D + half + at, x + 8);
    }
    if constexpr (FOUR) {
      unsigned char* tile = nullptr;
      int t = 0;
      if (!is_q && kept) {
        const long page = row >> a.page_shift;
        const int off = (int)(row & ((1L << a.page_shift) - 1));
        t = off & (TILE - 1);
        tile = (unsigned char*)(is_k ? kpool : vpool) + (page * a.G + h) * (((1L << a.page_shift) / TILE) * Tile4<DF>::BYTES) +
               off / TILE * Tile4<DF>::BYTES;
      }
      unsigned int lo, hi, lo_byte, hi_byte;
      if (is_k) {
        double y[16], sum = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          y[i] = here ? x[i] : 0.0f;
          sum += y[i] * y[i];
        }
        if (weights) sum = lanes_sum<L>(sum);
        norm_and_turn<T, double>(y, (const T*)a.wk, weights, a.narrow_weights, (const float*)a.wk, a.eps, 1.0 / DF, c, s, at, half, L, here, sum);
        lo = eight_codes(y, lo_byte);
        hi = eight_codes(y + 8, hi_byte);
        if (here && kept) {
          *reinterpret_cast<unsigned int*>(tile + Tile4<DF>::key_codes(t) + at / 2) = lo;
          *reinterpret_cast<unsigned int*>(tile + Tile4<DF>::key_codes(t) + (half + at) / 2) = hi;
          if ((l & 3) == 0) {
            tile[Tile4<DF>::key_scale(t, at / 32)] = (unsigned char)lo_byte;
            tile[Tile4<DF>::key_scale(t, (half + at) / 32)] = (unsigned char)hi_byte;
          }
        }
        continue;
      }
      if (!is_q) {
        if (!here) {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = 0.0f;
        }
        lo = eight_codes(x, lo_byte);
        hi = eight_codes(x + 8, hi_byte);
        if (here && kept) {
          if constexpr (DF == 64) {   // a lane's channels are four
            *reinterpret_cast<unsigned short*>(tile + Tile4<DF>::value_codes(t, at)) = (unsigned short)lo;
            *reinterpret_cast<unsigned short*>(tile + Tile4<DF>::value_codes(t, at + 4)) = (unsigned short)(lo >> 16);
            *reinterpret_cast<unsigned short*>(tile + Tile4<DF>::value_codes(t, half + at)) = (unsigned short)hi;
            *reinterpret_cast<unsigned short*>(tile + Tile4<DF>::value_codes(t, half + at + 4)) = (unsigned short)(hi >> 16);
          } else {
            *reinterpret_cast<unsigned int*>(tile + Tile4<DF>::value_codes(t, at)) = lo;
            *reinterpret_cast<unsigned int*>(tile + Tile4<DF>::value_codes(t, half + at)) = hi;
          }
          if ((l & 3) == 0) {
            tile[Tile4<DF>::value_scale(t, at / 32)] = (unsigned char)lo_byte;
            tile[Tile4<DF>::value_scale(t, (half + at) / 32)] = (unsigned char)hi_byte;
          }
        }
        continue;
      }
    }
    if (is_q || is_k) {
      float sum = 0.0f;
      if (here) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += x[i] * x[i];
      }
      if (weights) sum = lanes_sum<L>(sum);
      const void* w = is_q ? a.wq : a.wk;
      norm_and_turn<T, float>(x, (const T*)w, weights, a.narrow_weights, (const float*)w, (float)a.eps, 1.0f / (float)D, c, s, at, half, L,
                              here, sum);
    }
    if (!here || (!is_q && !kept)) continue;
    T* to = is_q ? out + (token * a.Hq + h) * D : (T*)(is_k ? kpool : vpool) + (row * a.G + h) * D;
    store8(to + at, x);
    store8(to + half + at, x + 8);
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
  check_act(q_in, "q");
  TORCH_CHECK(q_in.dim() == 3 && k_in.dim() == 3 && v_in.dim() == 3, who, "q, k and v must be [N, heads, D]");
  const c10::DeviceGuard guard(q_in.device());
  const at::Tensor q = head_rows(q_in), k = head_rows(k_in), v = head_rows(v_in);
  const int64_t N = q.size(0), Hq = q.size(1), D = q.size(2), G = k.size(1);
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == N && k.size(2) == D && k.scalar_type() == q.scalar_type() &&
              v.scalar_type() == q.scalar_type(), who, "keys and values are as many, of one size and of the queries' type");
  for (const at::Tensor& t : {k, v, kpool, vpool, rows, positions, table, wq.value_or(q), wk.value_or(q)})
    TORCH_CHECK(t.device() == q.device(), who, "tensors on ", q.device(), " and ", t.device());
  check_i32(rows, "rows");
  check_i32(positions, "positions");
  TORCH_CHECK(rows.numel() == N && positions.numel() == N, who, "rows and positions must be one a token");
  TORCH_CHECK(table.dim() == 2 && is_f32(table) && table.is_contiguous() && table.size(1) == D, who, "table must be float32 [positions, D]");
  TORCH_CHECK(wq.has_value() == wk.has_value(), who, "both weights or none");
  if (wq.has_value()) {
    TORCH_CHECK(wq->numel() == D && wk->numel() == D && wq->is_contiguous() && wk->is_contiguous() && wq->scalar_type() == wk->scalar_type() &&
                (is_f32(*wq) || wq->scalar_type() == q.scalar_type()), who, "weights must be [D], of the queries' type or float32");
  }
  const bool four = kpool.scalar_type() == at::kByte;
  Append a;
  if (four) {
    TORCH_CHECK(D == 64 || D == 128 || D == 256, who, "4-bit pools take heads of 64, 128 or 256 channels, got ", D);
    const int64_t ps = page_size_of(kpool, D);
    TORCH_CHECK(ps > 0 && kpool.size(1) == G && vpool.sizes() == kpool.sizes() && page_size_of(vpool, D) == ps, who,
                "4-bit pools must be contiguous uint8 [pages, ", G, ", page size * 17 * ", D, " / 32], page sizes powers of two from 16 on");
    a.page_shift = log2_of(ps);
    a.pool_rows = kpool.size(0) * ps;
  } else {
    TORCH_CHECK(kpool.dim() == 4 && kpool.is_contiguous() && vpool.is_contiguous() && kpool.sizes() == vpool.sizes() &&
                kpool.size(2) == G && kpool.size(3) == D && kpool.scalar_type() == q.scalar_type() && vpool.scalar_type() == q.scalar_type(),
                who, "pools must be contiguous [pages, page size, ", G, ", ", D, "] of the keys' type, or uint8");
    TORCH_CHECK(D % 16 == 0 && D <= 512, who, "head sizes are multiples of 16 up to 512, got ", D);
    TORCH_CHECK(reinterpret_cast<uintptr_t>(kpool.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(vpool.data_ptr()) % 16 == 0, who,
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
    const int64_t turns = (Hq + 2 * G + WAVE / L - 1) / (WAVE / L);
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
  TORCH_CHECK(D == 64 || D == 128 || D == 256, "kv4_read: 4-bit pools hold heads of 64, 128 or 256 channels, got ", D);
  const int64_t ps = page_size_of(kpool, D);
  TORCH_CHECK(kpool.is_cuda() && ps > 0 && vpool.sizes() == kpool.sizes() && page_size_of(vpool, D) == ps,
              "kv4_read: pools must be contiguous uint8 [pages, heads, page size * 17 * D / 32]");
  const c10::DeviceGuard guard(kpool.device());
  check_i32(rows, "rows");
  TORCH_CHECK(vpool.device() == kpool.device() && rows.device() == kpool.device(), "kv4_read: tensors on several devices");
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
